"""Cases of the paged-cache serving operators and of the rotary embedding: what they read,
their plain forms in elementary torch operations, their values in 64 bits, and the calls of
the library (include/cuda_bridge.h).

  rope       cb_rope                     rotary positions of a tensor, and its gradient
  append     cb_paged_append             a step's q, k, v: rotate, write k and v into the pages
  attention  cb_paged_attention          new tokens (one or a chunk) over the paged cache
  weights    cb_paged_attention_weights  add every slot's attention weight to its running sum
  evict      cb_paged_evict              keep the slots with the largest sums, fill the holes

A cache is [pages, kv_heads, page, 128]; sequence b uses the pages table[b], has len[b] slots
and its new tokens are rows row_start[b] .. row_start[b + 1] of the token arrays, the last
slots of the sequence. Rows behind the last sequence are padding that nobody writes.
"""
import ctypes
import math

import numpy as np
import torch

own = False

HD = 128
LOG2E = 1.4426950408889634
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # Q of a training step of the 600m-A model: 32 sequences of 512, whole heads rotated
        dict(name="rope_train", op="rope", dtype="f16", tokens=16384, heads=12, hd=128, rot=128,
             layout="interleaved", scaling="none", inverse=False, wide=False, far=0),
        # gradient of a partly rotated head inside fused QKV rows, far positions
        dict(name="rope_grad_partial", op="rope", dtype="bf16", tokens=5001, heads=32, hd=128,
             rot=64, layout="half", scaling="parts", inverse=True, wide=True, far=900_000),
        # one token of each of 64 sequences (the decode batch of 600m-A)
        dict(name="append_decode", op="append", dtype="f16", batch=64, heads=12, kv_heads=12,
             page=16, new=1, len=512, ragged=True, rot=128, layout="interleaved",
             scaling="none"),
        # prompts of up to 1000 tokens, grouped heads, positions stretched for a long context
        dict(name="append_prompts", op="append", dtype="bf16", batch=12, heads=32, kv_heads=8,
             page=64, new=1000, len=4000, ragged=True, rot=128, layout="half",
             scaling="parts"),
        # the same decode batch: its attention
        dict(name="attn_decode_batch", op="attention", dtype="f16", batch=64, heads=12,
             kv_heads=12, page=16, new=1, len=512, ragged=True),
        # few sequences with long caches, grouped heads
        dict(name="attn_decode_long", op="attention", dtype="bf16", batch=4, heads=32,
             kv_heads=8, page=32, new=1, len=32768, ragged=True),
        # chunks of ragged prompts behind a cached prefix
        dict(name="attn_chunks", op="attention", dtype="f16", batch=8, heads=12, kv_heads=12,
             page=16, new=512, len=2048, ragged=True),
        # a long prompt's last chunks, five query heads to a key head
        dict(name="attn_chunk_long", op="attention", dtype="bf16", batch=2, heads=40,
             kv_heads=8, page=128, new=2048, len=16384, ragged=False),
        # a decode step's weights
        dict(name="weights_decode", op="weights", dtype="f16", batch=16, heads=32, kv_heads=8,
             page=32, new=1, len=4097, ragged=True),
        # a chunk's weights
        dict(name="weights_chunk", op="weights", dtype="bf16", batch=3, heads=32, kv_heads=8,
             page=64, new=1024, len=8192, ragged=True),
        # one slot too many in each sequence of a decode batch
        dict(name="evict_step", op="evict", dtype="f16", batch=64, heads=12, kv_heads=12,
             page=16, len=513, budget=512, sinks=4, recent=64, ragged=False),
        # long prompts cut down to a quarter
        dict(name="evict_trim", op="evict", dtype="bf16", batch=4, heads=32, kv_heads=8,
             page=64, len=32768, budget=8192, sinks=4, recent=1024, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention", "weights", "evict"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rope":
        hd = rng.choice([64, 80, 128, 256])
        heads = rng.choice([1, 6, 8, 14, 16, 32, 40, 52])
        rot = rng.choice([hd, hd, hd // 2, 8 * rng.randint(1, hd // 8)])
        tokens = _log(rng, 32, max(32, 16384 * 32 * 128 // (heads * hd)))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, hd=hd, rot=rot,
                    layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "parts"]),
                    inverse=rng.choice([False, True]), wide=rng.choice([False, True]),
                    far=rng.choice([0, _log(rng, 1000, 2_000_000)]))
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    group = rng.choice([1, 2, 4, 5, 7, 8] if kv_heads <= 8 else [1, 3])
    case = dict(op=op, dtype=dtype, heads=kv_heads * group, kv_heads=kv_heads,
                page=rng.choice([16, 32, 64, 128]), ragged=rng.choice([True, True, False]))
    length = _log(rng, 24, 32768)
    if op == "evict":
        budget = max(8, int(length * rng.uniform(0.1, 1.0)))
        sinks = rng.randint(0, min(8, budget))
        return case | dict(
            batch=_log(rng, 1, max(1, min(96, 4 * 32768 * 8 // (length * kv_heads)))),
            len=length, budget=budget, sinks=sinks,
            recent=int((budget - sinks) * rng.uniform(0.0, 0.9)))
    new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 2048)])
    new = min(new, length)
    if op == "append":
        most = min(96, 12 * 1000 * 48 // (new * (case["heads"] + 2 * kv_heads)),
                   12 * 4000 * 8 // (length * kv_heads))
        return case | dict(batch=_log(rng, 1, max(1, most)), new=new, len=length,
                           rot=rng.choice([128, 128, 64, 8 * rng.randint(1, 16)]),
                           layout=rng.choice(["half", "interleaved"]),
                           scaling=rng.choice(["none", "linear", "base", "parts"]))
    if op == "weights":
        new = min(new, 1024)
    share = 1.0 if op == "attention" else 0.4
    pairs = 2 * 40 * 2048 * 16384 * share
    while case["heads"] * new * length > pairs:
        length = length // 2
        new = min(new, length)
    most = min(128, pairs // (case["heads"] * new * length),
               4 * 32768 * 8 * share // (length * kv_heads))
    return case | dict(batch=_log(rng, 1, max(1, most)), new=new, len=length)


def _sizes(case):
    """Every sequence's slots and new tokens: a fixed spread over a ragged batch, in which
    every seventh sequence has no new token in this step."""
    lens, news = [], []
    for b in range(case["batch"]):
        part = (b * 0.6180339887) % 1.0 if case["ragged"] else 0.0
        n = case.get("new", 0)
        if case["ragged"] and n > 1:
            n = max(1, int(n * (1.0 - 0.8 * ((b * 0.7548776662) % 1.0))))
        if case["ragged"] and n and b % 7 == 5:
            n = 0
        lens.append(max(n, 1, int(case["len"] * (1.0 - 0.9 * part))))
        news.append(n)
    return lens, news


def _pairs(case):
    return sum(n * (length - n) + n * (n + 1) // 2 for length, n in zip(*_sizes(case)))


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * case["hd"]
        return {"bytes": 4 * n + 4 * case["tokens"], "flops": 3 * n}
    lens, news = _sizes(case)
    h, g = case["heads"], case["kv_heads"]
    rows, slots = sum(news), sum(lens)
    if op == "append":
        return {"bytes": rows * ((h + 2 * g) * HD * 4 + 4 + 8 * g), "flops": 3 * rows * (h + g) * HD}
    if op == "attention":
        return {"bytes": slots * g * HD * 4 + rows * h * (HD * 4 + 4),
                "flops": 4.0 * HD * h * _pairs(case)}
    if op == "weights":
        return {"bytes": slots * g * (HD * 2 + 8) + rows * h * (HD * 2 + 4),
                "flops": 2.0 * HD * h * _pairs(case)}
    kept = sum(min(length, case["budget"]) for length in lens)
    # the kept slots behind the budget move down: a share of the budget as large as the
    # share of the slots that lies there
    moved = sum(case["budget"] * (length - case["budget"]) / length
                for length in lens if length > case["budget"])
    return {"bytes": g * (8 * slots + 8 * kept + moved * HD * 8), "flops": g * slots}


# ------------------------------------------------------------------------------ inputs
def _inv_freq(rot, scaling):
    """Radians per position of each rotated pair, and the factor of cos and sin."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    base, factor, trained = 10000.0, 8.0, 4096.0
    if scaling == "base":
        base = base * factor ** (rot / max(1, rot - 2))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling != "parts":
        return f, 1.0
    # pairs that turn over 32 times in the trained length stay, those under once are
    # divided by the factor, in between both are mixed
    def pair(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(0.0, math.floor(pair(32.0))), min(rot - 1.0, math.ceil(pair(1.0)))
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=dev, dtype=dt, generator=gen)

    op = case["op"]
    s = {"case": case}
    if "rot" in case:
        f, s["amplitude"] = _inv_freq(case["rot"], case["scaling"])
        s["inv_freq"] = f.to(dev)
    if op == "rope":
        t, h, hd = case["tokens"], case["heads"], case["hd"]
        width = (2 * h + 1) * hd if case["wide"] else h * hd  # columns of wider rows, or q alone
        s["x"] = randn(t, width)[:, :h * hd]
        s["y"] = torch.zeros(t, h * hd, device=dev, dtype=dt)
        s["positions"] = ((torch.arange(t, device=dev) % 512) if not case["far"] else
                          torch.randint(0, case["far"], (t,), device=dev, generator=gen)).int()
        return s

    lens, news = _sizes(case)
    batch, g, page = case["batch"], case["kv_heads"], case["page"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=dev, generator=gen).int()
    table = torch.full((batch, max(need)), -1, dtype=torch.int32)
    at = torch.cumsum(torch.tensor([0] + need), 0)
    col = torch.arange(max(need))[None, :]
    used = col < torch.tensor(need)[:, None]
    table[used] = (at[:-1, None] + col)[used].int()
    table = table.to(dev)
    s["table"] = torch.where(table >= 0, order[table.long().clamp(min=0)], table)
    s["len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["k"], s["v"] = randn(pages, g, page, HD), randn(pages, g, page, HD)
    s["pages"], s["max_len"], s["max_new"] = pages, max(lens), max(news)
    if op == "evict":
        # few slots carry most of the weight, a new token has none yet; the slots of a
        # cache that was evicted from before are in no order
        w = torch.exp(2.0 * torch.randn(pages, g, page, device=dev, generator=gen))
        s["weights"] = torch.where(torch.rand(w.shape, device=dev, generator=gen) < 0.05, 0.0, w)
        slot = torch.rand(batch, g, max(lens), device=dev, generator=gen)
        live = torch.arange(max(lens), device=dev) < s["len"][:, None, None]
        rank = torch.where(live, slot, 2.0).argsort(-1).argsort(-1).int() * 2
        ps = max(need) * page
        dense = torch.zeros(batch, g, ps, dtype=torch.int32, device=dev)
        dense[:, :, :max(lens)] = rank
        s["positions"] = torch.zeros(pages, g, page, dtype=torch.int32, device=dev)
        own_pages = used.to(dev)
        s["positions"][s["table"][own_pages].long()] = (
            dense.view(batch, g, -1, page).transpose(1, 2)[own_pages])
        s["next"] = s["len"] * 2
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["positions_out"] = torch.zeros_like(s["positions"])
        s["len_out"] = torch.zeros_like(s["len"])
        return s

    rows = -(-max(1, sum(news)) // 8) * 8  # token arrays are padded to a multiple of eight
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    s["row_start"] = torch.tensor(start, dtype=torch.int32, device=dev)
    s["rows"], h = rows, case["heads"]
    if op == "append":
        qkv = randn(rows, (h + 2 * g) * HD)
        s["q"], s["nk"], s["nv"] = qkv.split([h * HD, g * HD, g * HD], 1)
        s["q_out"] = torch.zeros(rows, h * HD, device=dev, dtype=dt)
        s["weights"] = torch.rand(pages, g, page, device=dev, generator=gen)
        s["slot_positions"] = torch.zeros(pages, g, page, dtype=torch.int32, device=dev)
        seq = torch.searchsorted(s["row_start"], torch.arange(rows, device=dev).int(), right=True) - 1
        seq = seq.clamp(0, batch - 1)
        # a cache that was evicted from: the token's position lies behind its slot
        s["positions"] = (s["len"][seq] - s["row_start"][seq + 1] + 7919
                          + torch.arange(rows, device=dev)).int()
        return s
    s["q"] = randn(rows, h * HD) * 1.5
    s["scale"] = 1.0 / math.sqrt(HD)
    if op == "attention":
        s["out"] = torch.zeros(rows, h * HD, device=dev, dtype=dt)
        s["lse"] = torch.zeros(rows, h, device=dev)
    else:
        # the log-sum-exp (base 2) that normal scores of that spread have, a little off
        seq = torch.searchsorted(s["row_start"], torch.arange(rows, device=dev).int(), right=True) - 1
        n = s["len"][seq.clamp(0, batch - 1)].float()
        s["lse"] = (torch.log(n)[:, None] + 1.125
                    + 0.1 * torch.randn(rows, h, device=dev, generator=gen)) * LOG2E
        s["weights"] = torch.exp(torch.randn(pages, g, page, device=dev, generator=gen))
    return s


# ------------------------------------------------------------------------- plain forms
def _rotate(x, positions, inv_freq, amplitude, layout, rot, inverse):
    """x [tokens, heads, hd] in 32 bits, angles in 64."""
    a = positions.double()[:, None] * inv_freq
    c, s = (torch.cos(a) * amplitude).float()[:, None], (torch.sin(a) * amplitude).float()[:, None]
    s = -s if inverse else s
    if layout == "half":
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], -1)
    else:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([x0 * c - x1 * s, x1 * c + x0 * s], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    x = s["x"].float().view(c["tokens"], c["heads"], c["hd"]) if s["x"].is_contiguous() else \
        s["x"].float().unflatten(1, (c["heads"], c["hd"]))
    y = _rotate(x, s["positions"], s["inv_freq"], s["amplitude"], c["layout"], c["rot"], c["inverse"])
    s["y"].copy_(y.flatten(1))
    return s["y"]


def _rows(s):
    """Of every row its sequence, its place among the new tokens and whether it is no padding."""
    r = torch.arange(s["rows"], device=s["len"].device)
    b = (torch.searchsorted(s["row_start"], r.int(), right=True) - 1).clamp(max=s["case"]["batch"] - 1)
    return b, r - s["row_start"][b], r < s["row_start"][-1]


def _plain_append(s):
    c = s["case"]
    h, g, page = c["heads"], c["kv_heads"], c["page"]
    b, i, real = _rows(s)
    q = _rotate(s["q"].float().unflatten(1, (h, HD)), s["positions"], s["inv_freq"],
                s["amplitude"], c["layout"], c["rot"], False)
    k = _rotate(s["nk"].float().unflatten(1, (g, HD)), s["positions"], s["inv_freq"],
                s["amplitude"], c["layout"], c["rot"], False)
    v = s["nv"].unflatten(1, (g, HD))
    s["q_out"].copy_(torch.where(real[:, None], q.flatten(1).to(s["q_out"].dtype), s["q_out"]))
    first = torch.where(real, torch.arange(s["rows"], device=real.device), 0)  # padding repeats row 0
    b, i = b[first], i[first]
    slot = (s["len"][b] - (s["row_start"][b + 1] - s["row_start"][b]) + i).long()
    page_id = s["table"][b, slot // page].long()
    at = slot % page
    s["k"][page_id, :, at] = k[first].to(s["k"].dtype)
    s["v"][page_id, :, at] = v[first]
    s["weights"][page_id, :, at] = 0.0
    s["slot_positions"][page_id, :, at] = s["positions"][first][:, None].expand(-1, g)
    return _append_outputs(s)


def _append_outputs(s):
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "weights": s["weights"],
            "positions": s["slot_positions"]}


def _gather(s, pool):
    """[batch, kv_heads, slots, 128] in 32 bits."""
    t = s["table"].long().clamp(min=0)
    return pool[t].transpose(1, 2).flatten(2, 3).float()


def _scores(s):
    """Scaled scores of the new tokens, [batch, kv_heads, group, new, slots], and their mask."""
    c = s["case"]
    g, group, n = c["kv_heads"], c["heads"] // c["kv_heads"], s["max_new"]
    i = torch.arange(n, device=s["len"].device)
    row = (s["row_start"][:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().view(c["batch"], n, g, group, HD).permute(0, 2, 3, 1, 4)
    k = _gather(s, s["k"])
    x = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (group, n)) * s["scale"]
    count = (s["row_start"][1:] - s["row_start"][:-1])[:, None]
    last = s["len"][:, None] - count + i  # the last slot that a new token sees
    slot = torch.arange(x.shape[-1], device=x.device)
    seen = (slot <= last[..., None]) & (i < count)[..., None]
    return x, seen[:, None, None]


def _plain_attention(s):
    c = s["case"]
    x, seen = _scores(s)
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    m0 = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m0)
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ _gather(s, s["v"])).view(*p.shape[:-1], HD)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (torch.log(total) + m0).squeeze(-1) * LOG2E
    b, i, real = _rows(s)
    i = i.clamp(max=s["max_new"] - 1)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 4)[b, i]
    lse = lse.permute(0, 3, 1, 2).flatten(2, 3)[b, i]
    s["out"].copy_(torch.where(real[:, None], o.to(s["out"].dtype), s["out"]))
    s["lse"].copy_(torch.where(real[:, None], lse, s["lse"]))
    return {"out": s["out"], "lse": s["lse"]}


def _plain_weights(s):
    c = s["case"]
    g, group, n = c["kv_heads"], c["heads"] // c["kv_heads"], s["max_new"]
    x, seen = _scores(s)
    row = (s["row_start"][:-1, None] + torch.arange(n, device=x.device)).clamp(max=s["rows"] - 1)
    lse = s["lse"][row].view(c["batch"], n, g, group).permute(0, 2, 3, 1)
    p = torch.exp(x - (lse / LOG2E)[..., None]).masked_fill(~seen, 0.0)
    w = p.sum((2, 3)).view(c["batch"], g, -1, c["page"]).transpose(1, 2)
    s["weights"].index_add_(0, s["table"].clamp(min=0).flatten(), w.flatten(0, 1))
    return s["weights"]


def _plain_evict(s):
    c = s["case"]
    g, page, budget = c["kv_heads"], c["page"], c["budget"]
    t = s["table"].long().clamp(min=0)
    w = s["weights"][t].transpose(1, 2).flatten(2, 3)
    pos = s["positions"][t].transpose(1, 2).flatten(2, 3)
    slot = torch.arange(w.shape[-1], device=w.device)
    live = slot < s["len"][:, None, None]
    must = (pos < c["sinks"]) | (pos >= (s["next"] - c["recent"])[:, None, None])
    key = torch.where(live, torch.where(must, math.inf, w), -math.inf)
    order = key.argsort(dim=-1, descending=True, stable=True)
    new_len = s["len"].clamp(max=budget)[:, None, None]
    keep = torch.zeros_like(key, dtype=torch.bool)
    keep = keep.scatter_(-1, order, (slot < new_len).expand_as(order)) & live
    hole, mover = (slot < new_len) & ~keep, (slot >= new_len) & keep
    # the i-th hole takes the i-th kept slot behind the budget
    source = (~mover).byte().argsort(dim=-1, stable=True)
    rank = (hole.cumsum(-1) - 1).clamp(min=0)
    source = torch.where(hole, source.gather(-1, rank), slot)
    # what a slot below the new length holds; the ones behind it repeat slot 0
    top = min(budget, slot.numel())
    to = torch.where(slot[:top] < new_len, slot[:top], 0).expand(-1, g, -1)
    fro = source.gather(-1, to)
    b = torch.arange(c["batch"], device=w.device)[:, None, None]
    head = torch.arange(g, device=w.device)[None, :, None]
    target = t[b, to // page], head, to % page
    origin = t[b, fro // page], head, fro % page
    s["k"][target] = s["k"][origin]
    s["v"][target] = s["v"][origin]
    s["weights_out"][target] = s["weights"][origin]
    s["positions_out"][target] = s["positions"][origin]
    s["len_out"].copy_(new_len.flatten())
    return _evict_outputs(s)


def _evict_outputs(s):
    return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "positions": s["positions_out"],
            "len": s["len_out"]}


# --------------------------------------------------------------------- the library's calls
def _plan(s):
    """What a program makes once for a cache and a batch shape: the descriptors of both and
    the workspace."""
    from rustane_b200 import bridge as B
    c = s["case"]
    lib = B.load_library()
    plan = {"lib": lib, "check": B.check}
    dtype = B.CB_DTYPE_F16 if c["dtype"] == "f16" else B.CB_DTYPE_BF16
    plan["dtype"] = dtype
    if "rot" in c:
        plan["rope"] = B.cb_rope_config(
            s["inv_freq"].data_ptr(), c["rot"],
            B.CB_ROPE_HALF if c["layout"] == "half" else B.CB_ROPE_INTERLEAVED, s["amplitude"])
        plan["rope_ref"] = ctypes.byref(plan["rope"])
    if c["op"] != "rope":
        plan["kv"] = B.cb_paged_kv(
            s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["len"].data_ptr(),
            s["row_start"].data_ptr() if "row_start" in s else None, dtype, s["pages"],
            c["kv_heads"], c["page"], c["batch"], s["table"].shape[1], s["max_len"],
            s.get("rows", 0), s["max_new"])
        plan["kv_ref"] = ctypes.byref(plan["kv"])
        size = ctypes.c_size_t()
        if c["op"] == "attention":
            B.check(lib.cb_paged_attention_workspace(plan["kv_ref"], c["heads"], ctypes.byref(size)))
        if c["op"] == "evict":
            B.check(lib.cb_paged_evict_workspace(plan["kv_ref"], c["budget"], ctypes.byref(size)))
        plan["workspace"] = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
    s["plan"] = plan
    return plan


def _own(s):
    c = s["case"]
    p = s.get("plan") or _plan(s)
    lib, check = p["lib"], p["check"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "rope":
        check(lib.cb_rope(p["rope_ref"], p["dtype"], s["x"].data_ptr(), s["x"].stride(0),
                          s["y"].data_ptr(), s["y"].stride(0), s["positions"].data_ptr(),
                          c["tokens"], c["heads"], c["hd"], int(c["inverse"]), stream))
        return s["y"]
    if c["op"] == "append":
        check(lib.cb_paged_append(p["kv_ref"], p["rope_ref"], c["heads"], s["q"].data_ptr(),
                                  s["q"].stride(0), s["q_out"].data_ptr(), s["q_out"].stride(0),
                                  s["nk"].data_ptr(), s["nk"].stride(0), s["nv"].data_ptr(),
                                  s["nv"].stride(0), s["positions"].data_ptr(),
                                  s["weights"].data_ptr(), s["slot_positions"].data_ptr(), stream))
        return _append_outputs(s)
    if c["op"] == "attention":
        check(lib.cb_paged_attention(p["kv_ref"], s["q"].data_ptr(), s["q"].stride(0), c["heads"],
                                     s["scale"], s["out"].data_ptr(), s["out"].stride(0),
                                     s["lse"].data_ptr(), p["workspace"].data_ptr(),
                                     p["workspace"].numel(), stream))
        return {"out": s["out"], "lse": s["lse"]}
    if c["op"] == "weights":
        check(lib.cb_paged_attention_weights(p["kv_ref"], s["q"].data_ptr(), s["q"].stride(0),
                                             c["heads"], s["scale"], s["lse"].data_ptr(),
                                             s["weights"].data_ptr(), stream))
        return s["weights"]
    check(lib.cb_paged_evict(p["kv_ref"], s["weights"].data_ptr(), s["weights_out"].data_ptr(),
                             s["positions"].data_ptr(), s["positions_out"].data_ptr(),
                             s["next"].data_ptr(), c["budget"], c["sinks"], c["recent"],
                             s["len_out"].data_ptr(), p["workspace"].data_ptr(),
                             p["workspace"].numel(), stream))
    return _evict_outputs(s)


PLAIN = {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention,
         "weights": _plain_weights, "evict": _plain_evict}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------- values in 64 bits
def _turn(x, positions, s):
    """Rotation of [tokens, heads, hd] as a product of complex numbers."""
    c = s["case"]
    rot = c["rot"]
    sign = -1.0 if c.get("inverse") else 1.0
    turn = s["amplitude"] * torch.exp(1j * sign * positions.double()[:, None] * s["inv_freq"])[:, None]
    y = x.double().clone()
    lanes = torch.arange(rot // 2, device=x.device)
    re, im = (lanes, lanes + rot // 2) if c["layout"] == "half" else (2 * lanes, 2 * lanes + 1)
    z = torch.complex(y[..., re], y[..., im]) * turn
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_append(s):
    c = s["case"]
    h, g, page = c["heads"], c["kv_heads"], c["page"]
    lens, news = _sizes(c)
    q, k, v = (s[n].unflatten(1, (-1, HD)) for n in ("q", "nk", "nv"))
    k_pool, v_pool = s["k"].double(), s["v"].double()
    w, where = s["weights"].clone(), s["slot_positions"].clone()
    q_out = torch.zeros(s["rows"], h, HD, dtype=torch.float64, device=q.device)
    row = 0
    for b in range(c["batch"]):
        span = slice(row, row + news[b])
        q_out[span] = _turn(q[span], s["positions"][span], s)
        slots = torch.arange(lens[b] - news[b], lens[b], device=q.device)
        at = s["table"][b].long()[slots // page], slots % page
        new_k = _turn(k[span], s["positions"][span], s)
        for head in range(g):
            k_pool[at[0], head, at[1]] = new_k[:, head]
            v_pool[at[0], head, at[1]] = v[span, head].double()
            w[at[0], head, at[1]] = 0.0
            where[at[0], head, at[1]] = s["positions"][span]
        row += news[b]
    return {"q": q_out.flatten(1), "k": k_pool, "v": v_pool, "weights": w, "positions": where}


def _exact_scores(s):
    """For each sequence and key head: its rows, slots, and masked scores in 64 bits."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    lens, news = _sizes(c)
    q = s["q"].unflatten(1, (c["kv_heads"], group, HD))
    row = 0
    for b in range(c["batch"]):
        n, length = news[b], lens[b]
        used = s["table"][b, :-(-length // c["page"])].long()
        for head in range(c["kv_heads"]):
            k = s["k"][used, head].flatten(0, 1)[:length].double()
            x = torch.einsum("igd,td->git", q[row:row + n, head].double(), k) * s["scale"]
            future = torch.ones(n, length, dtype=torch.bool, device=k.device).triu(length - n + 1)
            x[:, future] = -math.inf
            if n:
                yield b, head, slice(row, row + n), used, length, x
        row += n


def _exact_attention(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["rows"], c["kv_heads"], group, HD, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(s["rows"], c["kv_heads"], group, dtype=torch.float64, device=s["q"].device)
    for b, head, span, used, length, x in _exact_scores(s):
        v = s["v"][used, head].flatten(0, 1)[:length].double()
        total = torch.logsumexp(x, -1, keepdim=True)
        out[span, head] = (torch.exp(x - total) @ v).transpose(0, 1)
        lse[span, head] = total.squeeze(-1).T * LOG2E
    return {"out": out.flatten(1), "lse": lse.flatten(1)}


def _exact_weights(s):
    c = s["case"]
    group, page = c["heads"] // c["kv_heads"], c["page"]
    w = s["weights"].double()
    lse = s["lse"].double().unflatten(1, (c["kv_heads"], group))
    for b, head, span, used, length, x in _exact_scores(s):
        p = torch.exp2(x * LOG2E - lse[span, head].T[..., None]).sum((0, 1))
        slots = torch.arange(length, device=w.device)
        w[used[slots // page], head, slots % page] += p
    return w


def _exact_evict(s):
    c = s["case"]
    page = c["page"]
    lens, _ = _sizes(c)
    host = {n: s[n].cpu().numpy() for n in ("table", "weights", "positions", "next")}
    w_out = np.zeros(host["weights"].shape, np.float32)
    p_out = np.zeros(host["positions"].shape, np.int32)
    moves = []
    for b, length in enumerate(lens):
        slots = np.arange(length)
        pages, at = host["table"][b, slots // page], slots % page
        new = min(length, c["budget"])
        for head in range(c["kv_heads"]):
            w, pos = host["weights"][pages, head, at], host["positions"][pages, head, at]
            must = (pos < c["sinks"]) | (pos >= host["next"][b] - c["recent"])
            best = np.lexsort((slots, -w.astype(np.float64), ~must))[:new]
            keep = np.zeros(length, bool)
            keep[best] = True
            source = slots[:new].copy()
            source[~keep[:new]] = slots[new:][keep[new:]]
            w_out[pages[:new], head, at[:new]] = w[source]
            p_out[pages[:new], head, at[:new]] = pos[source]
            to = np.flatnonzero(source != slots[:new])
            fro = source[to]
            moves.append(np.stack([pages[to], np.full(len(to), head), at[to],
                                   pages[fro], at[fro]]))
    m = torch.from_numpy(np.concatenate(moves, 1).astype(np.int64)).to(s["k"].device)
    pools = {}
    for name in ("k", "v"):
        pools[name] = s[name].double()
        pools[name][m[0], m[1], m[2]] = s[name][m[3], m[1], m[4]].double()
    new_len = torch.tensor([min(n, c["budget"]) for n in lens], dtype=torch.int32)
    return pools | {"weights": torch.from_numpy(w_out).double(), "positions": torch.from_numpy(p_out),
                    "len": new_len}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        x = s["x"].unflatten(1, (case["heads"], case["hd"]))
        return _turn(x, s["positions"], s).flatten(1)
    return {"append": _exact_append, "attention": _exact_attention, "weights": _exact_weights,
            "evict": _exact_evict}[case["op"]](s)
