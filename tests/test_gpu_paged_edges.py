"""GPU tests of the paged-cache operators at the edges of what their calls allow, against
64-bit forms. Tolerances are derived beside each test."""
import ctypes as C
import math

import pytest
import torch

import paged_ref as R
from paged_ref import Cache, ptr, stream
from rustane_b200 import bridge as B

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- eviction and absent pages
def _evict(lib, c, w, wo, p, po, nxt, budget, sinks, recent, lo):
    d, size = c.desc(), C.c_size_t()
    assert lib.cb_paged_evict_workspace(C.byref(d), budget, C.byref(size)) == 0
    ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    rc = lib.cb_paged_evict(C.byref(d), ptr(w), ptr(wo), ptr(p), ptr(po), ptr(nxt), budget, sinks,
                            recent, ptr(lo), ptr(ws), size.value, stream())
    torch.cuda.synchronize()
    return rc


def _evict_absent_ref(w, p, absent, nxt, budget, sinks, recent):
    """{slot below the new length: the slot whose contents it gets} of one sequence and key
    head. Where a slot below the budget is absent, only slots that must stay move."""
    n = len(w)
    new = min(n, budget)
    slots = [s for s in range(n) if not absent[s]]
    if n <= budget:
        return {s: s for s in slots}
    held = any(absent[:new])

    def order(s):
        must = p[s] < sinks or (recent > 0 and p[s] >= nxt - recent)
        rank = 0 if must else 3 if held and s >= new else 2 if math.isnan(w[s]) else 1
        return rank, -w[s] if rank == 1 else 0.0, s
    keep = set(sorted(slots, key=order)[:new - sum(absent[:new])])
    movers = [s for s in slots if s >= new and s in keep]
    source = {s: s if s in keep else movers.pop(0) for s in slots if s < new}
    assert not movers
    return source


ABSENT = [
    # lens, kv_heads, page, budget, sinks, recent, absent pages of each sequence
    ([64, 64], 1, 16, 48, 0, 16, [[1], []]),
    ([64, 64, 64], 2, 16, 48, 4, 8, [[1], [3], [0, 2]]),
    ([52, 50, 49], 2, 16, 48, 2, 10, [[1], [3], [0, 1, 2]]),      # few slots go
    ([64, 64], 1, 16, 48, 8, 40, [[1], [0]]),                     # more must stay than have room
    ([64, 40], 1, 16, 48, 0, 48, [[0, 1, 2], [1]]),               # nothing below the budget is there
    ([700, 700], 3, 64, 300, 4, 100, [[0, 4, 9], [10]]),
    ([6000, 5500], 2, 64, 2000, 4, 900, [[3, 17, 90], [93]]),     # two CTAs
    ([5006, 5003], 1, 32, 5000, 4, 60, [[7], [156]]),             # few, two CTAs
    ([20000], 1, 128, 8000, 4, 3000, [[0, 30, 62, 100]]),         # eight CTAs
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,kv_heads,page,budget,sinks,recent,gone", ABSENT)
def test_evict_keeps_what_must_stay_beside_absent_pages(bridge_lib, lens, kv_heads, page, budget,
                                                        sinks, recent, gone, in_place):
    c = Cache(lens, [0] * len(lens), kv_heads, kv_heads, page, "f16", seed=sum(lens))
    shape = (c.pages, kv_heads, page)
    g = torch.Generator(device="cuda").manual_seed(budget)
    w = (torch.rand(shape, device="cuda", generator=g) * 50).floor() / 8
    odd = torch.randint(0, 20, shape, device="cuda", generator=g)
    for i, x in enumerate((math.nan, math.inf, -math.inf, -1.5)):
        w[odd == i] = x
    p = torch.zeros(shape, device="cuda", dtype=torch.int32)
    for b in range(c.batch):
        for h in range(kv_heads):
            at = c.place(b, torch.arange(lens[b], device="cuda"))
            p[at[0], h, at[1]] = torch.randperm(lens[b], device="cuda", generator=g).int()
    nxt = c.len.clone()
    for b, pages in enumerate(gone):
        for i, j in enumerate(pages):
            c.table[b, j] = (-1, c.pages, -2 ** 31, 2 ** 31 - 1)[i]
    wo = w if in_place else torch.full_like(w, 9.0)
    po = p if in_place else torch.full_like(p, 9)
    want = {"k": c.k.clone(), "v": c.v.clone(), "w": wo.clone(), "p": po.clone()}
    for b in range(c.batch):
        absent = [s // page in gone[b] for s in range(lens[b])]
        for h in range(kv_heads):
            pos = c.slots(p, b, h).tolist()
            source = _evict_absent_ref(c.slots(w, b, h).tolist(), pos, absent, lens[b], budget,
                                       sinks, recent)
            # what the call promises, apart from how: present positions that must stay do, as
            # far as there is room
            must = {x for x, a in zip(pos, absent)
                    if not a and (x < sinks or x >= lens[b] - recent)}
            if lens[b] > budget:
                stays = {pos[s] for s in source.values()}
                assert must <= stays or stays <= must
            to = c.place(b, torch.tensor(list(source), device="cuda", dtype=torch.long))
            fro = c.place(b, torch.tensor(list(source.values()), device="cuda", dtype=torch.long))
            for name, new, old in (("k", c.k, c.k), ("v", c.v, c.v), ("w", w, w), ("p", p, p)):
                want[name][to[0], h, to[1]] = old[fro[0], h, fro[1]]
    lo = torch.full_like(c.len, -1)
    assert _evict(bridge_lib, c, w, wo, p, po, nxt, budget, sinks, recent, lo) == 0
    assert lo.tolist() == [min(n, budget) for n in lens]
    for name, got in (("k", c.k), ("v", c.v)):
        assert torch.equal(got.view(torch.int16), want[name].view(torch.int16)), name
    assert torch.equal(wo.view(torch.int32), want["w"].view(torch.int32))
    assert torch.equal(po, want["p"])


# ------------------------------------------- keys with infinities in the weights of a chunk
@pytest.mark.parametrize("heads", [3, 5, 7, 100, 4, 128])
def test_weights_of_an_infinite_key_do_not_depend_on_the_group(bridge_lib, heads):
    """A key with one infinite element scores minus infinity with queries whose element there
    is negative: its slot gets 0 from them, also where the rows of a step are not all taken."""
    c = Cache([600], [150], heads, 1, 32, "bf16", seed=heads)
    q = c.tokens(heads * 128, scale=1.5)
    q.unflatten(1, (heads, 128))[:150, :, 9] = -0.5
    scale = 128 ** -0.5
    _, lse64, _, _ = R.attention_ref(c, q, scale)
    lse = torch.zeros(c.rows, heads, device="cuda")
    lse[:150] = lse64.float()
    clean, w = (torch.zeros(c.pages, 1, 32, device="cuda") for _ in range(2))
    d = c.desc()
    for x in (clean, w):
        assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), heads, scale,
                                                     ptr(lse), ptr(x), stream()) == 0
        torch.cuda.synchronize()
        for slot, value in ((5, math.inf), (70, -math.inf), (590, math.inf)):
            at = c.place(0, torch.tensor([slot], device="cuda"))
            c.k[at[0], 0, at[1], 9] = value
    want = clean.clone()
    for slot, total in ((5, 0.0), (70, math.inf), (590, 0.0)):
        at = c.place(0, torch.tensor([slot], device="cuda"))
        want[at[0], 0, at[1]] = total
    assert torch.equal(w, want)


# ------------------------------------------------------------- sums of many small weights
def _one_heavy_slot(n, new, batch, heads, behind, dtype):
    """Every sequence sees the same n slots, slot 0 with a score of `behind` (base 2) above
    the equal others and V = 0, the others' V = 1. (Many sequences, so that one worker walks all
    slots of one.) Returns out, lse, the others' sums and the error of a score."""
    c = Cache([n], [new], heads, 1, 64, dtype, seed=1, pad=0)
    c.k[c.live], c.v[c.live] = 0.0, 1.0
    first = c.place(0, torch.tensor([0], device="cuda"))
    c.k[first[0], 0, first[1]], c.v[first[0], 0, first[1]] = 1.0, 0.0
    c.table = c.table.expand(batch, -1).contiguous()
    c.len = c.len.expand(batch).contiguous()
    c.row_start = torch.arange(batch + 1, device="cuda", dtype=torch.int32) * new
    c.batch, c.rows = batch, batch * new
    q = torch.ones(c.rows, heads * 128, device="cuda", dtype=c.dt)
    out = torch.zeros_like(q)
    lse = torch.zeros(c.rows, heads, device="cuda")
    assert R.attention(B.load_library(), c, q, behind / (128 * R.LOG2E), out, lse) == 0
    others = torch.arange(n - new, n, dtype=torch.float64, device="cuda")
    # a score: its accumulation and scaling in 32 bits (paged_ref.attention_ref)
    delta = behind / R.LOG2E * 2.0 ** -19 + 2.0 ** -20 * (1 + behind / R.LOG2E)
    return (out.view(batch, new, -1).double(), lse.view(batch, new, -1).double(),
            (others * 2.0 ** -behind)[:, None], delta)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,new,batch", [(1, 1, 2400), (32, 1, 300), (2, 40, 150)])
@pytest.mark.parametrize("behind", [18.0, 20.3, 23.1, 25.6])
def test_the_log_sum_exp_counts_many_small_weights(bridge_lib, heads, new, batch, behind, dtype):
    """The sum itself, in 32 bits: off by half a step for each of its last additions (a step of
    128 keys each at most: n / 128 of them, and 32 within the first), not for each slot."""
    n = 30000
    _, lse, small, delta = _one_heavy_slot(n, new, batch, heads, behind, dtype)
    want = behind + torch.log2(1 + small)
    tol = delta * R.LOG2E + 2.0 ** -19 + (n / 128 + 32) * 2.0 ** -24 * R.LOG2E
    assert float((lse - want).abs().max()) <= tol


@pytest.mark.parametrize("heads,new,batch", [(1, 1, 2400), (32, 1, 300), (2, 40, 150)])
@pytest.mark.parametrize("behind", [20.3, 25.6])
def test_many_small_weights_in_fp16_add_up(bridge_lib, heads, new, batch, behind):
    """Each weight is far below fp16's normal range beside the largest, their sum is not. A
    weight is off by half a step of the type or by 2^-32 of the largest one."""
    n = 30000
    out, _, small, delta = _one_heavy_slot(n, new, batch, heads, behind, "f16")
    want = small / (1 + small)
    tol = 2 * 2.0 ** -11 * want + (2 * delta + 2.0 ** -18) * want + n * 2.0 ** -32 + 2.0 ** -25
    over = (out - want).abs() - tol
    assert float(over.max()) <= 0.0, (float(out.min()), float(out.max()), float(want[0, 0]))


# ----------------------------------------------- the exponential of the weights of a chunk
def test_exponentials_of_the_weights_over_their_whole_range(bridge_lib):
    """With q = 0 and one row of a step that counts (log-sum-exp -x, the others infinite) a
    slot's weight is 2^x. The columns of a step take 2^x from the special-function unit (relative
    error 2^-22) or from a polynomial (3.4e-7): each within that, 0 below 2^-126, infinite from
    2^128 on. Between 2^127.5 and there the polynomial is off by up to 7e-5."""
    n, heads, page = 8192, 128, 16
    dev = "cuda"
    own = 7 + torch.arange(n, device=dev, dtype=torch.int32)
    table = torch.cat([torch.arange(7, device=dev, dtype=torch.int32).expand(n, 7), own[:, None]], 1)
    table = table.contiguous()
    length = torch.full((n,), 128, device=dev, dtype=torch.int32)
    start = torch.arange(n + 1, device=dev, dtype=torch.int32)
    pages = n + 7
    k = torch.zeros(pages, 1, page, 128, device=dev, dtype=torch.float16)
    q = torch.zeros(n, heads * 128, device=dev, dtype=torch.float16)
    kv = B.cb_paged_kv(k.data_ptr(), k.data_ptr(), table.data_ptr(), length.data_ptr(),
                       start.data_ptr(), B.CB_DTYPE_F16, pages, 1, page, n, 8, 128, n, 1)
    row = torch.arange(n, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    special = [-126.0, -126.2, -126.49, -126.51, -127.0, -127.6, -149.0, -1e30, -math.inf,
               math.nextafter(-126.0, 0.0), 127.49, 127.51, 127.6, 127.99, 128.0, 128.01, 129.0,
               1e30, math.inf, math.nan, 0.0, -0.5, 0.5, 1.0, -1.0]
    for lo, hi in ((-127.0, -125.0), (126.5, 128.5), (-130.0, 129.0), (-1.0, 1.0), (-40.0, 2.0)):
        x = lo + (hi - lo) * torch.rand(n, device=dev, generator=g)
        x = torch.cat([torch.tensor(special, device=dev).repeat_interleave(8), x])[:n].float()
        lse = torch.full((n, heads), math.inf, device=dev)
        col = (row * 37 + row // 8) % 128
        col[:8 * len(special)] = (row % 8)[:8 * len(special)]  # every special value in 8 columns
        lse[row, col] = -x
        w = torch.zeros(pages, 1, page, device=dev)
        assert bridge_lib.cb_paged_attention_weights(C.byref(kv), ptr(q), q.stride(0), heads, 1.0,
                                                     ptr(lse), ptr(w), stream()) == 0
        torch.cuda.synchronize()
        got = w[own.long(), 0]
        assert bool(((got == got[:, :1]) | got.isnan()).all())  # all slots of a page alike
        got = got[:, 0]
        nan = x.isnan()
        assert bool(got[nan].isnan().all()) and not bool(got[~nan].isnan().any())
        assert bool((got[x < -126.0] == 0).all())
        assert bool(torch.isinf(got[x >= 128.001]).all())
        usual = (x >= -126.0) & (x <= 127.5)
        want = torch.exp2(x.double())
        error = ((got.double() - want).abs() / want)
        assert float(error[usual].max()) <= 3.4e-7
        top = (x > 127.5) & (x < 128.0)
        if bool(top.any()):
            assert float(error[top].max()) <= 7e-5


# ----------------------------------------------------------- bounds wider than what there is
@pytest.mark.parametrize("lens,news,heads,kv_heads,page", [
    ([700, 3, 0, 259], [1, 1, 0, 1], 8, 2, 32), ([400, 129, 64, 2], [129, 0, 1, 2], 4, 4, 128),
    ([5000, 20, 3000], [1, 1, 2], 8, 4, 16), ([90, 0, 17], [0, 0, 0], 4, 2, 16)])
def test_a_step_below_the_descriptors_bounds(bridge_lib, lens, news, heads, kv_heads, page):
    """What a graph captured for larger steps meets: max_len, max_new, rows and the table's rows
    far above the step's, ids behind a sequence's pages outside the pool. Up to a step in
    which no sequence has a token."""
    c = Cache(lens, news, heads, kv_heads, page, "bf16", seed=7, pad=600, max_len=40000, max_new=512,
              table_stride=40000 // page + 1)
    total, scale = c.starts[-1], 128 ** -0.5
    q = c.tokens(heads * 128)
    out = torch.full((c.rows, heads * 128), 3.0, device="cuda", dtype=c.dt)
    lse = torch.full((c.rows, heads), 3.0, device="cuda")
    assert R.attention(bridge_lib, c, q, scale, out, lse) == 0
    want, want_lse, tol, lse_tol = R.attention_ref(c, q, scale)
    over = (out[:total].unflatten(1, (heads, 128)).double() - want).abs() - tol
    assert total == 0 or float(over.max()) <= 0
    assert total == 0 or float(((lse[:total].double() - want_lse).abs() - lse_tol).max()) <= 0
    assert bool((out[total:] == 3.0).all()) and bool((lse[total:] == 3.0).all())
    w = torch.rand(c.pages, kv_heads, page, device="cuda")
    ref, w_tol = R.weights_ref(c, q, scale, lse, w)
    d = c.desc()
    assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), heads, scale,
                                                 ptr(lse), ptr(w), stream()) == 0
    torch.cuda.synchronize()
    assert float(((w.double() - ref).abs() - w_tol).max()) <= 0
    # append and evict of the same step: rows, and slots behind the sequences, as they were
    k, v = c.tokens(kv_heads * 128), c.tokens(kv_heads * 128)
    pool = c.k.clone()
    q_out = torch.full_like(q, 3.0)
    assert bridge_lib.cb_paged_append(C.byref(d), None, heads, ptr(q), q.stride(0), ptr(q_out),
                                      q_out.stride(0), ptr(k), k.stride(0), ptr(v), v.stride(0),
                                      None, None, None, stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(q_out[:total], q[:total]) and bool((q_out[total:] == 3.0).all())
    for b in range(c.batch):
        at = c.place(b, torch.arange(lens[b] - news[b], lens[b], device="cuda"))
        rows = k[c.starts[b]:c.starts[b + 1]].unflatten(1, (kv_heads, 128))
        for h in range(kv_heads):
            pool[at[0], h, at[1]] = rows[:, h]
    assert torch.equal(c.k.view(torch.int16), pool.view(torch.int16))
    p = torch.zeros(w.shape, device="cuda", dtype=torch.int32)
    lo = torch.full_like(c.len, -1)
    assert _evict(bridge_lib, c, w, w, p, p, c.len, 40000, 0, 0, lo) == 0
    assert lo.tolist() == lens and torch.equal(c.k.view(torch.int16), pool.view(torch.int16))


FIRST_CALLS = """
import ctypes as C, sys, torch
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import paged_ref as R
from paged_ref import Cache, ptr
from rustane_b200 import bridge as B
lib = B.load_library()
for lens, news, heads in (([300, 40], [1, 1], 4), ([300, 140], [120, 33], 4)):
    c = Cache(lens, news, heads, 2, 16, "f16")
    q, k, v = c.tokens(512), c.tokens(256), c.tokens(256)
    out, q_out = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.zeros(c.rows, heads, device="cuda")
    w = torch.zeros(c.pages, 2, 16, device="cuda")
    p = torch.zeros(c.pages, 2, 16, device="cuda", dtype=torch.int32)
    pos = torch.zeros(c.rows, device="cuda", dtype=torch.int32)
    inv = torch.ones(64, device="cuda", dtype=torch.float64)
    lo = torch.zeros_like(c.len)
    d, size, esize = c.desc(), C.c_size_t(), C.c_size_t()
    assert lib.cb_paged_attention_workspace(C.byref(d), heads, C.byref(size)) == 0
    assert lib.cb_paged_evict_workspace(C.byref(d), 64, C.byref(esize)) == 0
    ws = torch.zeros(size.value + esize.value + 64, dtype=torch.uint8, device="cuda")
    ews = ws[-(-size.value // 16) * 16:]
    rope = B.cb_rope_config(inv.data_ptr(), 128, B.CB_ROPE_HALF, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.cb_rope(C.byref(rope), 1, ptr(q), 512, ptr(out), 512, ptr(pos), c.rows, 4, 128, 0, st) == 0
        assert lib.cb_paged_append(C.byref(d), C.byref(rope), heads, ptr(q), 512, ptr(q_out), 512, ptr(k),
                                   256, ptr(v), 256, None, ptr(w), ptr(p), st) == 0
        assert lib.cb_paged_attention(C.byref(d), ptr(q_out), 512, heads, 0.1, ptr(out), 512, ptr(lse),
                                      ptr(ws), size.value, st) == 0
        assert lib.cb_paged_attention_weights(C.byref(d), ptr(q_out), 512, heads, 0.1, ptr(lse), ptr(w), st) == 0
        assert lib.cb_paged_evict(C.byref(d), ptr(w), ptr(w), ptr(p), ptr(p), ptr(c.len), 64, 0, 0,
                                  ptr(lo), ptr(ews), esize.value, st) == 0
    graph.replay()
    torch.cuda.synchronize()
    assert lo.tolist() == [min(n, 64) for n in lens]
    total = c.starts[-1]
    got = out[:total].unflatten(1, (heads, 128)).double()
    assert bool(torch.isfinite(got).all()) and float(got.abs().max()) > 0
    assert bool(torch.isfinite(lse[:total]).all())
print("captured first calls: fine")
"""


def test_the_first_calls_of_a_process_may_be_captured(bridge_lib):
    """No call needs one outside a capture before it."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=root)], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
