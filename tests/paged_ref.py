"""Plain 64-bit forms of the paged-cache operators, and caches to try them on.

A case's cache is poisoned: every slot that belongs to no sequence (unused pages, slots
behind a sequence's end) holds NaN, and so do the padding rows of the token arrays, so
whatever reads one of them shows.
"""
import ctypes as C
import math

import torch

from rustane_b200 import bridge as B

HD = 128
LOG2E = math.log2(math.e)
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f16": B.CB_DTYPE_F16, "bf16": B.CB_DTYPE_BF16}


class Cache:
    """Pages, table, lengths and a step's rows on the GPU, and the descriptor of them."""

    def __init__(self, lens, news, heads, kv_heads, page, dtype="f16", seed=0, pad=3,
                 max_len=None, max_new=None, spare=2, table_stride=None, dev="cuda"):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.dtype, self.dt, self.dev = dtype, DTYPES[dtype], dev
        self.lens, self.news, self.heads, self.kv_heads, self.page = lens, news, heads, kv_heads, page
        self.batch = len(lens)
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        stride = table_stride or max(1, max(need))
        order = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        rows = [[order.pop() for _ in range(n)] for n in need]
        self.page_lists = rows
        # ids behind a sequence's pages are not to be read: ones far outside the pool
        self.table = torch.tensor([r + [1 << 30] * (stride - len(r)) for r in rows],
                                  dtype=torch.int32, device=dev)
        self.len = torch.tensor(lens, dtype=torch.int32, device=dev)
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.row_start = torch.tensor(starts, dtype=torch.int32, device=dev)
        self.rows = starts[-1] + pad
        shape = (self.pages, kv_heads, page, HD)
        self.k = torch.randn(shape, generator=g, device=dev).to(self.dt)
        self.v = torch.randn(shape, generator=g, device=dev).to(self.dt)
        live = torch.zeros(self.pages, page, dtype=torch.bool, device=dev)
        for r, n in zip(rows, lens):
            for j, p in enumerate(r):
                live[p, :max(0, min(page, n - j * page))] = True
        self.live = live[:, None, :].expand(-1, kv_heads, -1)
        self.k[~self.live] = math.nan
        self.v[~self.live] = math.nan
        self.max_len = max_len or max(1, max(lens))
        self.max_new = max(news) if max_new is None else max_new
        self.gen = g

    def desc(self):
        return B.cb_paged_kv(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(),
                             self.len.data_ptr(), self.row_start.data_ptr(), CODES[self.dtype],
                             self.pages, self.kv_heads, self.page, self.batch,
                             self.table.shape[1], self.max_len, self.rows, self.max_new)

    def tokens(self, width, stride=None, scale=1.0):
        """A token array [rows, width] inside rows of `stride` elements; padding is NaN."""
        wide = torch.full((max(1, self.rows), stride or width), math.nan, device=self.dev, dtype=self.dt)
        x = wide[:self.rows, :width]
        x[:self.starts[-1]] = (torch.randn(self.starts[-1], width, generator=self.gen,
                                           device=self.dev) * scale).to(self.dt)
        return x

    def slots(self, pool, b, head):
        """The slots of a sequence, in order."""
        pages = torch.tensor(self.page_lists[b], dtype=torch.long, device=self.dev)
        return pool[pages, head].flatten(0, 1)[:self.lens[b]]

    def place(self, b, slots):
        pages = torch.tensor(self.page_lists[b], dtype=torch.long, device=self.dev)
        return pages[slots // self.page], slots % self.page


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def attention(lib, c, q, scale, out, lse=None, st=None):
    d = c.desc()
    size = C.c_size_t()
    rc = lib.cb_paged_attention_workspace(C.byref(d), c.heads, C.byref(size))
    if rc:
        return rc
    # exactly as long as asked for, with bytes behind it that must survive
    ws = torch.full((size.value + 64,), 0x5a, dtype=torch.uint8, device=c.dev)
    rc = lib.cb_paged_attention(C.byref(d), ptr(q), q.stride(0), c.heads, scale, ptr(out),
                                out.stride(0), ptr(lse), ptr(ws), size.value, st or stream())
    torch.cuda.synchronize()
    assert bool((ws[size.value:] == 0x5a).all())
    return rc


def scores(c, q, b, head, scale, group):
    """Scaled scores [group, n, len] of a sequence's rows in 64 bits, -inf where unseen, and
    the largest sum of the magnitudes of a dot product's terms."""
    n, length = c.news[b], c.lens[b]
    qs = q[c.starts[b]:c.starts[b] + n].double().view(n, -1, HD)[:, head * group:(head + 1) * group]
    k = c.slots(c.k, b, head).double()
    x = torch.einsum("igd,td->git", qs, k) * scale
    size = torch.einsum("igd,td->git", qs.abs(), k.abs()) * scale
    i = torch.arange(n, device=q.device)[:, None]
    t = torch.arange(length, device=q.device)[None]
    unseen = t > length - n + i
    return x.masked_fill(unseen, -math.inf), size.masked_fill(unseen, 0.0).amax(-1)


def attention_ref(c, q, scale):
    """out and lse of the valid rows in 64 bits, and how far a right kernel may be off."""
    group = c.heads // c.kv_heads
    total = c.starts[-1]
    half = torch.finfo(c.dt).eps / 2
    out = torch.zeros(total, c.heads, HD, dtype=torch.float64, device=q.device)
    lse = torch.full((total, c.heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(c.batch):
        n = c.news[b]
        if n == 0 or c.lens[b] == 0:
            continue
        span = slice(c.starts[b], c.starts[b] + n)
        for head in range(c.kv_heads):
            x, size = scores(c, q, b, head, scale, group)
            v = c.slots(c.v, b, head).double()
            m = x.amax(-1, keepdim=True)
            m = torch.where(m == -math.inf, 0.0, m)
            p = torch.exp(x - m)
            s = p.sum(-1, keepdim=True)
            hs = slice(head * group, (head + 1) * group)
            w = torch.where(s > 0, p / s, 0.0)
            o = w @ v
            out[span, hs] = o.transpose(0, 1)
            lse[span, hs] = ((torch.log(s) + m) * LOG2E).squeeze(-1).T
            # a score is off by its accumulation (eight steps of the matrix unit, each within
            # 2^-22 of the sum of magnitudes) and, scaled and shifted in 32 bits, by 2^-20
            delta = (size * 2.0 ** -19 + 2.0 ** -20 * (1 + m.squeeze(-1).abs()))[..., None]
            spread = w @ v.abs()
            # rounding of the output and of the weights; weights below the type's normal range
            # (fp16) lose up to 2^-25 of the largest one each
            t = half * o.abs() + (half + 2 * delta + 2.0 ** -18) * spread
            if c.dt == torch.float16:
                t = t + 2.0 ** -25 * (x.shape[-1] * v.abs().amax() + 1)
            tol[span, hs] = t.transpose(0, 1)
            lse_tol[span, hs] = (delta.squeeze(-1) * LOG2E + 2.0 ** -19).T
    return out, lse, tol, lse_tol


def weights_ref(c, q, scale, lse, weights):
    """The running sums after a step, and how far a right kernel may be off."""
    group = c.heads // c.kv_heads
    w = weights.double().clone()
    tol = weights.double().abs() * 2.0 ** -23
    for b in range(c.batch):
        n = c.news[b]
        if n == 0 or c.lens[b] == 0:
            continue
        span = slice(c.starts[b], c.starts[b] + n)
        for head in range(c.kv_heads):
            x, size = scores(c, q, b, head, scale, group)
            lg = lse[span, head * group:(head + 1) * group].double().T
            seen = x > -math.inf
            p = torch.where(seen, torch.exp2(x * LOG2E - lg[..., None]), 0.0)
            delta = (size * 2.0 ** -19 + 2.0 ** -19 * (1 + lg.abs()))[..., None]
            at = c.place(b, torch.arange(c.lens[b], device=q.device))
            w[at[0], head, at[1]] += p.sum((0, 1))
            # each term, and the additions of group * n terms in 32 bits
            tol[at[0], head, at[1]] += (p * (delta + 2.0 ** -20)).sum((0, 1)) + \
                p.sum((0, 1)) * (8 + group * n) * 2.0 ** -24
    return w, tol


def rotate_ref(x, positions, inv_freq, amplitude, layout, rot, inverse=False):
    """x [tokens, heads, hd] turned in 64 bits, and the sum of both terms' magnitudes."""
    a = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(a)[:, None] * amplitude, torch.sin(a)[:, None] * amplitude
    s = -s if inverse else s
    y, size = x.double().clone(), x.double().abs()
    i = torch.arange(rot // 2, device=x.device)
    i0, i1 = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    x0, x1 = x.double()[..., i0], x.double()[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    size[..., i0] = size[..., i1] = abs(amplitude) * (x0.abs() + x1.abs())
    return y, size


def rotate_tol(y, size, dt):
    """Rounding to the type (fp16: or half its smallest step), and cos, sin and two products
    in 32 bits."""
    least = 2.0 ** -25 if dt == torch.float16 else 0.0
    return torch.finfo(dt).eps / 2 * y.abs() + 2.0 ** -21 * size + least


def evict_ref(c, weights, positions, next_position, budget, sinks, recent):
    """keep order and moves of every sequence and head: {(b, head): (sources of the slots
    below the new length)}."""
    result = {}
    for b in range(c.batch):
        n = c.lens[b]
        new = min(n, budget)
        slots = list(range(n))
        for head in range(c.kv_heads):
            w = c.slots(weights, b, head).double().cpu().tolist()
            p = c.slots(positions, b, head).cpu().tolist()
            if n <= budget:
                result[b, head] = slots
                continue
            nxt = int(next_position[b])

            def order(s):
                must = p[s] < sinks or (recent > 0 and p[s] >= nxt - recent)
                nan = math.isnan(w[s])
                return (0 if must else 2 if nan else 1, 0.0 if must or nan else -w[s], s)
            keep = set(sorted(slots, key=order)[:new])
            movers = [s for s in slots[new:] if s in keep]
            source = []
            for s in range(new):
                source.append(s if s in keep else movers.pop(0))
            assert not movers
            result[b, head] = source
    return result
