"""GPU tests of the paged-cache operators against 64-bit forms (tests/paged_ref.py), whose
tolerances are derived there."""
import ctypes as C
import math

import pytest
import torch

import paged_ref as R
from paged_ref import Cache, ptr, stream
from rustane_b200 import bridge as B

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert not bool(torch.isnan(got).any()), f"{what}: NaN"
    inf = torch.isinf(want)
    assert bool((got[inf] == want[inf]).all()), f"{what}: infinities differ"
    over = ((got - want).abs() - tol)[~inf]
    assert over.numel() == 0 or float(over.max()) <= 0.0, \
        f"{what}: off by {float((got - want).abs()[~inf].max()):.3g}, over the bound by {float(over.max()):.3g}"


# ------------------------------------------------------------------------------- rope
def _inv(rot, scaling=0):
    lib = B.load_library()
    s = B.cb_rope_scaling(10000.0, scaling, 8.0, 4096.0, 32.0, 1.0)
    inv, amp = (C.c_double * (rot // 2))(), C.c_float()
    assert lib.cb_rope_frequencies(rot, C.byref(s), inv, C.byref(amp)) == 0
    return torch.tensor(list(inv), dtype=torch.float64, device="cuda"), amp.value


LAYOUT = {"half": B.CB_ROPE_HALF, "interleaved": B.CB_ROPE_INTERLEAVED}


def _rope(lib, x, y, pos, inv, amp, layout, rot, inverse, hd, dtype, st=None):
    t, w = x.shape
    cfg = B.cb_rope_config(inv.data_ptr(), rot, LAYOUT[layout], amp)
    return lib.cb_rope(C.byref(cfg), R.CODES[dtype], ptr(x), x.stride(0), ptr(y), y.stride(0),
                       ptr(pos), t, w // hd, hd, int(inverse), st or stream())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,tokens,heads,hd,rot,scaling,far", [
    ("f16", 1, 1, 8, 8, 0, 10),
    ("bf16", 3, 5, 64, 24, 1, 5000),
    ("f16", 129, 7, 128, 128, 0, 2_000_000),
    ("bf16", 257, 12, 128, 64, 3, 2_000_000),
    ("f16", 65, 3, 96, 96, 2, 100_000),
    ("bf16", 33, 2, 512, 512, 3, 2 ** 31 - 1),
    ("f16", 4096, 32, 128, 128, 3, 32768),   # enough work for four heads a thread
    ("bf16", 2048, 53, 128, 120, 0, 32768),  # a head count that four does not divide
])
def test_rope_and_its_gradient(bridge_lib, layout, dtype, tokens, heads, hd, rot, scaling, far):
    dt = R.DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(tokens + rot)
    inv, amp = _inv(rot, scaling)
    x = torch.randn(tokens, heads * hd + 16, device="cuda", generator=g).to(dt)[:, :heads * hd]
    pos = torch.randint(-far, far, (tokens,), device="cuda", generator=g).int()
    wide = torch.full((tokens, heads * hd + 24), 7.0, device="cuda", dtype=dt)
    y = wide[:, :heads * hd]
    for inverse in (False, True):
        assert _rope(bridge_lib, x, y, pos, inv, amp, layout, rot, inverse, hd, dtype) == 0
        torch.cuda.synchronize()
        want, size = R.rotate_ref(x.unflatten(1, (heads, hd)), pos, inv, amp, layout, rot, inverse)
        close(y.unflatten(1, (heads, hd)), want, R.rotate_tol(want, size, dt), f"inverse {inverse}")
        assert bool((wide[:, heads * hd:] == 7.0).all())
    in_place = x.clone()
    assert _rope(bridge_lib, in_place, in_place, pos, inv, amp, layout, rot, True, hd, dtype) == 0
    torch.cuda.synchronize()
    assert torch.equal(in_place, y)


def test_rope_gradient_is_the_transpose_and_agrees_with_differences(bridge_lib):
    """<R x, g> = <x, R^T g>, and the change of <R x, g> along a direction d is <d, R^T g>."""
    g = torch.Generator(device="cuda").manual_seed(3)
    inv, amp = _inv(64, 3)
    x, up, d = (torch.randn(50, 4 * 128, device="cuda", generator=g).half() for _ in range(3))
    pos = torch.randint(0, 100_000, (50,), device="cuda", generator=g).int()

    def run(a, inverse):
        y = torch.empty_like(a)
        assert _rope(bridge_lib, a, y, pos, inv, amp, "half", 64, inverse, 128, "f16") == 0
        return y.double()
    back = run(up, True)
    # both products round once per element: half a step of each of 25600 terms
    terms = (run(x, False) * up.double()).abs().sum() + (x.double() * back).abs().sum()
    assert abs((run(x, False) * up.double()).sum() - (x.double() * back).sum()) <= terms * 2.0 ** -11
    moved = (x.double() + d.double()).half()
    step = moved.double() - x.double()  # exact: the step that was taken
    change = ((run(moved, False) - run(x, False)) * up.double()).sum()
    terms = ((run(moved, False).abs() + run(x, False).abs()) * up.double().abs()).sum() \
        + (step * back).abs().sum()
    assert abs(change - (step * back).sum()) <= terms * 2.0 ** -11


def test_rope_matches_the_model_table(bridge_lib):
    """Interleaved, whole head, base 10000: the rotation that the model's forward uses."""
    inv, amp = _inv(128)
    t = torch.arange(512, device="cuda", dtype=torch.int32)
    x = torch.zeros(512, 128, device="cuda", dtype=torch.float16)
    x[:, 0::2] = 1.0
    y = torch.empty_like(x)
    assert _rope(bridge_lib, x, y, t, inv, amp, "interleaved", 128, False, 128, "f16") == 0
    i = torch.arange(64, device="cuda", dtype=torch.float64)
    a = t.double()[:, None] * 10000.0 ** (-2 * i / 128)
    torch.cuda.synchronize()
    assert float((y[:, 0::2].double() - torch.cos(a)).abs().max()) <= 2.0 ** -11
    assert float((y[:, 1::2].double() - torch.sin(a)).abs().max()) <= 2.0 ** -11


# ----------------------------------------------------------------------------- append
def _append(lib, c, rope, q, q_out, k, v, pos=None, w=None, sp=None, heads=None, st=None):
    d = c.desc()
    return lib.cb_paged_append(C.byref(d), C.byref(rope) if rope else None,
                               c.heads if heads is None else heads, ptr(q),
                               q.stride(0) if q is not None else 0, ptr(q_out),
                               q_out.stride(0) if q_out is not None else 0, ptr(k), k.stride(0),
                               ptr(v), v.stride(0), ptr(pos), ptr(w), ptr(sp), st or stream())


APPENDS = [
    # lens, news, heads, kv_heads, page, dtype, layout, rot, explicit positions
    ([1], [1], 1, 1, 16, "f16", "half", 128, False),
    ([5, 16, 17], [5, 1, 0], 4, 2, 16, "bf16", "interleaved", 128, True),
    ([100, 33, 1, 64], [37, 33, 0, 1], 8, 1, 32, "f16", "half", 40, True),
    ([300, 129], [300, 64], 6, 6, 128, "bf16", "half", 64, False),
    ([40 + i for i in range(70)], [i % 3 for i in range(70)], 3, 3, 64, "f16", "interleaved", 8, True),
    ([900, 1024, 700], [900, 1000, 640], 16, 16, 64, "bf16", "half", 128, True),
]


@pytest.mark.parametrize("lens,news,heads,kv_heads,page,dtype,layout,rot,explicit", APPENDS)
def test_append(bridge_lib, lens, news, heads, kv_heads, page, dtype, layout, rot, explicit):
    c = Cache(lens, news, heads, kv_heads, page, dtype, seed=len(lens) + heads)
    total = c.starts[-1]
    qkv = c.tokens((heads + 2 * kv_heads) * 128, stride=(heads + 2 * kv_heads) * 128 + 8)
    q, k, v = qkv.split([heads * 128, kv_heads * 128, kv_heads * 128], 1)
    q_out = torch.full((c.rows, heads * 128), 5.0, device="cuda", dtype=c.dt)
    inv, amp = _inv(rot, 3)
    rope = B.cb_rope_config(inv.data_ptr(), rot, LAYOUT[layout], amp)
    slots = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).int().cuda()
    pos = slots + 100_003 if explicit else slots
    given = torch.cat([pos, pos[:1].expand(c.rows - total)]).contiguous() if explicit else None
    w = torch.full((c.pages, kv_heads, page), 3.0, device="cuda")
    sp = torch.full((c.pages, kv_heads, page), -7, device="cuda", dtype=torch.int32)
    k0, v0 = c.k.clone(), c.v.clone()
    assert _append(bridge_lib, c, rope, q, q_out, k, v, given, w, sp) == 0
    torch.cuda.synchronize()

    def want(x, h):
        y, size = R.rotate_ref(x[:total].unflatten(1, (h, 128)), pos, inv, amp, layout, rot)
        return y, R.rotate_tol(y, size, c.dt)
    close(q_out[:total].unflatten(1, (heads, 128)), *want(q, heads), "q")
    assert bool((q_out[total:] == 5.0).all())  # padding
    want_k, tol_k = want(k, kv_heads)
    touched = torch.zeros(c.pages, kv_heads, page, dtype=torch.bool, device="cuda")
    for b in range(c.batch):
        span = slice(c.starts[b], c.starts[b + 1])
        at = c.place(b, torch.arange(lens[b] - news[b], lens[b], device="cuda"))
        for h in range(kv_heads):
            close(c.k[at[0], h, at[1]], want_k[span, h], tol_k[span, h], "k")
            assert torch.equal(c.v[at[0], h, at[1]], v[span].unflatten(1, (kv_heads, 128))[:, h])
            assert bool((w[at[0], h, at[1]] == 0).all())
            assert torch.equal(sp[at[0], h, at[1]], pos[span])
            touched[at[0], h, at[1]] = True
    for pool, before in ((c.k, k0), (c.v, v0)):
        assert torch.equal(torch.nan_to_num(pool[~touched], 9.0), torch.nan_to_num(before[~touched], 9.0))
    assert bool((w[~touched] == 3.0).all()) and bool((sp[~touched] == -7).all())


def test_append_in_place_without_rotation_and_without_q(bridge_lib):
    c = Cache([30, 9], [7, 9], 4, 2, 16, "f16", seed=2)
    total = c.starts[-1]
    q, k, v = c.tokens(512), c.tokens(256), c.tokens(256)
    q0 = q.clone()
    inv, amp = _inv(128)
    rope = B.cb_rope_config(inv.data_ptr(), 128, B.CB_ROPE_HALF, amp)
    apart = torch.zeros_like(q)
    assert _append(bridge_lib, c, rope, q, apart, k, v) == 0
    k_turned = c.k.clone()
    assert _append(bridge_lib, c, rope, q, q, k, v) == 0
    torch.cuda.synchronize()
    assert torch.equal(q[:total], apart[:total]) and bool(q[total:].isnan().all())
    assert _append(bridge_lib, c, rope, None, None, k, v, heads=0) == 0
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(c.k), torch.nan_to_num(k_turned))
    assert _append(bridge_lib, c, None, q0, q, k, v) == 0
    torch.cuda.synchronize()
    assert torch.equal(q[:total], q0[:total])
    at = c.place(1, torch.arange(9, device="cuda"))
    assert torch.equal(c.k[at[0], 1, at[1]], k[7:16, 128:])


# -------------------------------------------------------------------------- attention
ATTENTION = [
    # lens, news, heads, kv_heads, page
    ([1], [1], 1, 1, 16),
    ([17], [1], 2, 1, 16),
    ([5], [5], 1, 1, 16),
    ([64, 1, 33, 128], [1, 1, 1, 1], 12, 12, 16),
    ([700, 3, 0, 259], [1, 1, 0, 1], 8, 2, 32),
    ([513], [1], 32, 1, 64),             # 32 query heads to one key head
    ([40, 90, 300], [3, 0, 5], 6, 2, 32),
    ([130, 77], [130, 20], 5, 1, 16),    # a whole prompt, five heads to a key head
    ([400, 129, 64, 2], [129, 129, 1, 2], 4, 4, 128),
    ([1000, 1500], [200, 333], 7, 1, 64),
    ([9000], [1], 4, 4, 64),             # split over many parts
    ([5000, 20, 3000], [1, 1, 2], 8, 4, 16),
    ([4100, 260], [150, 256], 8, 2, 32),  # split with many rows
    ([65, 64, 63] * 30, [1] * 90, 2, 2, 16),
    ([300] * 40, [i % 4 for i in range(40)], 3, 1, 16),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,news,heads,kv_heads,page", ATTENTION)
def test_attention(bridge_lib, lens, news, heads, kv_heads, page, dtype):
    c = Cache(lens, news, heads, kv_heads, page, dtype, seed=heads + len(lens))
    total = c.starts[-1]
    q = c.tokens(heads * 128, stride=heads * 128 + 64, scale=1.5)
    wide = torch.full((c.rows, heads * 128 + 40), 3.0, device="cuda", dtype=c.dt)
    out = wide[:, :heads * 128]
    lse = torch.full((c.rows, heads), 3.0, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    want, want_lse, tol, lse_tol = R.attention_ref(c, q, SCALE)
    close(out[:total].unflatten(1, (heads, 128)), want, tol, "out")
    close(lse[:total], want_lse, lse_tol, "lse")
    assert bool((out[total:] == 3.0).all()) and bool((lse[total:] == 3.0).all())
    assert bool((wide[:, heads * 128:] == 3.0).all())
    # the same call without lse, and the same bits again
    again = torch.full((c.rows, heads * 128), 3.0, device="cuda", dtype=c.dt)
    assert R.attention(bridge_lib, c, q, SCALE, again) == 0
    assert torch.equal(again, out)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_rows_without_slots(bridge_lib, new):
    """A sequence whose length is below its new tokens: the first rows see nothing."""
    c = Cache([50, 50], [new, new], 4, 2, 16, "f16", seed=4)
    c.len[0] = new - 1  # token 0 sees no slot
    c.lens[0] = new - 1
    q = c.tokens(512)
    out = torch.full((c.rows, 512), 3.0, device="cuda", dtype=c.dt)
    lse = torch.full((c.rows, 4), 3.0, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    live = torch.isfinite(lse[:2 * new]).all(1)
    assert live.tolist() == [False] + [True] * (2 * new - 1)
    assert not bool(out[:2 * new].isnan().any())


@pytest.mark.parametrize("new", [1, 70])
def test_attention_skips_pages_outside_the_pool(bridge_lib, new):
    """Page ids outside 0 .. pages - 1 stand for absent slots: the result is that of a cache
    without them."""
    c = Cache([96], [new], 4, 2, 16, "bf16", seed=5)
    q = c.tokens(512)
    c.table[0, 1], c.table[0, 3] = -5, c.pages
    out = torch.zeros(c.rows, 512, device="cuda", dtype=c.dt)
    lse = torch.zeros(c.rows, 4, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    absent = torch.zeros(96, dtype=torch.bool, device="cuda")
    absent[16:32] = absent[48:64] = True
    for head in range(2):
        x, size = R.scores(c, q, 0, head, SCALE, 2)
        x = x.masked_fill(absent, -math.inf)
        w = torch.softmax(x, -1)
        v = c.slots(c.v, 0, head).double()
        want = (w @ v).transpose(0, 1)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * (w @ v.abs()).transpose(0, 1)
        close(out[:new].unflatten(1, (4, 128))[:, head * 2:head * 2 + 2], want, tol)


def test_attention_holds_to_the_descriptor(bridge_lib):
    """Lengths above max_len, more new tokens than max_new and row starts out of range: what
    lies behind the bounds is left alone."""
    c = Cache([64, 64], [4, 4], 2, 2, 16, "f16", seed=6, max_len=64, max_new=2)
    q = c.tokens(256)
    good = torch.full((c.rows, 256), 3.0, device="cuda", dtype=c.dt)
    assert R.attention(bridge_lib, c, q, SCALE, good) == 0
    assert bool((good[2:4] == 3.0).all()) and bool((good[6:] == 3.0).all())
    assert not bool((good[[0, 1, 4, 5]] == 3.0).all(1).any())
    c.len[:] = 2 ** 31 - 1
    c.row_start[:] = torch.tensor([-9, 4, 2 ** 31 - 1], dtype=torch.int32)
    out = torch.full((c.rows, 256), 3.0, device="cuda", dtype=c.dt)
    assert R.attention(bridge_lib, c, q, SCALE, out) == 0
    assert bool((out[[2, 3, 6, 7]] == 3.0).all())


def test_attention_extreme_scores(bridge_lib):
    """Scores of thousands, one key far above the others, and equal keys."""
    c = Cache([200, 200, 200], [1, 1, 17], 2, 1, 16, "f16", seed=7)
    q = c.tokens(256, scale=8.0)
    at = c.place(0, torch.arange(200, device="cuda"))
    c.k[at[0], 0, at[1]] *= 30
    at = c.place(1, torch.arange(200, device="cuda"))
    c.k[at[0], 0, at[1]] = 1.0
    at = c.place(2, torch.arange(150, 160, device="cuda"))
    c.k[at[0], 0, at[1]] *= 60
    out = torch.zeros(c.rows, 256, device="cuda", dtype=c.dt)
    lse = torch.zeros(c.rows, 2, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    want, want_lse, tol, lse_tol = R.attention_ref(c, q, SCALE)
    total = c.starts[-1]
    close(out[:total].unflatten(1, (2, 128)), want, tol, "out")
    close(lse[:total], want_lse, lse_tol, "lse")


# ---------------------------------------------------------------------------- weights
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,news,heads,kv_heads,page", ATTENTION)
def test_weights(bridge_lib, lens, news, heads, kv_heads, page, dtype):
    c = Cache(lens, news, heads, kv_heads, page, dtype, seed=heads + len(lens))
    q = c.tokens(heads * 128, stride=heads * 128 + 64, scale=1.5)
    _, lse64, _, _ = R.attention_ref(c, q, SCALE)
    lse = torch.full((c.rows, heads), math.nan, device="cuda")
    lse[:c.starts[-1]] = lse64.float()
    w = torch.rand(c.pages, kv_heads, page, device="cuda")
    before = w.clone()
    d = c.desc()
    assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), heads, SCALE,
                                                 ptr(lse), ptr(w), stream()) == 0
    torch.cuda.synchronize()
    want, tol = R.weights_ref(c, q, SCALE, lse, before)
    close(w, want, tol, "weights")
    assert torch.equal(w[~c.live], before[~c.live])
    w2 = before.clone()
    assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), heads, SCALE,
                                                 ptr(lse), ptr(w2), stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(w, w2)  # a fixed order of additions


@pytest.mark.parametrize("heads", [3, 5, 7, 100])
def test_weights_of_a_bad_key_stay_in_its_slot(bridge_lib, heads):
    """Groups that do not divide 128 leave rows of a step without a query; a key with NaN and
    infinities reaches its own slot's sum only."""
    c = Cache([600, 140], [150, 140], heads, 1, 32, "bf16", seed=heads)
    q = c.tokens(heads * 128, scale=1.5)
    _, lse64, _, _ = R.attention_ref(c, q, SCALE)
    lse = torch.zeros(c.rows, heads, device="cuda")
    lse[:c.starts[-1]] = lse64.float()
    d = c.desc()
    w = [torch.zeros(c.pages, 1, 32, device="cuda") for _ in range(2)]
    page = c.page_lists[0][1]
    for x in w:
        assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), heads, SCALE,
                                                     ptr(lse), ptr(x), stream()) == 0
        torch.cuda.synchronize()
        c.k[page, 0, 5, :64] = math.nan
        c.k[page, 0, 5, 64:] = math.inf
    assert bool(w[1][page, 0, 5].isnan()) and not bool(w[0].isnan().any())
    w[1][page, 0, 5] = w[0][page, 0, 5]
    assert torch.equal(w[0], w[1])


# ------------------------------------------------------------------------------ evict
def _evict(lib, c, w, wo, p, po, nxt, budget, sinks, recent, lo, st=None):
    d = c.desc()
    size = C.c_size_t()
    assert lib.cb_paged_evict_workspace(C.byref(d), budget, C.byref(size)) == 0
    ws = torch.full((size.value + 64,), 0x5a, dtype=torch.uint8, device="cuda")
    rc = lib.cb_paged_evict(C.byref(d), ptr(w), ptr(wo), ptr(p), ptr(po), ptr(nxt), budget, sinks,
                            recent, ptr(lo), ptr(ws), size.value, st or stream())
    torch.cuda.synchronize()
    assert bool((ws[size.value:] == 0x5a).all())
    return rc


EVICTS = [
    # lens, kv_heads, page, budget, sinks, recent, values of the weights
    ([1], 1, 16, 1, 0, 0, "random"),
    ([2], 1, 16, 1, 1, 0, "random"),
    ([33, 32, 31, 0], 2, 16, 32, 4, 8, "random"),
    ([100, 257, 40], 3, 32, 37, 0, 0, "equal"),
    ([513] * 5, 4, 16, 512, 4, 64, "random"),
    ([1000, 700], 2, 64, 300, 100, 200, "few"),
    ([1000, 700], 2, 64, 300, 0, 300, "odd"),
    ([1024, 1025], 2, 128, 1, 0, 0, "odd"),
    ([4096, 4097, 900], 1, 64, 2000, 4, 100, "few"),
    ([9000, 16384], 2, 128, 4000, 0, 64, "random"),
    ([20000], 1, 32, 19999, 8, 1000, "equal"),
    ([40000, 33000], 1, 128, 1000, 4, 0, "random"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,kv_heads,page,budget,sinks,recent,values", EVICTS)
def test_evict(bridge_lib, lens, kv_heads, page, budget, sinks, recent, values, in_place):
    c = Cache(lens, [0] * len(lens), kv_heads, kv_heads, page, "bf16", seed=sum(lens) + budget)
    shape = (c.pages, kv_heads, page)
    g = torch.Generator(device="cuda").manual_seed(budget)
    w = torch.rand(shape, device="cuda", generator=g)
    if values == "equal":
        w[:] = 0.25
    if values == "few":
        w = (w * 4).floor()
    if values == "odd":
        pick = torch.randint(0, 8, shape, device="cuda", generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, -1.5)):
            w[pick == i] = x
    p = torch.full(shape, -3, device="cuda", dtype=torch.int32)
    for b in range(c.batch):
        for h in range(kv_heads):
            at = c.place(b, torch.arange(lens[b], device="cuda"))
            p[at[0], h, at[1]] = torch.randperm(lens[b], device="cuda", generator=g).int() * 2
    nxt = c.len * 2
    wo = w if in_place else torch.full_like(w, 9.0)
    po = p if in_place else torch.full_like(p, 9)
    lo = torch.full_like(c.len, -1)
    before = {n: t.clone() for n, t in (("k", c.k), ("v", c.v), ("w", w), ("p", p), ("wo", wo), ("po", po))}
    moves = R.evict_ref(c, w, p, nxt, budget, sinks, recent)
    assert _evict(bridge_lib, c, w, wo, p, po, nxt, budget, sinks, recent, lo) == 0
    assert lo.tolist() == [min(n, budget) for n in lens]
    want = {n: before[n].clone() for n in ("k", "v", "wo", "po")}
    for (b, h), source in moves.items():
        to = c.place(b, torch.arange(len(source), device="cuda"))
        fro = c.place(b, torch.tensor(source, device="cuda", dtype=torch.long))
        for name, start in (("k", "k"), ("v", "v"), ("wo", "w"), ("po", "p")):
            want[name][to[0], h, to[1]] = before[start][fro[0], h, fro[1]]
    for name, got in (("k", c.k), ("v", c.v)):
        assert torch.equal(got.view(torch.int16), want[name].view(torch.int16)), name
    assert torch.equal(wo.view(torch.int32), want["wo"].view(torch.int32))
    assert torch.equal(po, want["po"])


def test_evict_with_pages_outside_the_pool(bridge_lib):
    """Absent slots go first and nothing is read from or written to them."""
    c = Cache([64, 64], [0, 0], 1, 1, 16, "f16", seed=9)
    w = torch.rand(c.pages, 1, 16, device="cuda") + 1
    p = torch.zeros(c.pages, 1, 16, device="cuda", dtype=torch.int32) + 50
    bad = int(c.table[0, 1])
    c.table[0, 1] = -1
    nxt = torch.full((2,), 1000, device="cuda", dtype=torch.int32)
    lo = torch.zeros_like(c.len)
    k0, w0 = c.k.clone(), w.clone()
    assert _evict(bridge_lib, c, w, w, p, p, nxt, 48, 0, 0, lo) == 0
    assert lo.tolist() == [48, 48]
    # the other 48 slots of sequence 0 stay: its holes are the absent ones, which take nothing
    for page in c.page_lists[0]:
        assert torch.equal(c.k[page], k0[page]) and torch.equal(w[page], w0[page])
    assert bad in c.page_lists[0]


@pytest.mark.parametrize("over", [1, 2, 7, 8, 9])
@pytest.mark.parametrize("budget,page", [(5, 16), (700, 16), (5000, 64), (20000, 128)])
def test_evict_of_a_few_slots(bridge_lib, over, budget, page):
    """Up to eight slots are looked for one by one, more of them by a threshold; equal
    weights, the highest slots of which go."""
    lens = [budget + over, budget, budget + 1]
    c = Cache(lens, [0] * 3, 2, 2, page, "f16", seed=over)
    g = torch.Generator(device="cuda").manual_seed(over)
    w = torch.randint(0, max(2, budget // 50), (c.pages, 2, page), device="cuda", generator=g).float()
    p = torch.randint(0, 10 * budget, w.shape, device="cuda", generator=g).int()
    nxt = torch.full((3,), 10 * budget, device="cuda", dtype=torch.int32)
    moves = R.evict_ref(c, w, p, nxt, budget, 1, budget // 4)
    lo = torch.zeros_like(c.len)
    k0, w0, p0 = c.k.clone(), w.clone(), p.clone()
    assert _evict(bridge_lib, c, w, w, p, p, nxt, budget, 1, budget // 4, lo) == 0
    assert lo.tolist() == [budget] * 3
    for (b, h), source in moves.items():
        to = c.place(b, torch.arange(len(source), device="cuda"))
        fro = c.place(b, torch.tensor(source, device="cuda", dtype=torch.long))
        k0[to[0], h, to[1]], w0[to[0], h, to[1]], p0[to[0], h, to[1]] = (
            x[fro[0], h, fro[1]].clone() for x in (k0, w0, p0))
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(w, w0) and torch.equal(p, p0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,news,heads,kv_heads,page", [
    ([40], [5], 3, 1, 16),               # the 16-row kernel
    ([300, 17], [4, 3], 4, 1, 32),
    ([500, 130], [200, 130], 4, 2, 16),  # the tcgen05 kernel: both tiles of a CTA
    ([3000], [300], 8, 1, 128),          # parts
])
def test_attention_keeps_what_a_row_does_not_see_out_of_it(bridge_lib, lens, news, heads,
                                                           kv_heads, page, dtype):
    """Infinities and NaN in K and V of new tokens reach the rows that see those tokens and no
    other row."""
    c = Cache(lens, news, heads, kv_heads, page, dtype, seed=11)
    q = c.tokens(heads * 128, scale=1.5)
    clean, clean_lse, tol, lse_tol = R.attention_ref(c, q, SCALE)
    bad = []  # (sequence, slot, element, value)
    for b in range(c.batch):
        n, length = news[b], lens[b]
        for k, (back, d, x) in enumerate([(0, 5, math.nan), (n // 3, 17, math.inf),
                                          (n // 2, 90, -math.inf), (n // 2, 91, math.nan)]):
            bad.append((b, length - 1 - back, d, x))
    for b, slot, d, x in bad:
        at = c.place(b, torch.tensor([slot], device="cuda"))
        c.v[at[0], :, at[1], d] = x
    out = torch.zeros(c.rows, heads * 128, device="cuda", dtype=c.dt)
    lse = torch.zeros(c.rows, heads, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    got = out[:c.starts[-1]].unflatten(1, (heads, 128))
    want = clean.clone()
    for b, slot, d, x in bad:
        first = slot - (lens[b] - news[b])  # the first token that sees it
        rows = slice(c.starts[b] + first, c.starts[b] + news[b])
        want[rows, :, d] += x
    odd = ~torch.isfinite(want)
    assert bool((torch.isnan(got) == torch.isnan(want)).all())
    assert bool((got[odd & ~torch.isnan(want)].double() == want[odd & ~torch.isnan(want)]).all())
    close(torch.where(odd, 0.0, got.double()), torch.where(odd, 0.0, want), tol, "out")
    close(lse[:c.starts[-1]], clean_lse, lse_tol, "lse")
    # K of the last token: only its own row sees it
    c.v[:] = torch.nan_to_num(c.v, 0.0, 0.0, 0.0)
    for b in range(c.batch):
        at = c.place(b, torch.tensor([lens[b] - 1], device="cuda"))
        c.k[at[0], :, at[1]] = math.nan
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    last = [c.starts[b + 1] - 1 for b in range(c.batch)]
    others = [r for r in range(c.starts[-1]) if r not in last]
    assert bool(out[last].isnan().all()) and not bool(out[others].isnan().any())
    assert not bool(lse[others].isnan().any())


# ------------------------------------------------------------------ how they are called
def test_more_sequences_than_are_added_up_at_a_time(bridge_lib):
    lens = [1 + (i * 37) % 50 for i in range(2500)]
    for news, heads in (([1] * 2500, 2), ([min(n, 1 + i % 20) for i, n in enumerate(lens)], 2)):
        c = Cache(lens, news, heads, 1, 16, "f16", seed=heads)
        q = c.tokens(heads * 128)
        out = torch.zeros(c.rows, heads * 128, device="cuda", dtype=c.dt)
        lse = torch.zeros(c.rows, heads, device="cuda")
        assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
        want, want_lse, tol, lse_tol = R.attention_ref(c, q, SCALE)
        close(out[:c.starts[-1]].unflatten(1, (heads, 128)), want, tol, "out")
        w = torch.zeros(c.pages, 1, 16, device="cuda")
        d = c.desc()
        assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), heads, SCALE,
                                                     ptr(lse), ptr(w), stream()) == 0
        want_w, tol_w = R.weights_ref(c, q, SCALE, lse, torch.zeros_like(w))
        torch.cuda.synchronize()
        close(w, want_w, tol_w, "weights")


@pytest.mark.parametrize("new", [1, 60])
def test_a_cache_of_more_than_2_to_the_31_elements(bridge_lib, new):
    """Every page in use lies behind element 2^31 of its array."""
    page, kv_heads = 64, 2
    pages = 2 ** 31 // (page * kv_heads * 128) + 100
    c = Cache([200], [new], 4, kv_heads, page, "f16", seed=3)
    far = torch.tensor([[pages - 5, pages - 1, pages - 17, pages - 3]], device="cuda", dtype=torch.int32)
    small_k, small_v = c.k, c.v
    c.k = torch.zeros(pages, kv_heads, page, 128, device="cuda", dtype=c.dt)
    c.v = torch.zeros_like(c.k)
    c.k[far[0].long()], c.v[far[0].long()] = small_k[c.page_lists[0]], small_v[c.page_lists[0]]
    c.table, c.page_lists, c.pages = far, [far[0].tolist()], pages
    q = c.tokens(512)
    out = torch.zeros(c.rows, 512, device="cuda", dtype=c.dt)
    lse = torch.zeros(c.rows, 4, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    want, want_lse, tol, lse_tol = R.attention_ref(c, q, SCALE)
    close(out[:new].unflatten(1, (4, 128)), want, tol, "out")
    d = c.desc()
    w = torch.zeros(pages, kv_heads, page, device="cuda")
    assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), 4, SCALE, ptr(lse),
                                                 ptr(w), stream()) == 0
    torch.cuda.synchronize()
    # every query row and head hands out a weight of one
    assert abs(float(w.double().sum()) - new * 4) < 1e-3 * new
    assert float(w[:pages - 20].abs().max()) == 0.0
    nk, nv = c.tokens(256), c.tokens(256)
    assert _append(bridge_lib, c, None, None, None, nk, nv, heads=0) == 0
    p = torch.arange(64, device="cuda", dtype=torch.int32).expand(pages, kv_heads, page).contiguous()
    lo = torch.zeros_like(c.len)
    assert _evict(bridge_lib, c, w, w, p, p, c.len, 100, 0, 0, lo) == 0
    at = c.place(0, torch.arange(200 - new, 200, device="cuda"))
    kept = at[0] * 0 + torch.arange(200 - new, 200, device="cuda") >= 100  # (others may be holes)
    assert torch.equal(c.v[at[0][kept], 1, at[1][kept]], nv[:new, 128:][kept])


def test_sequences_may_share_pages_for_attention(bridge_lib):
    """Two sequences with the same first pages; the weights of those collect from both."""
    c = Cache([70, 90], [1, 9], 4, 2, 16, "f16", seed=8)
    c.table[1, :3] = c.table[0, :3]
    c.page_lists[1][:3] = c.page_lists[0][:3]
    q = c.tokens(512)
    out = torch.zeros(c.rows, 512, device="cuda", dtype=c.dt)
    lse = torch.zeros(c.rows, 4, device="cuda")
    assert R.attention(bridge_lib, c, q, SCALE, out, lse) == 0
    want, _, tol, _ = R.attention_ref(c, q, SCALE)
    close(out[:10].unflatten(1, (4, 128)), want, tol)
    d = c.desc()
    w = torch.zeros(c.pages, 2, 16, device="cuda")
    assert bridge_lib.cb_paged_attention_weights(C.byref(d), ptr(q), q.stride(0), 4, SCALE, ptr(lse),
                                                 ptr(w), stream()) == 0
    want_w, tol_w = R.weights_ref(c, q, SCALE, lse, torch.zeros_like(w))
    torch.cuda.synchronize()
    close(w, want_w, tol_w + 2.0 ** -23 * want_w)


@pytest.mark.parametrize("seq,heads", [(512, 12), (320, 3)])
def test_a_prompt_through_pages_is_the_dense_attention(bridge_lib, seq, heads):
    """A whole prompt through the pages against the model's own attention kernel."""
    c = Cache([seq, seq], [seq, seq], heads, heads, 16, "f16", seed=1, pad=0)
    q = c.tokens(heads * 128)
    out = torch.zeros(c.rows, heads * 128, device="cuda", dtype=c.dt)
    assert R.attention(bridge_lib, c, q, SCALE, out) == 0
    dense = [q.view(2, seq, heads, 128).transpose(1, 2).contiguous()]
    for pool in (c.k, c.v):
        dense.append(torch.stack([torch.stack([c.slots(pool, b, h) for h in range(heads)])
                                  for b in range(2)]).contiguous())
    want = torch.empty_like(out)
    assert bridge_lib.cb_attention_f16(*(ptr(x) for x in dense), ptr(want), 2, heads, seq, stream()) == 0
    torch.cuda.synchronize()
    # both round their weights and their output to fp16
    _, _, tol, _ = R.attention_ref(c, q, SCALE)
    close(out, want, 2 * tol.flatten(1))


def test_pointers_that_are_not_device_memory_are_refused(bridge_lib):
    c = Cache([40], [2], 2, 1, 16, "f16")
    q = c.tokens(256)
    out = torch.zeros(c.rows, 256, device="cuda", dtype=c.dt)
    host = torch.zeros(c.rows, 256, dtype=c.dt)
    pinned = torch.zeros(c.rows, 256, dtype=c.dt).pin_memory()
    for bad in (host, pinned):
        assert R.attention(bridge_lib, c, bad, SCALE, out) == B.CB_ERR_INVALID_ARG
        assert R.attention(bridge_lib, c, q, SCALE, bad) == B.CB_ERR_INVALID_ARG
    d = c.desc()
    table = c.table.cpu()
    d.table = table.data_ptr()
    inv, amp = _inv(128)
    rope = B.cb_rope_config(inv.data_ptr(), 128, B.CB_ROPE_HALF, amp)
    k = c.tokens(128)
    assert bridge_lib.cb_paged_append(C.byref(d), C.byref(rope), 2, ptr(q), 256, ptr(out), 256, ptr(k),
                                      128, ptr(k), 128, None, None, None, stream()) == B.CB_ERR_INVALID_ARG
    inv_host = inv.cpu()
    cfg = B.cb_rope_config(inv_host.data_ptr(), 128, B.CB_ROPE_HALF, amp)
    pos = torch.zeros(c.rows, device="cuda", dtype=torch.int32)
    assert bridge_lib.cb_rope(C.byref(cfg), B.CB_DTYPE_F16, ptr(q), 256, ptr(out), 256, ptr(pos), 2,
                              2, 128, 0, stream()) == B.CB_ERR_INVALID_ARG


def test_calls_on_two_streams_at_once(bridge_lib):
    """Two caches, streams and workspaces; the same results as one after the other."""
    sides = []
    for seed, (lens, news) in enumerate([([3000, 40], [200, 1]), ([5000, 700], [1, 1])]):
        c = Cache(lens, news, 8, 2, 32, "bf16", seed=seed)
        q = c.tokens(1024)
        alone = torch.zeros(c.rows, 1024, device="cuda", dtype=c.dt)
        assert R.attention(bridge_lib, c, q, SCALE, alone) == 0
        size, d = C.c_size_t(), c.desc()
        assert bridge_lib.cb_paged_attention_workspace(C.byref(d), 8, C.byref(size)) == 0
        sides.append((c, q, alone, d, torch.empty(size.value, dtype=torch.uint8, device="cuda"),
                      torch.cuda.Stream(), torch.zeros_like(alone)))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, q, alone, d, ws, st, out in sides:
            assert bridge_lib.cb_paged_attention(C.byref(d), ptr(q), q.stride(0), 8, SCALE, ptr(out),
                                                 out.stride(0), None, ptr(ws), ws.numel(),
                                                 C.c_void_p(st.cuda_stream)) == 0
    torch.cuda.synchronize()
    for c, q, alone, d, ws, st, out in sides:
        assert torch.equal(out, alone)


class Serving:
    """One layer of a decode loop through all of the operators: dense 64-bit bookkeeping beside
    the calls, so that every step can be checked."""

    def __init__(self, lib, lens, heads, kv_heads, page, budget, dtype, seed):
        self.lib, self.budget = lib, budget
        self.sinks, self.recent = 2, budget // 4
        dev = "cuda"
        self.c = c = Cache([budget + 8] * len(lens), [1] * len(lens), heads, kv_heads, page, dtype,
                           seed=seed, pad=2)
        c.k.zero_(), c.v.zero_()
        self.real = list(lens)
        self.next = torch.tensor(lens, dtype=torch.int32, device=dev)  # position of the next token
        shape = (c.pages, kv_heads, page)
        self.w = torch.zeros(shape, device=dev)
        self.pos = torch.zeros(shape, dtype=torch.int32, device=dev)
        self.inv, self.amp = _inv(128, 3)
        self.rope = B.cb_rope_config(self.inv.data_ptr(), 128, B.CB_ROPE_INTERLEAVED, self.amp)
        g = kv_heads * 128
        self.qkv = c.tokens(heads * 128 + 2 * g)
        self.q, self.k, self.v = self.qkv.split([heads * 128, g, g], 1)
        self.row_pos = torch.zeros(c.rows, dtype=torch.int32, device=dev)
        self.q_out = torch.zeros(c.rows, heads * 128, device=dev, dtype=c.dt)
        self.out = torch.zeros_like(self.q_out)
        self.lse = torch.zeros(c.rows, heads, device=dev)
        self.len_after = torch.zeros_like(c.len)
        c.len.copy_(torch.tensor(lens, dtype=torch.int32))
        for b, n in enumerate(lens):  # a cached prefix, its tokens at positions 0 .. n - 1
            at = c.place(b, torch.arange(n, device=dev))
            for h in range(kv_heads):
                c.k[at[0], h, at[1]] = torch.randn(n, 128, device=dev, generator=c.gen).to(c.dt)
                c.v[at[0], h, at[1]] = torch.randn(n, 128, device=dev, generator=c.gen).to(c.dt)
                self.w[at[0], h, at[1]] = torch.rand(n, device=dev, generator=c.gen)
                self.pos[at[0], h, at[1]] = torch.arange(n, device=dev).int()
        self.d = c.desc()
        size = C.c_size_t()
        assert lib.cb_paged_attention_workspace(C.byref(self.d), heads, C.byref(size)) == 0
        self.ws = torch.empty(size.value, dtype=torch.uint8, device=dev)
        assert lib.cb_paged_evict_workspace(C.byref(self.d), budget, C.byref(size)) == 0
        self.evict_ws = torch.empty(size.value, dtype=torch.uint8, device=dev)

    def step(self):
        """Everything of a step is on the device: it can be captured and replayed."""
        c, lib, d = self.c, self.lib, C.byref(self.d)
        st = stream()
        c.len += 1  # the new token's slot
        self.row_pos[:c.batch] = self.next
        assert lib.cb_paged_append(d, C.byref(self.rope), c.heads, ptr(self.q), self.q.stride(0),
                                   ptr(self.q_out), self.q_out.stride(0), ptr(self.k),
                                   self.k.stride(0), ptr(self.v), self.v.stride(0),
                                   ptr(self.row_pos), ptr(self.w), ptr(self.pos), st) == 0
        assert lib.cb_paged_attention(d, ptr(self.q_out), self.q_out.stride(0), c.heads, SCALE,
                                      ptr(self.out), self.out.stride(0), ptr(self.lse), ptr(self.ws),
                                      self.ws.numel(), st) == 0
        assert lib.cb_paged_attention_weights(d, ptr(self.q_out), self.q_out.stride(0), c.heads,
                                              SCALE, ptr(self.lse), ptr(self.w), st) == 0
        self.next += 1
        assert lib.cb_paged_evict(d, ptr(self.w), ptr(self.w), ptr(self.pos), ptr(self.pos),
                                  ptr(self.next), self.budget, self.sinks, self.recent,
                                  ptr(self.len_after), ptr(self.evict_ws), self.evict_ws.numel(),
                                  st) == 0
        c.len.copy_(self.len_after)

    def expect(self):
        """The same step in 64 bits, from the state before it: the attention's output with its
        bounds, the new weights with theirs, and the lengths."""
        c = self.c
        lens = [n + 1 for n in self.real]
        ref = Cache.__new__(Cache)
        ref.__dict__.update(c.__dict__, lens=lens, k=c.k.clone(), v=c.v.clone())
        pos = self.next[:c.batch]

        def turned(x, h):
            return R.rotate_ref(x[:c.batch].unflatten(1, (h, 128)), pos, self.inv, self.amp,
                                "interleaved", 128)[0].to(c.dt)
        q, k = turned(self.q, c.heads), turned(self.k, c.kv_heads)
        v = self.v[:c.batch].unflatten(1, (c.kv_heads, 128))
        w = self.w.clone()
        for b in range(c.batch):
            at = ref.place(b, torch.tensor([lens[b] - 1], device="cuda"))
            ref.k[at[0], :, at[1]], ref.v[at[0], :, at[1]] = k[b], v[b]
            w[at[0], :, at[1]] = 0.0
        q = torch.cat([q.flatten(1), q.flatten(1)[:1].expand(c.rows - c.batch, -1)])
        out, lse, tol, lse_tol = R.attention_ref(ref, q, SCALE)
        weights, w_tol = R.weights_ref(ref, q, SCALE, lse, w)
        return out, tol, weights, w_tol, lens


def _check_serving(s, steps, advance):
    c = s.c
    for i in range(steps):
        s.qkv[:c.batch] = torch.randn(c.batch, s.qkv.shape[1], device="cuda", generator=c.gen).to(c.dt)
        out, tol, weights, w_tol, lens = s.expect()
        advance()
        torch.cuda.synchronize()
        # q and k rotated to the type by the operator may differ from the 64-bit ones by a step
        # of the type, which moves a score by that much of the sum of its terms' magnitudes
        step = torch.finfo(c.dt).eps
        slack = 2 * step * SCALE * 128 * 3
        got = s.out[:c.batch].unflatten(1, (c.heads, 128))
        close(got, out, tol + slack * tol / (step / 2), f"step {i}: out")
        s.real = [min(n, s.budget) for n in lens]
        assert c.len.tolist() == s.real
        for b in range(c.batch):
            for h in range(c.kv_heads):
                full = Cache.__new__(Cache)
                full.__dict__.update(c.__dict__, lens=lens)
                before = full.slots(weights, b, h)
                bound = (full.slots(w_tol, b, h) + slack * before.abs()).max()
                full.lens = s.real
                after = full.slots(s.w, b, h).double()
                positions = full.slots(s.pos, b, h)
                # no position twice, the sinks and the newest are there
                assert positions.unique().numel() == s.real[b]
                nxt = int(s.next[b])
                must = set(range(s.sinks)) | set(range(nxt - s.recent, nxt))
                assert must <= set(positions.tolist())
                # what stays has the largest weights: the sorted sums of what is left are the
                # largest of before, but for the ones that had to stay
                assert float(after.sum()) <= float(before.sum() + bound * len(before))
                if lens[b] > s.budget:
                    gone = float(before.sum() - after.sum())
                    free = after[(positions >= s.sinks) & (positions < nxt - s.recent)]
                    assert gone <= float(free.min() + 2 * bound * len(before))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,heads,kv_heads,page", [([20, 64, 61], 4, 2, 16), ([100, 127], 6, 6, 32)])
def test_a_decode_loop_through_all_operators(bridge_lib, lens, heads, kv_heads, page, dtype):
    s = Serving(bridge_lib, lens, heads, kv_heads, page, 64 if page == 16 else 128, dtype, seed=5)
    _check_serving(s, 8, s.step)


def test_a_captured_decode_loop_serves_every_step(bridge_lib):
    """One CUDA graph of a step, replayed while lengths and pages' contents move on, with
    another graph of another cache (and its own workspaces) between its replays."""
    graphs, loops = [], []
    for seed in (1, 2):
        s = Serving(bridge_lib, [20, 64, 61], 4, 2, 16, 64, "f16", seed=seed)
        keep = {n: x.clone() for n, x in dict(s.__dict__, **s.c.__dict__).items()
                if isinstance(x, torch.Tensor) and n != "live"}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.step()
        for n, x in dict(s.__dict__, **s.c.__dict__).items():  # back to the beginning
            if n in keep:
                x.copy_(keep[n])
        graphs.append(graph)
        loops.append(s)
    torch.cuda.synchronize()

    def advance():
        graphs[0].replay()
        graphs[1].replay()
    _check_serving(loops[0], 6, advance)
