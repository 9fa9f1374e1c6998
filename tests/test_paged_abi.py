"""CPU tests of the paged-cache entry points: refusals, workspaces and rotary frequencies."""
import ctypes as C
import math

import pytest

from rustane_b200 import bridge as B

BAD = B.CB_ERR_INVALID_ARG
A = 1 << 32  # an aligned address that is never read: every refusal comes before any use


def _kv(**change):
    f = dict(k=A, v=2 * A, table=3 * A, len=4 * A, row_start=5 * A, dtype=B.CB_DTYPE_F16, pages=8,
             kv_heads=2, page_size=16, batch=2, table_stride=4, max_len=64, rows=4, max_new=2)
    f.update(change)
    return B.cb_paged_kv(**f)


BAD_SIZES = [dict(dtype=0), dict(dtype=3), dict(pages=0), dict(kv_heads=0), dict(page_size=8),
             dict(page_size=48), dict(page_size=256), dict(batch=0), dict(table_stride=0),
             dict(max_len=0), dict(max_len=65), dict(rows=-1), dict(max_new=-1),
             dict(max_new=5), dict(pages=1 << 26), dict(pages=2 ** 31 - 1, kv_heads=2 ** 31 - 1)]
BAD_POINTERS = [dict(k=None), dict(v=None), dict(table=None), dict(len=None), dict(k=A + 8),
                dict(v=A + 2), dict(table=A + 1), dict(len=A + 2)]


def _attention(lib, kv, q=6 * A, q_stride=512, heads=4, scale=0.1, out=7 * A, out_stride=512,
               lse=8 * A, ws=9 * A, size=1 << 30):
    return lib.cb_paged_attention(C.byref(kv), q, q_stride, heads, scale, out, out_stride, lse, ws,
                                  size, None)


def _append(lib, kv, rope=None, heads=4, q=6 * A, qs=512, qo=7 * A, qos=512, k=8 * A, ks=256,
            v=9 * A, vs=256, pos=10 * A, w=11 * A, sp=12 * A):
    return lib.cb_paged_append(C.byref(kv), C.byref(rope) if rope else None, heads, q, qs, qo, qos,
                               k, ks, v, vs, pos, w, sp, None)


def _weights(lib, kv, q=6 * A, qs=512, heads=4, scale=0.1, lse=7 * A, w=8 * A):
    return lib.cb_paged_attention_weights(C.byref(kv), q, qs, heads, scale, lse, w, None)


def _evict(lib, kv, w=6 * A, wo=6 * A, p=7 * A, po=7 * A, nxt=8 * A, budget=32, sinks=2, recent=4,
           lo=9 * A, ws=10 * A, size=1 << 30):
    return lib.cb_paged_evict(C.byref(kv), w, wo, p, po, nxt, budget, sinks, recent, lo, ws, size,
                              None)


def _rope(lib, rope, dtype=B.CB_DTYPE_F16, x=A, xs=256, y=2 * A, ys=256, pos=3 * A, tokens=4,
          heads=2, hd=128, inverse=0):
    return lib.cb_rope(C.byref(rope) if rope else None, dtype, x, xs, y, ys, pos, tokens, heads,
                       hd, inverse, None)


def _config(inv=4 * A, rot=128, layout=B.CB_ROPE_HALF, amp=1.0):
    return B.cb_rope_config(inv, rot, layout, amp)


@pytest.mark.parametrize("change", BAD_SIZES + BAD_POINTERS, ids=str)
def test_bad_descriptors_are_refused(bridge_lib, change):
    kv = _kv(**change)
    assert _attention(bridge_lib, kv) == BAD
    assert _append(bridge_lib, kv) == BAD
    assert _weights(bridge_lib, kv) == BAD
    assert _evict(bridge_lib, kv) == BAD
    size = C.c_size_t()
    if change in BAD_SIZES:
        assert bridge_lib.cb_paged_attention_workspace(C.byref(kv), 4, C.byref(size)) == BAD
        assert bridge_lib.cb_paged_evict_workspace(C.byref(kv), 8, C.byref(size)) == BAD


@pytest.mark.parametrize("change", [
    dict(q=None), dict(out=None), dict(q=A + 2), dict(out=A + 8), dict(lse=A + 2), dict(ws=A + 8),
    dict(heads=0), dict(heads=3), dict(heads=-2), dict(q_stride=504), dict(out_stride=504),
    dict(q_stride=513), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
    dict(scale=math.inf), dict(out=6 * A), dict(out=6 * A + 16), dict(out=6 * A + 256, out_stride=512)],
    ids=str)
def test_attention_refusals(bridge_lib, change):
    assert _attention(bridge_lib, _kv(), **change) == BAD


def test_attention_needs_row_start_and_its_workspace(bridge_lib):
    assert _attention(bridge_lib, _kv(row_start=None)) == BAD
    # one long sequence: split, so a workspace is needed
    kv = _kv(batch=1, rows=1, max_new=1, table_stride=4096, max_len=65536, pages=5000)
    size = C.c_size_t()
    assert bridge_lib.cb_paged_attention_workspace(C.byref(kv), 4, C.byref(size)) == B.CB_OK
    assert size.value > 0 and size.value % 4 == 0
    assert _attention(bridge_lib, kv, size=size.value - 1) == BAD
    assert _attention(bridge_lib, kv, ws=None) == BAD
    assert bridge_lib.cb_paged_attention_workspace(C.byref(kv), 4, None) == BAD


@pytest.mark.parametrize("change", [
    dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(q=A + 8), dict(qo=A + 8),
    dict(k=A + 8), dict(v=A + 8), dict(heads=0), dict(heads=3), dict(qs=504), dict(qos=504),
    dict(ks=248), dict(vs=248), dict(ks=257), dict(pos=A + 1), dict(w=A + 1), dict(sp=A + 1),
    dict(qo=6 * A + 16), dict(qo=6 * A, qos=1024), dict(qo=8 * A), dict(qo=9 * A)], ids=str)
def test_append_refusals(bridge_lib, change):
    assert _append(bridge_lib, _kv(), **change) == BAD


@pytest.mark.parametrize("config", [
    _config(inv=None), _config(inv=A + 4), _config(rot=0), _config(rot=12), _config(rot=136),
    _config(layout=0), _config(layout=3), _config(amp=math.nan), _config(amp=math.inf)])
def test_rope_configs_are_checked(bridge_lib, config):
    assert _rope(bridge_lib, config) == BAD
    assert _append(bridge_lib, _kv(), rope=config) == BAD


@pytest.mark.parametrize("change", [
    dict(dtype=0), dict(x=None), dict(y=None), dict(pos=None), dict(pos=A + 2), dict(x=A + 8),
    dict(y=A + 2), dict(xs=248), dict(ys=260), dict(tokens=-1), dict(heads=0), dict(hd=0),
    dict(hd=132), dict(hd=520), dict(inverse=2), dict(inverse=-1), dict(y=A + 16),
    dict(y=A, ys=512), dict(hd=64)], ids=str)
def test_rope_refusals(bridge_lib, change):
    assert _rope(bridge_lib, _config(), **change) == BAD
    assert _rope(bridge_lib, None) == BAD


@pytest.mark.parametrize("change", [
    dict(q=None), dict(q=A + 2), dict(lse=None), dict(lse=A + 2), dict(w=None), dict(w=A + 2),
    dict(heads=3), dict(qs=504), dict(scale=0.0), dict(scale=math.nan)], ids=str)
def test_weights_refusals(bridge_lib, change):
    assert _weights(bridge_lib, _kv(), **change) == BAD
    assert _weights(bridge_lib, _kv(row_start=None)) == BAD


@pytest.mark.parametrize("change", [
    dict(w=None), dict(wo=None), dict(p=None), dict(po=None), dict(nxt=None), dict(lo=None),
    dict(ws=None), dict(w=A + 2), dict(po=A + 2), dict(ws=A + 4), dict(budget=0), dict(sinks=-1),
    dict(recent=-1), dict(sinks=20, recent=13), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1),
    dict(size=2 * 2 * 2 * 32 * 4 - 1), dict(wo=6 * A + 16), dict(po=7 * A + 16), dict(lo=4 * A),
    dict(wo=7 * A)], ids=str)
def test_evict_refusals(bridge_lib, change):
    assert _evict(bridge_lib, _kv(), **change) == BAD


@pytest.mark.parametrize("change", [
    dict(wo=9 * A, po=6 * A), dict(wo=7 * A, po=9 * A), dict(wo=7 * A + 4, po=9 * A)], ids=str)
def test_evict_refuses_an_output_over_the_other_input(bridge_lib, change):
    assert _evict(bridge_lib, _kv(), **change) == BAD


def test_calls_without_rows_take_null_token_arrays(bridge_lib):
    kv = _kv(rows=0, max_new=0)
    assert _attention(bridge_lib, kv, q=None, out=None, lse=None) == 0
    assert _weights(bridge_lib, kv, q=None, lse=None) == 0
    assert _append(bridge_lib, kv, q=None, qo=None, k=None, v=None, pos=None) == 0
    assert _rope(bridge_lib, _config(), x=None, y=None, pos=None, tokens=0) == 0
    assert _attention(bridge_lib, kv, ws=None) == BAD
    assert _weights(bridge_lib, kv, w=None) == BAD


@pytest.mark.parametrize("scale", [3e38, math.inf, -0.1])
def test_scales_whose_base_2_form_is_not_finite_are_refused(bridge_lib, scale):
    assert _attention(bridge_lib, _kv(), scale=scale) == BAD
    assert _weights(bridge_lib, _kv(), scale=scale) == BAD


def test_more_than_128_query_heads_to_a_key_head_are_refused(bridge_lib):
    kv = _kv(kv_heads=1)
    assert _attention(bridge_lib, kv, heads=129, q_stride=1 << 16, out_stride=1 << 16) == BAD
    assert _weights(bridge_lib, kv, heads=129, qs=1 << 16) == BAD


def test_evict_refuses_sequences_that_no_cluster_holds(bridge_lib):
    kv = _kv(max_len=262145, table_stride=20000, pages=20000)
    assert _evict(bridge_lib, kv) == B.CB_ERR_UNSUPPORTED


def test_empty_steps_need_no_gpu(bridge_lib):
    kv = _kv(rows=0, max_new=0)
    assert _attention(bridge_lib, kv) == B.CB_OK
    assert _append(bridge_lib, kv) == B.CB_OK
    assert _weights(bridge_lib, kv) == B.CB_OK
    assert _rope(bridge_lib, _config(), tokens=0) == B.CB_OK


def test_without_a_gpu_calls_fail_loudly(bridge_lib):
    n = C.c_int32()
    bridge_lib.cb_device_count(C.byref(n))
    if n.value > 0:
        pytest.skip("a GPU is present")
    assert _attention(bridge_lib, _kv()) == B.CB_ERR_CUDA
    assert _append(bridge_lib, _kv(), rope=_config()) == B.CB_ERR_CUDA
    assert _weights(bridge_lib, _kv()) == B.CB_ERR_CUDA
    assert _evict(bridge_lib, _kv()) == B.CB_ERR_CUDA
    assert _rope(bridge_lib, _config()) == B.CB_ERR_CUDA


# ------------------------------------------------------------------ rotary frequencies
def _frequencies(lib, rot, **f):
    s = B.cb_rope_scaling(**(dict(base=10000.0, kind=0, factor=0.0, original_len=0.0,
                                  fast_turns=0.0, slow_turns=0.0) | f))
    inv, amp = (C.c_double * (rot // 2))(), C.c_float()
    rc = lib.cb_rope_frequencies(rot, C.byref(s), inv, C.byref(amp))
    return rc, list(inv), amp.value


@pytest.mark.parametrize("rot", [8, 24, 64, 128])
def test_plain_linear_and_base_frequencies(bridge_lib, rot):
    want = [10000.0 ** (-2 * i / rot) for i in range(rot // 2)]
    rc, inv, amp = _frequencies(bridge_lib, rot)
    assert rc == 0 and amp == 1.0 and inv == pytest.approx(want, rel=1e-14)
    rc, inv, _ = _frequencies(bridge_lib, rot, kind=B.CB_ROPE_SCALE_LINEAR, factor=4.0)
    assert rc == 0 and inv == pytest.approx([w / 4 for w in want], rel=1e-14)
    rc, inv, _ = _frequencies(bridge_lib, rot, kind=B.CB_ROPE_SCALE_BASE, factor=4.0)
    assert rc == 0 and inv[0] == 1.0
    # the slowest pair turns `factor` times slower, as with linear scaling
    assert inv[-1] == pytest.approx(want[-1] / 4, rel=1e-12)


def test_frequencies_by_parts(bridge_lib):
    f = dict(kind=B.CB_ROPE_SCALE_PARTS, factor=8.0, original_len=4096.0, fast_turns=32.0,
             slow_turns=1.0)
    rc, inv, amp = _frequencies(bridge_lib, 128, **f)
    assert rc == 0 and amp == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-6)
    plain = [10000.0 ** (-i / 64) for i in range(64)]
    ratio = [a / b for a, b in zip(inv, plain)]
    turns = [4096.0 * p / (2 * math.pi) for p in plain]
    for r, t in zip(ratio, turns):
        if t > 40.0:
            assert r == 1.0
        elif t < 0.8:
            assert r == pytest.approx(1 / 8, rel=1e-14)
        assert 1 / 8 - 1e-15 <= r <= 1.0
    assert ratio == sorted(ratio, reverse=True)


@pytest.mark.parametrize("bad", [
    dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(kind=-1), dict(kind=4),
    dict(kind=1, factor=0.5), dict(kind=1, factor=math.nan), dict(kind=2, factor=math.inf),
    dict(kind=3, factor=2.0), dict(kind=3, factor=2.0, original_len=100.0, fast_turns=1.0,
                                   slow_turns=2.0)], ids=str)
def test_bad_scalings_are_refused(bridge_lib, bad):
    assert _frequencies(bridge_lib, 64, **bad)[0] == BAD


def test_bad_rot_dims_are_refused(bridge_lib):
    for rot in (0, -8, 12, 2):
        s = B.cb_rope_scaling(10000.0, 0, 1.0, 1.0, 1.0, 1.0)
        assert bridge_lib.cb_rope_frequencies(rot, C.byref(s), (C.c_double * 64)(), None) == BAD
    assert bridge_lib.cb_rope_frequencies(64, None, (C.c_double * 64)(), None) == BAD
