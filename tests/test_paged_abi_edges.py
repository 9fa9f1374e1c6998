"""CPU tests of refusals of the paged-cache entry points: arrays that lie over one another, and
sizes that no memory has. Addresses are never read."""
import ctypes as C

import pytest

from rustane_b200 import bridge as B
from test_paged_abi import A, BAD, _append, _attention, _config, _evict, _kv, _rope, _weights

# _kv(): k at A, v at 2 A, table 3 A, len 4 A, row_start 5 A; pools of 8 * 2 * 16 * 128 elements,
# weights and positions of 8 * 2 * 16 words
POOL, META = 8 * 2 * 16 * 128 * 2, 8 * 2 * 16 * 4


def _reached(rc):
    """Past the refusals: the call got as far as looking for a GPU."""
    return rc in (B.CB_ERR_CUDA, B.CB_ERR_UNSUPPORTED) or rc == BAD and _gpu_there()


def _gpu_there():
    n = C.c_int32()
    return B.load_library().cb_device_count(C.byref(n)) == 0 and n.value > 0


@pytest.mark.parametrize("change", [
    dict(lo=8 * A), dict(lo=8 * A + 4), dict(lo=8 * A - 4), dict(lo=3 * A), dict(lo=6 * A),
    dict(lo=7 * A + META - 4), dict(lo=A), dict(wo=9 * A, w=6 * A), dict(po=9 * A - META + 4),
    dict(wo=8 * A), dict(po=8 * A), dict(wo=3 * A), dict(po=4 * A), dict(wo=2 * A),
    dict(ws=6 * A), dict(ws=7 * A), dict(ws=9 * A), dict(ws=8 * A), dict(ws=A + POOL - 16),
    dict(ws=3 * A), dict(ws=4 * A), dict(w=A, wo=A), dict(p=2 * A, po=2 * A), dict(nxt=A),
    dict(nxt=2 * A + POOL - 4)], ids=str)
def test_evict_refuses_outputs_over_anything_else(bridge_lib, change):
    assert _evict(bridge_lib, _kv(), **change) == BAD


@pytest.mark.parametrize("change", [
    dict(lse=7 * A), dict(lse=7 * A + 3 * 512 * 2 + 1020), dict(lse=6 * A), dict(lse=9 * A),
    dict(lse=A), dict(lse=4 * A), dict(ws=6 * A), dict(ws=7 * A + 1024), dict(ws=2 * A),
    dict(ws=8 * A), dict(ws=5 * A), dict(out=A), dict(out=2 * A + POOL - 16), dict(out=3 * A),
    dict(out=4 * A), dict(out=5 * A)], ids=str)
def test_attention_refuses_outputs_over_anything_else(bridge_lib, change):
    assert _attention(bridge_lib, _kv(), **change) == BAD


@pytest.mark.parametrize("change", [
    dict(w=7 * A), dict(w=7 * A + 4 * 4 * 4 - 4), dict(w=6 * A), dict(w=A), dict(w=3 * A),
    dict(w=4 * A), dict(w=5 * A - META + 4)], ids=str)
def test_weights_refuse_sums_over_anything_else(bridge_lib, change):
    assert _weights(bridge_lib, _kv(), **change) == BAD


@pytest.mark.parametrize("change", [
    dict(w=12 * A), dict(sp=11 * A), dict(w=10 * A), dict(sp=10 * A), dict(sp=10 * A - META + 4),
    dict(w=8 * A), dict(sp=9 * A), dict(w=A), dict(sp=2 * A), dict(w=7 * A), dict(sp=6 * A),
    dict(w=3 * A), dict(sp=4 * A), dict(w=5 * A), dict(qo=A), dict(qo=2 * A), dict(qo=10 * A),
    dict(qo=3 * A), dict(pos=A), dict(pos=2 * A + POOL - 4)], ids=str)
def test_append_refuses_outputs_over_anything_else(bridge_lib, change):
    assert _append(bridge_lib, _kv(), **change) == BAD


def test_rope_refuses_an_output_over_its_positions_or_frequencies(bridge_lib):
    assert _rope(bridge_lib, _config(), pos=2 * A) == BAD
    assert _rope(bridge_lib, _config(), pos=2 * A + 4 * 256 * 2 - 4) == BAD
    assert _rope(bridge_lib, _config(inv=2 * A + 8)) == BAD
    assert _append(bridge_lib, _kv(), rope=_config(inv=7 * A)) == BAD
    assert _append(bridge_lib, _kv(), rope=_config(inv=A)) == BAD


def test_arrays_side_by_side_are_not_refused(bridge_lib):
    kv = _kv()
    row = 4 * 128 * 2
    assert _reached(_attention(bridge_lib, kv, q_stride=1024, out=6 * A + row, out_stride=1024))
    assert _reached(_attention(bridge_lib, kv, lse=7 * A + 4 * row))      # right behind out
    assert _reached(_evict(bridge_lib, kv, lo=8 * A + 8))                 # right behind next_position
    assert _reached(_evict(bridge_lib, kv, wo=6 * A + META, po=7 * A + META))
    assert _reached(_weights(bridge_lib, kv, w=7 * A + 4 * 4 * 4))
    assert _reached(_append(bridge_lib, kv, sp=11 * A + META))
    # q, k and v in one fused array, q rotated in place, and without weights and positions
    assert _reached(_append(bridge_lib, kv, q=6 * A, qs=1024, qo=6 * A, qos=1024, k=6 * A + row,
                            ks=1024, v=6 * A + row + 512, vs=1024, pos=None, w=None, sp=None))
    assert _reached(_attention(bridge_lib, _kv(v=A)))                     # one pool read as both


@pytest.mark.parametrize("rows", [1 << 23, (1 << 29) - 1])
def test_token_arrays_longer_than_any_memory_are_refused(bridge_lib, rows):
    """(rows - 1) * stride elements of two bytes pass 2^63: no address arithmetic on them."""
    kv, s = _kv(rows=rows), 1 << 40
    assert _attention(bridge_lib, kv, q_stride=s) == BAD
    assert _attention(bridge_lib, kv, out_stride=s) == BAD
    assert _weights(bridge_lib, kv, qs=s) == BAD
    for name in ("qs", "qos", "ks", "vs"):
        assert _append(bridge_lib, kv, **{name: s}) == BAD
    assert _rope(bridge_lib, _config(), xs=s, tokens=rows) == BAD
    assert _rope(bridge_lib, _config(), ys=s, tokens=rows) == BAD


@pytest.mark.parametrize("base,factor", [(10000.0, 1e306), (1e300, 1e10), (1e308, 2.0)])
def test_a_scaled_base_that_is_not_finite_is_refused(bridge_lib, base, factor):
    """All frequencies but the first would be 0."""
    s = B.cb_rope_scaling(base, B.CB_ROPE_SCALE_BASE, factor, 0.0, 0.0, 0.0)
    inv = (C.c_double * 32)(*[7.0] * 32)
    assert bridge_lib.cb_rope_frequencies(64, C.byref(s), inv, None) == BAD
    assert list(inv) == [7.0] * 32
