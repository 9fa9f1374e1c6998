"""The bounded waits of the paged-cache kernels, made to run out in an allowed form: the self-test
runs the kernels with loads that are never issued and waits of 1 ms. What they could not finish
has to be NaN, not what the arrays or the workspace held, and has to be reported."""
import ctypes as C
import math

import pytest
import torch

import paged_ref as R
from paged_ref import Cache, ptr, stream
from rustane_b200 import bridge as B

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)

STEPS = [
    # lens, news, heads, kv_heads, page
    ([64, 1, 33], [1, 1, 0], 4, 2, 16),    # the 16-row kernel, whole tiles
    ([9000, 40], [1, 3], 4, 4, 64),        # cut into parts
    ([500, 130], [200, 130], 4, 2, 16),    # the tcgen05 kernel
    ([5000, 300], [300, 5], 8, 2, 128),    # cut into parts
]


@pytest.mark.parametrize("lens,news,heads,kv_heads,page", STEPS)
def test_expired_waits_leave_nan_and_are_reported(bridge_lib, lens, news, heads, kv_heads, page):
    c = Cache(lens, news, heads, kv_heads, page, "f16", seed=heads)
    total = c.starts[-1]
    q = c.tokens(heads * 128)
    lse = torch.zeros(c.rows, heads, device="cuda")
    out = torch.full((c.rows, heads * 128), 3.0, device="cuda", dtype=c.dt)
    good, good_lse = out.clone(), lse.clone()
    d, size = c.desc(), C.c_size_t()
    assert bridge_lib.cb_paged_attention_workspace(C.byref(d), heads, C.byref(size)) == 0
    ws = torch.zeros(size.value, dtype=torch.uint8, device="cuda")
    w = torch.zeros(c.pages, kv_heads, page, device="cuda")

    def attention(o, ls):
        return bridge_lib.cb_paged_attention(C.byref(d), ptr(q), q.stride(0), heads, SCALE, ptr(o),
                                             o.stride(0), ptr(ls), ptr(ws), size.value, stream())
    def check():
        n = C.c_int32(-1)
        return bridge_lib.cb_paged_check_device_error(C.byref(n), stream()), n.value
    assert attention(good, good_lse) == 0
    assert check() == (B.CB_OK, 0)
    assert bridge_lib.cb_selftest_paged_timeout(C.byref(d), ptr(q), q.stride(0), heads, SCALE,
                                                ptr(out), out.stride(0), ptr(lse), ptr(w), ptr(ws),
                                                size.value, stream()) == B.CB_OK
    rc, expired = check()
    assert rc == B.CB_ERR_DEVICE_TIMEOUT and expired > 0
    assert check() == (B.CB_OK, 0)  # cleared
    assert bool(out[:total].isnan().all()) and bool(lse[:total].isnan().all())
    assert bool((out[total:] == 3.0).all()) and bool((lse[total:] == 0).all())
    if max(news) * heads // kv_heads > 16:
        assert bool(w[c.live].isnan().all())
    assert bool((w[~c.live] == 0).all())
    # everything works as before
    assert attention(out, lse) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[:total], good[:total]) and torch.equal(lse[:total], good_lse[:total])
    assert check() == (B.CB_OK, 0)


def test_the_selftest_takes_f16(bridge_lib):
    c = Cache([40], [1], 2, 1, 16, "bf16")
    q = c.tokens(256)
    out, lse = torch.zeros_like(q), torch.zeros(c.rows, 2, device="cuda")
    w = torch.zeros(c.pages, 1, 16, device="cuda")
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
    d = c.desc()
    assert bridge_lib.cb_selftest_paged_timeout(C.byref(d), ptr(q), q.stride(0), 2, SCALE, ptr(out),
                                                out.stride(0), ptr(lse), ptr(w), ptr(ws), ws.numel(),
                                                stream()) == B.CB_ERR_UNSUPPORTED
