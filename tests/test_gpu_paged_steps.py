"""GPU tests of whole decode steps through the paged-cache operators, each operator checked on what
the one before it wrote, with the tolerances of its own test (tests/paged_ref.py); and of caches
past 2^31 elements, bit for bit where rows are only moved."""
import ctypes as C

import pytest
import torch

import paged_ref as R
from paged_ref import Cache, ptr, stream
from rustane_b200 import bridge as B
from test_gpu_paged import LAYOUT, SCALE, Serving, _append, _evict, _inv, close

pytestmark = pytest.mark.gpu


def _same_bits(a, b, what):
    kind = torch.int16 if a.element_size() == 2 else torch.int32
    assert torch.equal(a.view(kind), b.view(kind)), what


def _can_fail(want, tol, what):
    """Most values are larger than their tolerance: zeros in their place would be found."""
    assert float((want.abs() > 4 * tol).double().mean()) > 0.5, what


def _moved(c, moves, pools):
    """What the pools hold after the moves {(b, head): sources of the slots below the new length}."""
    want = {n: x.clone() for n, x in pools.items()}
    for (b, h), source in moves.items():
        to = c.place(b, torch.arange(len(source), device="cuda"))
        fro = c.place(b, torch.tensor(source, device="cuda", dtype=torch.long))
        for n, x in pools.items():
            want[n][to[0], h, to[1]] = x[fro[0], h, fro[1]]
    return want


class Checked(Serving):
    """A step call by call, with every call's outputs checked before the next."""

    def checked_step(self):
        c, lib, d, st = self.c, self.lib, C.byref(self.d), stream()
        n, heads, g = c.batch, c.heads, c.kv_heads
        lens = [x + 1 for x in self.real]
        c.lens = lens
        at = [c.place(b, torch.tensor([lens[b] - 1], device="cuda")) for b in range(n)]
        want = {"k": c.k.clone(), "v": c.v.clone(), "w": self.w.clone(), "p": self.pos.clone()}
        c.len += 1
        self.row_pos[:n] = self.next
        assert lib.cb_paged_append(d, C.byref(self.rope), heads, ptr(self.q), self.q.stride(0),
                                   ptr(self.q_out), self.q_out.stride(0), ptr(self.k),
                                   self.k.stride(0), ptr(self.v), self.v.stride(0),
                                   ptr(self.row_pos), ptr(self.w), ptr(self.pos), st) == 0
        torch.cuda.synchronize()
        for x, got, h in ((self.q, self.q_out[:n].unflatten(1, (heads, 128)), heads),
                          (self.k, torch.cat([c.k[p, :, s] for p, s in at]), g)):
            turned, size = R.rotate_ref(x[:n].unflatten(1, (h, 128)), self.next, self.inv, self.amp,
                                        "interleaved", 128)
            tol = R.rotate_tol(turned, size, c.dt)
            _can_fail(turned, tol, "rotation")
            close(got, turned, tol, "rotation")
        for b, (p, s) in enumerate(at):
            want["k"][p, :, s] = c.k[p, :, s]  # checked above
            want["v"][p, :, s] = self.v[b].unflatten(0, (g, 128))
            want["w"][p, :, s] = 0.0
            want["p"][p, :, s] = self.next[b]
        for name, got in (("k", c.k), ("v", c.v), ("w", self.w), ("p", self.pos)):
            _same_bits(got, want[name], f"append: {name}")

        assert lib.cb_paged_attention(d, ptr(self.q_out), self.q_out.stride(0), heads, SCALE,
                                      ptr(self.out), self.out.stride(0), ptr(self.lse),
                                      ptr(self.ws), self.ws.numel(), st) == 0
        torch.cuda.synchronize()
        out, lse, tol, lse_tol = R.attention_ref(c, self.q_out, SCALE)
        _can_fail(out, tol, "attention")
        close(self.out[:n].unflatten(1, (heads, 128)), out, tol, "attention")
        close(self.lse[:n], lse, lse_tol, "log-sum-exp")

        w, w_tol = R.weights_ref(c, self.q_out, SCALE, self.lse, self.w)
        assert lib.cb_paged_attention_weights(d, ptr(self.q_out), self.q_out.stride(0), heads, SCALE,
                                              ptr(self.lse), ptr(self.w), st) == 0
        torch.cuda.synchronize()
        added = (w - want["w"].double())
        _can_fail(added[added != 0], w_tol[added != 0], "weights")
        close(self.w, w, w_tol, "weights")

        self.next += 1
        pools = {"k": c.k, "v": c.v, "w": self.w, "p": self.pos}
        want = _moved(c, R.evict_ref(c, self.w, self.pos, self.next, self.budget, self.sinks,
                                     self.recent), pools)
        assert lib.cb_paged_evict(d, ptr(self.w), ptr(self.w), ptr(self.pos), ptr(self.pos),
                                  ptr(self.next), self.budget, self.sinks, self.recent,
                                  ptr(self.len_after), ptr(self.evict_ws), self.evict_ws.numel(),
                                  st) == 0
        torch.cuda.synchronize()
        for name, got in pools.items():
            _same_bits(got, want[name], f"evict: {name}")
        self.real = [min(x, self.budget) for x in lens]
        assert self.len_after.tolist() == self.real
        c.len.copy_(self.len_after)

    def new_tokens(self):
        n = self.c.batch
        self.qkv[:n] = torch.randn(n, self.qkv.shape[1], device="cuda",
                                   generator=self.c.gen).to(self.c.dt)

    def state(self):
        own = {n: x for n, x in self.__dict__.items()
               if isinstance(x, torch.Tensor) and n not in ("ws", "evict_ws")}
        return own | {f"cache {n}": getattr(self.c, n) for n in ("k", "v", "len")}


SHAPES = [([20, 64, 61], 4, 2, 16, 64), ([100, 127], 6, 6, 32, 128), ([60, 63, 2], 40, 2, 16, 64)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,heads,kv_heads,page,budget", SHAPES)
def test_each_operator_of_a_decode_step_on_what_the_last_one_wrote(bridge_lib, lens, heads, kv_heads,
                                                                   page, budget, dtype):
    s = Checked(bridge_lib, lens, heads, kv_heads, page, budget, dtype, seed=7)
    for _ in range(6):
        s.new_tokens()
        s.checked_step()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_captured_steps_are_the_checked_ones(bridge_lib, dtype):
    """Two captured loops replayed in turn; both end every step with the bits of the same step
    made and checked call by call on a copy."""
    loops = []
    for lens, heads, kv_heads, page, budget in (SHAPES[0], SHAPES[2]):
        pair = [Checked(bridge_lib, lens, heads, kv_heads, page, budget, dtype, seed=heads)
                for _ in range(2)]
        graphed = pair[0]
        keep = {n: x.clone() for n, x in graphed.state().items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphed.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            graphed.step()
        for n, x in graphed.state().items():
            x.copy_(keep[n])
        loops.append((graph, *pair))
    for _ in range(5):
        for graph, graphed, checked in loops:
            checked.new_tokens()
            graphed.qkv.copy_(checked.qkv)
        torch.cuda.synchronize()
        for graph, _, _ in loops:
            graph.replay()
        torch.cuda.synchronize()
        for _, graphed, checked in loops:
            checked.checked_step()
            want = checked.state()
            for n, x in graphed.state().items():
                _same_bits(x, want[n], n)


@pytest.mark.parametrize("new,budget", [(1, 100), (60, 100), (60, 197)])
def test_append_and_evict_behind_2_to_the_31_elements(bridge_lib, new, budget):
    """Every page in use lies behind element 2^31 of the pools: all that append and evict write,
    and that they write nothing else."""
    page, kv_heads = 64, 2
    pages = 2 ** 31 // (page * kv_heads * 128) + 100
    c = Cache([200], [new], 4, kv_heads, page, "f16", seed=3)
    far = torch.tensor([[pages - 5, pages - 1, pages - 17, pages - 3]], device="cuda",
                       dtype=torch.int32)
    small_k, small_v, used = c.k, c.v, c.page_lists[0]
    c.k = torch.zeros(pages, kv_heads, page, 128, device="cuda", dtype=c.dt)
    c.v = torch.zeros_like(c.k)
    c.k[far[0].long()], c.v[far[0].long()] = small_k[used], small_v[used]
    c.table, c.page_lists, c.pages = far, [far[0].tolist()], pages
    w = torch.zeros(pages, kv_heads, page, device="cuda")
    p = torch.zeros(pages, kv_heads, page, device="cuda", dtype=torch.int32)
    old = c.place(0, torch.arange(200, device="cuda"))
    for h in range(kv_heads):
        w[old[0], h, old[1]] = torch.rand(200, device="cuda", generator=c.gen)
        p[old[0], h, old[1]] = torch.randperm(200, device="cuda", generator=c.gen).int()

    def tail(x):
        return x[pages - 20:].clone()
    pools = {"k": c.k, "v": c.v, "w": w, "p": p}
    want = {n: tail(x) for n, x in pools.items()}
    inv, amp = _inv(128)
    rope = B.cb_rope_config(inv.data_ptr(), 128, LAYOUT["half"], amp)
    nk, nv = c.tokens(256), c.tokens(256)
    slots = torch.arange(200 - new, 200, device="cuda")
    at = c.place(0, slots)
    near = at[0] - (pages - 20)
    assert _append(bridge_lib, c, rope, None, None, nk, nv, None, w, p, heads=0) == 0
    torch.cuda.synchronize()
    turned, size = R.rotate_ref(nk[:new].unflatten(1, (2, 128)), slots, inv, amp, "half", 128)
    for h in range(kv_heads):
        close(c.k[at[0], h, at[1]], turned[:, h], R.rotate_tol(turned, size, c.dt)[:, h], "k")
        want["k"][near, h, at[1]] = c.k[at[0], h, at[1]]
        want["v"][near, h, at[1]] = nv[:new].unflatten(1, (2, 128))[:, h]
        want["w"][near, h, at[1]] = 0.0
        want["p"][near, h, at[1]] = slots.int()
    for n, x in pools.items():
        _same_bits(tail(x), want[n], f"append: {n}")

    nxt = torch.tensor([200], device="cuda", dtype=torch.int32)
    moves = R.evict_ref(c, w, p, nxt, budget, 3, 20)
    near_pages = [[x - (pages - 20) for x in c.page_lists[0]]]
    small = Cache.__new__(Cache)
    small.__dict__.update(c.__dict__, page_lists=near_pages)
    want = _moved(small, moves, {n: tail(x) for n, x in pools.items()})
    lo = torch.zeros_like(c.len)
    assert _evict(bridge_lib, c, w, w, p, p, nxt, budget, 3, 20, lo) == 0
    assert lo.tolist() == [budget]
    for n, x in pools.items():
        _same_bits(tail(x), want[n], f"evict: {n}")
        assert not bool(x[:pages - 20].view(torch.int32).any()), n
