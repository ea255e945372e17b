"""Refusals and host-side checks of the router with balance loss and of the INT8 path: nothing here
needs a GPU."""
import ctypes

import pytest
import torch

from build_ext import lib_path

P = 1 << 20  # a 16-byte aligned address that is never dereferenced on these paths


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(str(lib_path()))


def test_public_names():
    import grouped_gemm_opt as g
    for name in ["moe_router", "MoERouting", "quantize_int8", "grouped_gemm_opt_int8",
                 "fused_moe_int8", "quantize_moe_weights_int8", "MoEInt8Weights"]:
        assert name in g.__all__ and hasattr(g, name)


def test_int8_quantiser_refusals(lib):
    q = lib.ggo_quantize_int8_rows
    q.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int] + \
        [ctypes.c_void_p] * 3
    assert q(P, 4, 64, 2, P, P, None) == 3          # fp32 input
    assert q(None, 4, 64, 0, P, P, None) == 1
    assert q(P, -1, 64, 0, P, P, None) == 1
    assert q(P, 4, 0, 0, P, P, None) == 1
    assert q(P, 4, 24, 0, P, P, None) == 4          # cols % 16
    assert q(P + 8, 4, 64, 0, P, P, None) == 4
    assert q(P, 1 << 31, 64, 0, P, P, None) == 2
    assert q(None, 0, 64, 0, None, None, None) == 0  # nothing to do


def test_int8_product_refusals(lib):
    f = lib.ggo_grouped_gemm_int8
    f.argtypes = [ctypes.c_void_p] * 6 + [ctypes.c_int] * 2 + [ctypes.c_int64] * 3 + \
        [ctypes.c_int] * 4 + [ctypes.c_void_p] * 3

    def call(a=P, sa=P, b=P, sb=P, out=P, counts=P, segs=8, e=8, t=256, n=1024, k=512, dt=0, glu=0,
             tc=4, ws=P):
        return f(a, sa, b, sb, out, counts, segs, e, t, n, k, dt, glu, tc, 1, ws, None, None)

    for name in ("a", "sa", "b", "sb", "out", "counts", "ws"):
        assert call(**{name: None}) == 1
    assert call(dt=2) == 3 and call(dt=7) == 3
    assert call(k=520) == 4 and call(n=1001) == 4 and call(a=P + 8) == 4 and call(b=P + 4) == 4
    assert call(k=131072) == 2                       # a sum could leave 32 bits
    assert call(e=1 << 20, n=1 << 12) == 2           # weight rows beyond 32-bit coordinates
    assert call(segs=2000, e=2000) == 5
    assert call(tc=9) == 1 and call(segs=0) == 1 and call(t=-1) == 1
    assert call(t=0) == 0


def test_int8_permute_refusals(lib):
    f = lib.ggo_moe_permute_int8
    f.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int] + \
        [ctypes.c_void_p] * 5 + [ctypes.c_int, ctypes.c_void_p]

    def call(x=P, t=16, h=64, e=8, k=2, ids=P, q=P, s=P, pos=P, scratch=P, dt=0):
        return f(x, t, h, e, k, ids, q, s, pos, scratch, dt, None)

    for name in ("x", "ids", "q", "s", "pos", "scratch"):
        assert call(**{name: None}) == 1
    assert call(h=72) == 4 and call(q=P + 8) == 4 and call(dt=2) == 3
    assert call(k=9) == 1 and call(k=17, e=64) == 1 and call(e=2000) == 1
    assert call(t=1 << 31) == 2 and call(t=0) == 0


def test_router_refusals(lib):
    f = lib.ggo_moe_router
    f.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int] + \
        [ctypes.c_void_p] * 10

    def call(l=P, dt=2, t=16, e=8, k=2, mask=None, ids=P, w=P, tpe=P, bc=P, loss=P, stat=P, coef=P,
             scratch=P):
        return f(l, dt, t, e, k, mask, ids, w, tpe, bc, loss, stat, coef, scratch, None)

    for name in ("l", "ids", "w", "tpe", "bc", "loss", "stat", "coef", "scratch"):
        assert call(**{name: None}) == 1
    assert call(dt=3) == 3 and call(k=9) == 1 and call(k=0) == 1 and call(e=1025) == 1
    assert call(k=17, e=64) == 1 and call(t=-1) == 1
    assert call(stat=P + 4) == 4 and call(t=1 << 30, k=4) == 2
    lib.ggo_moe_router_scratch_bytes.restype = ctypes.c_size_t
    lib.ggo_moe_router_scratch_bytes.argtypes = [ctypes.c_int64, ctypes.c_int]
    lib.ggo_moe_route_scratch_bytes.restype = ctypes.c_size_t
    lib.ggo_moe_route_scratch_bytes.argtypes = [ctypes.c_int64, ctypes.c_int]
    for t, e in [(1, 1), (33, 7), (16384, 256)]:  # its head is the dispatch's table
        assert lib.ggo_moe_router_scratch_bytes(t, e) > lib.ggo_moe_route_scratch_bytes(t, e)
    b = lib.ggo_moe_router_backward
    b.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int] + \
        [ctypes.c_void_p] * 8
    assert b(P, 2, 16, 8, 2, P, P, P, P, None, None, None, None) == 1  # no output
    assert b(P, 5, 16, 8, 2, P, P, P, P, None, None, P, None) == 3
    assert b(P, 2, 16, 8, 2, P, P, P + 4, P, None, None, P, None) == 4
    assert b(P, 2, 0, 8, 2, P, P, P, P, None, None, P, None) == 0


def test_python_refusals():
    import grouped_gemm_opt as g
    with pytest.raises(AssertionError):  # host logits
        g.moe_router(torch.randn(4, 8), 2)
    with pytest.raises(AssertionError):
        g.grouped_gemm_opt_int8(torch.zeros(4, 16, dtype=torch.int8), torch.ones(4),
                                torch.zeros(1, 8, 16, dtype=torch.int8), torch.ones(1, 8),
                                torch.tensor([4]))
    with pytest.raises(RuntimeError, match="CUDA"):
        g.quantize_int8(torch.randn(4, 16).to(torch.bfloat16))
    w = g.MoEInt8Weights(torch.zeros(8, 32, 16, dtype=torch.int8), torch.ones(8, 32),
                         torch.zeros(8, 16, 16, dtype=torch.int8), torch.ones(8, 16))
    with pytest.raises(AssertionError):  # host tokens
        g.fused_moe_int8(torch.randn(4, 16), torch.randn(4, 8), w, 2)


def test_routing_of_another_shape_is_refused():
    from grouped_gemm_opt.moe import MoERouting, fused_moe
    r = MoERouting(torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2),
                   torch.zeros(8, dtype=torch.int64), torch.tensor(0.0),
                   torch.zeros(8, dtype=torch.int64), torch.zeros(16, dtype=torch.int32))
    x, wgu, wd = torch.randn(4, 16), torch.randn(8, 32, 16), torch.randn(8, 16, 16)
    with pytest.raises(AssertionError, match="routing is for"):
        fused_moe(x, torch.randn(4, 8), wgu, wd, 3, routing=r)
    with pytest.raises(AssertionError, match="routing is for"):
        fused_moe(torch.randn(5, 16), torch.randn(5, 8), wgu, wd, 2, routing=r)


def test_given_routing_replaces_the_route_stage():
    """fused_moe with a routing runs the other stages on it and does not route again."""
    from grouped_gemm_opt.moe import MoEOps, MoERouting, fused_moe
    T, H, F, E, k = 6, 8, 16, 4, 2
    g = torch.Generator().manual_seed(0)
    x, logits = torch.randn(T, H, generator=g), torch.randn(T, E, generator=g)
    wgu, wd = torch.randn(E, 2 * F, H, generator=g), torch.randn(E, H, F, generator=g)
    ids = torch.sort(logits, dim=1, descending=True)[1][:, :k].to(torch.int32)
    w = torch.softmax(logits.gather(1, ids.long()), 1).requires_grad_(True)
    tpe = torch.bincount(ids.flatten().long(), minlength=E)
    r = MoERouting(ids, w, tpe, torch.tensor(1.0), tpe, torch.zeros(8, dtype=torch.int32))
    seen = []

    def permute(xs, i, scratch, experts):
        assert i is ids and scratch is r.scratch and experts == E
        order = torch.sort(ids.flatten(), stable=True)[1]
        pos = torch.empty(T * k, dtype=torch.int64)
        pos[order] = torch.arange(T * k)
        return xs[order // k], None, pos

    def no_route(*_):
        raise AssertionError("routed again")

    def experts(f):
        def stage(rows, weights, counts, n, sort):
            assert counts is tpe
            return torch.cat([f(a, weights[e]) for e, a in enumerate(rows.split(counts.tolist()))])
        return stage

    def glu(a, m):
        gate, up = (a @ m.t()).chunk(2, 1)
        return torch.nn.functional.silu(gate) * up

    def combine(y, weights, pos):
        assert not weights.requires_grad
        seen.append(True)
        return (y[pos].reshape(T, k, H) * weights[:, :, None]).sum(1)

    ops = MoEOps(no_route, permute, experts(glu), experts(lambda a, m: a @ m.t()), combine)
    out = fused_moe(x, logits, wgu, wd, k, ops=ops, routing=r)
    want = sum(w.detach()[:, j, None] * torch.stack(
        [wd[ids[t, j]] @ glu(x[t][None], wgu[ids[t, j]])[0] for t in range(T)]) for j in range(k))
    assert seen and torch.allclose(out, want, rtol=1e-4, atol=1e-4)
