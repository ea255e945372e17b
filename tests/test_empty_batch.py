"""Layers and their stages take a batch without tokens, as moe_router and the INT8 layer do: empty tensors
have no address, and there is nothing to read or write."""
import ctypes

import pytest
import torch

from build_ext import lib_path

P = 1 << 20
DEV = "cuda:0"


def test_stages_without_tokens_need_no_addresses():
    lib = ctypes.CDLL(str(lib_path()))
    v, i, l = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    f = lib.ggo_moe_permute
    f.argtypes = [v, l, l, i, i] + [v] * 5 + [i, v]
    assert f(None, 0, 64, 8, 2, None, None, None, None, P, 0, None) == 0
    assert f(None, 4, 64, 8, 2, P, P, P, P, P, 0, None) == 1
    assert f(P, 4, 64, 8, 2, P, None, P, P, P, 0, None) == 1
    assert f(None, -1, 64, 8, 2, P, P, P, P, P, 0, None) == 1
    f = lib.ggo_moe_combine
    f.argtypes = [v, v, v, l, l, i, v, i, v]
    assert f(None, None, None, 0, 64, 2, None, 0, None) == 0
    assert f(None, P, P, 4, 64, 2, P, 0, None) == 1 and f(P, P, P, 4, 64, 2, None, 0, None) == 1
    f = lib.ggo_quantize_fp8_rows
    f.argtypes = [v, l, l, i, v, v, v]
    assert f(None, 0, 64, 0, None, None, None) == 0 and f(None, 4, 64, 0, P, P, None) == 1
    f = lib.ggo_quantize_mxfp8
    f.argtypes = [v, i, v, i, l, l, v, v, v]
    assert f(None, 0, P, 8, 0, 128, None, P, None) == 0
    assert f(None, 0, P, 8, 4, 128, P, P, None) == 1


def test_route_scratch_without_tokens_holds_the_experts_starts():
    f = ctypes.CDLL(str(lib_path())).ggo_moe_route_scratch_bytes
    f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_int64, ctypes.c_int]
    assert f(0, 1024) == 4096 and f(0, 1) == 4 and f(1, 1024) == 8192


@pytest.mark.gpu
def test_routers_without_tokens():
    """Counts of zero for every expert, and the experts' starts behind an empty table."""
    from grouped_gemm_opt import _C, moe_router
    for E in (1, 8, 1024):
        l = torch.empty(0, E, device=DEV)
        ids, w, tpe, scratch = _C.moe_route(l, 1)
        assert ids.shape == w.shape == (0, 1) and tpe.tolist() == [0] * E
        assert scratch.numel() == E and torch.all(scratch == 0)
        assert moe_router(l, 1).tokens_per_expert.tolist() == [0] * E


@pytest.mark.gpu
def test_layers_without_tokens():
    import grouped_gemm_opt as ggo
    E, H, F, k = 8, 128, 256, 2
    x = torch.empty(0, H, dtype=torch.bfloat16, device=DEV)
    l = torch.empty(0, E, device=DEV)
    wgu = torch.randn(E, 2 * F, H, device=DEV).to(torch.bfloat16)
    wd = torch.randn(E, H, F, device=DEV).to(torch.bfloat16)
    outs = [ggo.fused_moe(x, l, wgu, wd, k),
            ggo.fused_moe(x, l, wgu, wd, k, routing=ggo.moe_router(l, k)),
            ggo.fused_moe_fp8(x, l, ggo.quantize_moe_weights(wgu, wd), k),
            ggo.fused_moe_mxfp8(x, l, ggo.quantize_moe_weights_mxfp8(wgu, wd), k),
            ggo.fused_moe_int8(x, l, ggo.quantize_moe_weights_int8(wgu, wd), k),
            ggo.fused_moe_host(x.cpu(), l.cpu(), wgu, wd, k)]
    for out in outs:
        assert out.shape == (0, H) and out.dtype == torch.bfloat16
    # one expert: the smallest tables
    r = ggo.moe_router(l[:, :1], 1)
    assert ggo.fused_moe(x, l[:, :1], wgu[:1], wd[:1], 1, routing=r).shape == (0, H)
    q, s = ggo.quantize_fp8(x)
    assert q.shape == (0, H) and s.shape == (0,)
    assert ggo.quantize_mxfp8(x, torch.zeros(E, dtype=torch.int64, device=DEV))[0].shape == (0, H)
    ggo.check_device_errors(0)
