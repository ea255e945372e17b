"""One rule for routing: the layers' own router, moe_router and the oracle choose the same experts with the
same weights for signed zeros, infinities and NaN too."""
import numpy as np
import pytest
import torch

import grouped_gemm_oracle as oracle

DEV = "cuda:0"
INF = float("inf")


def special_rows(E, seed=0):
    """Rows drawn from few values, zeros of both signs, infinities, NaN of both signs and the least
    number among them, and rows of one value only."""
    g = torch.Generator().manual_seed(seed + E)
    nan = torch.tensor([0x7fc00000, -0x400000], dtype=torch.int32).view(torch.float32)
    low = torch.finfo(torch.float32).min
    palettes = [[0.0, -0.0], [0.0, -0.0, 1.0, -1.0], [-INF, 0.0, -0.0], [-INF], [-INF, low],
                [INF, -INF, 1.0], [nan[0], nan[1], 0.0], [nan[0], nan[1], INF, -INF, -0.0, 0.0], [low],
                [nan[1], -INF], [-0.0], [1e-45, 0.0, -1e-45]]
    rows = []
    for p in palettes:
        p = torch.tensor([float(v) for v in p])
        for _ in range(12):
            rows.append(p[torch.randint(0, len(p), (E,), generator=g)])
    l = torch.stack(rows)
    # a float() of a NaN loses its sign: put negative NaN in by its bits
    l.view(torch.int32)[::7][torch.isnan(l[::7])] = -0x400000
    return l


def test_oracle_rule():
    l = np.array([[-0.0, 0.0, -1.0], [np.inf, np.nan, np.nan], [-np.inf] * 3,
                  [-np.inf, 2.0, -np.inf], [-0.0, -1.0, 0.0]], dtype=np.float32)
    ids, w, tpe = oracle.route(l, 2)
    assert ids.tolist() == [[0, 1], [1, 2], [0, 1], [1, 0], [0, 2]]
    assert w[0].tolist() == [0.5, 0.5] and w[2].tolist() == [0.0, 0.0] and w[3].tolist() == [1.0, 0.0]
    assert np.isnan(w[1]).all() and w[4].tolist() == [0.5, 0.5] and tpe.tolist() == [4, 4, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("E,k", [(2, 1), (3, 2), (8, 2), (33, 5), (64, 8), (256, 8), (500, 10),
                                 (1024, 16)])
@pytest.mark.parametrize("copies", [1, 3])
def test_both_routers_and_the_oracle_agree(E, k, copies):
    """copies: both launch forms of moe_router (up to 256 tokens, and more)."""
    from grouped_gemm_opt import _C, moe_router
    l = special_rows(E).repeat(copies, 1)
    ids, w, tpe = oracle.route(l.numpy(), k)
    a = moe_router(l.to(DEV), k)
    b = _C.moe_route(l.to(DEV), k)
    for got in (a.topk_ids, b[0]):
        assert np.array_equal(got.cpu().numpy(), ids)
    assert torch.equal(a.topk_weights.view(torch.int32), b[1].view(torch.int32)) or torch.equal(
        torch.nan_to_num(a.topk_weights, nan=-1.0), torch.nan_to_num(b[1], nan=-1.0))
    np.testing.assert_allclose(b[1].cpu().numpy(), w, rtol=2e-6, atol=1e-7)
    assert a.tokens_per_expert.tolist() == b[2].tolist() == tpe.tolist()
    assert torch.equal(a.scratch[:b[3].numel()], b[3])


@pytest.mark.gpu
def test_layers_with_and_without_a_given_routing():
    from grouped_gemm_opt import (fused_moe, fused_moe_fp8, fused_moe_int8, moe_router,
                                  quantize_moe_weights, quantize_moe_weights_int8)
    E, H, F, k = 8, 64, 128, 2
    l = special_rows(E).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(l.size(0), H, device=DEV, generator=g).to(torch.bfloat16)
    wgu = (torch.randn(E, 2 * F, H, device=DEV, generator=g) * 0.1).to(torch.bfloat16)
    wd = (torch.randn(E, H, F, device=DEV, generator=g) * 0.1).to(torch.bfloat16)
    r = moe_router(l, k)
    empty = (l == -INF).all(1)
    undefined = r.topk_weights.isnan().any(1)
    assert int(empty.sum()) >= 12 and int(undefined.sum()) >= 12
    qw = quantize_moe_weights_int8(wgu, wd)
    for out, given in ((fused_moe(x, l, wgu, wd, k), fused_moe(x, l, wgu, wd, k, routing=r)),
                       (fused_moe_int8(x, l, qw, k), fused_moe_int8(x, l, qw, k, routing=r)),
                       (fused_moe_fp8(x, l, quantize_moe_weights(wgu, wd), k), None)):
        assert torch.all(out[empty] == 0) and out[undefined].isnan().all()
        assert out[~undefined].isfinite().all()
        if given is not None:
            assert torch.equal(torch.nan_to_num(out, nan=-1.0), torch.nan_to_num(given, nan=-1.0))
