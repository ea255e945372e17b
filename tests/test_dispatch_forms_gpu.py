"""Forms that the sizes choose: every kernel of the dispatch with quantisation, rows longer than its
registers hold among them, and the router's scalar rows where a base is not 16-byte aligned."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,E,k", [(1300, 2048, 8, 2), (1300, 2064, 8, 2), (1300, 4096, 8, 2),
                                     (1300, 4112, 16, 2), (1300, 7168, 16, 2), (1300, 8192, 8, 1),
                                     (1300, 8208, 8, 2), (1300, 16400, 16, 3), (40, 8192, 8, 2),
                                     (40, 8208, 8, 2), (1184, 16400, 8, 2), (1185, 16400, 8, 2)])
def test_dispatch_with_quantisation(T, H, E, k, dtype):
    """Equal to the dispatch followed by the quantiser, the maximum of some rows at either end."""
    from grouped_gemm_opt import _C, quantize_int8
    g = torch.Generator(device=DEV).manual_seed(T + H)
    x = torch.randn(T, H, device=DEV, generator=g).to(dtype)
    x[0] = 0
    x[1, H - 1], x[2, 0], x[T - 1, H // 2] = 300.0, -300.0, 300.0
    x[3, H - 9] = float("nan")
    ids, _, _, scratch = _C.moe_route(torch.randn(T, E, device=DEV, generator=g), k)
    q, s, pos = _C.moe_permute_int8(x, ids, scratch, E)
    xs, _, want_pos = _C.moe_permute(x, ids, scratch, E)
    want_q, want_s = quantize_int8(xs)
    assert torch.equal(pos, want_pos) and torch.equal(q, want_q)
    assert torch.equal(s.view(torch.int32), want_s.view(torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [40, 300, 6000])
@pytest.mark.parametrize("E", [32, 64, 128, 256, 512, 1024])
def test_router_rows_off_their_alignment(T, E, dtype):
    """Logits that start one element behind an aligned address: the aligned copy's bits, gradient too.
    The sums of the forward are taken in the same order in both (lanes hold other experts, so the sum
    over all experts may differ in its last bits: loss and gradient within that)."""
    from grouped_gemm_opt import moe_router
    g = torch.Generator(device=DEV).manual_seed(T + E)
    base = torch.randn(T * E + 1, device=DEV, generator=g).to(dtype)
    off = base[1:].view(T, E).detach().requires_grad_(True)
    assert off.is_contiguous() and off.data_ptr() % 16
    plain = off.detach().clone().requires_grad_(True)
    assert plain.data_ptr() % 16 == 0
    k = 4
    gw = torch.randn(T, k, device=DEV, generator=g)
    a, b = moe_router(off, k), moe_router(plain, k)
    assert torch.equal(a.topk_ids, b.topk_ids) and torch.equal(a.topk_weights, b.topk_weights)
    assert torch.equal(a.tokens_per_expert, b.tokens_per_expert)
    # a sum of up to 1024 positive terms, in lanes of 32 terms and a tree of 5: 38 roundings a side
    tol = 2 * 38 * 2.0 ** -24
    assert abs(a.balance_loss.item() - b.balance_loss.item()) <= 2 * tol * b.balance_loss.item()
    one = torch.ones((), device=DEV)
    ga, = torch.autograd.grad((a.topk_weights, a.balance_loss), off, (gw, one))
    gb, = torch.autograd.grad((b.topk_weights, b.balance_loss), plain, (gw, one))
    # the balance part: E/T p (f - sum p f), p within tol, the bracket by absolute values; the weights'
    # part has the same bits; the sum is rounded once
    n = a.balance_counts.double() / (T * k)
    p = torch.softmax(plain.detach().double(), 1)
    size = E / T * p * (n + (p * n).sum(1, keepdim=True))
    step = torch.finfo(dtype).eps if dtype != torch.float32 else 2.0 ** -23
    least = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133
    assert torch.all((ga.double() - gb.double()).abs() <=
                     4 * tol * size + step * gb.double().abs() + least)
