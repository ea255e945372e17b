"""Router, quantiser, dispatch and INT8 product on tensors of more than 2^31 elements: rows behind the
32-bit border are checked against the same rows computed alone (rows and tokens are independent)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows_to_check(n):
    return torch.tensor([0, 1, n // 2, n - 33, n - 2, n - 1], device=DEV)


def test_router_past_32_bits():
    from grouped_gemm_opt import moe_router
    T, E, k = (1 << 21) + 37, 1024, 4
    g = torch.Generator(device=DEV).manual_seed(0)
    logits = torch.randn(T, E, device=DEV, generator=g, dtype=torch.bfloat16).requires_grad_(True)
    r = moe_router(logits, k)
    at = rows_to_check(T)
    small = moe_router(logits.detach()[at], k)
    assert torch.equal(r.topk_ids[at], small.topk_ids)
    assert torch.equal(r.topk_weights[at], small.topk_weights)
    assert int(r.tokens_per_expert.sum()) == T * k
    counts = torch.zeros(E, dtype=torch.int64, device=DEV)
    counts.scatter_add_(0, r.topk_ids.reshape(-1).long(), torch.ones(T * k, dtype=torch.int64,
                                                                   device=DEV))
    assert torch.equal(r.tokens_per_expert, counts)
    # without a preference every expert gets its share up to sqrt(1 / (T k / E)), about 1.1 %: the
    # loss is near 1 (f and p deviate together, quadratically)
    assert abs(r.balance_loss.item() - 1.0) < 1e-2
    gw = torch.zeros(T, k, device=DEV)
    gw[at] = torch.randn(len(at), k, device=DEV, generator=g)
    leaf = logits.detach()[at].requires_grad_(True)
    want, = torch.autograd.grad(moe_router(leaf, k).topk_weights, leaf, gw[at])
    got, = torch.autograd.grad(r.topk_weights, logits, gw)
    assert torch.equal(got[at], want)
    assert torch.count_nonzero(got[2:at[2]]) == 0


def test_quantiser_past_32_bits():
    from grouped_gemm_opt import quantize_int8
    for rows, cols in [(131075, 16400), (2100003, 1040)]:
        x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
        x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
        q, s = quantize_int8(x)
        at = rows_to_check(rows)
        want_q, want_s = quantize_int8(x[at])
        assert torch.equal(q[at], want_q) and torch.equal(s[at], want_s)
        del x, q, s


def test_product_past_32_bits():
    """Output offsets behind 2^31 elements and, in the second case, input offsets."""
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    g = torch.Generator(device=DEV).manual_seed(2)
    for counts, n, k in [([40000, 0, 30001], 32768, 64), ([131072, 7], 64, 16400)]:
        rows = sum(counts)
        x = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device=DEV, generator=g)
        w = torch.randint(-127, 128, (len(counts), n, k), dtype=torch.int8, device=DEV, generator=g)
        xs, ws = torch.rand(rows, device=DEV), torch.rand(len(counts), n, device=DEV)
        out = grouped_gemm_opt_int8(x, xs, w, ws, torch.tensor(counts, device=DEV))
        last = len(counts) - 1
        for at in (rows - 1, rows - 3, rows - counts[last], 5):
            e = last if at >= rows - counts[last] else 0
            one = torch.zeros(len(counts), dtype=torch.int64, device=DEV)
            one[e] = 1
            want = grouped_gemm_opt_int8(x[at:at + 1], xs[at:at + 1].clone(), w, ws, one)
            assert torch.equal(out[at:at + 1], want)
        check_device_errors(0)
        del x, w, out


def test_dispatch_past_32_bits():
    from grouped_gemm_opt import _C, moe_router, quantize_int8
    T, H, E, k = 70001, 4096, 16, 8
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(T, H, device=DEV, generator=g, dtype=torch.bfloat16)
    r = moe_router(torch.randn(T, E, device=DEV, generator=g), k)
    q, s, pos = _C.moe_permute_int8(x, r.topk_ids, r.scratch, E)
    at = rows_to_check(T)
    want_q, want_s = quantize_int8(x[at])
    for j in range(k):
        p = pos.view(T, k)[at, j].long()
        assert torch.equal(q[p], want_q) and torch.equal(s[p], want_s)
    assert torch.equal(torch.sort(pos)[0], torch.arange(T * k, dtype=torch.int32, device=DEV))
