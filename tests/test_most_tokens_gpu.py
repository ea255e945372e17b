"""The largest token count that the router, the dispatch with quantisation and the combine take, 2^31 - 1:
counters that step past the last token do not wrap. Only the ends of the large tensors are looked at;
needs up to 140 GB on the device."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = 2 ** 31 - 1
TAIL = 10000  # more than a step of every kernel's grid


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(DEV)[0] < 150 << 30:
        pytest.skip("needs 150 GB free on the device")
    yield
    torch.cuda.empty_cache()


def lopsided_logits():
    """Expert 0 by the tie for all tokens but the last TAIL, which prefer expert 1."""
    l = torch.zeros(T, 2, dtype=torch.bfloat16, device=DEV)
    l[-TAIL:, 1] = 1
    return l


def test_router():
    from grouped_gemm_opt import moe_router
    leaf = lopsided_logits().requires_grad_(True)
    r = moe_router(leaf, 1)
    assert r.tokens_per_expert.tolist() == r.balance_counts.tolist() == [T - TAIL, TAIL]
    for part, e in ((slice(0, TAIL), 0), (slice(T - 2 * TAIL, T - TAIL), 0), (slice(-TAIL, None), 1)):
        assert torch.all(r.topk_ids[part] == e) and torch.all(r.topk_weights[part] == 1)
    f = [(T - TAIL) / T, TAIL / T]
    p_tail = [1 / (1 + math.e), math.e / (1 + math.e)]
    p = [((T - TAIL) * 0.5 + TAIL * q) / T for q in p_tail]
    loss = 2 * (f[0] * p[0] + f[1] * p[1])
    assert abs(r.balance_loss.item() - loss) <= 2.0 ** -20 * loss
    grad, = torch.autograd.grad(r.balance_loss, leaf)
    for part, q in ((slice(0, TAIL), (0.5, 0.5)), (slice(T - 2 * TAIL, T - TAIL), (0.5, 0.5)),
                    (slice(-TAIL, None), p_tail)):
        mean = q[0] * f[0] + q[1] * f[1]
        want = torch.tensor([2 / T * q[e] * (f[e] - mean) for e in range(2)], dtype=torch.float64)
        # half a step of bf16 and some twenty roundings in fp32
        assert torch.all((grad[part].cpu().double() - want).abs() <=
                         (2.0 ** -8 + 20 * 2.0 ** -24) * want.abs())


def test_dispatch_with_quantisation():
    from grouped_gemm_opt import _C, moe_router, quantize_int8
    r = moe_router(lopsided_logits(), 1)
    ids = r.topk_ids
    table = r.scratch[:(-(-T // 32) + 1) * 2].clone()
    del r
    torch.cuda.empty_cache()
    x = torch.zeros(T, 16, dtype=torch.bfloat16, device=DEV)
    x[-2 * TAIL:] = torch.randn(2 * TAIL, 16, device=DEV).to(torch.bfloat16)
    q, s, pos = _C.moe_permute_int8(x, ids, table, 2)
    want_q, want_s = quantize_int8(x[-2 * TAIL:])
    assert torch.equal(q[-2 * TAIL:], want_q) and torch.equal(s[-2 * TAIL:], want_s)
    assert torch.equal(pos[-2 * TAIL:], torch.arange(T - 2 * TAIL, T, device=DEV,
                                                     dtype=torch.int32))
    assert torch.count_nonzero(q[:TAIL]) == 0 and torch.all(s[:TAIL] == 1)


def test_combine():
    from grouped_gemm_opt import _C
    y = torch.zeros(T, 8, dtype=torch.bfloat16, device=DEV)
    y[-TAIL:] = torch.randn(TAIL, 8, device=DEV).to(torch.bfloat16)
    w = torch.ones(T, 1, device=DEV)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    out = _C.moe_combine(y, w, pos)
    assert torch.equal(out[-2 * TAIL:], y[-2 * TAIL:]) and torch.count_nonzero(out[:TAIL]) == 0
