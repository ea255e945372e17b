"""SwiGLU of the INT8 products for gates far below zero, where e^-g passes the largest divisor of the
hardware's reciprocal (about -87.3) and then the largest number (-88.7), beside large up values.

Tolerance, relative: half a step of the result's type; g and u are within 3 * 2^-24, e^x is off by
(2 + 1.2 |x|) 2^-23 and its argument's error, twice where it is taken as two factors e^(g/2): in all
below (2 (4 + 1.2 |g|) + 3 (2 + |g|) + 10) 2^-24. Below the smallest number half of that."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
LARGEST = {torch.bfloat16: 3.3e38, torch.float16: 6.5e4}


@pytest.mark.parametrize("dtype,up", [(torch.bfloat16, 1e-3), (torch.bfloat16, 1e20),
                                      (torch.bfloat16, 1e32), (torch.float16, 1e-4)])
@pytest.mark.parametrize("counts,tc", [([5, 0, 40], 4), ([100, 70], 1), ([700, 300], 3)])
def test_far_gates(counts, tc, dtype, up):
    from grouped_gemm_opt import _C
    F, K = 264, 16
    g = torch.Generator().manual_seed(sum(counts))
    rows, experts = sum(counts), len(counts)
    x = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (experts, 2 * F, K), generator=g, dtype=torch.int8)
    xs = torch.rand(rows, generator=g) + 0.5
    ws = torch.cat([torch.rand(experts, F, generator=g) / 150, torch.full((experts, F), up)], 1)
    out = _C.grouped_gemm_int8(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV),
                               torch.tensor(counts, device=DEV), True, dtype, tc, True)
    at, far = 0, 0
    for e, c in enumerate(counts):
        s = x[at:at + c].double() @ w[e].double().t() * xs[at:at + c, None].double() * ws[e].double()
        gate, u = s[:, :F], s[:, F:]
        ref = gate * torch.sigmoid(gate) * u
        tol = (2 * (4 + 1.2 * gate.abs()) + 3 * (2 + gate.abs()) + 10) * 2.0 ** -24
        bound = ref.abs() * (HALF_STEP[dtype] + tol) + LEAST[dtype]
        fits = ref.abs() < LARGEST[dtype]
        got = out[at:at + c].cpu().double()
        assert torch.all(((got - ref).abs() <= bound)[fits])
        far += int(((gate < -87.3) & (gate > -120)).sum())
        at += c
    assert far > 100  # the range is met
