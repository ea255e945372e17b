"""The INT8 forms of the GEMM kernels return by themselves when a wait runs out, report it, and the next
call is right: the stall hook leaves the first tile's first pipeline stage unarmed (in every CTA of
the cluster that shares it) and lowers the waits' limit to about 10 ms. Nothing faults or hangs."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("counts,n,k,tc", [([700, 300, 1100, 20], 1024, 512, 1),   # one CTA a tile
                                           ([700, 300, 1100, 20], 1024, 512, 3),   # CTA pairs
                                           ([3, 0, 20, 9], 1024, 512, 4),          # thin
                                           ([5], 256, 8192, 4),                    # eight a tile
                                           ([40, 20], 1000, 8192, 4)])             # two or four
def test_timeout_is_reported_and_passes(counts, n, k, tc, monkeypatch):
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    g = torch.Generator(device=DEV).manual_seed(n + k)
    rows, experts = sum(counts), len(counts)
    x = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device=DEV, generator=g)
    w = torch.randint(-127, 128, (experts, n, k), dtype=torch.int8, device=DEV, generator=g)
    xs, ws = torch.rand(rows, device=DEV), torch.rand(experts, n, device=DEV)
    tpe = torch.tensor(counts, device=DEV)
    want = grouped_gemm_opt_int8(x, xs, w, ws, tpe, tc)
    check_device_errors(0)
    for _ in range(2):
        monkeypatch.setenv("GGO_TEST_INJECT_STALL", "1")
        t0 = time.time()
        grouped_gemm_opt_int8(x, xs, w, ws, tpe, tc)
        torch.cuda.synchronize()
        assert time.time() - t0 < 10.0
        with pytest.raises(RuntimeError, match="error code 8$"):
            check_device_errors(0)
        monkeypatch.delenv("GGO_TEST_INJECT_STALL")
        assert torch.equal(grouped_gemm_opt_int8(x, xs, w, ws, tpe, tc), want)
        check_device_errors(0)
