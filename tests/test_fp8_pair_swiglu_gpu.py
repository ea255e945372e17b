"""The FP8 gate/up product on CTA-pair tiles (segments long enough that the automatic choice takes
them): every output column is computed, as on single-CTA tiles."""
import pytest
import torch

import grouped_gemm_oracle as oracle
from gpu_util import assert_parity
from inputs import gemm_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("counts,f,k", [([2000, 0, 3000, 77], 2048, 256),
                                        ([1024] * 4, 1032, 128)])
def test_swiglu_fp8_on_pair_tiles(counts, f, k):
    from grouped_gemm_opt import _C, quantize_fp8
    x, w, tpe = gemm_inputs(counts, k, 2 * f, seed=2)
    xq, xs = quantize_fp8(x.to(DEV))
    wq, ws = quantize_fp8(w.to(DEV))
    h = _C.grouped_gemm_swiglu_fp8(xq, xs, wq, ws, tpe.to(DEV), len(counts), True)
    xd = xq.cpu().float() * xs.cpu().unsqueeze(1)
    wd = wq.cpu().float() * ws.cpu().unsqueeze(-1)
    assert_parity(h, oracle.swiglu_gemm(xd, wd, tpe, len(counts)), "swiglu fp8, pair tiles")
