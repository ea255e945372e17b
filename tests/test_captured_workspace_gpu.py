"""The first call on a stream may be a captured one: the stream's workspace is then ready for eager
calls and later graphs, whether or not the first graph has been replayed."""
import pytest
import torch

from inputs import gemm_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_eager_call_after_a_first_captured_one():
    import grouped_gemm_opt as ggo
    x, w, tpe = gemm_inputs([300, 0, 513, 17, 256], 256, 512, seed=3)
    xd, wd, td = x.to(DEV), w.to(DEV), tpe.to(DEV)
    want = ggo.grouped_gemm_opt(xd, wd, td)
    torch.cuda.synchronize()
    # a stream that no call has used: priority -1 streams come from a pool of their own
    s = torch.cuda.Stream(priority=-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = ggo.grouped_gemm_opt(xd, wd, td)
    with torch.cuda.stream(s):
        filler = torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV)
        eager = ggo.grouped_gemm_opt(xd, wd, td)
        torch.cuda.synchronize()
        assert torch.equal(eager, want)
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(captured, want) and int(filler[0]) == 255
