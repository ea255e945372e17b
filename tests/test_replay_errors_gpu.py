"""check_device_errors waits for replays on other streams before it reads their errors."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_replay_still_running_on_another_stream_is_waited_for():
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(32, 64, device=DEV, generator=g).to(torch.bfloat16)
    w = torch.randn(2, 64, 64, device=DEV, generator=g).to(torch.bfloat16)
    counts = torch.tensor([20, 12], device=DEV)
    grouped_gemm_opt(x, w, counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grouped_gemm_opt(x, w, counts)
    check_device_errors(0)
    side = torch.cuda.Stream()
    busy = torch.randn(8192, 8192, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):  # some tens of milliseconds before the replay starts
            busy = busy @ busy * 1e-2
        counts[1] = 11
        graph.replay()
    with pytest.raises(RuntimeError):
        check_device_errors(0)
    torch.cuda.synchronize()
    check_device_errors(0)
