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


def test_errors_go_to_the_word_that_a_call_names():
    """The C entry's error_dev: the workspace's own error word stays clear."""
    import ctypes

    from build_ext import lib_path
    lib = ctypes.CDLL(str(lib_path()))
    f = lib.ggo_grouped_gemm_int8
    f.argtypes = [ctypes.c_void_p] * 6 + [ctypes.c_int] * 2 + [ctypes.c_int64] * 3 + \
        [ctypes.c_int] * 4 + [ctypes.c_void_p] * 3
    word = lib.ggo_workspace_error_word
    word.argtypes, word.restype = [ctypes.c_void_p], ctypes.c_void_p
    read = lib.ggo_workspace_error
    read.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]
    x = torch.ones(32, 64, dtype=torch.int8, device=DEV)
    w = torch.ones(2, 64, 64, dtype=torch.int8, device=DEV)
    xs, ws = torch.ones(32, device=DEV), torch.ones(2, 64, device=DEV)
    out = torch.empty(32, 64, dtype=torch.bfloat16, device=DEV)
    counts = torch.tensor([20, 11], device=DEV)  # one row short
    own, other = (torch.zeros(256, dtype=torch.uint8, device=DEV) for _ in range(2))
    stream = torch.cuda.current_stream().cuda_stream
    assert f(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), out.data_ptr(),
             counts.data_ptr(), 2, 2, 32, 64, 64, 0, 0, 4, 1, own.data_ptr(),
             word(other.data_ptr()), stream) == 0
    code = ctypes.c_int(-1)
    assert read(own.data_ptr(), stream, ctypes.byref(code)) == 0 and code.value == 0
    assert read(other.data_ptr(), stream, ctypes.byref(code)) == 0 and code.value == 9
    assert read(other.data_ptr(), stream, ctypes.byref(code)) == 0 and code.value == 0
