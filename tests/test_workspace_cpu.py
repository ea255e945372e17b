"""Refusals of the workspaces' error report; nothing here needs a GPU."""
import ctypes

from build_ext import lib_path

P = 1 << 20


def test_collect_errors_refusals():
    f = ctypes.CDLL(str(lib_path())).ggo_workspace_collect_errors
    f.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]
    assert f(None, P, 1, None) == 1 and f(P, None, 1, None) == 1 and f(P, P, -1, None) == 1
    assert f(P, P, 1 << 40, None) == 2
    assert f(P, None, 0, None) == 0
