"""A routing given to a layer is refused unless its parts are of the layer's shape, device and types:
the dispatch and the combine read and write by them. Nothing here needs a GPU."""
import ctypes
from dataclasses import replace

import pytest
import torch

from build_ext import lib_path

P = 1 << 20  # an aligned address that is never dereferenced on these paths


def _fitting(T=40, E=8, k=2):
    from grouped_gemm_opt import MoERouting
    return MoERouting(torch.zeros(T, k, dtype=torch.int32), torch.ones(T, k),
                      torch.zeros(E, dtype=torch.int64), torch.tensor(0.0),
                      torch.zeros(E, dtype=torch.int64),
                      torch.zeros(((T + 31) // 32 + 1) * E, dtype=torch.int32))


def test_a_fitting_routing_is_taken():
    from grouped_gemm_opt.moe import _routing_of
    r = _fitting()
    ids, w, tpe, scratch = _routing_of(r, torch.randn(40, 8), 2)
    assert ids is r.topk_ids and tpe is r.tokens_per_expert and scratch is r.scratch
    assert torch.equal(w, r.topk_weights)
    _routing_of(replace(_fitting(0, 1, 1), scratch=torch.zeros(3, dtype=torch.int32)),
                torch.randn(0, 1), 1)


@pytest.mark.parametrize("change,match", [
    (dict(topk_weights=torch.ones(39, 2)), "routing is for"),
    (dict(topk_weights=torch.ones(40, 3)), "routing is for"),
    (dict(topk_weights=torch.ones(40, 2, dtype=torch.bfloat16)), "topk_weights must be"),
    (dict(topk_weights=torch.ones(2, 40).t()), "topk_weights must be"),
    (dict(topk_ids=torch.zeros(40, 2, dtype=torch.int64)), "topk_ids must be"),
    (dict(topk_ids=torch.zeros(2, 40, dtype=torch.int32).t()), "topk_ids must be"),
    (dict(tokens_per_expert=torch.zeros(8, dtype=torch.int32)), "tokens_per_expert must be"),
    (dict(tokens_per_expert=torch.zeros(16, dtype=torch.int64)[::2]), "tokens_per_expert must be"),
    (dict(tokens_per_expert=torch.zeros(7, dtype=torch.int64)), "routing is for"),
    (dict(scratch=torch.zeros(24)), "scratch must be"),
    (dict(scratch=torch.zeros(23, dtype=torch.int32)), "scratch is not"),
    (dict(scratch=torch.zeros(24, dtype=torch.int32, device="meta")), "another device"),
    (dict(tokens_per_expert=torch.zeros(8, dtype=torch.int64, device="meta")), "another device"),
    (dict(topk_weights=torch.ones(40, 2, device="meta")), "another device"),
])
def test_a_routing_that_does_not_fit_is_refused(change, match):
    from grouped_gemm_opt import fused_moe
    r = replace(_fitting(), **change)
    x, wgu, wd = torch.randn(40, 16), torch.randn(8, 32, 16), torch.randn(8, 16, 16)
    with pytest.raises(AssertionError, match=match):
        fused_moe(x, torch.randn(40, 8), wgu, wd, 2, routing=r)


def test_bounded_dispatch_refusals():
    f = ctypes.CDLL(str(lib_path())).ggo_ep_dispatch_bounded
    f.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int] + \
        [ctypes.c_void_p] * 3 + [ctypes.c_int, ctypes.c_int, ctypes.c_int64] + \
        [ctypes.c_void_p] * 3 + [ctypes.c_int, ctypes.c_void_p]
    two = (ctypes.c_void_p * 2)(P, P)

    def call(x=P, t=16, h=64, e=8, k=2, ids=P, scratch=P, counts=P, world=2, rank=0, cap=64,
             recv=two, origin=two, pos=P, dt=0):
        return f(x, t, h, e, k, ids, scratch, counts, world, rank, cap, recv, origin, pos, dt, None)

    assert call(cap=-1) == 1 and call(rank=2) == 1 and call(world=3) == 1 and call(counts=None) == 1
    assert call(recv=(ctypes.c_void_p * 2)(P, None)) == 1 and call(h=60) == 4 and call(dt=2) == 3
    assert call(t=0) == 0
