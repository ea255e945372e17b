"""fused_moe over expert-parallel ranks with a given routing (CPU gloo ranks, the stages by the oracle):
no stage routes again, and the result is that of the layer that routes itself."""
import datetime
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import grouped_gemm_oracle as oracle
from test_ep_gloo import E, K, _inputs, _port, _weights, cpu_ops


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=30))
    try:
        from grouped_gemm_opt import MoERouting, fused_moe
        x, logits = _inputs(rank)
        wgu, wd = _weights()
        el = E // world
        mine = slice(rank * el, (rank + 1) * el)
        ops = cpu_ops({})
        ids, w, tpe, _ = ops.route(logits, K)

        def no_route(*_):
            raise AssertionError("routed again")

        ops.route = no_route
        r = MoERouting(ids, w, tpe, torch.tensor(1.0), tpe, torch.zeros(2 * E, dtype=torch.int32))
        out = fused_moe(x, logits, wgu[mine].contiguous(), wd[mine].contiguous(), K,
                        ep_group=dist.group.WORLD, ops=ops, routing=r)
        q.put((rank, out.float().numpy()))
    except Exception as exc:  # noqa: BLE001 - reported to the parent
        q.put((rank, repr(exc)))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_given_routing(world):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in range(world))
    for p in procs:
        p.join(timeout=60)
        if p.is_alive():
            p.kill()
    wgu, wd = _weights()
    for r in range(world):
        assert not isinstance(got[r], str), got[r]
        x, logits = _inputs(r)
        ref = oracle.moe_layer(x, logits, wgu, wd, K, round_to=torch.bfloat16).numpy()
        np.testing.assert_allclose(got[r], ref, rtol=1e-5, atol=1e-5)
