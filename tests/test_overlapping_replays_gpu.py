"""Graphs captured apart replay at the same time, beside eager calls: every product of a captured call
has tile counters of its own, which go back when the graph is gone, and its errors are reported."""
import gc
import subprocess
import sys
import time
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T, H, F, E, K = 2048, 512, 1024, 8, 2


def inputs(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, H, device=DEV, generator=g).to(torch.bfloat16)
    logits = torch.randn(T, E, device=DEV, generator=g)
    wgu = (torch.randn(E, 2 * F, H, device=DEV, generator=g) * 0.02).to(torch.bfloat16)
    wd = (torch.randn(E, H, F, device=DEV, generator=g) * 0.02).to(torch.bfloat16)
    return x, logits, wgu, wd


def bf16_layer(seed):
    import grouped_gemm_opt as ggo
    x, l, wgu, wd = inputs(seed)
    r = ggo.moe_router(l, K)
    return lambda: ggo.fused_moe(x, l, wgu, wd, K, routing=r)


def fp8_layer(seed):
    import grouped_gemm_opt as ggo
    x, l, wgu, wd = inputs(seed)
    qw = ggo.quantize_moe_weights(wgu, wd)
    return lambda: ggo.fused_moe_fp8(x, l, qw, K)


def mxfp8_layer(seed):
    import grouped_gemm_opt as ggo
    x, l, wgu, wd = inputs(seed)
    qw = ggo.quantize_moe_weights_mxfp8(wgu, wd)
    return lambda: ggo.fused_moe_mxfp8(x, l, qw, K)


def int8_layer(seed):
    import grouped_gemm_opt as ggo
    x, l, wgu, wd = inputs(seed)
    qw = ggo.quantize_moe_weights_int8(wgu, wd)
    return lambda: ggo.fused_moe_int8(x, l, qw, K)


def products(seed):
    """The plain products of every kind and the backward ones, as one tensor."""
    import grouped_gemm_opt as ggo
    from grouped_gemm_opt import _C
    x, _, wgu, _ = inputs(seed)
    counts = torch.tensor([300, 0, 17, 513, 256, 700, 1, 261], device=DEV)
    xq, xs = ggo.quantize_fp8(x)
    wq, ws = ggo.quantize_fp8(wgu)
    mx, ms = ggo.quantize_mxfp8(x, counts)
    mw, mws = ggo.quantize_mxfp8(wgu)

    def step():
        y = ggo.grouped_gemm_opt(x, wgu, counts)
        return torch.cat([t.flatten() for t in (
            y, _C.grouped_gemm_dgrad(y, wgu, counts), _C.grouped_gemm_wgrad(x, y, counts),
            ggo.grouped_gemm_opt_fp8(xq, xs, wq, ws, counts),
            ggo.grouped_gemm_opt_mxfp8(mx, ms, mw, mws, counts))])
    return step


@pytest.mark.parametrize("make", [bf16_layer, fp8_layer, mxfp8_layer, int8_layer, products])
def test_replays_at_the_same_time(make):
    from grouped_gemm_opt import check_device_errors
    steps = [make(0), make(1), make(2)]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    graphs = []
    for s in steps[:2]:  # both on the default capture stream
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = s()
        graphs.append((g, out, torch.cuda.Stream()))
    eager_stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        for g, out, s in graphs:
            with torch.cuda.stream(s):
                out.zero_()
                for _ in range(3):
                    g.replay()
        with torch.cuda.stream(eager_stream):
            eager = steps[2]()
        torch.cuda.synchronize()
        assert torch.equal(eager, want[2])
        for (_, out, _), w in zip(graphs, want):
            assert torch.equal(out, w)
    check_device_errors(0)


def test_workspaces_go_back_with_their_graph():
    import grouped_gemm_opt as ggo
    from grouped_gemm_opt import _C
    step = bf16_layer(3)
    want = step()
    gc.collect()
    torch.cuda.synchronize()
    made = []
    for _ in range(100):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del g, out
        made.append(_C.captured_workspaces(0)[1])
    end = time.time() + 10
    while _C.captured_workspaces(0)[0] > 0 and time.time() < end:
        gc.collect()  # graphs of other tests too
        time.sleep(0.01)
    assert _C.captured_workspaces(0)[0] == 0
    assert made[-1] <= made[0] + 64  # give-backs may lag behind
    ggo.check_device_errors(0)


def test_errors_of_replayed_products_are_reported():
    import grouped_gemm_opt as ggo
    x, _, wgu, _ = inputs(4)
    counts = torch.tensor([300, 0, 17, 513, 256, 700, 1, 261], device=DEV)
    want = ggo.grouped_gemm_opt(x, wgu, counts)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ggo.grouped_gemm_opt(x, wgu, counts)
    ggo.check_device_errors(0)
    counts[0] = 299
    g.replay()
    with pytest.raises(RuntimeError):
        ggo.check_device_errors(0)
    # an eager error and a replayed one are both read by one check
    ggo.grouped_gemm_opt(x, wgu, counts)
    g.replay()
    with pytest.raises(RuntimeError):
        ggo.check_device_errors(0)
    ggo.check_device_errors(0)
    counts[0] = 300
    g.replay()
    ggo.check_device_errors(0)
    assert torch.equal(out, want)


FRESH = """
import gc, sys, torch
sys.path[:0] = %r
from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
g = torch.Generator().manual_seed(0)
x = torch.randint(-127, 128, (32, 64), generator=g, dtype=torch.int8).cuda()
w = torch.randint(-127, 128, (2, 64, 64), generator=g, dtype=torch.int8).cuda()
a = x, torch.ones(32).cuda(), w, torch.ones(2, 64).cuda(), torch.tensor([20, 12]).cuda()
torch.cuda.synchronize()
first = torch.cuda.CUDAGraph()
with torch.cuda.graph(first):  # the first product of the process
    out = grouped_gemm_opt_int8(*a)
first.replay()
torch.cuda.synchronize()
once = out.clone()
del first, out
gc.collect()
torch.cuda.empty_cache()
filler = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
second = torch.cuda.CUDAGraph()
with torch.cuda.graph(second):
    out = grouped_gemm_opt_int8(*a)
check_device_errors(0)
a[4][1] = 11
second.replay()
try:
    check_device_errors(0)
except RuntimeError:
    pass
else:
    sys.exit("the mismatch was not reported")
a[4][1] = 12
second.replay()
check_device_errors(0)
assert torch.equal(out, once) and torch.equal(grouped_gemm_opt_int8(*a), once)
assert int(filler.min()) == 255
print("fine")
"""


def test_first_product_of_a_process_is_a_captured_one():
    """Its workspace is made during the capture and lasts beyond that graph and its memory pool."""
    import grouped_gemm_opt
    path = [str(Path(grouped_gemm_opt.__file__).resolve().parent.parent)]
    r = subprocess.run([sys.executable, "-c", FRESH % path], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
