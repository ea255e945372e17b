"""INT8 path: the quantiser against exact arithmetic (bit for bit), the grouped products against
integer sums, the layer against the same steps on the CPU.

Tolerances. A product's sum is an exact integer S (|S| < 2^31); the kernel rounds S to fp32, multiplies
by two fp32 scales and rounds to the result type: relative error below half a step of the type plus
4 * 2^-24 (scales of the reference are the same fp32 numbers), or half the smallest subnormal."""
import pytest
import torch

import grouped_gemm_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def ref_quant(x):
    """127 x / max|x| in 64 bits: 127 x is exact and so are ties; with significands of at most 11 bits
    every other quotient is at least 2^-20 from a tie, so rounding it decides nothing."""
    xd = x.double()
    top = xd.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    q = torch.where((top > 0) & ~bad, torch.round(127 * xd / top), 0.0)
    s = torch.where(top > 0, top.float() / 127, torch.ones_like(top, dtype=torch.float32))
    s = torch.where(bad, float("nan"), s)
    return torch.nan_to_num(q).to(torch.int8), s[..., 0]


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-1.0), torch.nan_to_num(b, nan=-1.0))


def check_quant(x):
    from grouped_gemm_opt import quantize_int8
    q, s = quantize_int8(x.to(DEV))
    rq, rs = ref_quant(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == x.shape[:-1]
    assert same(s.cpu(), rs)
    assert torch.equal(q.cpu(), rq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 16), (7, 48), (333, 1024), (37, 14336), (5, 16384),
                                       (3, 16400), (2, 40000), (64, 1040), (1000, 2048),
                                       (9, 4096), (70001, 16)])
def test_quantize_exact(rows, cols, dtype):
    g = torch.Generator().manual_seed(cols + rows)
    x = (torch.randn(rows, cols, generator=g) *
         torch.logspace(-3, 3, rows).unsqueeze(1)).to(dtype)
    if rows > 5:
        x[5] = 0
    check_quant(x)


@pytest.mark.parametrize("cols", [32, 64, 80, 256, 272, 512, 528, 1008, 2032, 2064, 4080, 4112, 8192,
                                  8208, 16368])
def test_quantize_row_widths(cols):
    """Both sides of every border between the forms for short, medium and long rows."""
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(131, cols, generator=g).to(torch.bfloat16)
    x[77, cols - 1] = 100.0  # the maximum in the last piece
    x[130] = 0
    check_quant(x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_every_value(dtype):
    """Every finite value of the type in rows whose maximum is one of many: ties (x = max / 2 among
    them), subnormals and the largest numbers."""
    bits = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    values = bits[torch.isfinite(bits)]
    g = torch.Generator().manual_seed(0)
    tops = values[torch.randint(1, values.numel(), (60,), generator=g)].tolist()
    tops += [values[1].item(), values[2].item(), values[-1].item(), 1.0, 2.0, 1.984375, 0.9921875]
    for top in tops:
        some = values[values <= top]
        some = torch.cat([some, -some])[-16384:]
        some = torch.cat([some, torch.zeros((-some.numel()) % 16, dtype=dtype)])
        some[0] = top
        check_quant(some.view(1, -1))


def test_quantize_nonfinite_rows():
    x = torch.randn(6, 64).to(torch.bfloat16)
    x[1, 3], x[2, 60], x[3, 5], x[3, 6] = float("inf"), float("nan"), -float("inf"), float("nan")
    x[4] = -float("inf")
    check_quant(x)


def test_quantize_strided_empty_and_3d():
    from grouped_gemm_opt import quantize_int8
    x = torch.randn(64, 96).to(torch.bfloat16)
    q, s = quantize_int8(x.to(DEV).t())
    rq, rs = ref_quant(x.t())
    assert torch.equal(q.cpu(), rq) and same(s.cpu(), rs)
    check_quant(torch.randn(3, 40, 32).to(torch.float16))
    q, s = quantize_int8(torch.empty(0, 32, dtype=torch.bfloat16, device=DEV))
    assert q.shape == (0, 32) and s.shape == (0,)


def codes(shape, g):
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)


def operands(counts, n, k, seed=0):
    g = torch.Generator().manual_seed(seed + k + n)
    rows, experts = sum(counts), len(counts)
    x, w = codes((rows, k), g), codes((experts, n, k), g)
    xs = torch.rand(rows, generator=g) * 0.02 + 1e-3
    ws = torch.rand(experts, n, generator=g) * 0.02 + 1e-3
    return x, xs, w, ws


def reference(counts, x, xs, w, ws):
    """Sums of the codes in 64 bits (exact: below 2^53), times the scales."""
    out, at = [], 0
    for e, c in enumerate(counts):
        s = x[at:at + c].to(DEV).double() @ w[e].to(DEV).double().t()
        out.append(s.cpu() * xs[at:at + c, None].double() * ws[e][None].double())
        at += c
    return torch.cat(out)


def assert_product(out, ref, dtype):
    bound = ref.abs() * (HALF_STEP[dtype] + 4 * 2.0 ** -24) + LEAST[dtype]
    assert out.dtype == dtype
    assert torch.all((out.cpu().double() - ref).abs() <= bound)


CASES = [([1], 8, 16), ([3], 1000, 1104), ([32] * 8, 1024, 512),
         ([1, 7, 8, 127, 128, 129, 0], 384, 256), ([700, 300, 1100, 20], 2048, 1024),
         ([0, 0, 5, 0], 264, 48), ([17], 4096, 14336), ([2] * 64, 128, 64),
         ([2000, 0, 3000, 77, 129, 1], 512, 272)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,n,k", CASES)
def test_grouped_product(counts, n, k, dtype):
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    x, xs, w, ws = operands(counts, n, k)
    tpe = torch.tensor(counts)
    ref = reference(counts, x, xs, w, ws)
    args = [t.to(DEV) for t in (x, xs, w, ws)]
    for tc in (4, 0, 1, 3):
        out = grouped_gemm_opt_int8(*args, tpe.to(DEV), tc, out_dtype=dtype)
        assert_product(out, ref, dtype)
    out = grouped_gemm_opt_int8(*args, tpe, sort_by_m=False, out_dtype=dtype)  # counts on the CPU
    assert_product(out, ref, dtype)
    check_device_errors(0)


LONG = [([1], 256, 4096), ([16], 4096, 4096), ([64], 1000, 2064), ([3, 0, 30, 31], 264, 8192),
         ([2] * 8, 14336, 4096), ([65], 128, 16384), ([200, 0, 90], 520, 3088), ([128], 256, 4096),
         ([1000], 64, 9008), ([5] * 12, 1024, 1040)]


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts,n,k", LONG)
def test_few_tiles_and_a_long_sum(counts, n, k, swiglu):
    """Few output tiles and long sums, in every tile width; repeated calls agree to the bit."""
    from grouped_gemm_opt import _C, check_device_errors
    x, xs, w, ws = operands(counts, 2 * n if swiglu else n, k, seed=11)
    dtype = torch.float16 if n % 16 else torch.bfloat16
    if swiglu:
        xs = xs * 4 / k ** 0.5
        ref, g = swiglu_reference(counts, x, xs, w, ws)
        tol = (2 * (2 + 1.2 * g.abs()) + 3 * (2 + g.abs()) + 8) * 2.0 ** -24
    else:
        ref, tol = reference(counts, x, xs, w, ws), 4 * 2.0 ** -24
    dev = [t.to(DEV) for t in (x, xs, w, ws, torch.tensor(counts))]
    for tc in (4, 0, 1):
        out = _C.grouped_gemm_int8(*dev, swiglu, dtype, tc, True)
        assert torch.all((out.cpu().double() - ref).abs() <=
                         ref.abs() * (HALF_STEP[dtype] + tol) + LEAST[dtype])
        for _ in range(10):
            assert torch.equal(out, _C.grouped_gemm_int8(*dev, swiglu, dtype, tc, True))
    check_device_errors(0)


@pytest.mark.parametrize("counts", [[1], [24], [27], [28], [64], [0, 3, 0, 9], [1] * 20])
@pytest.mark.parametrize("n,k", [(8, 16384), (136, 8192), (512, 4112), (2048, 10000), (4104, 6144)])
def test_sums_dealt_out_to_clusters(counts, n, k):
    """Few tiles and long sums: a cluster of two, four or eight CTAs per tile, over several tiles each,
    in turn with launches in one piece on the same stream."""
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    x, xs, w, ws = operands(counts, n, k, seed=3)
    ref = reference(counts, x, xs, w, ws)
    dev = [t.to(DEV) for t in (x, xs, w, ws, torch.tensor(counts))]
    other = [t.to(DEV) for t in operands([70, 3], 64, 64)] + [torch.tensor([70, 3], device=DEV)]
    want_other = grouped_gemm_opt_int8(*other)
    first = grouped_gemm_opt_int8(*dev)
    assert_product(first, ref, torch.bfloat16)
    for _ in range(20):
        assert torch.equal(grouped_gemm_opt_int8(*dev), first)
        assert torch.equal(grouped_gemm_opt_int8(*other), want_other)
    check_device_errors(0)


def test_longest_sum_does_not_wrap():
    """K = 131056 products of -128 with -128: 2147221504, just inside 32 bits, rounded to fp32."""
    from grouped_gemm_opt import grouped_gemm_opt_int8
    k = 131056
    x = torch.full((3, k), -128, dtype=torch.int8)
    x[1] = 127
    w = torch.full((1, 8, k), -128, dtype=torch.int8)
    xs, ws = torch.ones(3), torch.full((1, 8), 2.0 ** -20)
    out = grouped_gemm_opt_int8(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), torch.tensor([3]))
    assert_product(out, reference([3], x, xs, w, ws), torch.bfloat16)
    with pytest.raises(RuntimeError, match="shape"):
        grouped_gemm_opt_int8(torch.zeros(1, k + 16, dtype=torch.int8, device=DEV),
                              torch.ones(1, device=DEV),
                              torch.zeros(1, 8, k + 16, dtype=torch.int8, device=DEV),
                              torch.ones(1, 8, device=DEV), torch.tensor([1]))


def test_nan_scale_stays_in_its_row():
    from grouped_gemm_opt import grouped_gemm_opt_int8, quantize_int8
    x = torch.randn(40, 64, device=DEV).to(torch.bfloat16)
    x[11, 5] = float("nan")
    w = torch.randn(2, 48, 64, device=DEV).to(torch.bfloat16)
    out = grouped_gemm_opt_int8(*quantize_int8(x), *quantize_int8(w), torch.tensor([25, 15]))
    assert out[11].isnan().all()
    assert out[:11].isfinite().all() and out[12:].isfinite().all()


def test_device_errors_are_reported():
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    x, xs, w, ws = (t.to(DEV) for t in operands([20, 12], 64, 64))
    check_device_errors(0)
    grouped_gemm_opt_int8(x, xs, w, ws, torch.tensor([20, 11], device=DEV))
    with pytest.raises(RuntimeError):
        check_device_errors(0)
    grouped_gemm_opt_int8(x, xs, w, ws, torch.tensor([20, 12], device=DEV))
    check_device_errors(0)


def swiglu_reference(counts, x, xs, w, ws):
    gu = reference(counts, x, xs, w, ws)
    f = gu.size(1) // 2
    g, u = gu[:, :f], gu[:, f:]
    return g * torch.sigmoid(g) * u, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,f,k", [([1], 8, 16), ([5, 0, 70, 130], 200, 80),
                                        ([2000, 0, 3000, 77], 512, 256),
                                        ([1300, 700], 4096, 128), ([9], 14336, 4096)])
def test_swiglu(counts, f, k, dtype):
    """silu(g) u: g and u within 3 * 2^-24; e^-g is off by (2 + 1.2 |g|) 2^-23 + its argument's error
    |g| 3 * 2^-24, of which silu takes at most all; then a division, two products and the rounding.
    Scales keep |g| below about 40."""
    from grouped_gemm_opt import _C
    x, xs, w, ws = operands(counts, 2 * f, k, seed=7)
    xs = xs * 4 / k ** 0.5
    ref, g = swiglu_reference(counts, x, xs, w, ws)
    h = _C.grouped_gemm_int8(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV),
                             torch.tensor(counts, device=DEV), True, dtype, 4, True)
    assert h.dtype == dtype and h.shape == ref.shape
    tol = (2 * (2 + 1.2 * g.abs()) + 3 * (2 + g.abs()) + 8) * 2.0 ** -24
    bound = ref.abs() * (HALF_STEP[dtype] + tol) + LEAST[dtype]
    assert torch.all((h.cpu().double() - ref).abs() <= bound)


@pytest.mark.parametrize("T,H,E,k", [(1, 64, 4, 2), (33, 144, 7, 3), (700, 4096, 16, 2),
                                     (4097, 256, 256, 8)])
def test_permute_codes(T, H, E, k):
    """The dispatch with quantisation equals the dispatch followed by the quantiser."""
    from grouped_gemm_opt import _C, quantize_int8
    g = torch.Generator(device=DEV).manual_seed(T)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(T, H, device=DEV, generator=g).to(dtype)
        x[0] = 0
        ids, _, _, scratch = _C.moe_route(torch.randn(T, E, device=DEV, generator=g), k)
        q, s, pos = _C.moe_permute_int8(x, ids, scratch, E)
        xs, _, want_pos = _C.moe_permute(x, ids, scratch, E)
        want_q, want_s = quantize_int8(xs)
        assert torch.equal(pos, want_pos) and torch.equal(q, want_q) and torch.equal(s, want_s)


def layer_inputs(T, H, F, E, dtype, seed=9):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).to(dtype)
    logits = torch.randn(T, E, generator=g)
    wgu = (torch.randn(E, 2 * F, H, generator=g) * 0.02).to(torch.bfloat16)
    wd = (torch.randn(E, H, F, generator=g) * 0.02).to(torch.bfloat16)
    return x, logits, wgu, wd


def layer_reference(x, logits, qw, k, dtype):
    """The layer's steps in 64 bits on the CPU, with h and y rounded to the layer's type."""
    ids, w, tpe = oracle.route(logits.numpy(), k)
    st, pos = oracle.permute_indices(ids, logits.size(1))
    counts = tpe.tolist()
    xq, xs = ref_quant(x[torch.from_numpy(st).long()])
    ref, _ = swiglu_reference(counts, xq, xs, qw.w_gate_up_q.cpu(), qw.w_gate_up_scale.cpu())
    hq, hs = ref_quant(ref.to(dtype))
    y = reference(counts, hq, hs, qw.w_down_q.cpu(), qw.w_down_scale.cpu()).to(dtype)
    pos = torch.from_numpy(pos).long().reshape(x.size(0), k)
    return (y.double()[pos] * torch.from_numpy(w).double()[:, :, None]).sum(1), y[pos].double()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,F,E,k", [(1, 64, 32, 4, 2), (37, 144, 80, 5, 3),
                                       (512, 512, 1024, 8, 2), (3000, 256, 512, 2, 1)])
def test_layer(T, H, F, E, k, dtype):
    """An element of h may round to the neighbouring number of its type (the reference's 64-bit value
    and the kernel's fp32 one lie on two sides of a tie), which moves its code by at most one where it
    does (half a step of the type is at most 127 * 2^-8 < 1/2 code, a tie apart). Of F elements those
    are rare, about one in 2^-8 / 2^-20; F / 256 + 4 are allowed, each worth 127 codes' share of one
    weight. y may round the other way once (one step), and so does the result."""
    from grouped_gemm_opt import fused_moe_int8, moe_router, quantize_moe_weights_int8
    x, logits, wgu, wd = layer_inputs(T, H, F, E, dtype)
    qw = quantize_moe_weights_int8(wgu.to(DEV), wd.to(DEV))
    out = fused_moe_int8(x.to(DEV), logits.to(DEV), qw, k)
    assert out.dtype == dtype and out.shape == (T, H)
    ref, y = layer_reference(x, logits, qw, k, dtype)
    # one code of h times one weight: at most (max|h| / 127) * max|w|; max|h| <= 127 hs below
    gu_scale = qw.w_down_scale.max().item() * 127
    h_code = _largest_h_scale(x, logits, qw, k, dtype)
    flips = (F / 256 + 4) * h_code * gu_scale
    step = 2 * HALF_STEP[dtype]
    bound = flips + step * y.abs().amax(1) + step * ref.abs() + 4 * LEAST[dtype]
    assert torch.all((out.cpu().double() - ref).abs() <= bound)
    if T >= 512:
        # over many rows: about 2.5e-4 F changed codes a row, each 16 / (127 sqrt(F)) of it, which is
        # 0.2 % in the 2-norm, and the two roundings
        assert (out.cpu().double() - ref).norm() <= 2.0 ** -7 * ref.norm()
    r = moe_router(logits.to(DEV), k)
    assert torch.equal(out, fused_moe_int8(x.to(DEV), logits.to(DEV), qw, k, routing=r))


def _largest_h_scale(x, logits, qw, k, dtype):
    ids, _, tpe = oracle.route(logits.numpy(), k)
    st, _ = oracle.permute_indices(ids, logits.size(1))
    xq, xs = ref_quant(x[torch.from_numpy(st).long()])
    h, _ = swiglu_reference(tpe.tolist(), xq, xs, qw.w_gate_up_q.cpu(), qw.w_gate_up_scale.cpu())
    return ref_quant(h.to(dtype))[1].max().item()


def test_layer_close_to_the_unquantised_one():
    """Codes of normal values with 127 steps to the maximum (about 4 sigma): a relative error of
    about 4 / 127 / sqrt(12) = 0.9 % per operand; gate times up doubles it, and h, whose maximum is
    some 8 times its size, adds 1.8 %: 3 to 4 % in all."""
    from grouped_gemm_opt import fused_moe_int8, quantize_moe_weights_int8
    x, logits, wgu, wd = layer_inputs(512, 512, 1024, 8, torch.bfloat16)
    qw = quantize_moe_weights_int8(wgu.to(DEV), wd.to(DEV))
    out = fused_moe_int8(x.to(DEV), logits.to(DEV), qw, 2).float().cpu()
    ref = oracle.moe_layer(x, logits, wgu, wd, 2, round_to=torch.bfloat16)
    assert (out - ref).norm() <= 0.06 * ref.norm()


def test_router_then_layer_together():
    """Serving with load figures: one routing feeds the layer and reports counts and balance; masked
    (padding) tokens change the figures, not the layer. Empty batches pass."""
    from grouped_gemm_opt import fused_moe_int8, moe_router, quantize_moe_weights_int8
    T, H, F, E, k = 300, 128, 256, 8, 2
    x, logits, wgu, wd = layer_inputs(T, H, F, E, torch.bfloat16)
    qw = quantize_moe_weights_int8(wgu.to(DEV), wd.to(DEV))
    mask = torch.arange(T, device=DEV) < 250
    r = moe_router(logits.to(DEV), k, mask)
    assert int(r.tokens_per_expert.sum()) == T * k and int(r.balance_counts.sum()) == 250 * k
    whole = fused_moe_int8(x.to(DEV), logits.to(DEV), qw, k)
    assert torch.equal(fused_moe_int8(x.to(DEV), logits.to(DEV), qw, k, routing=r), whole)
    r = moe_router(logits[:0].to(DEV), k)
    none = fused_moe_int8(x[:0].to(DEV), logits[:0].to(DEV), qw, k, routing=r)
    assert none.shape == (0, H)
    assert fused_moe_int8(x[:0].to(DEV), logits[:0].to(DEV), qw, k).shape == (0, H)


def test_layer_graph_and_overlapping_replays():
    """Two captured layers replay on two streams beside an eager call; each has its own counters. The
    graphs are captured on streams that no call has used before."""
    from grouped_gemm_opt import check_device_errors, fused_moe_int8, quantize_moe_weights_int8
    T, H, F, E, k = 2048, 512, 1024, 8, 2
    x, logits, wgu, wd = layer_inputs(T, H, F, E, torch.bfloat16)
    qw = quantize_moe_weights_int8(wgu.to(DEV), wd.to(DEV))
    xd, ld = x.to(DEV), logits.to(DEV)
    want = fused_moe_int8(xd, ld, qw, k)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            out = fused_moe_int8(xd, ld, qw, k)
        graphs.append((g, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        eager = fused_moe_int8(xd, ld, qw, k)
        torch.cuda.synchronize()
        assert torch.equal(eager, want)
        for _, out, _ in graphs:
            assert torch.equal(out, want)
            out.zero_()
        torch.cuda.synchronize()
    check_device_errors(0)


def test_first_call_on_a_stream_is_a_captured_one():
    """The stream's workspace is made during the capture and must be usable eagerly afterwards, also
    when the graph is replayed late or never."""
    from grouped_gemm_opt import grouped_gemm_opt_int8
    counts = [300, 0, 513, 17, 256]
    x, xs, w, ws = (t.to(DEV) for t in operands(counts, 512, 256))
    tpe = torch.tensor(counts, device=DEV)
    want = grouped_gemm_opt_int8(x, xs, w, ws, tpe)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = grouped_gemm_opt_int8(x, xs, w, ws, tpe)
    with torch.cuda.stream(s):
        eager = grouped_gemm_opt_int8(x, xs, w, ws, tpe)
    torch.cuda.synchronize()
    assert torch.equal(eager, want)
    with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_host_counts_are_refused_in_a_capture():
    from grouped_gemm_opt import grouped_gemm_opt_int8
    x, xs, w, ws = (t.to(DEV) for t in operands([20, 12], 64, 64))
    tpe = torch.tensor([20, 12])
    grouped_gemm_opt_int8(x, xs, w, ws, tpe)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="captured"):
            grouped_gemm_opt_int8(x, xs, w, ws, tpe)


def test_errors_of_a_replayed_call_are_reported():
    """Counts that stop matching between capture and replay: the replay records it, wherever it runs."""
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    x, xs, w, ws = (t.to(DEV) for t in operands([20, 12], 64, 64))
    tpe = torch.tensor([20, 12], device=DEV)
    want = grouped_gemm_opt_int8(x, xs, w, ws, tpe)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = grouped_gemm_opt_int8(x, xs, w, ws, tpe)
    g.replay()
    check_device_errors(0)
    assert torch.equal(out, want)
    tpe[1] = 11
    g.replay()
    with pytest.raises(RuntimeError):
        check_device_errors(0)
    tpe[1] = 12
    g.replay()
    check_device_errors(0)
    assert torch.equal(out, want)


def test_nan_token_stays_alone_in_the_layer():
    from grouped_gemm_opt import fused_moe_int8, quantize_moe_weights_int8
    x, logits, wgu, wd = layer_inputs(90, 64, 128, 4, torch.bfloat16)
    qw = quantize_moe_weights_int8(wgu.to(DEV), wd.to(DEV))
    xd, ld = x.to(DEV), logits.to(DEV)
    want = fused_moe_int8(xd, ld, qw, 2)
    xd[17, 3] = float("nan")
    xd[40, 9] = float("inf")
    out = fused_moe_int8(xd, ld, qw, 2)
    hit = torch.zeros(90, dtype=torch.bool, device=DEV)
    hit[[17, 40]] = True
    assert out[hit].isnan().all() and torch.equal(out[~hit], want[~hit])


def test_layer_with_logits_of_other_types():
    """The layer routes on whatever float type the logits have, as the others do."""
    from grouped_gemm_opt import fused_moe_int8, quantize_moe_weights_int8
    x, logits, wgu, wd = layer_inputs(70, 64, 128, 4, torch.bfloat16)
    qw = quantize_moe_weights_int8(wgu.to(DEV), wd.to(DEV))
    half = logits.to(torch.float16)
    want = fused_moe_int8(x.to(DEV), half.float().to(DEV), qw, 2)
    for l in (half, half.double(), half.float().t().contiguous().t()):
        assert torch.equal(fused_moe_int8(x.to(DEV), l.to(DEV), qw, 2), want)
    strided = x.to(DEV).t().contiguous().t()
    assert torch.equal(fused_moe_int8(strided, half.to(DEV), qw, 2), want)


def test_products_on_two_streams_at_once():
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt_int8
    counts = [500, 0, 900, 33]
    dev = [t.to(DEV) for t in operands(counts, 2048, 1024)] + [torch.tensor(counts, device=DEV)]
    want = grouped_gemm_opt_int8(*dev)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(grouped_gemm_opt_int8(*dev))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    check_device_errors(0)


@pytest.mark.parametrize("experts,rows", [(256, 40), (257, 64), (300, 63), (1024, 50), (1000, 2500)])
def test_many_experts(experts, rows):
    """Both ways of ordering the segments, in thin and ordinary launches; most experts have no rows."""
    from grouped_gemm_opt import check_device_errors, grouped_gemm_opt, grouped_gemm_opt_int8
    g = torch.Generator().manual_seed(experts)
    which = torch.randint(0, experts, (rows,), generator=g)
    which[: rows // 4] = experts - 1
    counts = torch.bincount(which, minlength=experts).tolist()
    x, xs, w, ws = operands(counts, 48, 64, seed=1)
    ref = reference(counts, x, xs, w, ws)
    dev = [t.to(DEV) for t in (x, xs, w, ws, torch.tensor(counts))]
    for sort in (True, False):
        out = grouped_gemm_opt_int8(*dev, sort_by_m=sort)
        assert_product(out, ref, torch.bfloat16)
    # the bf16 product of the same codes (whole numbers up to 127 are exact in bf16)
    plain = grouped_gemm_opt(dev[0].to(torch.bfloat16), dev[2].to(torch.bfloat16), dev[4])
    one = [torch.ones_like(dev[1]), torch.ones_like(dev[3])]
    assert torch.equal(plain, grouped_gemm_opt_int8(dev[0], one[0], dev[2], one[1], dev[4]))
    check_device_errors(0)
