"""moe_router against the definition in 64 bits: routing, counts, balance loss, and both gradients.

Tolerances. ids and counts are whole numbers and must be equal. A weight or a probability p is
exp(d) / sum: d = l - max is one rounding (2^-24 |d|), expf is within 2 ulp (2^-22), a sum of n <= 1024
positive terms by a tree of per-lane chains of at most 32 + 5 additions loses (37 + 1) 2^-24, the
reciprocal and product 2^-23: relative error below (|d| + 4 + 38 + 4) 2^-24, P_TOL for |d| <= 40."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
P_TOL = 86 * 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(logits, k, mask=None):
    """ids, weights, counts, kept counts, loss as 64-bit functions of `logits` (a CPU leaf)."""
    l = logits.double()
    T, E = l.shape
    ids = torch.sort(l.detach(), dim=1, descending=True, stable=True)[1][:, :k]
    live = (l.detach() > -float("inf")).any(1) | l.detach().isnan().any(1)
    safe = torch.where(live[:, None], l, torch.zeros_like(l))
    w = torch.softmax(safe.gather(1, ids), 1) * live[:, None]
    keep = live if mask is None else live & mask
    p = torch.softmax(safe, 1)[keep]
    chosen = torch.zeros(T, E, dtype=torch.float64).scatter_(1, ids, 1.0)
    n = int(keep.sum())
    kept = chosen[keep].sum(0)
    loss = E * (kept / max(1, n * k) * p.sum(0) / max(1, n)).sum()
    return ids, w, chosen.sum(0).long(), kept.long(), loss


def make(T, E, k, dtype, masked, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed + T * 31 + E)
    logits = (torch.randn(T, E, generator=g) * scale).to(dtype)
    mask = torch.rand(T, generator=g) < 0.7 if masked else None
    gw = torch.randn(T, k, generator=g)
    return logits, mask, gw


SHAPES = [(1, 1, 1), (1, 8, 2), (33, 7, 3), (31, 64, 1), (64, 256, 8), (257, 60, 4), (5, 33, 5),
          (100, 1024, 16), (1000, 512, 2), (4099, 8, 2), (2500, 160, 6)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_router_forward_and_gradient(T, E, k, dtype, masked):
    from grouped_gemm_opt import moe_router
    logits, mask, gw = make(T, E, k, dtype, masked)
    ref_leaf = logits.clone().double().requires_grad_(True)
    ids, w, counts, kept, loss = reference(ref_leaf, k, mask)
    gl = 0.25
    ref_grad, = torch.autograd.grad((w * gw.double()).sum() + gl * loss, ref_leaf)
    leaf = logits.to(DEV).requires_grad_(True)
    r = moe_router(leaf, k, None if mask is None else mask.to(DEV))
    assert r.topk_ids.dtype == torch.int32 and r.topk_weights.dtype == torch.float32
    assert torch.equal(r.topk_ids.cpu().long(), ids)
    assert torch.equal(r.tokens_per_expert.cpu(), counts)
    assert torch.equal(r.balance_counts.cpu(), kept)
    assert torch.all((r.topk_weights.cpu().double() - w).abs() <= P_TOL * w)
    # a sum of positive terms each within P_TOL, added in blocks of four and eight, then in 64 bits
    assert abs(r.balance_loss.item() - loss.item()) <= (P_TOL + 16 * 2.0 ** -24) * loss.item()
    got, = torch.autograd.grad((r.topk_weights, r.balance_loss), leaf,
                               (gw.to(DEV), torch.tensor(gl, device=DEV)))
    assert got.dtype == dtype and got.shape == logits.shape
    # balance part: c p_e (f_e - sum p f), both terms of the bracket at most max f; weights part:
    # w (u - sum w u). A factor p or w is within P_TOL; the dot of up to 1024 terms and the products
    # add fewer than 50 roundings: below 3 (P_TOL + 12 * 2^-24) in all, before the last rounding.
    tol = P_TOL + 12 * 2.0 ** -24
    l = logits.double()
    p = torch.softmax(l, 1)
    n = max(1, int(kept.sum()) // k)
    f = kept.double() / (n * k)
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask
    size = gl * E / n * p * (f + (p * f).sum(1, keepdim=True)) * keep[:, None]
    u = gw.double().abs()
    size = size.scatter_add(1, ids, w.detach() * (u + (w.detach() * u).sum(1, keepdim=True)))
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134  # half of the smallest number
    bound = 4 * tol * size + HALF_STEP[dtype] * ref_grad.abs() + least
    assert torch.all((got.cpu().double() - ref_grad).abs() <= bound)


def test_gradient_against_differences():
    """Directional differences of the kernel's own loss and weights. Logits are spaced so that the
    step changes no choice (f stays constant). The difference quotient along a unit direction is off by
    h^2 / 6 of the third derivative (below 6 for a softmax value) and by the error of the two values
    over h: 20 roundings each (|d| <= 3.5 and 8 experts in the count at the top of this file)."""
    from grouped_gemm_opt import moe_router
    T, E, k, h = 6, 8, 2, 2.0 ** -7
    g = torch.Generator().manual_seed(3)
    base = torch.stack([torch.randperm(E, generator=g).float() for _ in range(T)]) * 0.5
    gw = torch.randn(T, k, generator=g).to(DEV)

    def value(l):
        r = moe_router(l, k)
        return 3.0 * r.balance_loss.double() + (r.topk_weights.double() * gw.double()).sum()

    leaf = base.to(DEV).requires_grad_(True)
    grad, = torch.autograd.grad(value(leaf), leaf)
    for _ in range(8):
        d = torch.randn(T, E, generator=g)
        d = (d / d.norm()).to(DEV)
        with torch.no_grad():
            diff = (value(leaf + h * d) - value(leaf - h * d)) / (2 * h)
        size = 3 * E + gw.abs().sum().item()
        bound = h * h / 6 * 6 * size + 20 * 2.0 ** -24 * size / h
        assert abs(diff.item() - (grad.double() * d.double()).sum().item()) <= bound
    # and the bound says something: it is well below the gradient itself
    assert bound < 0.2 * grad.norm().item()


def test_ties_and_signed_zeros():
    from grouped_gemm_opt import moe_router
    l = torch.zeros(3, 40)
    l[0, ::2] = -0.0
    l[1, 35] = 1.0
    l[2, 39] = -1.0
    r = moe_router(l.to(DEV), 4)
    assert r.topk_ids.cpu().tolist() == [[0, 1, 2, 3], [35, 0, 1, 2], [0, 1, 2, 3]]


def test_excluded_experts_and_empty_rows():
    """-inf logits are experts a token may not use; a row of nothing else has no distribution."""
    from grouped_gemm_opt import moe_router
    g = torch.Generator().manual_seed(1)
    l = torch.randn(70, 12, generator=g)
    l[:, 3] = -float("inf")
    l[5] = -float("inf")
    l[6, 1:] = -float("inf")  # one expert left, two asked for
    l[7] = torch.finfo(torch.float32).min
    ref_leaf = l.clone().double().requires_grad_(True)
    ids, w, counts, kept, loss = reference(ref_leaf, 2)
    leaf = l.to(DEV).requires_grad_(True)
    r = moe_router(leaf, 2)
    assert torch.equal(r.topk_ids.cpu().long(), ids)
    assert torch.equal(r.tokens_per_expert.cpu(), counts) and int(counts.sum()) == 140
    assert torch.equal(r.balance_counts.cpu(), kept) and int(kept.sum()) == 138
    assert r.topk_weights[5].tolist() == [0.0, 0.0] and r.topk_weights[6].tolist() == [1.0, 0.0]
    assert torch.all((r.topk_weights.cpu().double() - w).abs() <= P_TOL * w)
    assert abs(r.balance_loss.item() - loss.item()) <= 2 * P_TOL * loss.item()
    got, = torch.autograd.grad(r.balance_loss + r.topk_weights[:, 0].sum(), leaf)
    want, = torch.autograd.grad(loss + w[:, 0].sum(), ref_leaf)
    assert torch.isfinite(got).all() and torch.all(got[5] == 0) and torch.all(got[:7, 3] == 0)
    assert torch.all((got.cpu().double() - want).abs() <= 4 * P_TOL)


def test_nothing_kept_and_no_tokens():
    from grouped_gemm_opt import moe_router
    leaf = torch.randn(40, 16, device=DEV, requires_grad=True)
    r = moe_router(leaf, 3, torch.zeros(40, dtype=torch.bool, device=DEV))
    assert r.balance_loss.item() == 0.0 and int(r.balance_counts.sum()) == 0
    assert int(r.tokens_per_expert.sum()) == 120
    got, = torch.autograd.grad(r.balance_loss, leaf)
    assert torch.all(got == 0)
    leaf = torch.empty(0, 16, device=DEV, requires_grad=True)
    r = moe_router(leaf, 3)
    assert r.topk_ids.shape == (0, 3) and r.balance_loss.item() == 0.0
    assert r.tokens_per_expert.tolist() == [0] * 16
    got, = torch.autograd.grad(r.balance_loss, leaf)
    assert got.shape == (0, 16)


def test_nan_reaches_the_loss():
    from grouped_gemm_opt import moe_router
    l = torch.randn(10, 6, device=DEV)
    l[4, 2] = float("nan")
    l[4, 3] = -float("nan")
    r = moe_router(l, 2)
    assert r.balance_loss.isnan().item() and r.topk_weights[4].isnan().all()
    assert r.topk_ids[4].tolist() == [2, 3]
    assert r.topk_weights[:4].isfinite().all() and r.topk_weights[5:].isfinite().all()
    masked = torch.ones(10, dtype=torch.bool, device=DEV)
    masked[4] = False
    assert moe_router(l, 2, masked).balance_loss.isfinite().item()


def test_only_one_gradient_and_strided_arguments():
    from grouped_gemm_opt import moe_router
    wide = torch.randn(64, 40, device=DEV)
    leaf = wide.t()[:24].detach().requires_grad_(True)  # [24, 64], columns far apart
    plain = leaf.detach().contiguous().requires_grad_(True)
    mask = (torch.arange(48, device=DEV) % 3 > 0)[::2]
    a, b = moe_router(leaf, 4, mask), moe_router(plain, 4, mask.contiguous())
    assert torch.equal(a.topk_ids, b.topk_ids) and torch.equal(a.balance_loss, b.balance_loss)
    gw = torch.randn(4, 24, device=DEV).t()
    ga, = torch.autograd.grad(a.topk_weights, leaf, gw, retain_graph=True)
    gb, = torch.autograd.grad(b.topk_weights, plain, gw.contiguous(), retain_graph=True)
    assert torch.equal(ga, gb)
    # the gradient of a sum is a broadcast one (stride 0)
    ga, = torch.autograd.grad(a.topk_weights.sum(), leaf, retain_graph=True)
    assert ga.abs().max().item() <= 64 * 2.0 ** -24  # the weights sum to one
    la, = torch.autograd.grad(a.balance_loss, leaf)
    lb, = torch.autograd.grad(b.balance_loss, plain)
    assert torch.equal(la, lb) and torch.all(la[~mask] == 0)


def test_equal_bits_and_layer_routing():
    """Two calls agree to the bit, and the routing is the layers' own: ids, weights, counts and the
    dispatch's offset table."""
    from grouped_gemm_opt import _C, fused_moe, moe_router
    g = torch.Generator(device=DEV).manual_seed(5)
    for T, E, k in [(1, 4, 2), (333, 16, 2), (4096, 256, 8)]:
        l = torch.randn(T, E, device=DEV, generator=g)
        a, b = moe_router(l, k), moe_router(l, k)
        assert torch.equal(a.balance_loss, b.balance_loss)
        ids, w, tpe, scratch = _C.moe_route(l, k)
        assert torch.equal(a.topk_ids, ids) and torch.equal(a.topk_weights, w)
        assert torch.equal(a.tokens_per_expert, tpe)
        assert torch.equal(a.scratch[:scratch.numel()], scratch)
    T, H, F, E, k = 200, 128, 256, 16, 2
    x = torch.randn(T, H, device=DEV, generator=g).to(torch.bfloat16)
    l = torch.randn(T, E, device=DEV, generator=g)
    wgu = (torch.randn(E, 2 * F, H, device=DEV, generator=g) * 0.05).to(torch.bfloat16)
    wd = (torch.randn(E, H, F, device=DEV, generator=g) * 0.05).to(torch.bfloat16)
    assert torch.equal(fused_moe(x, l, wgu, wd, k),
                       fused_moe(x, l, wgu, wd, k, routing=moe_router(l, k)))


def test_training_step_through_the_grouped_gemm():
    """Router, gathered rows, grouped_gemm_opt and the weighted sum as one differentiable step, with
    the balance loss added: gradients against the same step in 64 bits."""
    from grouped_gemm_opt import grouped_gemm_opt, moe_router
    T, H, N, E, k = 96, 64, 32, 6, 2
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    wr = torch.randn(E, H, generator=g) * 0.2
    we = (torch.randn(E, N, H, generator=g) * 0.1).to(torch.bfloat16)
    target = torch.randn(T, N, generator=g)

    def combine(y, order, weights):
        back = torch.zeros(T * k, N, dtype=y.dtype, device=y.device).index_copy(0, order, y)
        return (back.reshape(T, k, N) * weights[:, :, None]).sum(1)

    rd, xd, wd = wr.to(DEV).requires_grad_(True), x.to(DEV), we.to(DEV).requires_grad_(True)
    r = moe_router(xd.float() @ rd.t(), k)
    order = torch.sort(r.topk_ids.reshape(-1), stable=True)[1]
    y = grouped_gemm_opt(xd[order // k], wd, r.tokens_per_expert)
    out = combine(y.float(), order, r.topk_weights)
    loss = ((out - target.to(DEV)) ** 2).mean() + 0.1 * r.balance_loss
    got = torch.autograd.grad(loss, (rd, wd))

    r64, w64 = wr.double().requires_grad_(True), we.double().requires_grad_(True)
    ids, w, _, _, bal = reference(x.double() @ r64.t(), k)
    assert torch.equal(ids, r.topk_ids.cpu().long())
    order = torch.sort(ids.reshape(-1), stable=True)[1]
    rows, expert = x.double()[order // k], ids.reshape(-1)[order]
    y = torch.einsum("rh,rnh->rn", rows, w64[expert])
    out = combine(y, order, w)
    want = torch.autograd.grad(((out - target.double()) ** 2).mean() + 0.1 * bal, (r64, w64))
    # Roundings to bf16: y (2^-8), which also moves d out = 2 (out - target) / (T N), then dy and
    # dW. Their effect, term by term in absolute values, with a tenth for all that is in fp32.
    with torch.no_grad():
        by_slot = torch.zeros(T * k, N, dtype=torch.float64).index_copy(0, order, y.abs())
        by_slot = by_slot.reshape(T, k, N)
        dout = (2 * (out - target.double()) / (T * N)).abs()
        moved = 2 / (T * N) * (by_slot * w[:, :, None]).sum(1)      # |change of dout| / 2^-8
        u = ((dout + moved)[:, None, :] * by_slot).sum(2)           # |change of dL/dw| / 2^-8
        dlogit = torch.zeros(T, E, dtype=torch.float64).scatter_(
            1, ids, w * (u + (w * u).sum(1, keepdim=True)))
        bound_r = 1.1 * 2.0 ** -8 * dlogit.t() @ x.double().abs()
        dy = ((dout + moved)[:, None, :] * w[:, :, None]).reshape(T * k, N)[order]
        per_row = torch.einsum("rn,rh->rnh", dy, rows.abs())
        bound_w = torch.zeros_like(w64).index_add_(0, expert, per_row)
        bound_w = 1.1 * 2.0 ** -8 * (bound_w + want[1].abs())
    assert torch.all((got[0].cpu().double() - want[0]).abs() <= bound_r)
    assert torch.all((got[1].cpu().double() - want[1]).abs() <= bound_w)


def test_captured_step_replays():
    """Forward and backward in one graph; the replay follows the logits' new contents. An eager graph
    of another leaf is alive meanwhile."""
    from grouped_gemm_opt import moe_router
    T, E, k = 130, 40, 4
    leaf = torch.randn(T, E, device=DEV, requires_grad=True)
    gw = torch.randn(T, k, device=DEV)
    one = torch.ones((), device=DEV)

    def step(l):
        r = moe_router(l, k)
        return r, torch.autograd.grad((r.topk_weights, r.balance_loss), l, (gw, one))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        static = leaf.detach().clone().requires_grad_(True)
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    alive = moe_router(leaf, k)  # an eager graph that outlives the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, grad = step(static)
    for i in range(3):
        fresh = torch.randn(T, E, device=DEV)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        want, want_grad = step(fresh.requires_grad_(True))
        assert torch.equal(r.topk_ids, want.topk_ids) and torch.equal(grad, want_grad)
        assert torch.equal(r.balance_loss, want.balance_loss)
    alive.balance_loss.backward()
    assert leaf.grad.isfinite().all()


def test_other_stream():
    from grouped_gemm_opt import moe_router
    l = torch.randn(5000, 64, device=DEV)
    want = moe_router(l, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = moe_router(l, 6)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got.balance_loss, want.balance_loss)
    assert torch.equal(got.topk_ids, want.topk_ids)


def test_second_derivatives_are_refused():
    from grouped_gemm_opt import moe_router
    leaf = torch.randn(20, 8, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(moe_router(leaf, 2).balance_loss, leaf, create_graph=True)
    assert g.isfinite().all()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(g.sum(), leaf)


@pytest.mark.parametrize("E", [8, 40, 256, 1000])
def test_nearly_equal_logits_are_ordered_exactly(E):
    """fp32 logits that agree in their leading bits, among them equal ones: the order is that of all
    their bits, ties to the lower index."""
    from grouped_gemm_opt import moe_router
    g = torch.Generator().manual_seed(E)
    steps = torch.randint(0, 12, (300, E), generator=g).float()
    for base in (1.0, -1.0, 100.0):
        l = base * (1 + steps * 2.0 ** -22)
        l[:50] = l[:50] + torch.randn(50, E, generator=g)
        k = min(8, E)
        want = torch.sort(l, dim=1, descending=True, stable=True)[1][:, :k]
        assert torch.equal(moe_router(l.to(DEV), k).topk_ids.cpu().long(), want)


def test_capture_over_a_live_eager_graph_is_refused():
    from grouped_gemm_opt import moe_router
    leaf = torch.randn(40, 16, device=DEV, requires_grad=True)
    alive = moe_router(leaf, 2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="still alive"):
            moe_router(leaf, 2)
        with torch.no_grad():
            moe_router(leaf, 2)  # without a gradient there is nothing to refuse
    alive.balance_loss.backward()
    assert leaf.grad.isfinite().all()
    del alive
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        moe_router(leaf, 2)


@pytest.mark.parametrize("T", [1, 31, 32, 33, 255, 256, 257])
@pytest.mark.parametrize("E", [2, 32, 33, 255, 256, 257])
def test_both_sides_of_the_one_launch_form(T, E):
    """Up to 256 tokens and 256 experts the forward is one launch, beyond it two: the same routing,
    offset table, counts and loss."""
    from grouped_gemm_opt import _C, moe_router
    g = torch.Generator().manual_seed(T * E)
    l = torch.randn(T, E, generator=g)
    mask = torch.rand(T, generator=g) < 0.8
    k = min(E, 5)
    ids, w, counts, kept, loss = reference(l, k, mask)
    for rows, m in ((l, mask), (torch.cat([l, torch.full((257, E), -float("inf"))]), None)):
        r = moe_router(rows.to(DEV), k, None if m is None else m.to(DEV))
        assert torch.equal(r.topk_ids[:T].cpu().long(), ids)
        assert torch.all((r.topk_weights[:T].cpu().double() - w).abs() <= P_TOL * w)
        if m is not None:
            assert torch.equal(r.balance_counts.cpu(), kept)
            assert torch.equal(r.tokens_per_expert.cpu(), counts)
            assert abs(r.balance_loss.item() - loss.item()) <= (P_TOL + 2.0 ** -20) * loss.item()
            scratch = _C.moe_route(rows.to(DEV), k)[3]
            assert torch.equal(r.scratch[:scratch.numel()], scratch)
        else:  # rows without a distribution add nothing to the loss
            want = reference(l, k)
            assert torch.equal(r.balance_counts.cpu(), want[3])
            assert abs(r.balance_loss.item() - want[4].item()) <= (P_TOL + 2.0 ** -20) * want[4].item()


@pytest.mark.parametrize("T,E,k", [(64, 8, 1), (300, 12, 3), (4096, 64, 4), (1024, 512, 2)])
def test_balanced_router_has_no_balance_gradient(T, E, k):
    """Every expert chosen equally often: the gradient is zero, not the rounding of a difference; one
    choice moved away leaves it as exact as the small imbalance is."""
    from grouped_gemm_opt import moe_router
    g = torch.Generator().manual_seed(E)
    T = T // E * E
    base = torch.rand(T, E, generator=g)
    chosen = (torch.arange(T)[:, None] + torch.arange(k)[None]) % E
    base.scatter_add_(1, chosen, 2.0 + torch.rand(T, k, generator=g))
    leaf = base.to(DEV).requires_grad_(True)
    r = moe_router(leaf, k)
    assert torch.equal(r.balance_counts.cpu(), torch.full((E,), T * k // E))
    grad, = torch.autograd.grad(r.balance_loss, leaf)
    assert torch.count_nonzero(grad) == 0
    base[0, chosen[0, 0]] = -3.0  # token 0 takes another expert instead
    ref_leaf = base.clone().double().requires_grad_(True)
    _, _, _, kept, loss = reference(ref_leaf, k)
    want, = torch.autograd.grad(loss, ref_leaf)
    leaf = base.to(DEV).requires_grad_(True)
    grad, = torch.autograd.grad(moe_router(leaf, k).balance_loss, leaf)
    p = torch.softmax(base.double(), 1)
    off = (kept.double() / (T * k) - 1.0 / E).abs()
    size = E / T * p * (off + (p * off).sum(1, keepdim=True))
    assert torch.all((grad.cpu().double() - want).abs() <= 4 * (P_TOL + 12 * 2.0 ** -24) * size +
                     2.0 ** -140)
