"""Timing cases of the router with its balance loss and of the INT8 expert products.

Four operators, each with a plain form in elementary torch operations and the call a user makes:

  router    moe_router: top-k routing, per-expert counts and the balance loss, with the gradient
  quantize  quantize_int8: one scale per row, signed 8-bit codes
  product   grouped_gemm_opt_int8: grouped matrix product with row and channel scales
  layer     moe_router followed by fused_moe_int8: the MoE layer over INT8 expert weights

`own` picks the form that `run` uses. Whole numbers are defined exactly: ties of the top-k go to the
lowest expert index, and an INT8 code is the quotient 127 x / max|row| rounded half to even, a
quotient of numbers that 32 bits hold exactly.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BALANCE_WEIGHT = 0.01  # what a training loss multiplies the balance loss by


def listed():
    return [
        # one training step's router over 8 experts: the whole of a 16384-token batch
        dict(name="router-train-8", op="router", tokens=16384, experts=8, top_k=2, dtype="fp32",
             masked=False, train=True),
        # fine-grained experts in bf16 with padding tokens: the largest router step
        dict(name="router-train-256", op="router", tokens=32768, experts=256, top_k=8,
             dtype="bf16", masked=True, train=True),
        # a decode step's router: latency only
        dict(name="router-serve-256", op="router", tokens=256, experts=256, top_k=8, dtype="fp32",
             masked=False, train=False),
        # odd expert and token counts, half precision, padding
        dict(name="router-train-60", op="router", tokens=5003, experts=60, top_k=4, dtype="fp16",
             masked=True, train=True),
        # the activations between the two expert products of a 16384-token, top-2 layer
        dict(name="quantize-prefill", op="quantize", rows=32768, cols=14336, dtype="bf16"),
        # a handful of decode rows
        dict(name="quantize-decode", op="quantize", rows=7, cols=4096, dtype="fp16"),
        # the down projection of a 16384-token, top-2 layer
        dict(name="product-prefill", op="product", rows=32768, experts=8, n=4096, k=14336,
             spread="even", dtype="bf16"),
        # heavy-tailed counts over 64 experts, some of them empty
        dict(name="product-skewed", op="product", rows=8192, experts=64, n=14336, k=4096,
             spread="zipf", dtype="bf16"),
        # eight decoding sequences, two experts each: the weights' bytes are the cost
        dict(name="product-decode", op="product", rows=16, experts=8, n=14336, k=4096,
             spread="even", dtype="bf16"),
        # widths that fill no tile, half-precision result
        dict(name="product-odd", op="product", rows=1003, experts=5, n=1000, k=1104,
             spread="zipf", dtype="fp16"),
        # the whole layer over 8 experts
        dict(name="layer-prefill-8", op="layer", tokens=16384, experts=8, top_k=2, hidden=4096,
             ffn=14336, dtype="bf16"),
        # the whole layer over 256 experts at a decode batch
        dict(name="layer-decode-256", op="layer", tokens=256, experts=256, top_k=8, hidden=7168,
             ffn=2048, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["router", "router", "quantize", "product", "product", "layer"])
    if op == "router":
        experts = _log(rng, 2, 1024)
        return dict(op=op, tokens=_log(rng, 1, max(1, min(65536, (1 << 24) // experts))),
                    experts=experts, top_k=rng.randint(1, min(16, experts)),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), masked=rng.random() < 0.5,
                    train=rng.random() < 0.7)
    if op == "quantize":
        cols = 16 * _log(rng, 1, 1536)
        return dict(op=op, rows=_log(rng, 1, min(65536, (1 << 28) // cols)), cols=cols,
                    dtype=rng.choice(["bf16", "fp16"]))
    if op == "product":
        experts, n, k = _log(rng, 1, 128), 8 * _log(rng, 4, 2048), 16 * _log(rng, 4, 1024)
        while experts * n * k > 1 << 32:
            experts = max(1, experts // 2)
        return dict(op=op, rows=_log(rng, 1, max(1, min(32768, (1 << 40) // (n * k)))),
                    experts=experts, n=n, k=k, spread=rng.choice(["even", "zipf"]),
                    dtype=rng.choice(["bf16", "fp16"]))
    experts, hidden, ffn = _log(rng, 2, 128), 16 * _log(rng, 8, 448), 16 * _log(rng, 8, 896)
    while experts * hidden * ffn > 1 << 30:
        experts = max(2, experts // 2)
        ffn = max(128, ffn // 32 * 16)
    top_k = rng.randint(1, min(8, experts))
    most = max(1, min(8192, (1 << 40) // (top_k * hidden * ffn)))
    return dict(op=op, tokens=_log(rng, 1, most), experts=experts, top_k=top_k, hidden=hidden,
                ffn=ffn, dtype=rng.choice(["bf16", "fp16"]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _counts(case):
    """Rows of each expert: sizes of the case, the same for every seed."""
    experts, rng = case["experts"], random.Random(case["rows"] * 1009 + case["experts"])
    weight = [1.0 / (e + 1) ** 1.2 if case["spread"] == "zipf" else 1.0 for e in range(experts)]
    counts = [0] * experts
    for e in rng.choices(range(experts), weight, k=case["rows"]):
        counts[e] += 1
    return counts


def _codes(rows, cols, g):
    """INT8 codes and scales of normally distributed rows, as weights and activations have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    top = x.abs().amax(1, keepdim=True)
    return torch.round(x * 127 / top).to(torch.int8), top[:, 0] * (0.02 / 127)


def _weights(experts, n, k, g):
    q = torch.empty(experts, n, k, dtype=torch.int8, device="cuda")
    s = torch.empty(experts, n, device="cuda")
    for e in range(experts):
        q[e], s[e] = _codes(n, k, g)
    return q, s


def _logits(tokens, experts, dtype, g):
    """Router logits with a preference for some experts, as a router in training has."""
    lean = torch.randn(experts, generator=g, device="cuda") * 0.5
    return (torch.randn(tokens, experts, generator=g, device="cuda") + lean).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case=case)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "router":
        tokens, k = case["tokens"], case["top_k"]
        state["logits"] = _logits(tokens, case["experts"], dtype, g)
        state["mask"] = None
        if case["masked"]:  # about one token in eight is padding
            state["mask"] = torch.rand(tokens, generator=g, device="cuda") < 0.875
        if case["train"]:
            state["logits"].requires_grad_(True)
            state["weights_grad"] = torch.randn(tokens, k, generator=g, device="cuda") / tokens
            state["loss_grad"] = torch.full((), BALANCE_WEIGHT, device="cuda")
    elif case["op"] == "quantize":
        rows = torch.exp(torch.randn(case["rows"], 1, generator=g, device="cuda"))
        x = torch.empty(case["rows"], case["cols"], dtype=dtype, device="cuda")
        for at in range(0, case["rows"], 4096):
            part = torch.randn(x[at:at + 4096].shape, generator=g, device="cuda")
            x[at:at + 4096] = (part * rows[at:at + 4096]).to(dtype)
        state["x"] = x
    elif case["op"] == "product":
        state["x"], state["x_scale"] = _codes(case["rows"], case["k"], g)
        state["w"], state["w_scale"] = _weights(case["experts"], case["n"], case["k"], g)
        state["host_counts"] = _counts(case)
        state["counts"] = torch.tensor(state["host_counts"], device="cuda")
    else:
        e, h, f = case["experts"], case["hidden"], case["ffn"]
        state["x"] = torch.randn(case["tokens"], h, generator=g, device="cuda").to(dtype)
        state["logits"] = _logits(case["tokens"], e, torch.float32, g)
        state["gate_up"], state["gate_up_scale"] = _weights(e, 2 * f, h, g)
        state["down"], state["down_scale"] = _weights(e, h, f, g)
    return state


def _route(logits, top_k):
    """Top-k of the logits (ties to the lowest index) and the softmax over the chosen ones."""
    values, order = torch.sort(logits, dim=1, descending=True, stable=True)
    values, ids = values[:, :top_k], order[:, :top_k]
    weights = torch.exp(values - values[:, :1])
    return ids, weights / weights.sum(1, keepdim=True)


def _count(ids, keep, experts):
    ones = keep[:, None].expand_as(ids).to(torch.int64)
    zero = torch.zeros(experts, dtype=torch.int64, device=ids.device)
    return zero.scatter_add(0, ids.reshape(-1), ones.reshape(-1))


def _router(logits, mask, top_k):
    """ids, weights, counts of all tokens, counts of the unmasked ones, their number, the softmax
    over all experts (zero for masked tokens) and the loss E sum_e f_e p_e, f_e the share of the
    unmasked tokens' choices that fell on e and p_e the mean probability of e."""
    lg = logits.detach().float()
    tokens, experts = lg.shape
    ids, weights = _route(lg, top_k)
    every = torch.ones(tokens, dtype=torch.bool, device=lg.device)
    keep = every if mask is None else mask
    p = torch.exp(lg - lg.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True) * keep[:, None]
    kept_counts = _count(ids, keep, experts)
    kept = keep.sum().clamp(min=1).float()
    share = kept_counts.float() / (kept * top_k)
    loss = experts * (share * p.sum(0) / kept).sum()
    return ids, weights, _count(ids, every, experts), kept_counts, kept, p, share, loss


def _router_gradient(state, ids, weights, kept, p, share):
    """d loss / d logit_e = (E / T) p_e (f_e - sum p f); through the weights, w_j (g_j - sum w g)."""
    gw = state["weights_grad"]
    mean = (p * share).sum(1, keepdim=True)
    grad = state["loss_grad"] * (p.shape[1] / kept) * p * (share - mean)
    chosen = weights * (gw - (weights * gw).sum(1, keepdim=True))
    return grad.scatter_add(1, ids, chosen).to(state["logits"].dtype)


def _quantize(x):
    """Codes round(127 x / max|row|) (both products and their quotient's rounding as 32 bits hold
    them, half to even) and scales max|row| / 127; a zero row has scale 1."""
    xf = x.float()
    top = xf.abs().amax(-1, keepdim=True)
    some = top > 0
    q = torch.round(xf * 127 / torch.where(some, top, 1.0))
    return q.to(torch.int8), torch.where(some, top / 127, 1.0)[..., 0]


def _products(x, counts, w):
    """Rows of each expert times its weights, of codes in 32 bits: sums of whole numbers."""
    out = x.new_empty(x.shape[0], w.shape[1], dtype=torch.float32)
    at = 0
    for e, c in enumerate(counts):
        if c:
            torch.matmul(x[at:at + c].float(), w[e].float().t(), out=out[at:at + c])
            at += c
    return out


def _expert_of_row(counts):
    return torch.repeat_interleave(torch.arange(len(counts), device="cuda"),
                                   torch.tensor(counts, device="cuda"), output_size=sum(counts))


def _layer(state, ids, weights, counts, dtype):
    """Rows sorted by expert, then token; each stage hands on activations of the layer's type, as
    the layer is defined: h = silu(gate) up and the expert's output y are values of that type."""
    k = ids.shape[1]
    order = torch.sort(ids.reshape(-1), stable=True)[1]
    counts = counts.tolist()
    expert = _expert_of_row(counts)
    xq, xs = _quantize(state["x"])
    token = order // k
    gu = _products(xq[token], counts, state["gate_up"])
    gu = gu * xs[token][:, None] * state["gate_up_scale"][expert]
    gate, up = gu.chunk(2, dim=1)
    h = (gate / (1 + torch.exp(-gate)) * up).to(dtype)
    del gu, gate, up
    hq, hs = _quantize(h)
    y = _products(hq, counts, state["down"])
    y = (y * hs[:, None] * state["down_scale"][expert]).to(dtype)
    rows = torch.empty_like(y)
    rows[order] = y  # back to (token, choice) order
    rows = rows.float().reshape(*ids.shape, -1)
    return (rows * weights[:, :, None]).sum(1).to(dtype)


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "groupedgemm-opt_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import grouped_gemm_opt
    return grouped_gemm_opt


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return _run_plain(case, state)


def _run_own(case, state):
    ggo = _package()
    if case["op"] == "router":
        if not case["train"]:
            with torch.no_grad():
                r = ggo.moe_router(state["logits"], case["top_k"], token_mask=state["mask"])
        else:
            r = ggo.moe_router(state["logits"], case["top_k"], token_mask=state["mask"])
        out = dict(ids=r.topk_ids, weights=r.topk_weights, counts=r.tokens_per_expert,
                   balance_counts=r.balance_counts, loss=r.balance_loss)
        if case["train"]:
            out["grad"], = torch.autograd.grad((r.topk_weights, r.balance_loss),
                                               (state["logits"],),
                                               (state["weights_grad"], state["loss_grad"]))
        return out
    if case["op"] == "quantize":
        q, s = ggo.quantize_int8(state["x"])
        return dict(q=q, scale=s)
    if case["op"] == "product":
        return ggo.grouped_gemm_opt_int8(state["x"], state["x_scale"], state["w"],
                                         state["w_scale"], state["counts"],
                                         out_dtype=DTYPES[case["dtype"]])
    weights = ggo.MoEInt8Weights(state["gate_up"], state["gate_up_scale"], state["down"],
                                 state["down_scale"])
    r = ggo.moe_router(state["logits"], case["top_k"])
    y = ggo.fused_moe_int8(state["x"], state["logits"], weights, case["top_k"], routing=r)
    return dict(y=y, counts=r.tokens_per_expert, loss=r.balance_loss)


def _run_plain(case, state):
    if case["op"] == "router":
        ids, weights, counts, kept_counts, kept, p, share, loss = _router(
            state["logits"], state["mask"], case["top_k"])
        out = dict(ids=ids.to(torch.int32), weights=weights, counts=counts,
                   balance_counts=kept_counts, loss=loss)
        if case["train"]:
            out["grad"] = _router_gradient(state, ids, weights, kept, p, share)
        return out
    if case["op"] == "quantize":
        q, s = _quantize(state["x"])
        return dict(q=q, scale=s)
    if case["op"] == "product":
        acc = _products(state["x"], state["host_counts"], state["w"])
        expert = _expert_of_row(state["host_counts"])
        acc = acc * state["x_scale"][:, None] * state["w_scale"][expert]
        return acc.to(DTYPES[case["dtype"]])
    ids, weights, counts, _, _, _, _, loss = _router(state["logits"], None, case["top_k"])
    return dict(y=_layer(state, ids, weights, counts, DTYPES[case["dtype"]]), counts=counts,
                loss=loss)


def work(case):
    if case["op"] == "router":
        t, e, k, size = case["tokens"], case["experts"], case["top_k"], BYTES[case["dtype"]]
        passes = 2 if case["train"] else 1  # logits in, their gradient out
        return dict(bytes=t * e * size * passes + t * k * (8 + 4 * (passes - 1)) +
                    (t if case["masked"] else 0) + 16 * e,
                    flops=t * e * 8 * passes)
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return dict(bytes=3 * n + 4 * case["rows"], flops=3 * n)
    if case["op"] == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        live = sum(c > 0 for c in _counts(case))
        return dict(bytes=rows * (k + 4 + 2 * n) + live * n * (k + 4), flops=2 * rows * n * k)
    t, e, k, h, f = (case[x] for x in ("tokens", "experts", "top_k", "hidden", "ffn"))
    live = e * (1 - (1 - k / e) ** t)  # experts that some token chose, in expectation
    return dict(bytes=int(4 * t * h + 4 * t * e + live * (3 * f * h + 4 * (2 * f + h))),
                flops=6 * t * k * f * h)


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_router(state, top_k):
    logits = state["logits"].detach().double().requires_grad_(True)
    tokens, experts = logits.shape
    ids = torch.argsort(logits.detach(), dim=1, descending=True, stable=True)[:, :top_k]
    weights = torch.softmax(logits.gather(1, ids), dim=1)
    p = torch.softmax(logits, dim=1)
    chosen = torch.zeros(tokens, experts, dtype=torch.float64, device="cuda")
    chosen.scatter_(1, ids, 1.0)
    mask = state.get("mask")
    if mask is None:
        kept_p, kept_chosen, n = p, chosen, tokens
    else:
        kept_p, kept_chosen, n = p[mask], chosen[mask], max(1, int(mask.sum()))
    share = kept_chosen.sum(0) / (n * top_k)
    loss = experts * torch.dot(share, kept_p.sum(0) / n)
    return logits, ids, weights, chosen.sum(0).long(), kept_chosen.sum(0).long(), loss


def _exact_quantize(x):
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(127 * x / top), 0.0)
    return q, torch.where(top > 0, top / 127, 1.0).squeeze(1)


def _exact_layer(state, ids, weights, dtype):
    x, xs = _exact_quantize(state["x"])
    out = torch.zeros_like(x)
    for e in range(state["gate_up"].shape[0]):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if not len(token):
            continue
        gu = (x[token] @ state["gate_up"][e].double().t()) * xs[token, None]
        gate, up = (gu * state["gate_up_scale"][e].double()).chunk(2, dim=1)
        # the activations between the stages are of the layer's type
        h, hs = _exact_quantize((torch.nn.functional.silu(gate) * up).to(dtype))
        y = (h @ state["down"][e].double().t()) * hs[:, None] * state["down_scale"][e].double()
        out.index_add_(0, token, y.to(dtype).double() * weights[token, choice][:, None])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "router":
        logits, ids, weights, counts, kept_counts, loss = _exact_router(state, case["top_k"])
        out = dict(ids=ids.int(), weights=weights.detach(), counts=counts,
                   balance_counts=kept_counts, loss=loss.detach())
        if case["train"]:
            total = (weights * state["weights_grad"].double()).sum() + \
                loss * state["loss_grad"].double()
            out["grad"], = torch.autograd.grad(total, logits)
        return out
    if case["op"] == "quantize":
        parts = [_exact_quantize(p) for p in state["x"].split(4096)]
        return dict(q=torch.cat([q.to(torch.int8) for q, _ in parts]),
                    scale=torch.cat([s for _, s in parts]))
    if case["op"] == "product":
        out, at = [], 0
        for e, c in enumerate(state["host_counts"]):
            x = state["x"][at:at + c].double() * state["x_scale"][at:at + c, None].double()
            out.append(x @ (state["w"][e].double() * state["w_scale"][e, :, None].double()).t())
            at += c
        return torch.cat(out)
    _, ids, weights, counts, _, loss = _exact_router(state, case["top_k"])
    y = _exact_layer(state, ids, weights.detach(), DTYPES[case["dtype"]])
    return dict(y=y, counts=counts, loss=loss.detach())
