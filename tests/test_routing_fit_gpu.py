"""Ids and offset tables that do not belong together: the dispatches drop the choices that the table has
no place for, every other row arrives where it should, nothing outside the buffers is touched, and the
token of a dropped choice is NaN. The peer-memory layer with a given routing, its ranks one after the
other on one GPU with every wait's flag posted before the wait is launched."""
from dataclasses import replace
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def routing(T, E, k, seed=0):
    from grouped_gemm_opt import moe_router
    g = torch.Generator(device=DEV).manual_seed(seed + T)
    logits = torch.randn(T, E, device=DEV, generator=g)
    return logits, moe_router(logits, k)


def places(ids, scratch, E):
    """The dispatch's rule, entry by entry: sorted position of every choice, -1 for a dropped one."""
    T, k = ids.shape
    nb = (T + 31) // 32
    table = scratch.cpu()[:(nb + 1) * E].view(nb + 1, E).tolist()
    out = torch.full((T, k), -1, dtype=torch.int32)
    for b in range(nb):
        at = list(table[b])
        end = table[b + 1] if b + 1 < nb else table[nb][1:] + [T * k]
        for t in range(32 * b, min(T, 32 * b + 32)):
            for j in range(k):
                e = int(ids[t, j])
                if 0 <= e < E:
                    if at[e] < end[e]:
                        out[t, j] = at[e]
                    at[e] += 1
    return out


def edited(ids, E):
    """Choices dropped by a negative id, ids behind the last expert, choices moved to another expert and
    the same expert twice."""
    ids = ids.clone()
    for t, j, e in [(3, 0, -1), (17, 1, E), (18, 0, 2 ** 31 - 1), (2, 1, -2 ** 31)]:
        if t < ids.size(0):
            ids[t, j] = e
    if ids.size(0) > 30:
        ids[25:30, 0] = (ids[25:30, 0] + 1) % E
        ids[24, 1] = ids[24, 0]
    return ids


@pytest.mark.parametrize("T,H,E,k", [(5, 64, 8, 2), (100, 64, 8, 2), (1300, 128, 60, 4),
                                     (700, 64, 1024, 2)])
def test_choices_without_a_place_are_dropped(T, H, E, k):
    from grouped_gemm_opt import _C, quantize_int8
    _, r = routing(T, E, k)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    for ids in (r.topk_ids, edited(r.topk_ids, E)):
        want = places(ids.cpu(), r.scratch, E)
        kept = want.flatten() >= 0
        where = want.flatten()[kept].long().to(DEV)
        rows = torch.arange(T, device=DEV).repeat_interleave(k)[kept.to(DEV)]
        assert torch.unique(where).numel() == where.numel()
        xs, token, pos = _C.moe_permute(x, ids, r.scratch, E)
        assert torch.equal(pos.cpu(), want.flatten())
        assert torch.equal(xs[where], x[rows]) and torch.equal(token[where].long(), rows)
        q, s, pos = _C.moe_permute_int8(x, ids, r.scratch, E)
        wq, ws = quantize_int8(x)
        assert torch.equal(pos.cpu(), want.flatten())
        assert torch.equal(q[where], wq[rows]) and torch.equal(s[where], ws[rows])
        if ids is r.topk_ids:
            assert bool(kept.all())


def test_a_table_of_another_routing_stays_inside_the_rows():
    """Offsets from elsewhere, in range and far out of it."""
    from grouped_gemm_opt import _C
    T, H, E, k = 200, 64, 16, 2
    _, r = routing(T, E, k)
    _, other = routing(T, E, k, seed=99)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    far = torch.randint(-2 ** 31, 2 ** 31 - 1, r.scratch.shape, device=DEV, dtype=torch.int32)
    for scratch in (other.scratch, far, torch.full_like(far, 2 ** 31 - 1), torch.zeros_like(far)):
        for pos in (_C.moe_permute(x, r.topk_ids, scratch, E)[2],
                    _C.moe_permute_int8(x, r.topk_ids, scratch, E)[2]):
            assert int(pos.min()) >= -1 and int(pos.max()) < T * k
    with pytest.raises(RuntimeError, match="scratch"):
        _C.moe_permute(x, r.topk_ids, r.scratch[:8 * E - 1].clone(), E)
    with pytest.raises(RuntimeError, match="topk_ids"):
        _C.moe_permute(x, r.topk_ids[:-1].contiguous(), r.scratch, E)
    with pytest.raises(RuntimeError, match="slot_pos"):
        _C.moe_combine(x.repeat(2, 1), r.topk_weights[:-1].contiguous(),
                       torch.zeros(T * k, dtype=torch.int32, device=DEV))


def layer(T=100, H=64, F=128, E=8, k=2):
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, H, device=DEV, generator=g).to(torch.bfloat16)
    wgu = (torch.randn(E, 2 * F, H, device=DEV, generator=g) * 0.1).to(torch.bfloat16)
    wd = (torch.randn(E, H, F, device=DEV, generator=g) * 0.1).to(torch.bfloat16)
    logits, r = routing(T, E, k)
    return x, logits, wgu, wd, r


def test_edited_ids_make_their_tokens_nan_and_no_other():
    """The INT8 layer's sums are exact, so that a row's result does not depend on its place: the other
    tokens keep their bits."""
    from grouped_gemm_opt import fused_moe, fused_moe_int8, quantize_moe_weights_int8
    x, logits, wgu, wd, r = layer()
    ids = r.topk_ids.clone()
    ids[3, 0], ids[70, 1], ids[99, 0] = -1, 8, -77
    hit = torch.zeros(100, dtype=torch.bool, device=DEV)
    hit[[3, 70, 99]] = True
    out = fused_moe(x, logits, wgu, wd, 2, routing=replace(r, topk_ids=ids))
    assert out[hit].isnan().all() and out[~hit].isfinite().all()
    qw = quantize_moe_weights_int8(wgu, wd)
    want = fused_moe_int8(x, logits, qw, 2, routing=r)
    out = fused_moe_int8(x, logits, qw, 2, routing=replace(r, topk_ids=ids))
    assert out[hit].isnan().all() and torch.equal(out[~hit], want[~hit])


def test_peer_dispatch_stays_inside_the_buffers():
    """Counts that do not belong to the ids, as every rank publishes them: rows whose place lies behind
    the receive buffer are dropped, and the rows behind its end keep what they held. Where the counts
    keep the experts' places apart, each place holds the row that its origin names. Places that dropped
    choices left are named as their own."""
    from grouped_gemm_opt import _C
    T, H, E, k, cap = 100, 64, 8, 2, 230
    _, r = routing(T, E, k)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16)
    tpe = r.tokens_per_expert
    for counts, ids, apart in ((torch.stack([tpe, tpe]), edited(r.topk_ids, E), True),
                               (torch.stack([tpe * 3, tpe]), r.topk_ids, True),
                               (torch.stack([(tpe + 1) << 40, tpe]), r.topk_ids, True),
                               (torch.stack([tpe - 60, tpe]), r.topk_ids, False)):
        for rank in range(2):
            recv = [torch.full((cap + 400, H), 7.0, dtype=torch.bfloat16, device=DEV)
                    for _ in range(2)]
            org = [torch.full((cap + 400,), -5, dtype=torch.int32, device=DEV) for _ in range(2)]
            pos = _C.ep_dispatch(x, ids, r.scratch, counts.contiguous(), rank,
                                 [t.data_ptr() for t in recv], [t.data_ptr() for t in org], cap)
            named = torch.cat([o[o != -5] & 0x0fffffff for o in org])
            if ids is not r.topk_ids:  # all places lie in the buffer: every one is named once
                assert torch.equal(named.sort()[0], torch.arange(T * k, device=DEV,
                                                                 dtype=torch.int32))
            for a, o in zip(recv, org):
                assert torch.all(a[cap:] == 7.0) and torch.all(o[cap:] == -5)
                word = o[:cap][o[:cap] != -5]
                assert torch.all(word >> 28 == rank)
                token = torch.full((T * k,), -1, dtype=torch.int64, device=DEV)
                ok = pos >= 0
                token[pos[ok].long()] = torch.arange(T, device=DEV).repeat_interleave(k)[ok]
                token = token[(word & 0x0fffffff).long()]
                rows = a[:cap][o[:cap] != -5]
                assert torch.all(rows[token < 0] == 7.0)
                assert not apart or torch.equal(rows[token >= 0], x[token[token >= 0]])


class Ranks:
    """The ranks of the peer-memory layer in one process, one after the other: `run` calls the layer of
    every rank in turn with the flags of all posted before each call, so that no kernel waits. Rows
    and results are complete after the second turn."""

    def __init__(self, world, T, H, E, k):
        from grouped_gemm_opt import _C
        self.C, self.world, self.T, self.H, self.E, self.k = _C, world, T, H, E, k
        self.cap = world * T * k
        z = dict(device=DEV)
        self.mem = {
            "recv": [torch.zeros(self.cap, H, dtype=torch.bfloat16, **z) for _ in range(world)],
            "origin": [torch.zeros(self.cap, dtype=torch.int32, **z) for _ in range(world)],
            "back": [torch.zeros(T * k, H, dtype=torch.bfloat16, **z) for _ in range(world)],
            "board": [torch.zeros(int(_C.ep_board_bytes(E)) // 8, dtype=torch.int64, **z)
                      for _ in range(world)]}

    def run(self, xs, ls, wgu, wd, rs):
        from grouped_gemm_opt.moe import _fused_moe_p2p
        ptrs = {n: [t.data_ptr() for t in ts] for n, ts in self.mem.items()}
        el, outs = self.E // self.world, [None] * self.world
        for _ in range(2):
            for rank in range(self.world):
                for b in self.mem["board"]:
                    b[:self.world * self.E] = torch.stack([r.tokens_per_expert for r in rs]).flatten()
                    b[8 * self.E:] = 1 << 40
                bufs = SimpleNamespace(
                    _C=self.C, world=self.world, rank=rank, max_tokens=self.T, hidden=self.H,
                    top_k=self.k, num_experts=self.E, dtype=torch.bfloat16, epoch=0,
                    capacity=self.cap, ptrs=ptrs, _own={n: p[rank] for n, p in ptrs.items()},
                    wait_limit_cycles=1 << 24, recv=self.mem["recv"][rank],
                    origin=self.mem["origin"][rank], back=self.mem["back"][rank],
                    board_counts=self.mem["board"][rank][:8 * self.E].view(8, self.E))
                local = slice(rank * el, (rank + 1) * el)
                outs[rank] = _fused_moe_p2p(xs[rank], ls[rank], wgu[local], wd[local], self.k, bufs,
                                            True, routing=rs[rank])
        return outs


def rank_inputs(world, T, H, F, E, k):
    from grouped_gemm_opt import moe_router
    g = torch.Generator(device=DEV).manual_seed(0)
    wgu = (torch.randn(E, 2 * F, H, device=DEV, generator=g) * 0.1).to(torch.bfloat16)
    wd = (torch.randn(E, H, F, device=DEV, generator=g) * 0.1).to(torch.bfloat16)
    xs = [torch.randn(T, H, device=DEV, generator=g).to(torch.bfloat16) for _ in range(world)]
    ls = [torch.randn(T, E, device=DEV, generator=g) for _ in range(world)]
    return xs, ls, wgu, wd, [moe_router(l, k) for l in ls]


def other_rounding(x, wgu, wd, r, out):
    """How far two layers over the same products may be apart that add them up in other orders: an
    element of h, of y or of the result rounds the other way, a step of 2^-7 each."""
    bound = 2.0 ** -7 * out.double().abs()
    for j in range(r.topk_ids.size(1)):
        e = r.topk_ids[:, j].long()
        gate, up = torch.einsum("th,tfh->tf", x.double(), wgu[e].double()).chunk(2, 1)
        h = (torch.nn.functional.silu(gate) * up).abs()
        y = torch.einsum("tf,thf->th", h, wd[e].double().abs())  # at least |y|
        bound += r.topk_weights[:, j, None].double() * 2 * 2.0 ** -7 * y
    return bound


@pytest.mark.parametrize("T", [40, 700])
def test_peer_layer_with_a_given_routing(T):
    """Equal to the single-GPU layer, whose tiles are of other sizes, but for roundings."""
    from grouped_gemm_opt import check_device_errors, fused_moe
    H, F, E, k, world = 64, 128, 8, 2, 2
    xs, ls, wgu, wd, rs = rank_inputs(world, T, H, F, E, k)
    outs = Ranks(world, T, H, E, k).run(xs, ls, wgu, wd, rs)
    check_device_errors(0)
    for rank in range(world):
        want = fused_moe(xs[rank], ls[rank], wgu, wd, k, routing=rs[rank])
        bound = other_rounding(xs[rank], wgu, wd, rs[rank], want)
        assert torch.all((outs[rank].double() - want.double()).abs() <= bound)


@pytest.mark.parametrize("T", [40, 700])
def test_dropped_choices_in_the_peer_layer(T):
    """The places that dropped choices leave in a peer's buffer hold a row of an earlier layer, whose
    result must not be sent to where that row came from. The other tokens' rows may move up by a place,
    no more."""
    from grouped_gemm_opt import check_device_errors
    H, F, E, k, world = 64, 128, 8, 2, 2
    xs, ls, wgu, wd, rs = rank_inputs(world, T, H, F, E, k)
    ranks = Ranks(world, T, H, E, k)
    before = [o.clone() for o in ranks.run(xs, ls, wgu, wd, rs)]
    cut, hit = [], []
    for r in rs:
        ids = r.topk_ids.clone()
        drop = torch.zeros(T, dtype=torch.bool, device=DEV)
        drop[[1, T // 2, T - 1]] = True
        ids[1, 0], ids[T // 2, 1], ids[T - 1, 0] = -1, E, -9
        cut.append(replace(r, topk_ids=ids))
        hit.append(drop)
    for b in ranks.mem["back"]:
        b.fill_(float("nan"))  # results that nobody sends stay NaN
    outs = ranks.run(xs, ls, wgu, wd, cut)
    check_device_errors(0)
    for x, r, out, want, drop in zip(xs, rs, outs, before, hit):
        assert out[drop].isnan().all() and out[~drop].isfinite().all()
        near = (out.double() - want.double()).abs() <= other_rounding(x, wgu, wd, r, want)
        assert torch.all(near[~drop])
