"""Shaped attention at its edges on the kernels: prefixes and query positions at the ends of their types, constants that change before the backward
pass, what rounding takes from the output, dropout, shards of two runs and sharded caches."""
import math

import pytest
import torch
from shaped_plain import HALF, SLACK, attention, check, slopes_for, visible
from test_gpu_shaped import _inputs, _rand, _train

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ prefixes
@pytest.mark.parametrize("cbs", [1, 4])
@pytest.mark.parametrize("prefix", [-(2 ** 31), -(2 ** 31) + 130, -1, torch.tensor([torch.iinfo(torch.int64).min, 2 ** 62]),
                                    torch.tensor([-(2 ** 31), 2 ** 31 - 1], dtype=torch.int32)])
def test_prefixes_at_the_ends_of_their_type(cbs, prefix):
    """Far below zero nothing is open, far behind the end everything: over several key tiles, forward and backward."""
    B, S, H, D = 2, 400, 2, 64
    prefix = prefix.to(DEV) if isinstance(prefix, torch.Tensor) else prefix
    for cap in (0.0, 20.0):
        _train(*_inputs(B, S, S, H, D, seed=4), cap, None, prefix, cbs, what=f"cap {cap}")


# ------------------------------------------------------------------------------------------------ query positions
FAR = [2 ** 29, 2 ** 30 - 1, torch.tensor([2 ** 31 - 1, -(2 ** 31), 2 ** 30 + 77, 505], dtype=torch.int32),
       torch.tensor([2 ** 62, -(2 ** 62), 2 ** 33, -3])]


@pytest.mark.parametrize("Q,grad", [(1, False), (3, False), (8, False), (9, False), (40, False), (1, True), (40, True)])
@pytest.mark.parametrize("pos", FAR)
def test_queries_beyond_either_end_of_the_cache(Q, grad, pos):
    """All keys are on one side of such a query: its weights are those of a query at that end, however far it is. So the oracle's positions are moved to
    the end, which changes a row's scores by one number for all its keys, and its bound counts distances within the cache alone."""
    B, S, H, D, cap = 4, 500, 3, 64, 20.0
    pos = pos.to(DEV) if isinstance(pos, torch.Tensor) else pos
    q, k, v, dout = _inputs(B, Q, S, H, D)
    slopes = torch.tensor([0.5, 0.07, 2.0 ** -8], device=DEV)
    leaves = [t.requires_grad_(grad) for t in (q, k, v)]
    with torch.set_grad_enabled(grad):
        out = rab.ringattention_inference(*leaves, logit_cap=cap, alibi_slopes=slopes, query_pos=pos)
    rows = torch.as_tensor(pos, device=DEV).long().reshape(-1, 1) + torch.arange(Q, device=DEV)
    dist = rows.clamp(0, S - 1)[:, None, :, None] - torch.arange(S, device=DEV)
    want = attention(q, k, v, cap, slopes, dist, None, torch.ones(B, 1, Q, S, dtype=torch.bool, device=DEV), dout if grad else None)
    check(out, want[0], want[1], "out")
    if grad:
        for n, a, b, c in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout), want[2], want[3]):
            check(a, b, c, n)


# ------------------------------------------------------------------------------------------------ constants of a call
@pytest.mark.parametrize("which", ["alibi_slopes", "prefix_lens", "none", "prefix_lens in 64 bits"])
def test_constants_that_change_before_the_backward_pass(which):
    """The backward reads the slopes and prefixes again: a change in place in between is an error, as it is for any saved tensor. (A copy in another type
    is the call's own.)"""
    B, S, H, D = 2, 200, 3, 64
    q, k, v, dout = _inputs(B, S, S, H, D)
    prefix = torch.tensor([20, 90], device=DEV, dtype=torch.int64 if which.endswith("64 bits") else torch.int32)
    kw = dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, alibi_slopes=slopes_for(H, DEV), prefix_lens=prefix)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(rab.ringattention(*leaves, blockwise_kwargs=kw), leaves, dout)
    out = rab.ringattention(*leaves, blockwise_kwargs=kw)
    if which in kw:
        kw[which].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, leaves, dout)
        return
    if which.endswith("64 bits"):
        prefix.mul_(2)
    for a, b in zip(torch.autograd.grad(out, leaves, dout), want):
        assert (a.float() - b.float()).norm() <= 2.0 ** -7 * b.float().norm()  # (dq is reduced in no fixed order)


def test_query_positions_that_change_before_the_backward_pass():
    q, k, v, dout = _inputs(2, 20, 300, 2, 64)
    pos = torch.tensor([280, 100], device=DEV, dtype=torch.int32)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = rab.ringattention_inference(*leaves, alibi_slopes=slopes_for(2, DEV), query_pos=pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, dout)


def test_constants_made_in_inference_mode():
    with torch.inference_mode():
        slopes, prefix = slopes_for(2, DEV), torch.tensor([5], device=DEV, dtype=torch.int32)
    _train(*_inputs(1, 150, 150, 2, 64), 0.0, slopes, prefix)


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("Q", [1, 8, 20])
def test_forward_mode_derivatives_are_refused(which, Q):
    from torch.autograd import forward_ad

    x = list(_inputs(1, Q, 100, 2, 64)[:3])
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="forward mode"):
            rab.ringattention_inference(*x, alibi_slopes=slopes_for(2, DEV))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            rab.ringattention_inference(*x)


# ------------------------------------------------------------------------------------------------ what rounding takes from the output
def _launch(form, H, D, shape):
    """A launch of this form: its arguments, the last step's carry included."""
    from ringattention_b200.ops import flash
    from ringattention_b200.ops.flash import MaskSpec, Positions

    B, Sq, Sk = {"pairs": (2, 1300, 1300), "halves": (1, 500, 600), "split": (1, 140, 9000), "carry": (2, 300, 300)}[form]
    H = 40 if form == "pairs" else H
    q, k, v, dout = _inputs(B, Sq, Sk, H, D, seed=3)
    shape = dict(shape, slopes=slopes_for(H, DEV)) if shape.pop("sloped", False) else shape
    kw = {}
    if form == "carry":
        first = MaskSpec(1, Positions(Sk), Positions(0), **shape)
        kw["o_prev"], kw["lse_prev"] = flash.flash_fwd(q, _rand(B, Sk, H, D, seed=8), _rand(B, Sk, H, D, seed=9), first, out_fp32=True)
    return q, k, v, dout, MaskSpec(1, Positions(Sk if form == "carry" else Sk - Sq), Positions(Sk if form == "carry" else 0), **shape), kw


@pytest.mark.parametrize("form", ["pairs", "halves", "split", "carry"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [dict(logit_cap=25.0), dict(sloped=True), dict(logit_cap=25.0, sloped=True)])
def test_what_rounding_took_is_kept_and_used(form, D, shape):
    """The same launch in fp32 tells what the bf16 output left out; delta is the sum over both."""
    from ringattention_b200.ops import _lib, flash

    q, k, v, dout, ms, kw = _launch(form, 2, D, dict(shape))
    lo = torch.full_like(q, 7.0)
    out, lse = flash.flash_fwd(q, k, v, ms, out_lo=lo, **kw)
    full, lse_full = flash.flash_fwd(q, k, v, ms, out_fp32=True, **kw)
    _lib.check_status()
    assert torch.equal(lse, lse_full) and torch.equal(out, full.bfloat16())
    left = full.double() - out.double()
    # rounded to bf16: half a step of itself; one multiplication may or may not have been rounded ahead of the subtraction: half a step of fp32
    assert bool(((lo.double() - left).abs() <= left.abs() * HALF + full.double().abs() * 2.0 ** -24 + 1e-38).all())
    assert float(left.abs().max()) > 2.0 ** -10 * float(full.abs().max())  # (there is something to keep)
    _, delta = flash.flash_bwd_prep(out, dout, lse, out_lo=lo)
    terms = (dout.double() * (out.double() + lo.double())).transpose(1, 2)
    off = (delta[:, :, :q.shape[1]].double() - terms.sum(-1)).abs()
    # fp32: 2^-24 for out + lo and for each product, and as much for each of the additions that a term goes through (no more than D)
    assert bool((off <= (D + 2) * 2.0 ** -24 * terms.abs().sum(-1) + 1e-30).all())


def _dominant(S, D, cap):
    """One key has nearly all of every row's weight; the bounds for dq and dk count that its probability is 1 but for what the others have."""
    H = 2
    q, k, v, dout = _inputs(1, S, S, H, D, seed=6, std=0.5)
    with torch.no_grad():
        k[:, 5] = 4.0 * q[:, :1].float().sign().bfloat16()[:, 0]
        q.copy_(q.abs() * q[:, :1].sign())
    g, kk, vv = (t.double().transpose(1, 2) for t in (dout, k, v))
    want = attention(q, k, v, cap, seen=torch.ones(1, 1, S, S, dtype=torch.bool, device=DEV), dout=dout)
    x = q.double().transpose(1, 2) @ kk.transpose(2, 3) / math.sqrt(D)
    steep = 1 - torch.tanh(x / cap) ** 2
    x = cap * torch.tanh(x / cap)
    p = torch.softmax(x, -1)
    assert float(p[..., 5].min()) > 0.95
    rel = HALF + SLACK * (1 + x.abs().amax(3, keepdim=True))
    rest = p.clone()
    rest[..., 5] = 0
    rest = rest * rel  # errors of the other weights; the large one's is their sum, the weights of a row being normalised
    weight = rest @ vv.abs() + rest.sum(3, keepdim=True) * vv[:, :, 5:6].abs()
    out = want[0].transpose(1, 2)
    off = (g.abs() * (weight + 2.0 ** -16 * out.abs())).sum(3, keepdim=True) + SLACK * (g.abs() @ vv.abs().transpose(2, 3))
    ds = p * steep * (g @ vv.transpose(2, 3) - (g * out).sum(3, keepdim=True)) / math.sqrt(D)
    dds = ds.abs() * 2 * rel + p * steep * off / math.sqrt(D)
    bound = [(dds @ kk.abs()).transpose(1, 2) + HALF * want[2][0].abs() + 1e-6,
             (dds.transpose(2, 3) @ q.double().transpose(1, 2).abs()).transpose(1, 2) + HALF * want[2][1].abs() + 1e-6]
    return (q, k, v, dout), want[2][:2], bound


@pytest.mark.parametrize("S,D", [(100, 64), (700, 128)])
def test_gradients_of_rows_that_one_key_has(S, D):
    """dP - delta is then the small difference of numbers as large as dO O, and delta out of the rounded output would be most of it."""
    from ringattention_b200.ops import flash
    from ringattention_b200.ops.flash import MaskSpec, Positions

    cap = 40.0
    (q, k, v, dout), want, bound = _dominant(S, D, cap)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = rab.ringattention(*leaves, blockwise_kwargs=dict(query_chunk_size=S, key_chunk_size=S, logit_cap=cap))
    for n, a, w, b in zip(("dq", "dk"), torch.autograd.grad(out, leaves, dout), want, bound):
        check(a, w, b, n)
    got = torch.autograd.grad(rab.ringattention_inference(*leaves, logit_cap=cap), leaves, dout) if S > 8 else None
    for n, a, w, b in zip(("dq", "dk"), got, want, bound):
        check(a, w, b, "inference " + n)
    # without what rounding took the bound is not kept: the test sees it
    ms = MaskSpec(0, Positions(0), Positions(0), logit_cap=cap)
    out, lse = flash.flash_fwd(q, k, v, ms)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    flash.flash_bwd_run(q, k, v, out, lse, dout, ms, dq, dk, dv)
    assert float(((dq.double() - want[0]).abs() / bound[0]).max()) > 1


# ------------------------------------------------------------------------------------------------ dropout, rings, sharded caches
@pytest.mark.parametrize("cap,sloped,prefix", [(20.0, False, None), (0.0, True, None), (20.0, True, 90)])
def test_dropout(cap, sloped, prefix):
    from ringattention_b200.ops import reference as R

    B, S, H, D, p, seed = 2, 333, 3, 64, 0.3, 1234567
    q, k, v, dout = _inputs(B, S, S, H, D)
    slopes = slopes_for(H, DEV) if sloped else None
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = rab.ringattention(*leaves, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, deterministic=False, dropout_rng=seed,
                                                           attn_pdrop=p, logit_cap=cap or None, alibi_slopes=slopes, prefix_lens=prefix))
    at = torch.arange(S, device=DEV)
    seen = visible(at, at, B, 1, prefix) & ~R.dropped(seed, p, B, H, at, at)
    want = attention(q, k, v, cap, slopes, (at[:, None] - at)[None, None], None, seen, dout)
    check(out, want[0], want[1], "out")
    for n, a, w, b in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout), want[2], want[3]):
        check(a, w, b, n)


@pytest.mark.parametrize("layout", ["contiguous", "zigzag", "pairs:0-3,1-2,4-7,5-6"])
@pytest.mark.parametrize("cap,sloped,prefix", [(20.0, True, [0, 700]), (0.0, False, [130, 1100]), (20.0, False, None), (0.0, True, None)])
def test_every_rank_of_a_ring_by_its_plan(layout, cap, sloped, prefix):
    """The launches that a ring's ranks make, one rank after another on one device: plans over shards of one and of two runs, prefixes that reach into later
    ranks' blocks, documents, gradients of the blocks added up in fp32."""
    from ringattention_b200.config import BlockwiseKwargs
    from ringattention_b200.ops import _lib, attention as A, flash
    from ringattention_b200.ops import reference as R

    world, n, B, H, D = 4, 256, 2, 2, 64
    S = world * n
    x = _inputs(B, S, S, H, D, seed=11)
    slopes = slopes_for(H, DEV) if sloped else None
    pre = None if prefix is None else torch.tensor(prefix, device=DEV, dtype=torch.int32)
    seg = (torch.arange(S, device=DEV) // 600).int().expand(B, S).contiguous()
    kw = BlockwiseKwargs.from_any(dict(causal_block_size=1, query_chunk_size=n, key_chunk_size=n, logit_cap=cap or None, alibi_slopes=slopes, prefix_lens=pre,
                                       layout=layout))
    q, k, v, dout = ([t.contiguous() for t in R.to_layout(t, world, layout).split(n, 1)] for t in x)
    outs, dqs, acc = [], [], torch.zeros(world, B, n, 2, H, D, device=DEV)
    for rank in range(world):
        plan = A.make_plan(rank, world, B, n, n, H, kw, segment_ids=seg, device=torch.device(DEV))
        o = lse = None
        lo = torch.empty_like(q[rank])
        for i, st in enumerate(plan.active):
            last = i + 1 == len(plan.active)
            o, lse = flash.flash_fwd(q[rank], k[st.block], v[st.block], st.mask, o_prev=o, lse_prev=lse, out_fp32=not last, out_lo=lo if last else None)
        dq = torch.empty(B, n, H, D, device=DEV)
        lse2, delta = flash.flash_bwd_prep(o, dout[rank], lse, dq, out_lo=lo)
        for st in plan.active:
            t = acc[st.block]
            flash.flash_bwd(q[rank], k[st.block], v[st.block], dout[rank], lse2, delta, st.mask, dq, t[:, :, 0], t[:, :, 1], flash.DKV_REDUCE_FP32)
        outs.append(o)
        dqs.append(dq)
    _lib.check_status()
    at = torch.arange(S, device=DEV)
    want = attention(*x[:3], cap, slopes, (at[:, None] - at)[None, None], None, visible(at, at, B, 1, pre, seg, seg), x[3])
    whole = lambda parts: R.from_layout(torch.cat(list(parts), 1), world, layout)
    check(whole(outs), want[0], want[1], "out")
    for what, got, w, b in zip(("dq", "dk", "dv"), (whole(dqs), whole(acc[:, :, :, 0]), whole(acc[:, :, :, 1])), want[2], want[3]):
        check(got, w, b, what)


class _Axis:
    def __init__(self, rank, size):
        self.rank, self.size, self.group = rank, size, None


@pytest.mark.parametrize("Q", [1, 3, 8, 30])
@pytest.mark.parametrize("cap,sloped", [(20.0, True), (0.0, True), (20.0, False)])
def test_a_cache_in_shards(Q, cap, sloped, monkeypatch):
    """Every rank's call over its part of the cache, one after another; the parts are put together here as the ranks' exchange puts them together."""
    from ringattention_b200.ops import decode as Dk
    from ringattention_b200.ops import inference as Inf

    world, n, B, H, D = 3, 200, 2, 3, 64
    S = world * n
    q, k, v, dout = _inputs(B, Q, S, H, D, seed=Q)
    pos = torch.tensor([S - Q, 250], device=DEV, dtype=torch.int32)
    at = torch.arange(S, device=DEV)
    mask = (at <= pos[:, None, None] + torch.arange(Q, device=DEV)[:, None])[:, None]
    slopes = slopes_for(H, DEV) if sloped else None
    shape = lambda: Inf.inference_shape(q, k[:, :n], world, cap or None, slopes, pos)
    want = attention(q, k, v, cap, slopes, pos[:, None, None, None] + torch.arange(Q, device=DEV)[:, None] - at, None, mask, dout)
    parts = []
    shards = [(k[:, r * n:(r + 1) * n], v[:, r * n:(r + 1) * n]) for r in range(world)]
    if Q <= 8:
        monkeypatch.setattr(Dk, "merge_exchange", lambda o, lse, H, QL, out, ring: parts.append((o, lse, H, QL)))
        with torch.no_grad():
            for r, (kk, vv) in enumerate(shards):
                Inf.ring_inference_attention(q, kk, vv, mask, _Axis(r, world), object(), shape())
        out = torch.empty(B, parts[0][3], H, D, device=DEV, dtype=torch.bfloat16)
        Dk.merge_partials(torch.cat([p[0] for p in parts], 1), torch.cat([p[1] for p in parts], 1), H, parts[0][3], out=out)
        check(out[:, :Q], want[0], want[1], "out")
        return
    monkeypatch.setattr(Inf, "_exchange_and_merge", lambda o, lse, axis, ring: (parts.append((o, lse)), (o.bfloat16(), lse))[1])
    with torch.no_grad():
        for r, (kk, vv) in enumerate(shards):
            Inf.ring_inference_attention(q, kk, vv, mask, _Axis(r, world), object(), shape())
    lses = torch.stack([p[1] for p in parts])
    lse = torch.logsumexp(lses, 0)
    out = sum(p[0] * torch.exp(l - lse).transpose(1, 2)[..., None] for p, l in zip(parts, lses)).bfloat16()
    check(out, want[0], want[1], "out")
    monkeypatch.setattr(Inf, "_exchange_and_merge", lambda o, lse_, axis, ring: (out.clone(), lse))
    monkeypatch.setattr(torch.distributed, "all_reduce", lambda *a, **kw: None)
    grads = []
    for r, (kk, vv) in enumerate(shards):
        leaves = [t.detach().clone().requires_grad_() for t in (q, kk, vv)]
        got = Inf.ring_inference_attention(*leaves, mask, _Axis(r, world), object(), shape())
        grads.append(torch.autograd.grad(got, leaves, dout))
    # delta comes out of the rounded output here, and dq is the sum of as many roundings as there are ranks
    g, o = dout.double().abs(), want[0].abs()
    delta_off = (HALF * g * o).sum(-1).amax() / math.sqrt(D)
    for i, what in ((1, "dk"), (2, "dv")):
        extra = (delta_off * q.double().abs().amax() * Q) if i == 1 else 0.0
        check(torch.cat([x[i] for x in grads], 1), want[2][i], want[3][i] + extra, what)
    dq = sum(x[0].double() for x in grads)
    check(dq, want[2][0], want[3][0] + delta_off * k.double().abs().amax() + HALF * sum(x[0].double().abs() for x in grads), "dq")


def test_nan_in_hidden_and_in_seen_places():
    """A key of NaN reaches the rows and the head that see it; a value of NaN likewise; both stay away from rows ahead of their tile."""
    S, D = 400, 64
    for where in ("key", "value"):
        q, k, v, _ = _inputs(1, S, S, 2, D)
        (k if where == "key" else v)[0, 300, 0] = float("nan")
        with torch.no_grad():
            out = rab.ringattention(q, k, v, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=30.0))
        bad = out.isnan()[0]
        assert not bad[:, 1].any() and not bad[:256].any() and bool(bad[300:, 0].any(-1).all()), where
        if where == "key":  # a hidden score is replaced whatever it is
            assert not bad[:300].any()


# ------------------------------------------------------------------------------------------------ layouts
@pytest.mark.parametrize("Q", [1, 2, 3, 8])
@pytest.mark.parametrize("cap,sloped", [(0.0, False), (20.0, True)])
def test_caches_of_any_layout(Q, cap, sloped):
    """Views that start off 16 bytes, whose rows do, that are not contiguous in D, heads ahead of rows, heads that share one row."""
    from test_shaped_edges_cpu import _layouts

    B, S, H, D = 2, 300, 3, 64
    q, k, v, _ = _inputs(B, Q, S, H, D)
    slopes = slopes_for(H, DEV) if sloped else None
    dist = torch.arange(S - Q, S, device=DEV)[:, None] - torch.arange(S, device=DEV)
    seen = torch.ones(B, 1, Q, S, dtype=torch.bool, device=DEV)
    call = lambda *x: rab.ringattention_inference(*x, logit_cap=cap or None, alibi_slopes=slopes)
    with torch.no_grad():
        want = call(q, k, v)
        check(want, *attention(q, k, v, cap, slopes, dist[None, None], None, seen))
        for (name, a), b, c in zip(_layouts(q).items(), _layouts(k).values(), _layouts(v).values()):
            assert torch.equal(call(a, k, v), want) and torch.equal(call(q, b, v), want) and torch.equal(call(q, k, c), want), name
        one = k[:, :, :1].expand(B, S, H, D)
        assert torch.equal(call(q, one, v), call(q, one.contiguous(), v))


@pytest.mark.parametrize("name", ["off", "rows", "by_column", "by_head"])
@pytest.mark.parametrize("cap,sloped", [(0.0, False), (20.0, True)])
def test_training_and_prompts_of_any_layout(name, cap, sloped):
    """The same, and gradients of the outputs that lie so, for the attention kernels with tiles."""
    from test_shaped_edges_cpu import _layouts

    B, S, H, D = 2, 150, 3, 64
    q, k, v, dout = _inputs(B, S, S, H, D)
    slopes = slopes_for(H, DEV) if sloped else None
    kw = dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=cap or None, alibi_slopes=slopes)
    calls = (lambda *x: rab.ringattention(*x, blockwise_kwargs=kw), lambda *x: rab.ringattention_inference(*x, logit_cap=cap or None, alibi_slopes=slopes))
    for call in calls:
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = call(*leaves)
        want = torch.autograd.grad(out, leaves, dout)
        # (queries and keys so, values as they are: gradients of keys and values in layouts of their own)
        leaves = [_layouts(t)[name].detach().requires_grad_() for t in (q, k)] + [leaves[2]]
        again = call(*leaves)
        assert torch.equal(again, out)
        got = torch.autograd.grad(again, leaves, _layouts(dout)[name])
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert (got[0].float() - want[0].float()).norm() <= 2.0 ** -7 * want[0].float().norm()  # (dq is reduced in no fixed order)


def test_heads_that_share_keys_and_values():
    """One head's keys and values for all query heads, as an expanded view: gradients add up over them."""
    B, S, H, D = 2, 200, 4, 64
    q, k, v, dout = _inputs(B, S, S, H, D)
    kw = dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=20.0)
    at = torch.arange(S, device=DEV)
    k1, v1 = (t[:, :, :1].contiguous().requires_grad_() for t in (k, v))
    q.requires_grad_()
    out = rab.ringattention(q, k1.expand(B, S, H, D), v1.expand(B, S, H, D), blockwise_kwargs=kw)
    want = attention(q, k1.expand(B, S, H, D), v1.expand(B, S, H, D), 20.0, seen=visible(at, at, B, 1), dout=dout)
    check(out, want[0], want[1], "out")
    got = torch.autograd.grad(out, (q, k1, v1), dout)
    check(got[0], want[2][0], want[3][0], "dq")
    for i in (1, 2):  # the sum of H gradients in bf16 is rounded once more, at most once for each
        check(got[i], want[2][i].sum(2, keepdim=True), want[3][i].sum(2, keepdim=True) + H * HALF * want[2][i].abs().sum(2, keepdim=True), f"{i}")


def test_gradients_of_queries_keys_and_values_in_layouts_of_their_own():
    """Heads ahead of rows in some of them: the inference backward's results are contiguous whatever its inputs are."""
    B, S, H, D = 2, 150, 3, 64
    q, k, v, dout = _inputs(B, S, S, H, D)
    by_head = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(rab.ringattention_inference(*leaves, logit_cap=20.0), leaves, dout)
    for turned in ((0,), (1,), (2,), (0, 1, 2)):
        leaves = [(by_head(t) if i in turned else t).detach().requires_grad_() for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(rab.ringattention_inference(*leaves, logit_cap=20.0), leaves, dout)
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert (got[0].float() - want[0].float()).norm() <= 2.0 ** -7 * want[0].float().norm()  # (dq is reduced in no fixed order)


@pytest.mark.parametrize("Q", [1, 3, 8, 20])
@pytest.mark.parametrize("shape", ["1", "B111", "1H11", "BHQ1", "S", "QS", "B1QS", "longer"])
def test_masks_that_broadcast(Q, shape):
    """Along the keys too; a longer one is cut."""
    B, S, H, D = 2, 300, 3, 64
    q, k, v, _ = _inputs(B, Q, S, H, D)
    dims = {"1": (1,), "B111": (B, 1, 1, 1), "1H11": (1, H, 1, 1), "BHQ1": (B, H, Q, 1), "S": (S,), "QS": (Q, S), "B1QS": (B, 1, Q, S), "longer": (B, 1, 1, S + 50)}
    g = torch.Generator(device=DEV)
    g.manual_seed(Q)
    mask = torch.rand(dims[shape], device=DEV, generator=g) > 0.4
    with torch.no_grad():
        out = rab.ringattention_inference(q, k, v, mask, logit_cap=20.0)
    check(out, *attention(q, k, v, 20.0, seen=mask[..., :S].expand(B, H, Q, S)))


def test_documents_and_a_bias_that_all_rows_share():
    B, S, H, D = 3, 300, 2, 64
    x = _inputs(B, S, S, H, D)
    seg = (torch.arange(S, device=DEV) // 70).int()[None]
    bias = torch.zeros(1, 1, 1, S, device=DEV)
    bias[..., 250:] = float("-inf")
    kw = dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=20.0)
    with torch.no_grad():
        got = rab.ringattention(*x[:3], bias, seg, blockwise_kwargs=kw)
        want = rab.ringattention(*x[:3], bias.expand(B, H, 1, S).contiguous(), seg.expand(B, S).contiguous(), blockwise_kwargs=kw)
    assert torch.equal(got, want)


@pytest.mark.parametrize("B,S,H", [(1, 200, 3), (2, 1, 3), (2, 200, 1), (1, 1, 1)])
def test_axes_of_one_element_may_have_any_step(B, S, H):
    """Rows ahead of the batch, or heads ahead of rows, where there is one of them: contiguous with other strides than a new tensor's."""
    x = _inputs(B, S, S, H, 64)
    for cap, turn in ((0.0, (0, 1)), (20.0, (0, 1)), (20.0, (1, 2))):
        turned = [t.transpose(*turn).clone(memory_format=torch.contiguous_format).transpose(*turn) for t in x]
        _train(*turned, cap, slopes_for(H, DEV) if cap else None)
        leaves = [t.detach().requires_grad_() for t in turned[:3]]
        out = rab.ringattention_inference(*leaves, logit_cap=cap or None)
        got = torch.autograd.grad(out, leaves, turned[3])
        want = attention(*x[:3], cap, seen=torch.ones(B, 1, S, S, dtype=torch.bool, device=DEV), dout=x[3])
        check(out, want[0], want[1], "out")
        for a, w, b in zip(got, want[2], want[3]):
            check(a, w, b)


@pytest.mark.parametrize("cap,sloped,prefix", [(0.0, True, None), (20.0, False, None), (20.0, True, 5000)])
def test_more_tiles_than_the_lists_hold(cap, sloped, prefix):
    """Over 2^20 keys, or queries, tiles are looked for as the walk goes: in falling order with slopes, in the backward over the queries."""
    from ringattention_b200.ops import _lib, flash
    from ringattention_b200.ops.flash import MaskSpec, Positions

    n, few, D = (1 << 20) + 300, 70, 64
    far = _rand(1, n, 1, D, seed=1, std=1.4)
    near, v = _rand(1, few, 1, D, seed=2, std=1.4), _rand(1, n, 1, D, seed=3)
    slopes = torch.tensor([2.0 ** -14], device=DEV) if sloped else None
    pre = None if prefix is None else torch.tensor([prefix], device=DEV, dtype=torch.int32)
    qp, kp = torch.arange(n - few, n, device=DEV), torch.arange(n, device=DEV)
    out, lse = flash.flash_fwd(near, far, v, MaskSpec(1, Positions(n - few), Positions(0), logit_cap=cap, slopes=slopes, prefix=pre))
    check(out, *attention(near, far, v, cap, slopes, (qp[:, None] - kp)[None, None], None, visible(qp, kp, 1, 1, pre)), "keys")
    # few keys in the middle of many queries: only the gradients of the keys, whose sums go over all queries
    at, dout = Positions(n // 2), _rand(1, n, 1, D, seed=4)
    ms, val = MaskSpec(1, Positions(0), at, logit_cap=cap, slopes=slopes, prefix=pre), v[:, :few].contiguous()
    lo = torch.empty_like(far)
    out, lse = flash.flash_fwd(far, near, val, ms, out_lo=lo)
    dq = torch.empty(1, n, 1, D, device=DEV)
    lse2, delta = flash.flash_bwd_prep(out, dout, lse, dq, out_lo=lo)
    dk, dv = torch.empty_like(near), torch.empty_like(val)
    flash.flash_bwd(far, near, val, dout, lse2, delta, ms, dq, dk, dv)
    _lib.check_status()
    kp = torch.arange(n // 2, n // 2 + few, device=DEV)
    qp = torch.arange(n, device=DEV)
    want = attention(far, near, val, cap, slopes, (qp[:, None] - kp)[None, None], None, visible(qp, kp, 1, 1, pre), dout)
    check(out, want[0], want[1], "queries")
    for what, a, w, b in zip(("dq", "dk", "dv"), (dq, dk, dv), want[2], want[3]):
        check(a, w, b, what)


def test_second_derivatives_are_refused():
    x = [t.requires_grad_() for t in _inputs(1, 40, 40, 2, 64)[:3]]
    gains = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
    ids = torch.zeros(40, 3, device=DEV, dtype=torch.int32)
    for f, of in ((lambda: rab.ringattention(*x, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=40, key_chunk_size=40, logit_cap=2.0)), x),
                  (lambda: rab.ringattention_inference(*x, logit_cap=2.0), x), (lambda: rab.qk_norm_rope(*x[:2], *gains)[0], x[:1]),
                  (lambda: rab.distillation_loss(x[0][0, :, 0], ids, torch.zeros(40, 3, device=DEV)), x[:1])):
        want = torch.autograd.grad(f().float().sum(), of)
        grads = torch.autograd.grad(f().float().sum(), of, create_graph=True)
        assert torch.equal(grads[-1], want[-1])
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (grads[0].float().sum() + x[0].float().square().sum()).backward()
        assert x[0].grad is None
