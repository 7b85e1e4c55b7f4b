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
