"""Shaped attention over random calls of what its documentation allows, against 64 bits: sizes, layouts, documents, biases, dropout, prefixes, caches,
positions and masks in combinations that no other test names. Seeds are fixed."""
import math
import random

import pytest
import torch
from shaped_plain import attention, check, slopes_for, visible

import ringattention_b200 as rab
from ringattention_b200.ops import reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _laid_out(rng, t):
    """The same values, or one slice's for all, in a layout that callers have."""
    B, S, H, D = t.shape
    kind = rng.choice(["plain", "heads first", "packed", "wide", "off 16 bytes", "by column", "shared"])
    if kind == "heads first":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "by column":
        return t.transpose(1, 3).contiguous().transpose(1, 3)
    if kind == "shared":
        axis = rng.choice([0, 2])
        return t.narrow(axis, 0, 1).expand(t.shape)
    if kind == "plain":
        return t
    buf = {"packed": torch.zeros(B, S, 3, H, D, device=DEV, dtype=t.dtype), "wide": torch.full((B, S + 5, H + 1, D), math.nan, device=DEV, dtype=t.dtype),
           "off 16 bytes": torch.zeros(t.numel() + 3, device=DEV, dtype=t.dtype)}[kind]
    view = {"packed": lambda: buf[:, :, 1], "wide": lambda: buf[:, 2:S + 2, :H], "off 16 bytes": lambda: buf[3:].view(t.shape)}[kind]()
    return view.copy_(t)


def _shape(rng, H):
    """A cap and slopes, and the deviation of queries and keys. (Where nearly all scores are far beyond the cap its derivative, 1 - tanh^2, is the rounding of
    the tanh and no bound relative to the gradient holds; so small caps come with small scores.)"""
    cap, slopes = rng.choice([0.0, 0.0, 0.5, 5.0, 20.0, 50.0, 54.0, 60.0, 300.0]), None
    if rng.random() < 0.5:
        slopes = rng.choice([slopes_for(H, DEV), -0.02 * slopes_for(H, DEV), torch.zeros(H, device=DEV), 3 * torch.rand(H, device=DEV)])
    return cap, slopes, 0.1 if 0 < cap < 1 else rng.choice([0.3, 1.4]) if cap < 20 else rng.choice([0.3, 1.4, 3.0])


def _inputs(rng, B, Sq, Sk, H, D, std):
    rand = lambda S, std: _laid_out(rng, (torch.randn(B, S, H, D, device=DEV) * std).bfloat16())
    return rand(Sq, std), rand(Sk, std), rand(Sk, 1.0), torch.randn(B, Sq, H, D, device=DEV).bfloat16()


def _compare(leaves, out, dout, want, what):
    check(out, want[0], want[1], f"out {what}")
    if len(want) > 2:
        for name, a, w, b in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout), want[2], want[3]):
            check(a, w, b, f"{name} {what}")


@pytest.mark.parametrize("seed", range(60))
def test_training(seed):
    rng = random.Random(seed)
    torch.manual_seed(seed)
    B, H, D, Sq = rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 5]), rng.choice([64, 128]), _log_int(rng, 1, 1200)
    Sk, first = (Sq, None) if rng.random() < 0.7 else (_log_int(rng, 1, 4000), 0)
    first = None if first is None else rng.randrange(Sk)
    cap, slopes, std = _shape(rng, H)
    q, k, v, dout = _inputs(rng, B, Sq, Sk, H, D, std)
    cbs, prefix, seg, bias, drop = rng.choice([0, 1, 1, 2, 64, 300]), None, None, None, rng.choice([0.0, 0.0, 0.1, 0.5])
    if rng.random() < 0.5:
        prefix = torch.randint(-5, Sk + 20, (B,), device=DEV, dtype=rng.choice([torch.int32, torch.int64])) if rng.random() < 0.7 else rng.randrange(-3, Sk + 3)
    if first is None and rng.random() < 0.4:
        seg = (torch.rand(B, Sq, device=DEV) < rng.choice([0.5, 0.02, 0.003])).int().cumsum(1).int()
    if rng.random() < 0.4:
        bias = torch.randn(B, rng.choice([1, H]), 1, Sk, device=DEV) * rng.choice([0.0, 4.0])
        bias.masked_fill_(torch.rand(bias.shape, device=DEV) < rng.choice([0.0, 0.3]), rng.choice([-math.inf, torch.finfo(torch.float32).min]))
    kw = dict(causal_block_size=cbs or None, query_chunk_size=Sq, key_chunk_size=Sk, logit_cap=cap or None, alibi_slopes=slopes, prefix_lens=prefix)
    if drop:
        kw.update(deterministic=False, dropout_rng=seed, attn_pdrop=drop)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = rab.ringattention(*leaves, bias, seg, first, blockwise_kwargs=kw)
    qp, kp = torch.arange(Sq, device=DEV) + (first or 0), torch.arange(Sk, device=DEV)
    seen = visible(qp, kp, B, cbs, prefix, seg, seg, bias)
    if drop:
        seen = seen.expand(B, H, Sq, Sk) & ~R.dropped(seed, drop, B, H, qp, kp)
    want = attention(q, k, v, cap, slopes, (qp[:, None] - kp)[None, None], None if bias is None else bias.clamp_min(-1e30), seen, dout)
    _compare(leaves, out, dout, want, f"{(B, Sq, Sk, H, D)} cap {cap} blocks {cbs}")


@pytest.mark.parametrize("seed", range(90))
def test_inference(seed):
    rng = random.Random(1000 + seed)
    torch.manual_seed(seed)
    B, H, D = rng.choice([1, 2, 3, 8]), rng.choice([1, 3, 8]), rng.choice([64, 128])
    Q, S = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 9, 17, 130]), _log_int(rng, 1, 3000)
    cap, slopes, std = _shape(rng, H)
    q, k, v, dout = _inputs(rng, B, Q, S, H, D, std)
    pos = rng.choice([None, rng.randrange(S + 50), torch.randint(-Q - 3, S + 5, (B,), device=DEV, dtype=rng.choice([torch.int32, torch.int64]))])
    lens = torch.randint(0, S + 1, (B,), device=DEV)
    mask = rng.choice([None, torch.rand(rng.choice([1, B]), rng.choice([1, H]), rng.choice([1, Q]), S, device=DEV) < rng.choice([0.02, 0.5, 0.98]),
                       (torch.arange(S, device=DEV) < lens[:, None])[:, None, None],
                       (torch.arange(S, device=DEV) <= torch.arange(S - Q, S, device=DEV)[:, None])[None, None]])
    grad = rng.random() < 0.3
    leaves = [t.detach().requires_grad_(grad) for t in (q, k, v)]
    out = rab.ringattention_inference(*leaves, mask, logit_cap=cap or None, alibi_slopes=slopes, query_pos=pos)
    first = torch.as_tensor(max(0, S - Q) if pos is None else pos, device=DEV).long().reshape(-1, 1, 1, 1)
    dist = (first + torch.arange(Q, device=DEV)[:, None]).clamp(0, S - 1) - torch.arange(S, device=DEV)  # (beyond an end all keys are further by one number)
    seen = torch.ones(B, 1, Q, S, dtype=torch.bool, device=DEV) if mask is None else mask.expand(B, -1, Q, S)
    want = attention(q, k, v, cap, slopes, dist, None, seen, dout if grad else None)
    _compare(leaves, out, dout, want, f"{(B, Q, S, H, D)} cap {cap}")
