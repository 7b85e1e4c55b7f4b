"""Shaped attention at its edges without a GPU: query positions far away, plans and what they refuse, rings of the PyTorch path."""
import pytest
import torch
from shaped_plain import attention

import ringattention_b200 as rab


def _rand(B, S, H, D, n=3, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, S, H, D, generator=g, dtype=torch.float64).to(dtype) for _ in range(n)]


@pytest.mark.parametrize("pos", [2 ** 29, 2 ** 30 - 1, torch.tensor([2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32), torch.tensor([2 ** 62, -(2 ** 62)])])
def test_queries_beyond_either_end_of_the_cache(pos):
    """In 32 bits as in 64 bits from the end of the cache on: 50 keys, slopes up to 0.5, so 2^-24 of scores up to 25 and a few roundings of sums."""
    B, Q, S, H, D = 2, 3, 50, 2, 8
    q, k, v = _rand(B, S, H, D)
    q, slopes = q[:, :Q], torch.tensor([0.5, 0.1])
    got = rab.ringattention_inference(q, k, v, logit_cap=5.0, alibi_slopes=slopes, query_pos=pos)
    rows = torch.as_tensor(pos).long().reshape(-1, 1) + torch.arange(Q)
    dist = rows.clamp(0, S - 1)[:, None, :, None] - torch.arange(S)
    want, _ = attention(q, k, v, 5.0, slopes, dist, None, torch.ones(B, 1, Q, S, dtype=torch.bool))
    assert torch.allclose(got.double(), want, atol=2e-5)


@pytest.mark.parametrize("which", ["alibi_slopes", "prefix_lens", "query_pos"])
def test_constants_that_change_before_the_backward_pass(which):
    q, k, v = (t.requires_grad_() for t in _rand(2, 12, 2, 4))
    const = dict(alibi_slopes=torch.tensor([0.5, 0.1]), prefix_lens=torch.tensor([3, 5], dtype=torch.int32), query_pos=torch.tensor([2, 7], dtype=torch.int32))
    if which == "query_pos":
        call = lambda: rab.ringattention_inference(q, k, v, alibi_slopes=const["alibi_slopes"], query_pos=const[which])
    else:
        call = lambda: rab.ringattention(q, k, v, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=12, key_chunk_size=12,
                                                                        **{c: const[c] for c in ("alibi_slopes", "prefix_lens")}))
    torch.autograd.grad(call().sum(), (q, k, v))
    out = call()
    const[which].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), (q, k, v))


def test_constants_made_in_inference_mode():
    q, k, v = (t.requires_grad_() for t in _rand(2, 12, 2, 4))
    with torch.inference_mode():
        const = dict(alibi_slopes=torch.tensor([0.5, 0.1]), prefix_lens=torch.tensor([3, 5], dtype=torch.int32))
    kw = dict(causal_block_size=1, query_chunk_size=12, key_chunk_size=12)
    a = torch.autograd.grad(rab.ringattention(q, k, v, blockwise_kwargs=dict(kw, **const)).sum(), (q, k, v))
    b = torch.autograd.grad(rab.ringattention(q, k, v, blockwise_kwargs=dict(kw, **{n: t.clone() for n, t in const.items()})).sum(), (q, k, v))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_forward_mode_derivatives_are_noticed():
    from torch.autograd import forward_ad

    from ringattention_b200.ops import _lib

    x, y = torch.ones(3), torch.ones(3)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, y)
        assert _lib.has_tangent(y, d) and not _lib.has_tangent(x, y) and not d.requires_grad
    assert not _lib.has_tangent(d)


@pytest.mark.parametrize("causal", [None, 1])
@pytest.mark.parametrize("bad", [torch.zeros(3, dtype=torch.int32), torch.zeros(2), True, 2.5])
def test_a_plan_checks_prefixes_with_and_without_a_causal_rule(bad, causal):
    from ringattention_b200.config import BlockwiseKwargs
    from ringattention_b200.ops.attention import make_plan

    kw = dict(causal_block_size=causal, query_chunk_size=6, key_chunk_size=6)
    with pytest.raises(ValueError):
        make_plan(0, 1, 2, 6, 6, 2, BlockwiseKwargs.from_any(dict(kw, prefix_lens=bad)), device="cpu")
    plan = make_plan(0, 1, 2, 6, 6, 2, BlockwiseKwargs.from_any(dict(kw, prefix_lens=torch.tensor([1, 2]))), device="cpu")
    assert (plan.shape is None) == (causal is None) and (plan.steps[0].mask.prefix is None) == (causal is None)
