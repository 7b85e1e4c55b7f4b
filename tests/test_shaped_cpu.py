"""Shaped attention scores on the PyTorch path (any device and type): against 64 bits and differences, over rings, and what is refused."""
import pytest
import torch
from shaped_plain import attention, slopes_for, visible

import ringattention_b200 as rab
from ringattention_b200.config import BlockwiseKwargs
from ringattention_b200.ops import reference as R
from ringattention_b200.parallel.comm import SingleComm, run_fake_ring


def _rand(B, S, H, D, n=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, S, H, D, generator=g, dtype=torch.float64) * 1.5 for _ in range(n)]


@pytest.mark.parametrize("cap,sloped,prefix,cbs", [(2.0, False, None, 1), (0.0, True, None, None), (3.0, True, [0, 20], 1), (0.0, False, [9, 40], 4)])
def test_reference_path_matches_64_bits(cap, sloped, prefix, cbs):
    B, S, H, D = 2, 36, 4, 8
    q, k, v, g = _rand(B, S, H, D)
    seg = (torch.arange(S) // 13).expand(B, S)
    prefix = None if prefix is None else torch.tensor(prefix)
    slopes = slopes_for(H) if sloped else None
    kw = dict(causal_block_size=cbs, query_chunk_size=12, key_chunk_size=9, logit_cap=cap or None, alibi_slopes=slopes, prefix_lens=prefix)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = rab.ringattention(*leaves, None, seg, blockwise_kwargs=kw)
    at = torch.arange(S)
    want, _, grads, _ = attention(q, k, v, cap, slopes, (at[:, None] - at)[None, None], None, visible(at, at, B, cbs, prefix, seg, seg), g)
    assert torch.allclose(out, want, atol=1e-10)
    for a, b in zip(torch.autograd.grad(out, leaves, g), grads):
        assert torch.allclose(a, b, atol=1e-9)


def test_gradients_against_differences():
    q, k, v = (t[:, :7, :2, :3].clone().requires_grad_() for t in _rand(1, 7, 2, 3, n=3))
    kw = dict(causal_block_size=1, query_chunk_size=7, key_chunk_size=7, logit_cap=1.5, alibi_slopes=slopes_for(2), prefix_lens=3)
    assert torch.autograd.gradcheck(lambda *x: rab.ringattention(*x, blockwise_kwargs=kw), (q, k, v))
    f = lambda *x: rab.ringattention_inference(*x, logit_cap=1.5, alibi_slopes=slopes_for(2), query_pos=torch.tensor([2]))
    assert torch.autograd.gradcheck(f, (q[:, :2].detach().requires_grad_(), k, v))


@pytest.mark.parametrize("layout", ["contiguous", "zigzag"])
def test_ring_equals_one_device(layout):
    world, B, S, H, D = 4, 2, 64, 2, 8
    q, k, v, g = _rand(B, S, H, D, seed=3)
    shape = dict(causal_block_size=1, query_chunk_size=8, key_chunk_size=8, logit_cap=2.5, alibi_slopes=slopes_for(H), prefix_lens=torch.tensor([0, 37]))

    def one(q, k, v, g, comm, layout):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = R.RingAttentionRef.apply(*leaves, None, None, None, comm, True, BlockwiseKwargs.from_any(dict(shape, layout=layout)))
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    want = one(q, k, v, g, SingleComm(), "contiguous")
    parts = [R.to_layout(t, world, layout) for t in (q, k, v, g)]
    n = S // world
    got = run_fake_ring(world, lambda comm: one(*(t[:, comm.rank * n:(comm.rank + 1) * n] for t in parts), comm, layout))
    for i, w in enumerate(want):
        assert torch.allclose(R.from_layout(torch.cat([r[i] for r in got], 1), world, layout), w, atol=1e-9)


def test_inference_positions():
    B, Q, S, H, D = 3, 2, 30, 2, 8
    q, k, v = _rand(B, S, H, D, n=3, seed=5)
    q = q[:, :Q]
    at = torch.arange(S)
    for pos in (None, 11, torch.tensor([28, 5, 0])):
        first = torch.as_tensor(S - Q if pos is None else pos).reshape(-1, 1, 1, 1)
        dist = first + torch.arange(Q)[:, None] - at
        mask = (dist >= 0).expand(B, 1, Q, S)
        got = rab.ringattention_inference(q, k, v, mask, logit_cap=3.0, alibi_slopes=slopes_for(H), query_pos=pos)
        want, _ = attention(q, k, v, 3.0, slopes_for(H), dist, None, mask)
        assert torch.allclose(got, want, atol=1e-10)


@pytest.mark.parametrize("bad", [dict(logit_cap=0.0), dict(logit_cap=-1.0), dict(logit_cap=float("nan")), dict(logit_cap=float("inf")), dict(logit_cap=True),
                                 dict(logit_cap="30"), dict(alibi_slopes=torch.zeros(3)), dict(alibi_slopes=torch.zeros(2, 1)),
                                 dict(alibi_slopes=torch.zeros(2, dtype=torch.int32)), dict(alibi_slopes=torch.zeros(2, requires_grad=True)),
                                 dict(prefix_lens=torch.zeros(2)), dict(prefix_lens=torch.zeros(2, dtype=torch.int32)), dict(prefix_lens=True),
                                 dict(prefix_lens=2.5)])
def test_what_is_refused(bad):
    q, k, v = _rand(1, 6, 2, 4, n=3)
    with pytest.raises(ValueError):
        rab.ringattention(q, k, v, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=6, key_chunk_size=6, **bad))
    if "prefix_lens" not in bad:
        with pytest.raises(ValueError):
            rab.ringattention_inference(q, k, v, **bad)


@pytest.mark.parametrize("cap", [1e-3, 1e30])
def test_caps_at_the_ends_of_their_range(cap):
    import ringattention_b200 as rab

    q = torch.randn(1, 6, 2, 8)
    kw = dict(causal_block_size=1, query_chunk_size=6, key_chunk_size=6)
    assert rab.ringattention(q, q, q, blockwise_kwargs=dict(kw, logit_cap=cap)).isfinite().all()
    with pytest.raises(ValueError):
        rab.ringattention(q, q, q, blockwise_kwargs=dict(kw, logit_cap=cap / 2 if cap < 1 else cap * 2))


@pytest.mark.parametrize("pos", [-1, 1 << 30, True, 2.0, torch.zeros(1), torch.zeros(2, dtype=torch.int32)])
def test_query_positions_that_are_refused(pos):
    q, k, v = _rand(1, 6, 2, 4, n=3)
    with pytest.raises(ValueError):
        rab.ringattention_inference(q, k, v, alibi_slopes=torch.ones(2), query_pos=pos)


def test_a_validated_object_is_checked_too():
    q, k, v = _rand(1, 6, 2, 4, n=3)
    with pytest.raises(ValueError):
        rab.ringattention(q, k, v, blockwise_kwargs=BlockwiseKwargs(query_chunk_size=6, key_chunk_size=6, logit_cap=-2.0))
