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


@pytest.mark.parametrize("pos", [None, 13, torch.tensor([27, 4])])
def test_a_cache_in_shards_on_the_pytorch_ring(pos):
    from ringattention_b200.ops import reference as R
    from ringattention_b200.ops.inference import inference_shape
    from ringattention_b200.parallel.comm import SingleComm, run_fake_ring

    world, B, Q, S, H, D = 3, 2, 3, 30, 2, 8
    q, k, v, g = _rand(B, S, H, D, n=4, dtype=torch.float64)
    q, g, n = q[:, :Q], g[:, :Q], S // 3
    slopes, mask = torch.tensor([0.5, 0.1]), torch.rand(B, 1, Q, S, generator=torch.Generator().manual_seed(1)) > 0.2

    def one(k, v, comm):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = R.RingAttentionInferenceRef.apply(*leaves, mask, comm, True, inference_shape(q, k, comm.size, 3.0, slopes, pos))
        # every rank's output is the whole one, and what its gradient says of keys and values travels to their owners: a share of it each
        return (out.detach(), *torch.autograd.grad(out, leaves, g / comm.size))

    want = one(k, v, SingleComm())
    got = run_fake_ring(world, lambda comm: one(*(t[:, comm.rank * n:(comm.rank + 1) * n] for t in (k, v)), comm))
    for r in got:
        assert torch.allclose(r[0], want[0], atol=1e-10) and torch.allclose(r[1] * world, want[1], atol=1e-10)
    for i in (2, 3):
        assert torch.allclose(torch.cat([r[i] for r in got], 1), want[i], atol=1e-10)


def test_a_ring_keeps_what_rounding_took_at_its_last_step(monkeypatch):
    """Of the launches of a rank the last one alone, which writes the bf16 output, gets the place for it; the backward's preparation reads it."""
    from ringattention_b200.config import BlockwiseKwargs
    from ringattention_b200.ops import attention as A
    from ringattention_b200.ops import flash
    from ringattention_b200.parallel.symm import SymmRing

    world, B, n, H, D = 3, 1, 128, 2, 64
    ring = object.__new__(SymmRing)
    ring.rank, ring.overlap, ring.copy_ctas, ring._local, ring.device = 1, True, 4, {}, torch.device("cpu")
    own = type("Own", (), dict(peer_ptrs=[0] * world))
    monkeypatch.setattr(SymmRing, "_stage_kv", lambda self, k, v: (own, 0, 0, torch.zeros(1)))
    monkeypatch.setattr(SymmRing, "_slab_views", lambda self, *a: (k, v))
    monkeypatch.setattr(SymmRing, "barrier", lambda self: None)
    monkeypatch.setattr(SymmRing, "backward", lambda self, *a: None)
    calls, preps = [], []
    monkeypatch.setattr(flash, "flash_fwd", lambda *a, **kw: calls.append(kw))
    monkeypatch.setattr(flash, "flash_bwd_prep", lambda out, dout, lse, dq, out_lo=None: (preps.append(out_lo), (None, None))[1])
    monkeypatch.setattr(A.K, "cast_f32_to_bf16", lambda *a: None)
    q, k, v = (torch.zeros(B, n, H, D, dtype=torch.bfloat16) for _ in range(3))
    for kw, steps in ((dict(logit_cap=5.0), 2), (dict(prefix_lens=300), 3), (dict(), 2)):  # (a prefix opens the block ahead, too)
        calls.clear()
        preps.clear()
        plan = A.make_plan(1, world, B, n, n, H, BlockwiseKwargs.from_any(dict(causal_block_size=1, query_chunk_size=n, key_chunk_size=n, **kw)), device="cpu")
        leaf = q.clone().requires_grad_()
        out = A.RingFlashAttention.apply(leaf, k, v, plan, ring)
        assert len(calls) == steps and all(c["out_lo"] is None for c in calls[:-1])
        assert (calls[-1]["out_lo"] is not None) == bool(kw) and calls[-1]["out"].dtype == torch.bfloat16
        out.backward(torch.zeros_like(out))
        assert preps[0] is calls[-1]["out_lo"]


def _layouts(t, seed=0):
    """The same values behind layouts that a caller may have."""
    B, S, H, D = t.shape
    off = torch.zeros(t.numel() + 3, dtype=t.dtype, device=t.device)[3:].view(t.shape)
    off.copy_(t)
    rows = torch.zeros(B, S, H, D + 4, dtype=t.dtype, device=t.device)[..., :D]
    rows.copy_(t)
    return dict(off=off, rows=rows, by_column=t.transpose(1, 3).contiguous().transpose(1, 3), by_head=t.transpose(1, 2).contiguous().transpose(1, 2))


def test_few_query_rows_read_aligned_rows_whatever_the_cache_is(monkeypatch):
    """The decode kernels read 16 bytes at a time: views that start elsewhere or are not contiguous in D are copied ahead of the launch."""
    import struct

    from ringattention_b200.ops import _lib, flash
    from ringattention_b200.ops import decode as Dk

    launches, copies, real = [], [], flash.ready
    monkeypatch.setattr(Dk, "default_splits", lambda *a, **kw: 1)
    monkeypatch.setattr(Dk, "merge_partials", lambda *a, **kw: None)
    monkeypatch.setattr(flash, "ready", lambda t: (copies.append(real(t)), copies[-1])[1])
    monkeypatch.setattr(_lib, "stream_handle", lambda: 0)
    monkeypatch.setattr(_lib, "call", lambda name, args: launches.append(struct.unpack_from("@3P6q", args)))
    axis = type("Axis", (), dict(rank=0, size=1))
    q, k, v = _rand(2, 8, 3, 64, dtype=torch.bfloat16)
    k, v = torch.cat([k, k, v], 1), torch.cat([v, k, v], 1)
    for n in (1, 2, 4, 8):
        for a, b, c in zip(_layouts(q[:, :n]).values(), _layouts(k).values(), _layouts(v).values()):
            copies.clear()
            Dk.ring_decode_attention(a, b, c, None, axis)
            at = launches[-1]
            assert not any(p % 16 for p in at[:3]) and not any(s % 8 for s in at[3:])
            kk, vv = copies or (b, c)
            assert at[1:] == (kk.data_ptr(), vv.data_ptr(), *kk.stride()[:3], *vv.stride()[:3])
            assert torch.equal(kk, k) and torch.equal(vv, v) and kk.stride(3) == vv.stride(3) == 1
    copies.clear()
    Dk.ring_decode_attention(q[:, :1].contiguous(), k, v, None, axis)
    assert not copies and launches[-1][1:3] == (k.data_ptr(), v.data_ptr())


@pytest.mark.parametrize("bad", [dict(q=6), dict(k=2), dict(v=8), dict(k_s=4), dict(v_s=12)])
def test_the_decode_launcher_refuses_rows_off_16_bytes(bad):
    from ringattention_b200.ops import _lib
    from ringattention_b200.ops import decode as Dk

    at = [4096 + bad.get(n, 0) for n in "qkv"]
    strides = [6400, 64 + bad.get("k_s", 0), 64, 6400, 64 + bad.get("v_s", 0), 64]
    args = Dk._DECODE_ARGS.pack(*at, *strides, 4096, 4096, 0, 0, 0, 0, 1, 1, 1, 100, 64, 1, 0.125, -1, 0, 0, 0, 0, 0, 0, 0, 3, 0, 0, 0.0, 0, 0, 0, 0, 0)
    with pytest.raises(_lib.KernelError, match="start on 16 bytes"):
        _lib.call("ra_decode_splitkv", args)


def test_inference_checks_that_queries_keys_and_values_belong_together():
    q, k, v = _rand(2, 12, 3, 8)
    rab.ringattention_inference(q[:, :2], k, v)
    for bad in ((q[0], k, v), (q, k, v[:, :11]), (q[:1], k, v), (q, k[:1], v[:1]), (q[:, :, :1], k, v), (q[..., :4], k, v), (q, k, v[..., :4]),
                (q, k.to("meta"), v), (q, k, v.to("meta"))):
        with pytest.raises(ValueError):
            rab.ringattention_inference(*bad)


def test_few_query_rows_take_keys_and_values_of_their_type():
    from ringattention_b200.ops.inference import ring_inference_attention

    q, k, v = _rand(1, 4, 2, 64, dtype=torch.bfloat16)
    axis = type("Axis", (), dict(rank=0, size=1))
    for bad in ((q, k.float(), v), (q, k, v.half())):
        with pytest.raises(ValueError, match="one type"):
            ring_inference_attention(*bad, None, axis)


@pytest.mark.parametrize("bad", [(3, 1, 2, 12), (2, 2, 2, 12), (2, 3, 3, 12), (1, 1, 4, 12), (2, 3, 2, 11), (2, 1, 2, 0), (1, 2, 3, 2, 12), ()])
def test_masks_that_do_not_broadcast_are_refused(bad):
    q, k, v = _rand(2, 12, 3, 8)
    with pytest.raises(ValueError, match="attn_mask"):
        rab.ringattention_inference(q[:, :2], k, v, torch.ones(bad, dtype=torch.bool))


def test_masks_of_another_type_or_device_are_refused():
    q, k, v = _rand(2, 12, 3, 8)
    for bad in (torch.zeros(2, 12), torch.zeros(2, 12, dtype=torch.complex64), torch.ones(2, 12, dtype=torch.bool, device="meta")):
        with pytest.raises(ValueError, match="attn_mask"):
            rab.ringattention_inference(q[:, :2], k, v, bad)


@pytest.mark.parametrize("shape", [(1,), (12,), (15,), (1, 1), (2, 1), (2, 12), (3, 1, 12), (3, 2, 1), (2, 1, 1, 1), (2, 3, 2, 12), (1, 3, 1, 12)])
def test_masks_that_broadcast(shape):
    q, k, v = _rand(2, 12, 3, 8, dtype=torch.float64)
    q = q[:, :2]
    mask = torch.rand(shape, generator=torch.Generator().manual_seed(3)) > 0.4
    whole = mask[..., :12].expand(2, 3, 2, 12)
    want, _ = attention(q, k, v, seen=whole)
    assert torch.allclose(rab.ringattention_inference(q, k, v, mask), want, atol=1e-10)


def _plan(B=3, S=6, H=2, **kw):
    from ringattention_b200.config import BlockwiseKwargs
    from ringattention_b200.ops.attention import make_plan

    return make_plan(0, 1, B, S, S, H, BlockwiseKwargs(query_chunk_size=S, key_chunk_size=S), device="cpu", **kw)


@pytest.mark.parametrize("bad", [dict(segment_ids=torch.zeros(2, 6, dtype=torch.int32)), dict(segment_ids=torch.zeros(6, dtype=torch.int32)),
                                 dict(attn_bias=torch.zeros(2, 1, 1, 6)), dict(attn_bias=torch.zeros(3, 3, 1, 6)), dict(attn_bias=torch.zeros(1, 0, 1, 6))])
def test_documents_and_biases_of_another_batch_or_heads_are_refused(bad):
    with pytest.raises(ValueError):
        _plan(**bad)


def test_documents_and_biases_that_all_rows_share():
    seg, bias = torch.arange(6)[None] // 2, torch.randn(1, 2, 1, 6)
    ms = _plan(segment_ids=seg, attn_bias=bias).steps[0].mask
    assert torch.equal(ms.seg_q, seg.int().expand(3, 6)) and ms.seg_q.is_contiguous() and ms.seg_q_mm.shape == (3, 1, 2)
    assert torch.equal(ms.bias, bias[:, :, 0].expand(3, 2, 6)) and ms.bias.is_contiguous()


def test_second_derivatives_are_refused():
    """The backward passes are not differentiable themselves: their results would count as constants."""
    q, k, v = (t.requires_grad_() for t in _rand(1, 6, 2, 4, dtype=torch.float64))
    calls = (lambda: rab.ringattention(q, k, v, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=6, key_chunk_size=6, logit_cap=2.0)),
             lambda: rab.ringattention_inference(q, k, v, alibi_slopes=torch.ones(2)))
    for call in calls:
        grads = torch.autograd.grad(call().sum(), (q, k, v), create_graph=True)
        grads[2].mul_(2.0)  # (as after any other backward)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            sum(g.square().sum() for g in grads).backward()
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (grads[0].sum() + q.square().sum()).backward()


def test_constants_made_in_inference_mode_without_gradients():
    q, k, v = _rand(2, 12, 2, 4)
    with torch.inference_mode():
        slopes, pos = torch.tensor([0.5, 0.1]), torch.tensor([3, 5], dtype=torch.int32)
    want = rab.ringattention_inference(q, k, v, alibi_slopes=slopes.clone(), query_pos=pos.clone())
    with torch.no_grad():
        assert torch.equal(rab.ringattention_inference(q, k, v, alibi_slopes=slopes, query_pos=pos), want)
    with torch.inference_mode():
        assert torch.equal(rab.ringattention_inference(q, k, v, alibi_slopes=slopes, query_pos=pos), want)
