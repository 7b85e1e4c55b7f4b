"""Public API: ``ringattention``, ``blockwise_feedforward``, ``ringattention_inference`` and the
pure-PyTorch ``ringattention_ref`` (the same four names the reference exports,
ringattention/__init__.py:23-27, with ``ringattention_jax`` -> ``ringattention_ref``), and beside them what a decoder needs
around its attention: ``qk_norm_rope``, ``distillation_loss`` and ``distillation_loss_and_grad``.

Dispatch (the reference picks an implementation per XLA platform, __init__.py:12-21):

* CUDA bf16 tensors with head_dim 64 or 128 and at most a key bias -> the fused sm_100a kernels.
  On a multi-rank axis KV blocks are pulled from peer memory inside the kernels.
* anything else (CPU, fp32/fp64, a bias with query rows) -> the PyTorch restatement, which rotates
  KV through the axis' communicator (gloo, NCCL or the in-process fake ring).

The GPU path never silently degrades: if the kernel library cannot be loaded the call raises.
"""
from __future__ import annotations

import warnings
from typing import Any, Callable, Optional, Sequence

import torch
import torch.utils.checkpoint

from .config import POLICY_NOTHING_SAVEABLE, BlockwiseKwargs, _policy_name
from .ops import _lib
from .ops import reference as R
from .parallel.mesh import AxisContext, resolve_axis


_WARNED: set = set()


def _warn_fallback(q: torch.Tensor, why: str) -> None:
    """Tell the user, once per reason, that CUDA tensors are being served by the PyTorch restatement."""
    if q.is_cuda and why not in _WARNED:
        _WARNED.add(why)
        warnings.warn(f"ringattention_b200: {why}; this call runs on the PyTorch path, far slower than the "
                      "sm_100a kernels (which take bf16 tensors with head_dim 64 or 128 and at most a key bias)",
                      RuntimeWarning, stacklevel=3)


def _fallback_reason(q: torch.Tensor, attn_bias) -> str:
    if q.dtype != torch.bfloat16:
        return f"dtype {q.dtype} is not bfloat16"
    if q.shape[-1] not in (64, 128):
        return f"head_dim {q.shape[-1]} is not 64 or 128"
    return "attn_bias has query rows (only a key bias (B, 1|H, 1, S_total) is fused)"


def _fused_ok(q: torch.Tensor, attn_bias) -> bool:
    if not q.is_cuda or q.dtype != torch.bfloat16 or q.shape[-1] not in (64, 128):
        return False
    if attn_bias is not None and (attn_bias.dim() != 4 or attn_bias.shape[-2] != 1):
        return False
    return True


def _symm_ring_for(axis: AxisContext, device):
    if axis.size == 1:
        return None
    if axis.symm_ring is None:
        from .parallel.symm import SymmRing

        axis.symm_ring = SymmRing(axis.group, device)
    return axis.symm_ring


def _check_qkv(q, k, v) -> None:
    a, b = q.shape, k.shape
    if len(a) != 4 or len(b) != 4 or b != v.shape or a[0] != b[0] or a[2] != b[2] or a[3] != b[3]:
        raise ValueError("q must be (B,Sq,H,D) and k, v (B,Sk,H,D) with matching B, H, D")
    d = q.device
    if k.device != d or v.device != d:
        raise ValueError("q, k and v must be on one device")


def ringattention(q, k, v, attn_bias=None, segment_ids=None, cache_idx=None, axis_name=None,
                  float32_logits: bool = True, blockwise_kwargs=None):
    """Blockwise ring attention over the mesh axis ``axis_name``.

    Arguments follow ringattention/ringattention_jax.py:93 (README.md:20-36):

    ``q, k, v``  per-rank shards ``(B, S_local, H, D)``; rank r owns tokens ``[r*S_local,
    (r+1)*S_local)`` (or the zig-zag chunks when ``blockwise_kwargs["layout"] == "zigzag"``).
    ``attn_bias``  additive, global along keys: ``(B, 1|H, 1|S, S_total)``, or ``None``.
    ``segment_ids``  global ``(B, S_total)`` ints; tokens attend only inside equal ids.
    ``cache_idx``  ``None`` for training; otherwise the global position of the first query on
    *every* rank (q replicated, KV cache sequence-sharded). Taken as an exact token offset.
    ``axis_name``  registered axis name (``"sp"``), a communicator, or ``None`` for one device.
    ``float32_logits``  accepted for compatibility; logits and softmax state are always fp32
    (bf16 x bf16 products are exact in the fp32 accumulator).
    ``blockwise_kwargs``  the reference's dict (see :class:`~ringattention_b200.config.BlockwiseKwargs`).

    ``blockwise_kwargs`` may also shape the scores (``logit_cap``, ``alibi_slopes``) and open a prefix (``prefix_lens``).

    Returns ``(B, S_local, H, D)`` in ``v.dtype``; differentiable w.r.t. q, k, v only, once.
    """
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return ringattention(q, k, v, attn_bias, segment_ids, cache_idx, axis_name, float32_logits, blockwise_kwargs)
    kw = BlockwiseKwargs.from_any(blockwise_kwargs)
    axis = resolve_axis(axis_name)
    _check_qkv(q, k, v)
    if _fused_ok(q, attn_bias):
        from .ops import attention as A
        from .ops.flash import ready

        B, Sq, H, D = q.shape
        plan = A.make_plan(axis.rank, axis.size, B, Sq, k.shape[1], H, kw, segment_ids=segment_ids,
                           attn_bias=attn_bias, cache_idx=cache_idx, device=q.device)
        qq, kk, vv = (ready(t) for t in (q, k, v))
        return A.RingFlashAttention.apply(qq, kk, vv, plan, _symm_ring_for(axis, q.device))
    _warn_fallback(q, _fallback_reason(q, attn_bias))
    return R.RingAttentionRef.apply(q, k, v, attn_bias, segment_ids, cache_idx, axis.comm,
                                    float32_logits, kw)


def ringattention_ref(q, k, v, attn_bias=None, segment_ids=None, cache_idx=None, axis_name=None,
                      float32_logits: bool = True, blockwise_kwargs=None):
    """Same contract as :func:`ringattention`, always on the PyTorch restatement (any device or
    dtype). It is the CPU path, the oracle of the tests and, with NCCL, the rotation baseline."""
    kw = BlockwiseKwargs.from_any(blockwise_kwargs)
    axis = resolve_axis(axis_name)
    return R.RingAttentionRef.apply(q, k, v, attn_bias, segment_ids, cache_idx, axis.comm,
                                    float32_logits, kw)


def ringattention_inference(q, k, v, attn_mask=None, axis_name=None, float32_logits: bool = True, *, logit_cap=None,
                            alibi_slopes=None, query_pos=None):
    """Decoding attention over a sequence-sharded KV cache
    (ringattention/ringattention_inference.py:67-73).

    ``q (B, q_len, H, D)`` is replicated, ``k, v (B, kv_len, H, D)`` are this rank's cache shard and
    ``attn_mask`` is boolean (True = attend), broadcastable to ``(B, H, q_len, S_total)`` and global
    on its last axis. On CUDA bf16 the KV cache stays where it is: every rank computes a partial
    ``(o, lse)`` over its shard (the split-KV decode kernel for up to 8 query rows without gradients, the
    flash-attention kernel with the mask as a bitmap for longer queries or when gradients are needed) and
    the partials are merged through peer memory; all ranks return the same result as the reference's
    rotation. Differentiable w.r.t. q, k, v (ringattention_inference.py:38-64): ``dk``/``dv`` belong to the
    local shard, ``dq`` is the full gradient of the replicated queries on every rank.

    ``logit_cap`` and ``alibi_slopes`` shape the scores as in :func:`ringattention`'s ``blockwise_kwargs``. Key j of the whole cache sits
    at position j and query row i at ``query_pos + i``; ``query_pos`` is an int below 2^30 or a ``(B,)`` integer tensor of any values (a batch of
    caches that are filled up to places of their own), by default the one that ends the queries with the cache. A query beyond either end of the cache
    gets the weights of one at that end: its distances to all keys differ by one number. Masked rows of the cache may hold anything in
    calls of up to 8 query rows; in longer ones their values have to be finite (their weight is 0, and 0 times NaN is NaN).
    """
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return ringattention_inference(q, k, v, attn_mask, axis_name, float32_logits, logit_cap=logit_cap, alibi_slopes=alibi_slopes,
                                           query_pos=query_pos)
    axis = resolve_axis(axis_name)
    _check_qkv(q, k, v)
    if attn_mask is not None:
        attn_mask = _whole_mask(attn_mask, q, k.shape[1] * axis.size)
    shape = None
    if not (logit_cap is None and alibi_slopes is None and query_pos is None):
        from .ops.inference import inference_shape

        shape = inference_shape(q, k, axis.size, logit_cap, alibi_slopes, query_pos)
    if q.is_cuda and q.dtype == torch.bfloat16 and q.shape[-1] in (64, 128):
        from .ops import inference as Inf

        return Inf.ring_inference_attention(q, k, v, attn_mask, axis, _symm_ring_for(axis, q.device), shape=shape)
    _warn_fallback(q, _fallback_reason(q, None))
    return R.RingAttentionInferenceRef.apply(q, k, v, attn_mask, axis.comm, float32_logits, shape)


def _whole_mask(mask, q, S: int):
    """The mask of an inference call, checked, with all its ``S`` keys (their axis may be one that broadcasts)."""
    B, ql, H, _ = q.shape
    if mask.device != q.device or (mask.dtype != torch.bool and (mask.is_floating_point() or mask.is_complex())):
        raise ValueError("attn_mask must be a boolean tensor on the device of the queries")
    if not 1 <= mask.dim() <= 4:
        raise ValueError("attn_mask must broadcast to (B, H, q_len, S_total)")
    while mask.dim() < 4:
        mask = mask[None]
    b, h, m, n = mask.shape
    if (b != 1 and b != B) or (h != 1 and h != H) or (m != 1 and m != ql):
        raise ValueError("attn_mask must broadcast to (B, H, q_len, S_total)")
    if n >= S:
        return mask
    if n != 1:
        raise ValueError("attn_mask is too short along the keys: its last axis is global (all shards)")
    return mask.expand(b, h, m, S)


def _elsewhere(x: torch.Tensor) -> bool:
    """Whether ``x`` is on another CUDA device than the current one, whose stream launches go to."""
    return x.is_cuda and x.get_device() != torch._C._cuda_getDevice()


def qk_norm_rope(q, k, q_gain, k_gain, positions=None, *, theta: float = 10000.0, eps: float = 1e-6, q_out=None, k_out=None):
    """RMS norm of each head's queries and keys and their rotation by position, in one pass:
    ``R(position) (gain * x / sqrt(mean(x^2) + eps))`` over the last axis of ``q (B, S, H, D)`` and ``k (B, S, G, D)``. R turns the pairs
    ``(i, i + D/2)`` by ``position * theta^(-2i/D)``, with the angles made in 64 bits.

    ``q_gain, k_gain``  ``(D,)``, of one type (that of ``q``, or fp32).
    ``positions``  of the S tokens: a ``(S,)`` or ``(B, S)`` tensor of int32 or int64, the first one's (an int), a
    :class:`~ringattention_b200.ops.flash.Positions` map of a shard, or ``None`` for 0, 1, ...
    ``q_out, k_out``  views that receive the results instead of new tensors, without gradients (rows of a cache, or ``q`` and ``k``
    themselves; other overlaps are not allowed).

    Returns ``(q', k')`` in the type of ``q``; differentiable w.r.t. both and the gains. On CUDA bf16 and fp32 with head dims 64, 128 and 256 run on
    the sm_100a kernels (others are refused), on the CPU any type runs in PyTorch.
    """
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return qk_norm_rope(q, k, q_gain, k_gain, positions, theta=theta, eps=eps, q_out=q_out, k_out=k_out)
    from .ops import qknorm as N

    pos, theta, eps = N.check(q, k, q_gain, k_gain, positions, theta, eps)
    needs_grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_gain.requires_grad or k_gain.requires_grad)
    needs_grad = needs_grad or (q.is_cuda and _lib.has_tangent(q, k, q_gain, k_gain))  # (refused by autograd: the kernels have no forward mode)
    if q_out is not None or k_out is not None:
        if needs_grad:
            raise ValueError("q_out and k_out are for calls without gradients")
        N.check_outputs(q, k, q_out, k_out, (q_gain, k_gain, pos) if isinstance(pos, torch.Tensor) else (q_gain, k_gain))
    if not q.is_cuda:
        got = N.plain(q, k, q_gain, k_gain, pos, theta, eps)
        return tuple(x if y is None else y.copy_(x) for x, y in zip(got, (q_out, k_out)))
    q_gain, k_gain = q_gain.contiguous(), k_gain.contiguous()
    if needs_grad:
        return N.QkNormRope.apply(q, k, q_gain, k_gain, pos, theta, eps)
    got = N.norm_rope_fwd(N.as_ready(q), N.as_ready(k), q_gain, k_gain, pos, theta, eps, q_out, k_out)
    _lib.wrote(q_out, k_out)
    return got


def distillation_loss(logits, teacher_ids, teacher_logits, *, temperature: float = 1.0, reduction: str = "mean"):
    """Distillation from a teacher's top logits. ``logits (..., V)`` are the student's; ``teacher_ids`` (int32 or int64) and ``teacher_logits``
    ``(..., K)`` a few entries of the teacher's for each row. Ids outside ``[0, V)`` mark absent entries; entries of the same id add up.

    With ``p = softmax(teacher_logits / T)`` over a row's entries and ``q = softmax(logits / T)`` over the vocabulary a row's loss is
    ``T^2 sum p (log p - log q)``; a row without entries (padding) has none. ``reduction``: ``"mean"`` over the rows that have entries, ``"sum"``, or
    ``"none"`` for the ``(...)`` losses; fp32. Differentiable w.r.t. ``logits`` (bf16 or fp32 on CUDA, any type on the CPU). In 32 bits a loss is off
    by some T^2 2^-21 at most (of logits up to 2^29 T), and rows of fewer than 2 K logits above T = 4, whose p and q hardly differ, are taken in 64 bits.
    """
    if _elsewhere(logits):
        with torch.cuda.device(logits.device):
            return distillation_loss(logits, teacher_ids, teacher_logits, temperature=temperature, reduction=reduction)
    from .ops import distill as Ds

    T = Ds.check(logits, teacher_ids, teacher_logits, temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none'")
    if logits.numel() == 0:
        raise ValueError("there are no rows")
    if not logits.is_cuda:
        loss, some = Ds.plain_rows(logits, teacher_ids, teacher_logits, T)
        return loss if reduction == "none" else loss.sum() / (some.sum().clamp_min(1) if reduction == "mean" else 1)
    return Ds.DistillLoss.apply(logits, teacher_ids, teacher_logits, T, reduction)


@torch.no_grad()
def distillation_loss_and_grad(logits, teacher_ids, teacher_logits, *, temperature: float = 1.0, grad_scale: float = 1.0, out=None):
    """The ``(...)`` losses of :func:`distillation_loss` and ``grad_scale`` times the gradient of their sum, in one pass over the logits, for
    training loops with a backward of their own. ``out`` receives the gradient: a tensor like ``logits`` (which may be ``logits``) with a contiguous
    last axis. Returns ``(losses, gradient)``."""
    if _elsewhere(logits):
        with torch.cuda.device(logits.device):
            return distillation_loss_and_grad(logits, teacher_ids, teacher_logits, temperature=temperature, grad_scale=grad_scale, out=out)
    from .ops import distill as Ds

    T = Ds.check(logits, teacher_ids, teacher_logits, temperature)
    if logits.numel() == 0:
        raise ValueError("there are no rows")
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device):
        raise ValueError("out must have the shape, type and device of the logits")
    if not logits.is_cuda:
        with torch.enable_grad():
            x = logits.detach().requires_grad_()
            loss, _ = Ds.plain_rows(x, teacher_ids, teacher_logits, T)
            grad, = torch.autograd.grad(loss.sum(), x)
        grad = grad * grad_scale
        return loss.detach(), grad if out is None else out.copy_(grad)
    x = Ds._rows(logits)
    grad = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype) if out is None else out
    try:
        g2 = grad.view(-1, grad.shape[-1])
    except RuntimeError:
        raise ValueError("out must be a tensor whose rows lie an equal distance apart") from None
    if g2.stride(1) != 1 and g2.shape[1] > 1:
        raise ValueError("out must have a contiguous last axis")
    ids, teacher = Ds._rows(teacher_ids), Ds._rows(teacher_logits)
    if out is not None and not (_lib.writable(g2) and (_lib.same_place(g2, x) or _lib.apart(g2, x)) and _lib.apart(g2, ids) and _lib.apart(g2, teacher)):
        raise ValueError("out overlaps itself or another argument (it may be the logits, as they are)")
    loss = Ds.distill_rows(x, ids, teacher, T, grad=g2, grad_scale=float(grad_scale))
    _lib.wrote(out)
    return loss.view(logits.shape[:-1]), grad


def blockwise_feedforward(feedforward: Callable, inputs: torch.Tensor, chunk_size: int,
                          static_argnums: Sequence[int] = (1,), policy: Any = POLICY_NOTHING_SAVEABLE,
                          pre_remat: bool = True, *extra_args):
    """Apply a position-wise ``feedforward`` to ``inputs (B, S, D)`` in chunks of ``chunk_size``
    tokens (ringattention/ringattention_jax.py:333-352).

    Peak activation memory is that of one chunk. With ``pre_remat=False`` each chunk is wrapped in
    activation checkpointing when ``policy`` is ``nothing_saveable`` (the reference wraps with
    ``partitioning.remat``; the default ``pre_remat=True`` assumes the caller already did).
    ``static_argnums`` is accepted for signature compatibility. A
    :class:`~ringattention_b200.ops.ffn.FusedSwiGLU` module as ``feedforward`` runs its chunks on the sm_100a
    GEMM kernels (activation in the GEMM epilogue, per-chunk recomputation in the backward unless ``policy``
    with ``pre_remat=False`` says everything is saveable); any other callable is looped over in PyTorch.
    """
    if inputs.dim() != 3:
        raise ValueError("inputs must be (B, S, D)")
    B, S, D = inputs.shape
    if chunk_size <= 0 or S % chunk_size:
        raise ValueError(f"chunk_size {chunk_size} must divide the sequence length {S}")
    from .ops.ffn import FusedSwiGLU

    if isinstance(feedforward, FusedSwiGLU) and inputs.is_cuda and inputs.dtype == torch.bfloat16:
        # kernel-backed chunk loop with the policy's recomputation built in (a chunk holds chunk_size tokens
        # of every batch row, like one scan step of the reference)
        return feedforward.blockwise(inputs, chunk_size * B if B > 1 else chunk_size,
                                     policy if not pre_remat else POLICY_NOTHING_SAVEABLE)
    remat = (not pre_remat) and _policy_name(policy) == POLICY_NOTHING_SAVEABLE
    outs = []
    for s0 in range(0, S, chunk_size):
        chunk = inputs[:, s0:s0 + chunk_size]
        if remat and torch.is_grad_enabled():
            y = torch.utils.checkpoint.checkpoint(feedforward, chunk, *extra_args, use_reentrant=False)
        else:
            y = feedforward(chunk, *extra_args)
        outs.append(y)
    return torch.cat(outs, dim=1)
