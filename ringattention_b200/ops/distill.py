"""Distillation from a teacher's top logits on ``distill.cu``: the loss with its backward pass, and both at once.

With ``p`` the softmax of a row's teacher logits over the entries it has, and ``q`` the softmax of the student's logits over the vocabulary, both at a
temperature T, a row's loss is ``T^2 sum p (log p - log q)`` and the gradient of its logits ``T (q - p)``.
"""
from __future__ import annotations

import math
import struct

import torch

from . import _lib
from ._lib import address, stream_handle
from .reference import once_differentiable

# ``RaDistillArgs`` (distill.cu): logits ld, grad ldg, ids ld_ids, teacher ld_t, f32 ids64 teacher_f32, rows, V K, temperature grad_scale, loss,
# stats, dloss dloss_s per_row, stream
_ARGS = struct.Struct("@PqPqPqPq3iq2i2fPPPiPP")

MAX_ENTRIES = 1024  # of a teacher's row
WIDE_FROM = 4.0     # temperature from which on rows of fewer logits than twice the entries are taken in 64 bits (see distill.cu)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``(..., n)`` as ``(rows, n)`` with a contiguous last dim."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return t2 if t2.stride(1) == 1 or t2.shape[1] == 1 else t2.contiguous()


def check(logits, teacher_ids, teacher_logits, temperature) -> float:
    if logits.dim() < 1 or teacher_ids.shape != teacher_logits.shape or teacher_ids.dim() < 1 or teacher_ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError("logits (..., V), teacher_ids and teacher_logits (..., K) must agree in their leading dimensions")
    if logits.shape[-1] < 1 or not 1 <= teacher_ids.shape[-1] <= MAX_ENTRIES:
        raise ValueError(f"a row has at least one logit and 1 to {MAX_ENTRIES} teacher entries")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_ids must be int32 or int64")
    if not logits.is_floating_point() or not teacher_logits.is_floating_point():
        raise ValueError("logits must be floating-point numbers")
    if not (logits.device == teacher_ids.device == teacher_logits.device):
        raise ValueError("logits, teacher_ids and teacher_logits must be on one device")
    if teacher_logits.requires_grad:
        raise ValueError("there is no gradient for the teacher's logits: detach them")
    if isinstance(temperature, bool) or not isinstance(temperature, (int, float)) or not 0.0 < temperature < math.inf:
        raise ValueError("temperature must be a positive number")
    if logits.is_cuda:
        if logits.dtype not in (torch.bfloat16, torch.float32) or teacher_logits.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("the kernels take logits in bf16 or fp32")
        if not 1e-6 <= temperature <= 1e6:
            raise ValueError("the kernels take temperatures from 1e-6 to 1e6")
    return float(temperature)


def _pack(x, grad, ids, teacher, T, grad_scale, loss, stats, dloss=0, dloss_s=0, per_row=0) -> bytes:
    return _ARGS.pack(x.data_ptr(), x.stride(0), address(grad), 0 if grad is None else grad.stride(0), ids.data_ptr(), ids.stride(0), teacher.data_ptr(),
                      teacher.stride(0), int(x.dtype == torch.float32), int(ids.dtype == torch.int64), int(teacher.dtype == torch.float32), x.shape[0],
                      x.shape[1], ids.shape[1], T, grad_scale, address(loss), address(stats), dloss, dloss_s, per_row, stream_handle())


def distill_rows(x, ids, teacher, T: float, *, stats=None, grad=None, grad_scale: float = 1.0, loss=None):
    """Losses (fp32) of the rows of ``x (rows, V)``; ``grad`` (its type and shape, ``x`` itself allowed) receives their gradient times
    ``grad_scale``, ``stats (rows, 2)`` what :func:`distill_rows_bwd` needs."""
    if loss is None:
        loss = torch.empty(x.shape[0], device=x.device, dtype=torch.float32)
    assert x.stride(1) == 1 or x.shape[1] == 1
    assert grad is None or (grad.shape == x.shape and grad.dtype == x.dtype and (grad.stride(1) == 1 or x.shape[1] == 1))
    _lib.call("ra_distill", _pack(x, grad, ids, teacher, T, grad_scale, loss, stats))
    return loss


def distill_rows_bwd(x, ids, teacher, T: float, stats, dloss, per_row=None):
    """Gradient of ``x`` for ``dloss`` (fp32, ``(rows,)`` or one number on the device), times the number ``per_row`` points at."""
    grad = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    _lib.call("ra_distill_bwd", _pack(x, grad, ids, teacher, T, 1.0, None, stats, dloss.data_ptr(), 0 if dloss.dim() == 0 else dloss.stride(0),
                                      address(per_row)))
    return grad


class DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, T, reduction):
        x, i2, t2 = _rows(logits), _rows(ids), _rows(teacher)
        stats = torch.empty(x.shape[0], 2, device=x.device, dtype=torch.float32)
        loss = distill_rows(x, i2, t2, T, stats=stats)
        total = per_row = None
        if reduction != "none":
            total, per_row = torch.empty((), device=x.device, dtype=torch.float32), torch.empty((), device=x.device, dtype=torch.float32)
            _lib.call("ra_distill_reduce", loss.data_ptr(), stats.data_ptr(), x.shape[0], int(reduction == "mean"), total.data_ptr(), per_row.data_ptr(),
                      stream_handle())
        ctx.save_for_backward(logits, ids, teacher, stats, per_row)
        ctx.T = T
        return loss.view(logits.shape[:-1]) if total is None else total

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        logits, ids, teacher, stats, per_row = ctx.saved_tensors
        d = dloss.reshape(-1) if per_row is None else dloss
        grad = distill_rows_bwd(_rows(logits), _rows(ids), _rows(teacher), ctx.T, stats, d, per_row)
        return grad if logits.dim() == 2 else grad.view(logits.shape), None, None, None, None


def plain_rows(logits, ids, teacher, T: float):
    """The losses in plain PyTorch (any device and type; 32 bits at least), and which rows have entries."""
    V = logits.shape[-1]
    kept = torch.promote_types(logits.dtype, torch.float32)
    acc = torch.float64 if V < 2 * ids.shape[-1] and T > WIDE_FROM else kept
    there = (ids >= 0) & (ids < V)
    u = torch.where(there, teacher.detach().to(acc) / T, -math.inf)
    some = u.amax(-1) != -math.inf  # (NaN too)
    log_p = torch.log_softmax(torch.where(some[..., None], u, 0.0), -1)
    p = torch.where(there & some[..., None], log_p.exp(), 0.0)
    x = torch.where(some[..., None], logits.to(acc), 0.0)
    log_q = torch.log_softmax(x / T, -1).gather(-1, ids.long().clamp(0, V - 1))
    part = torch.where(p == 0, 0.0, p * (log_p - torch.where(p == 0, 0.0, log_q)))
    return torch.where(some, T * T * part.sum(-1), 0.0).to(kept), some
