"""RMS norm of each head's queries and keys with their rotation by position, on ``qk_norm_rope.cu``.

``y = R(pos) (gain * x / sqrt(mean(x^2) + eps))`` for every row of ``D`` values; R turns the pairs ``(i, i + D/2)`` by ``pos * theta^(-2i/D)``, as
:func:`ringattention_b200.ops.kernels.rope_` does. The gains' gradients are sums over all rows.
"""
from __future__ import annotations

import math
import struct

import torch

from . import _lib
from ._lib import address, stream_handle
from .flash import Positions
from .reference import once_differentiable

_SIDE = "P3qP3qP3qPi0P"
# ``RaQkNormArgs`` (qk_norm_rope.cu): queries and keys (x, dy, y with strides, gain, heads), B S D, f32 gain_f32, pos pos64 and its strides,
# off0 off1 half, eps, theta, part parts, dgain, stream
_ARGS = struct.Struct("@" + _SIDE + _SIDE + "5iPi2q3ifdPiPP")


def ready(t: torch.Tensor) -> bool:
    """Whether the kernels take a ``(B, S, H, D)`` view as it is: contiguous ``D``, strides and base of whole 16 bytes."""
    sb, ss, sh, sd = t.stride()
    n = 16 // t.element_size()
    return sd == 1 and not (sb % n or ss % n or sh % n) and not t.data_ptr() & 15


def _side(x, dy, y, gain) -> tuple:
    d = (0, 0, 0, 0) if dy is None else (dy.data_ptr(), *dy.stride()[:3])
    return (x.data_ptr(), *x.stride()[:3], *d, y.data_ptr(), *y.stride()[:3], gain.data_ptr(), x.shape[2])


def _call(name, q, k, dq, dk, yq, yk, gq, gk, pos, theta, eps, part=None, parts=0, dgain=None, n_kernels=1) -> None:
    B, S, _, D = q.shape
    if isinstance(pos, torch.Tensor):
        at = (pos.data_ptr(), int(pos.dtype == torch.int64), pos.stride(0) if pos.shape[0] > 1 else 0, pos.stride(1), 0, 0, 0)
    else:
        at = (0, 0, 0, 0, pos.off0, pos.off1, min(pos.half, 1 << 30))
    _lib.call(name, _ARGS.pack(*_side(q, dq, yq, gq), *_side(k, dk, yk, gk), B, S, D, int(q.dtype == torch.float32), int(gq.dtype == torch.float32), *at,
                               eps, theta, address(part), parts, address(dgain), stream_handle()), n_kernels=n_kernels)


def norm_rope_fwd(q, k, gq, gk, pos, theta: float, eps: float, yq=None, yk=None):
    """``q (B, S, H, D)``, ``k (B, S, G, D)`` (:func:`ready` views of one type), gains ``(D,)`` of one type, ``pos`` a ``(1|B, S)`` integer tensor or a
    :class:`~ringattention_b200.ops.flash.Positions` map. Returns the results, or fills ``yq`` and ``yk`` (which may be ``q`` and ``k``)."""
    yq = torch.empty(q.shape, device=q.device, dtype=q.dtype) if yq is None else yq
    yk = torch.empty(k.shape, device=k.device, dtype=k.dtype) if yk is None else yk
    _call("ra_qk_norm_rope", q, k, None, None, yq, yk, gq, gk, pos, theta, eps)
    return yq, yk


def norm_rope_bwd(q, k, gq, gk, dyq, dyk, pos, theta: float, eps: float):
    """Returns ``(dq, dk, dgq, dgk)``, contiguous, in the types of what they are gradients of."""
    D = q.shape[3]
    dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    dk = torch.empty(k.shape, device=k.device, dtype=k.dtype)
    parts = _lib.lib().ra_qk_norm_parts()
    part = torch.empty(parts, D, device=q.device, dtype=torch.float32)
    dgain = torch.empty(2, D, device=q.device, dtype=gq.dtype)
    _call("ra_qk_norm_rope_bwd", q, k, dyq, dyk, dq, dk, gq, gk, pos, theta, eps, part, parts, dgain, n_kernels=2)
    return dq, dk, dgain[0], dgain[1]


def as_ready(t):
    return t if ready(t) else t.contiguous() if not t.is_contiguous() else t.clone()


class QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, gq, gk, pos, theta, eps):
        qq, kk = as_ready(q), as_ready(k)
        yq, yk = norm_rope_fwd(qq, kk, gq, gk, pos, theta, eps)
        ctx.save_for_backward(qq, kk, gq, gk, pos if isinstance(pos, torch.Tensor) else None)
        ctx.pos, ctx.theta, ctx.eps = None if isinstance(pos, torch.Tensor) else pos, theta, eps
        return yq, yk

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, gq, gk, pos = ctx.saved_tensors
        grads = norm_rope_bwd(q, k, gq, gk, as_ready(dyq), as_ready(dyk), pos if ctx.pos is None else ctx.pos, ctx.theta, ctx.eps)
        return (*grads, None, None, None)


def _plain_one(x, gain, pos, theta: float, eps: float):
    acc = torch.promote_types(x.dtype, torch.float32)
    D = x.shape[-1]
    y = x.to(acc)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * gain.to(acc)
    angle = pos.to(torch.float64)[:, :, None, None] * theta ** (-2.0 * torch.arange(D // 2, device=x.device, dtype=torch.float64) / D)
    cos, sin = angle.cos().to(acc), angle.sin().to(acc)
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def plain(q, k, gq, gk, pos, theta: float, eps: float):
    """The same in plain PyTorch (any device and type; 32 bits at least)."""
    if not isinstance(pos, torch.Tensor):
        pos = pos.tensor(q.shape[1], q.device)[None]
    return _plain_one(q, gq, pos, theta, eps), _plain_one(k, gk, pos, theta, eps)


def check_outputs(q, k, yq, yk, read=()) -> None:
    """Refuses given outputs that are not like their inputs, or share memory with what the launch still reads, with one another or with themselves."""
    for name, y, x, other, other_y in (("q_out", yq, q, k, yk), ("k_out", yk, k, q, yq)):
        if y is None:
            continue
        if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device or (y.is_cuda and not ready(y)):
            raise ValueError(f"{name} must have its input's shape, type and device, and rows that start on 16 bytes")
        if not _lib.writable(y) or not (_lib.same_place(y, x) or _lib.apart(y, x)) or not _lib.apart(y, other) or (
                other_y is not None and not _lib.apart(y, other_y)):
            raise ValueError(f"{name} overlaps itself or another argument (it may be its input, as it is)")
        if any(_lib.meet(y, t) for t in read):  # (gains, positions)
            raise ValueError(f"{name} overlaps the gains or the positions")


def check(q, k, q_gain, k_gain, positions, theta, eps):
    """Checks the arguments of :func:`ringattention_b200.qk_norm_rope`; returns the positions as the functions above take them, theta and eps."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.shape[3] % 2 or 0 in q.shape or 0 in k.shape:
        raise ValueError("q must be (B, S, H, D) and k (B, S, G, D) with an even D")
    B, S, _, D = q.shape
    if q.dtype != k.dtype or not q.is_floating_point():
        raise ValueError("q and k must be of one floating-point type")
    if q_gain.shape != (D,) or k_gain.shape != (D,) or q_gain.dtype != k_gain.dtype or not q_gain.is_floating_point():
        raise ValueError(f"the gains must be ({D},) floating-point numbers of one type")
    if not (q.device == k.device == q_gain.device == k_gain.device):
        raise ValueError("queries, keys and gains must be on one device")
    if isinstance(theta, bool) or not isinstance(theta, (int, float)) or not 0.0 < theta < math.inf:
        raise ValueError("theta must be a positive number")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0.0 <= eps < math.inf:
        raise ValueError("eps must be a non-negative number")
    if positions is None:
        positions = 0
    if isinstance(positions, int) and not isinstance(positions, bool):
        if not 0 <= positions <= 2**31 - 1 - S:
            raise ValueError("positions must be in [0, 2^31)")
        positions = Positions(positions)
    elif isinstance(positions, torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((S,), (1, S), (B, S)):
            raise ValueError(f"positions must be a ({S},) or ({B}, {S}) tensor of int32 or int64")
        if positions.device != q.device:
            raise ValueError("positions must be on the device of the queries")
        positions = positions.reshape(-1, S)
    elif isinstance(positions, Positions):  # the kernels count in 32 bits
        runs = ((positions.off0, min(S, positions.half)), (positions.off1, S - positions.half))
        if positions.half < 0 or any(not -(2**31) <= off <= 2**31 - max(n, 1) for off, n in runs):
            raise ValueError("a Positions map must stay in [-2^31, 2^31)")
    else:
        raise ValueError("positions must be an int, an integer tensor or a Positions map")
    if q.is_cuda:
        if q.dtype not in (torch.bfloat16, torch.float32) or q_gain.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("the kernels take bf16 or fp32")
        if D not in (64, 128, 256):
            raise ValueError("the kernels take head dims 64, 128 and 256")
    return positions, float(theta), float(eps)
