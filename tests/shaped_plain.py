"""Shaped attention in 64 bits, written out from its definition, and how far a kernel that rounds to bf16 may be from it."""
import math

import torch

HALF = 2.0 ** -8     # largest relative error of a rounding to bf16
SLACK = 2.0 ** -18   # 32-bit scores, exponentials and sums


def slopes_for(H, device="cpu"):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=device)


def visible(q_pos, k_pos, B, cbs=0, prefix=None, seg_q=None, seg_k=None, bias=None, mask=None):
    """``(B, 1|H, Sq, Sk)``: who sees whom."""
    m = torch.ones(B, 1, q_pos.numel(), k_pos.numel(), dtype=torch.bool, device=q_pos.device)
    if cbs:
        m = m & (torch.div(k_pos, cbs, rounding_mode="floor")[None] <= torch.div(q_pos, cbs, rounding_mode="floor")[:, None])
        if prefix is not None:
            m = m | (k_pos[None, None, None] < torch.as_tensor(prefix, device=k_pos.device).expand(B)[:, None, None, None])
    if seg_q is not None:
        m = m & (seg_q[:, None, :, None] == seg_k[:, None, None, :])
    if bias is not None:
        m = m & (bias > -1e30)
    return m if mask is None else m & mask


def attention(q, k, v, cap=0.0, slopes=None, dist=None, bias=None, seen=None, dout=None):
    """``q (B, Sq, H, D)``, ``dist (B|1, 1, Sq, Sk)``. Returns ``out`` and its bound, with ``dout`` also ``[dq, dk, dv]`` and theirs."""
    q, k, v = (x.detach().double().transpose(1, 2) for x in (q, k, v))
    scale = 1.0 / math.sqrt(q.shape[3])
    x = q @ k.transpose(2, 3) * scale
    steep = torch.ones_like(x)
    if cap:
        steep = 1 - torch.tanh(x / cap) ** 2
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias.double()
    if slopes is not None:
        x = x - slopes.double()[None, :, None, None] * dist.double().abs()
    big = x.abs().masked_fill(~seen, 0).amax(3, keepdim=True)
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(m.isfinite(), m, 0.0))
    p = p / p.sum(3, keepdim=True).clamp_min(1e-300)
    out = p @ v
    rel = HALF + SLACK * (1 + big)  # of a weight, and of a sum with them
    weight = (p * rel) @ v.abs()
    back = lambda t: t.transpose(1, 2)
    tiny = 1e-6
    if dout is None:
        return back(out), back(weight + HALF * out.abs() + tiny)
    g = dout.detach().double().transpose(1, 2)
    dv, ddv = p.transpose(2, 3) @ g, (p * rel).transpose(2, 3) @ g.abs()
    dp = g @ v.transpose(2, 3)
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * steep * (dp - delta) * scale
    # delta comes out of the rounded product of the weights with v; dp of 32-bit sums
    off = (g.abs() * (weight + 2.0 ** -16 * out.abs())).sum(3, keepdim=True) + SLACK * (g.abs() @ v.abs().transpose(2, 3))
    dds = ds.abs() * 2 * rel + p * steep * off * scale
    dq, ddq = ds @ k, dds @ k.abs()
    dk, ddk = ds.transpose(2, 3) @ q, dds.transpose(2, 3) @ q.abs()
    return (back(out), back(weight + HALF * out.abs() + tiny), [back(x) for x in (dq, dk, dv)],
            [back(e + HALF * x.abs() + tiny) for x, e in ((dq, ddq), (dk, ddk), (dv, ddv))])


def check(got, want, bound, what=""):
    off = (got.detach().double() - want).abs()
    assert got.detach().isfinite().all(), what
    worst = (off / bound).max()
    assert worst <= 1, f"{what}: {float(worst):.2f} of the bound"
