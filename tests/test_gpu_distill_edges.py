"""Distillation at its edges on the kernels: temperatures far from 1."""
import pytest
import torch
from test_gpu_distill import _inputs

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plain(logits, ids, teacher, T):
    """Losses and gradients of their sum in 64 bits, the terms they are sums of, and the row's largest exponent (from the row's largest logit on)."""
    V = logits.shape[-1]
    x, t, ids = logits.detach().double(), teacher.detach().double(), ids.long()
    used = (ids >= 0) & (ids < V)
    some = used.any(-1)
    u = torch.where(used, (t - t.masked_fill(~used, -torch.inf).amax(-1, keepdim=True).clamp_min(-1e300)) / T, -torch.inf)
    log_p = torch.log_softmax(torch.where(some[:, None], u, 0.0), -1)
    p = torch.where(used, log_p.exp(), 0.0)
    log_q = torch.log_softmax((x - x.amax(-1, keepdim=True)) / T, -1)
    at = log_q.gather(-1, ids.clamp(0, V - 1))
    loss = T * T * torch.where(p > 0, p * (log_p - at), 0.0).sum(-1)
    target = torch.zeros_like(x).scatter_add_(-1, ids.clamp(0, V - 1), p)
    size = T * T * torch.where(p > 0, p * (log_p.abs() + at.abs()), 0.0).sum(-1)
    grad = T * (log_q.exp() - target)
    reach = 1 + torch.where(log_q > -120, -log_q, 0.0).amax(-1) + torch.where(log_p > -120, -log_p, 0.0).amax(-1)
    zero = lambda v: torch.where(some.reshape(-1, *[1] * (v.dim() - 1)), v, 0.0)
    return zero(loss), zero(grad), zero(size), zero(T * (log_q.exp() + target)), zero(reach)


def _within(got, want, bound, what):
    off = (got.detach().double() - want).abs()
    assert got.detach().isfinite().all(), what
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.2f} of the bound"


@pytest.mark.parametrize("T", [1e-6, 1e-4, 1e-2, 0.3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,K", [(7, 3), (1003, 40), (9001, 300)])
def test_low_temperatures(T, dtype, V, K):
    """Logits that lie as close as the temperature is low, some way from 0, in rows whose ends are cut from 16 bytes: what an exponent is off by must be
    relative to the distance of two logits, not to a logit over T."""
    rows = 9
    x, ids, t = _inputs(rows, V + 1, K, torch.float32, torch.float32, seed=V)
    x, t = (19.3 + x * T).to(dtype)[:, 1:], (17.7 + t * T).to(dtype)
    ids[ids == V] = 0
    loss, grad, size, gsize, reach = _plain(x, ids, t, T)
    # 32 bits: 2^-22 of each exponent and of each exponential, sums of them; T itself is rounded to 2^-24
    rel = 2.0 ** -20
    half = torch.finfo(dtype).eps / 2
    got = rab.distillation_loss_and_grad(x, ids, t, temperature=T)
    _within(got[0], loss, (size + T * T * reach) * rel + 1e-30, "loss")
    bound = grad.abs() * half + gsize * reach[:, None] * rel + 1e-30 + (torch.finfo(dtype).tiny if dtype == torch.bfloat16 else 0)
    _within(got[1], grad, bound, "gradient at once")
    leaf = x.detach().requires_grad_()
    each = rab.distillation_loss(leaf, ids, t, temperature=T, reduction="none")
    assert torch.equal(each.detach(), got[0])
    _within(torch.autograd.grad(each.sum(), leaf)[0], grad, bound, "gradient")
