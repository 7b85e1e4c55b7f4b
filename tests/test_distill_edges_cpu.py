"""Distillation at its edges on the CPU."""
import pytest
import torch

import ringattention_b200 as rab


@pytest.mark.parametrize("T", [5.0, 300.0, 1e4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_high_temperatures_with_entries_for_much_of_the_vocabulary(T, dtype):
    """p and q hardly differ: in 32 bits the loss, of the order of the logits' variance at any T, would be off by T^2 2^-22. What is left here is the
    rounding of the result to 32 bits and of the gradient to its type, and 2^-47 of what cancels."""
    g = torch.Generator().manual_seed(0)
    rows, V = 6, 40
    x, t = ((torch.randn(rows, V, generator=g, dtype=torch.float64) * 2.5).to(dtype) for _ in range(2))
    ids = torch.stack([torch.randperm(V, generator=g) for _ in range(rows)])
    log_q, log_p = torch.log_softmax(x.double() / T, -1), torch.log_softmax(t.double() / T, -1)
    p = log_p.exp()
    want = T * T * (p * (log_p - log_q.gather(-1, ids))).sum(-1)
    grad = T * (log_q.exp() - torch.zeros(rows, V, dtype=torch.float64).scatter_add_(-1, ids, p))
    loss, got = rab.distillation_loss_and_grad(x, ids, t, temperature=T)
    assert loss.dtype == torch.float32 and got.dtype == dtype
    assert bool(((loss.double() - want).abs() <= want * 2.0 ** -23 + T * T * 2.0 ** -45).all())
    assert bool(((got.double() - grad).abs() <= grad.abs() * torch.finfo(dtype).eps + T * 2.0 ** -45).all())


def test_a_view_in_the_same_place():
    from ringattention_b200.ops import _lib

    x = torch.zeros(3, 20)[:, 4:14]
    assert _lib.same_place(x, x) and _lib.same_place(x[:1], x[:1].view(-1, 10)) and _lib.same_place(x[1, 2:3], x[1:2, 2])
    assert not _lib.same_place(x[:2], x[1:]) and not _lib.same_place(x[:, :5], x[:, ::2]) and not _lib.same_place(x[:1], x[0])
