"""Distillation at its edges on the kernels: temperatures far from 1."""
import json
import os
import subprocess
import sys

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


@pytest.mark.parametrize("T", [5.0, 100.0, 1000.0, 1e4, 1e6])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,K,rows", [(1, 1, 3), (7, 7, 5), (300, 256, 40), (1024, 1024, 3), (2047, 1024, 9), (999, 500, 20)])
def test_high_temperatures_with_entries_for_much_of_the_vocabulary(T, dtype, V, K, rows):
    """p and q are then nearly the same, and the loss, T^2 times the sum of what hardly differs, is of the order of the logits' variance whatever T is."""
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    x, _, t = _inputs(rows, V, K, dtype, dtype, seed=V)
    ids = torch.stack([torch.randperm(V, device=DEV, generator=g)[:K] for _ in range(rows)])
    if rows > 3:
        ids[1, K // 2:] = -1
        ids[2] = V
        x[2, 0] = float("nan")
        ids[3, :K // 3] = ids[3, -1]
    where = x.nan_to_num(nan=0.0)  # (the row without entries holds a NaN)
    loss, grad, size, gsize, reach = _plain(where, ids, t, T)
    # 64 bits in both, where T^2 (and T) multiply what cancels, rounded to fp32 and to the gradient's type
    slack = 2.0 ** -47
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny if dtype == torch.bfloat16 else 0
    bound = lambda scale: grad.abs() * scale * (half + 2.0 ** -22) + gsize * scale * slack + 1e-30 + tiny
    got = rab.distillation_loss_and_grad(x, ids, t, temperature=T, grad_scale=0.25)
    _within(got[0], loss, loss.abs() * 2.0 ** -22 + (size + T * T * reach) * slack + 1e-30, "loss")
    _within(got[1], grad * 0.25, bound(0.25), "gradient at once")
    over = x.clone()
    same = rab.distillation_loss_and_grad(over, ids.int(), t, temperature=T, grad_scale=0.25, out=over)
    assert torch.equal(same[0], got[0]) and torch.equal(over, got[1])
    leaf = x.detach().requires_grad_()
    each = rab.distillation_loss(leaf, ids, t, temperature=T, reduction="none")
    assert torch.equal(each.detach(), got[0])
    d = torch.rand(rows, device=DEV) + 0.5
    _within(torch.autograd.grad(each, leaf, d)[0], grad * d.double()[:, None], bound(d.double()[:, None]), "gradient")
    one = rab.distillation_loss(leaf, ids, t, temperature=T)
    n = rows - (rows > 3)
    assert abs(float(one.detach()) - float(got[0].double().sum() / n)) <= 2.0 ** -22 * float(got[0].double().abs().sum() / n)
    _within(torch.autograd.grad(one, leaf)[0], grad / n, bound(1 / n), "gradient of the mean")


@pytest.mark.parametrize("T", [5.0, 1000.0, 1e6])
def test_high_temperatures_with_few_entries(T):
    x, ids, t = _inputs(20, 2048, 1024, torch.float32, torch.float32)
    loss, grad, size, gsize, reach = _plain(x, ids, t, T)
    got = rab.distillation_loss_and_grad(x, ids, t, temperature=T)
    _within(got[0], loss, (size + T * T) * 2.0 ** -20, "loss")
    _within(got[1], grad, grad.abs() * 2.0 ** -24 + gsize * 2.0 ** -20, "gradient")


def test_nan_and_infinities_at_a_high_temperature():
    x, ids, t = _inputs(6, 100, 80, torch.float32, torch.float32)
    ids[:, 0] = 3
    x[1, 77] = float("nan")
    x[2, 3] = float("-inf")
    t[3, 0] = float("-inf")
    t[4] = float("-inf")
    ids[5] = 100
    x[5] = float("inf")
    loss, grad = rab.distillation_loss_and_grad(x, ids, t, temperature=50.0)
    assert bool(loss[1].isnan()) and bool(grad[1].isnan().all())
    assert float(loss[2]) == float("inf") and bool(grad[2].isfinite().all())
    assert bool(loss[[0, 3]].isfinite().all()) and bool(grad[[0, 3]].isfinite().all())
    assert bool((loss[4:] == 0).all()) and bool((grad[4:] == 0).all())


def test_a_captured_step_at_a_high_temperature():
    x, ids, t = _inputs(30, 500, 400)

    def step():
        leaf = x.detach().requires_grad_()
        loss = rab.distillation_loss(leaf, ids, t, temperature=20.0)
        return loss, torch.autograd.grad(loss, leaf)[0], *rab.distillation_loss_and_grad(x, ids, t, temperature=20.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        for dst, src in zip((x, ids, t), _inputs(30, 500, 400, seed=seed)):
            dst.copy_(src)
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("checked", [True, False])
def test_no_access_out_of_range_and_canaries_survive(checked):
    """In the checked build of the library and in the plain one, in a child process."""
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "edges_bounds_worker.py")
    p = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=900,
                       env=dict(os.environ, RINGATTN_B200_BOUNDS_CHECK="1" if checked else "0"))
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-3000:]
    rep = json.loads([ln for ln in p.stdout.splitlines() if ln.startswith("BOUNDS ")][-1][len("BOUNDS "):])
    assert rep["clean"]["checked"] is checked and rep["clean"]["violations"] == 0, rep["clean"]
    assert rep["canaries_intact"] is True


@pytest.mark.parametrize("rows,V", [(1, 40), (1, 1), (5, 1), (5, 40)])
def test_the_gradient_over_logits_that_are_part_of_wider_rows(rows, V):
    wide = torch.randn(rows, 60, device=DEV)
    x, ids, t = wide[:, 3:3 + V], torch.zeros(rows, 2, device=DEV, dtype=torch.int32), torch.randn(rows, 2, device=DEV)
    want, kept = rab.distillation_loss_and_grad(x, ids, t), wide.clone()
    got = rab.distillation_loss_and_grad(x, ids, t, out=x)
    assert torch.equal(got[0], want[0]) and torch.equal(x, want[1])
    assert torch.equal(wide[:, :3], kept[:, :3]) and torch.equal(wide[:, 3 + V:], kept[:, 3 + V:])
    by_batch = wide[:, None, 3:3 + V]
    assert rab.distillation_loss_and_grad(by_batch, ids[:, None], t[:, None], out=by_batch)[1] is by_batch
