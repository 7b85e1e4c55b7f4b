"""Distillation from a teacher's top logits on the kernels against 64 bits: sizes, alignments, absent and repeated entries, extreme logits."""
import pytest
import torch

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plain(logits, ids, teacher, T):
    """Losses, gradients of their sum in 64 bits, and what their errors are relative to."""
    V = logits.shape[-1]
    x, t, ids = logits.detach().double(), teacher.detach().double(), ids.long()
    used = (ids >= 0) & (ids < V)
    u = torch.where(used, t / T, -torch.inf)
    some = u.amax(-1) > -torch.inf
    p = torch.where(used & some[:, None], torch.softmax(torch.where(some[:, None], u, 0.0), -1), 0.0)
    log_q = torch.log_softmax(x / T, -1)
    at = log_q.gather(-1, ids.clamp(0, V - 1))
    loss = torch.where(some, T * T * torch.where(p > 0, p * (p.log() - at), 0.0).sum(-1), 0.0)
    target = torch.zeros_like(x).scatter_add_(-1, ids.clamp(0, V - 1), p)
    grad = torch.where(some[:, None], T * (log_q.exp() - target), 0.0)
    # 32-bit exponents: a relative error of 2^-22 for each unit of the exponent (fp32 products and the exponential's own 2^-22). A logit
    # 120 below the largest counts nothing in that: its weight is below 2^-149 and 0 in 32 bits, off by no more than the 1e-30 that every bound
    # has; so a logit of -inf or of the type's lowest value does not make the bound of its row infinite.
    reach = 1 + torch.where(log_q > -120, (x / T).abs(), 0.0).amax(-1) * 1.45
    loss_size = torch.where(some, T * T * (torch.where(p > 0, p * (p.log().abs() + at.abs()), 0.0).sum(-1) + reach), 0.0)
    return loss, grad, loss_size, torch.where(some[:, None], T * (log_q.exp() + target) * reach[:, None], 0.0), some


def _check(got, want, size, what, scale=1.0):
    half = torch.finfo(got.dtype).eps / 2
    off = (got.detach().double() - want).abs()
    bound = want.abs() * half + size * 2.0 ** -20 + 1e-30 + (torch.finfo(torch.bfloat16).tiny if got.dtype == torch.bfloat16 else 0)
    assert got.detach().isfinite().all(), what
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.2f} of the bound"


def _inputs(rows, V, K, dtype=torch.bfloat16, tdtype=torch.bfloat16, seed=0, std=2.5):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    logits = (torch.randn(rows, V, device=DEV, generator=g) * std).to(dtype)
    ids = torch.randint(0, V, (rows, K), device=DEV, generator=g, dtype=torch.int32)
    ids[torch.rand(rows, K, device=DEV, generator=g) < 0.2] = -1
    teacher = (torch.randn(rows, K, device=DEV, generator=g) * std + 3).to(tdtype)
    return logits, ids, teacher


def _run(logits, ids, teacher, T=1.0):
    rows = logits.shape[0]
    loss, grad, ls, gs, some = _plain(logits, ids, teacher, T)
    # both at once, with a scale, into a new tensor and over the logits
    got = rab.distillation_loss_and_grad(logits, ids, teacher, temperature=T, grad_scale=0.25)
    _check(got[0], loss, ls, "losses")
    _check(got[1], grad * 0.25, gs * 0.25, "gradient at once")
    over = logits.detach().clone(memory_format=torch.contiguous_format)
    same = rab.distillation_loss_and_grad(over, ids, teacher, temperature=T, grad_scale=0.25, out=over)
    assert same[1] is over
    if logits.is_contiguous():
        assert torch.equal(same[0], got[0]) and torch.equal(over, got[1])
    else:  # rows that start elsewhere within 16 bytes are cut elsewhere: sums of another order, so no equal bits
        _check(same[0], loss, ls, "losses of a copy")
        _check(over, grad * 0.25, gs * 0.25, "gradient of a copy")
    # the loss and its backward
    x = logits.detach().requires_grad_()
    d = torch.rand(rows, device=DEV) + 0.5
    each = rab.distillation_loss(x, ids, teacher, temperature=T, reduction="none")
    assert torch.equal(each.detach(), got[0])
    g, = torch.autograd.grad(each, x, d)
    _check(g, grad * d.double()[:, None], gs * d.double()[:, None], "gradient")
    n = max(1, int(some.sum()))
    for reduction, per in (("mean", 1.0 / n), ("sum", 1.0)):
        one = rab.distillation_loss(x, ids, teacher, temperature=T, reduction=reduction)
        assert abs(float(one.detach()) - float(loss.sum() * per)) <= float((ls * 2.0 ** -20).sum() * per + loss.sum().abs() * per * 2.0 ** -20) + 1e-30
        g, = torch.autograd.grad(one * 2, x)
        _check(g, grad * (2 * per), gs * (2 * per), reduction)
    assert bool((got[1].reshape(rows, -1)[~some] == 0).all()) and bool((got[0][~some] == 0).all())


@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (3, 7, 2), (5, 300, 40), (64, 1000, 3), (17, 4097, 64), (2, 32000, 100), (9, 40001, 5), (2, 150000, 256), (1, 270000, 33)])
@pytest.mark.parametrize("dtype,tdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
def test_against_64_bits(rows, V, K, dtype, tdtype):
    """Every number of shares of a row, rows that are held and rows that are read again, rows that start anywhere in 16 bytes."""
    _run(*_inputs(rows, V, K, dtype, tdtype, seed=V))


@pytest.mark.parametrize("rows,V,K,dtype", [(3, 34, 2, torch.bfloat16), (500, 1000, 20, torch.bfloat16), (161, 4098, 64, torch.float32), (310, 32000, 64, torch.bfloat16),
                                            (300, 32766, 3, torch.bfloat16), (170, 50002, 300, torch.bfloat16), (90, 70001, 10, torch.float32),
                                            (40, 131072, 1024, torch.bfloat16), (21, 200002, 40, torch.bfloat16), (20, 262144, 7, torch.bfloat16)])
def test_rows_of_every_length(rows, V, K, dtype):
    """Few and many pieces a thread, one and more rounds of them, in place and not, with rows that have no entries, one id many times, or half of
    the vocabulary at -inf."""
    from ringattention_b200.ops import distill as Ds

    x, ids, t = _inputs(rows, V, K, dtype, dtype, seed=V)
    ids[rows // 2] = -1
    ids[1] = ids[1, 0]
    x[rows - 1, : V // 2] = float("-inf")
    ids[rows - 1] = V - 1
    loss, grad, ls, gs, _ = _plain(x, ids, t, 1.5)
    stats, g = torch.empty(rows, 2, device=DEV), torch.full_like(x, 7.0)
    got = Ds.distill_rows(x, ids, t, 1.5, stats=stats)
    _check(got, loss, ls, "losses")
    assert torch.equal(Ds.distill_rows(x, ids, t, 1.5, grad=g, grad_scale=2.0), got)
    _check(g, grad * 2, gs * 2, "gradient")
    _check(Ds.distill_rows_bwd(x, ids, t, 1.5, stats, torch.ones(rows, device=DEV)), grad, gs, "gradient by the stats")
    over = x.clone()
    assert torch.equal(Ds.distill_rows(over, ids, t, 1.5, grad=over, grad_scale=2.0), got) and torch.equal(over, g)


@pytest.mark.parametrize("T", [0.5, 2.0, 7.0])
def test_temperatures(T):
    _run(*_inputs(33, 5000, 20, torch.float32, torch.float32), T)


def test_many_entries_and_ids_of_64_bits():
    x, ids, t = _inputs(4, 9000, 1024)
    _run(x, ids.long(), t)
    ids = ids.long()
    ids[0, :7] = torch.tensor([2 ** 40, -(2 ** 40), 9000, 8999, 0, -1, 2 ** 31], device=DEV)
    _run(x, ids, t)


def test_the_same_id_many_times():
    x, ids, t = _inputs(6, 500, 30)
    ids[:, 3:20] = 7
    ids[1] = 499
    _run(x, ids, t)


def test_rows_without_entries_whatever_they_hold():
    x, ids, t = _inputs(8, 1000, 10)
    ids[2] = -1
    ids[5] = 1000
    t[6] = float("-inf")
    _run(x, ids, t)
    x[2] = float("nan")
    x[5, ::2] = float("inf")
    x[6] = float("-inf")
    loss, grad = rab.distillation_loss_and_grad(x, ids, t)
    leaf = x.clone().requires_grad_()
    mean = rab.distillation_loss(leaf, ids, t)
    g, = torch.autograd.grad(mean, leaf)
    for r in (2, 5, 6):
        assert float(loss[r]) == 0 and bool((grad[r] == 0).all()) and bool((g[r] == 0).all())
    assert bool(grad.isfinite().all()) and bool(g.isfinite().all()) and bool(mean.isfinite())


def test_no_row_has_entries():
    x, ids, t = _inputs(5, 100, 3)
    ids[:] = -1
    x.requires_grad_()
    loss = rab.distillation_loss(x, ids, t)
    loss.backward()
    assert float(loss.detach()) == 0 and bool((x.grad == 0).all())


def test_masked_and_outsized_logits():
    """Part of the vocabulary at -inf or the type's lowest value, logits of 1e4, teacher entries of -inf beside others."""
    x, ids, t = _inputs(8, 3001, 12, torch.float32, torch.float32)
    ids = ids.clamp_min(0) % 1500 * 2
    x[:, 1::2] = float("-inf")
    x[3, 1::2] = torch.finfo(torch.float32).min
    t[:, 2] = float("-inf")
    _run(x, ids, t)
    x, ids, t = _inputs(4, 2000, 6, torch.float32, torch.float32, std=3000.0)
    _run(x, ids, t / 100)


def test_what_the_student_rules_out_costs_without_end():
    x, ids, t = _inputs(2, 100, 3, torch.float32, torch.float32)
    ids[:] = torch.tensor([4, 9, 30], device=DEV)
    x[0, 9] = float("-inf")
    loss, grad = rab.distillation_loss_and_grad(x, ids, t)
    assert float(loss[0]) == float("inf") and bool(loss[1].isfinite())
    p = torch.softmax(t.double(), -1)
    assert abs(float(grad[0, 9]) + float(p[0, 1])) < 1e-6


def test_nan_stays_in_its_row():
    x, ids, t = _inputs(3, 900, 4)
    ids[:, 0] = 3
    x[1, 77] = float("nan")
    loss, grad = rab.distillation_loss_and_grad(x, ids, t)
    assert bool(loss[1].isnan()) and bool(grad[1].isnan().all())
    assert bool(loss[[0, 2]].isfinite().all()) and bool(grad[[0, 2]].isfinite().all())


def test_layouts():
    x, ids, t = _inputs(12, 1003, 8)
    wide = torch.zeros(12, 1100, device=DEV, dtype=torch.bfloat16)
    view = wide[:, 5:1008]
    view.copy_(x)
    _run(view, torch.cat([ids, ids], 1)[:, 3:11], t)
    by_batch = rab.distillation_loss(x.view(3, 4, -1), ids.view(3, 4, -1), t.view(3, 4, -1), reduction="none")
    assert by_batch.shape == (3, 4) and torch.equal(by_batch.view(-1), rab.distillation_loss(x, ids, t, reduction="none"))
    turned = x.t().contiguous().t()
    _run(turned, ids.t().contiguous().t(), t)
    # a gradient into a view of another alignment, next to values that stay
    wide.fill_(9.0)
    _, grad = rab.distillation_loss_and_grad(x, ids, t, out=view)
    assert torch.equal(view, rab.distillation_loss_and_grad(x, ids, t)[1])
    assert bool((wide[:, :5] == 9).all()) and bool((wide[:, 1008:] == 9).all())
    one = rab.distillation_loss(x[0], ids[0], t[0], reduction="none")
    assert one.shape == () and torch.equal(one, by_batch[0, 0])


def test_results_do_not_differ_from_call_to_call():
    x, ids, t = _inputs(40, 50000, 64)
    a, b = (rab.distillation_loss_and_grad(x, ids, t) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_step_follows_its_inputs():
    x, ids, t = (torch.zeros_like(v) for v in _inputs(30, 2000, 8))

    def step():
        leaf = x.detach().requires_grad_()
        loss = rab.distillation_loss(leaf, ids, t)
        return loss, torch.autograd.grad(loss, leaf)[0], *rab.distillation_loss_and_grad(x, ids, t)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        for dst, src in zip((x, ids, t), _inputs(30, 2000, 8, seed=seed)):
            dst.copy_(src)
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_what_the_kernels_refuse():
    x, ids, t = _inputs(2, 50, 3)
    for bad in ((x.half(), ids, t), (x, ids, t.double()), (x, ids.cpu(), t), (x, ids, t.cpu())):
        with pytest.raises(ValueError):
            rab.distillation_loss(*bad)
    with pytest.raises(ValueError):
        rab.distillation_loss_and_grad(x, ids, t, out=torch.zeros(50, 2, device=DEV, dtype=torch.bfloat16).t())
    with pytest.raises(ValueError):
        rab.distillation_loss(x, ids, t, temperature=1e-9)


def test_gradients_that_overlap_their_inputs_are_refused():
    x, ids, t = _inputs(4, 64, 3)
    wide = torch.zeros(4, 160, device=DEV, dtype=torch.bfloat16)
    wide[:, :64] = x
    for out in (wide[:, 8:72], x[:1].expand(4, 64), wide.flatten()[:256].view(4, 64)):
        with pytest.raises(ValueError, match="overlaps"):
            rab.distillation_loss_and_grad(wide[:, :64] if out.data_ptr() != x.data_ptr() else x, ids, t, out=out)
    want = rab.distillation_loss_and_grad(x, ids, t)[1]
    assert torch.equal(rab.distillation_loss_and_grad(wide[:, :64], ids, t, out=wide[:, 64:128])[1], want)
    assert torch.equal(rab.distillation_loss_and_grad(wide[:, :64], ids, t, out=wide[:, :64])[1], want)


def test_autograd_sees_that_a_given_tensor_changed():
    x, ids, t = _inputs(4, 64, 3)
    y = torch.tanh(x.float().requires_grad_())  # its backward reads y
    rab.distillation_loss_and_grad(y, ids, t, out=y)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
