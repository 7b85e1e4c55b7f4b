"""``qk_norm_rope`` on the kernels against 64 bits: types, head dims, layouts, positions, gradients, output views, graphs and streams."""
import pytest
import torch

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plain(x, gain, pos, theta, eps, dy=None):
    """One of queries and keys in 64 bits: the result, with ``dy`` the gradients too, and for each what errors are relative to."""
    x, gain, D = x.detach().double(), gain.detach().double(), x.shape[-1]
    a = pos.double()[..., None, None] * theta ** (-torch.arange(0, D, 2, device=x.device, dtype=torch.float64) / D)
    cos, sin = torch.cat([a.cos()] * 2, -1), torch.cat([a.sin()] * 2, -1)
    swap = lambda t: torch.cat([-t[..., D // 2:], t[..., :D // 2]], -1)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    m = n * gain
    y, size = m * cos + swap(m) * sin, m.abs() + swap(m).abs()
    if dy is None:
        return [(y, size)]
    dy = dy.detach().double()
    u = dy * cos - swap(dy) * sin
    us = dy.abs() + swap(dy).abs()
    w = u * gain
    dx = r * (w - n * (w * n).mean(-1, keepdim=True))
    ws = us * gain.abs()
    return [(y, size), (dx, r * (ws + n.abs() * (ws * n.abs()).mean(-1, keepdim=True))), ((u * n).sum((0, 1, 2)), (us * n.abs()).sum((0, 1, 2)))]


def _check(got, want, size, what, rel=2.0 ** -19):
    half = torch.finfo(got.dtype).eps / 2
    bound = want.abs() * half + size * rel + 1e-30
    off = (got.detach().double() - want).abs()
    assert got.detach().isfinite().all(), what
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.2f} of the bound"


def _rand(*shape, dtype, seed=0, std=1.7):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def _gains(D, dtype):
    return (1 + 0.2 * _rand(D, dtype=torch.float32, seed=7)).to(dtype), (1 + 0.2 * _rand(D, dtype=torch.float32, seed=8)).to(dtype)


def _run(q, k, gq, gk, positions, theta=10000.0, eps=1e-6):
    B, S = q.shape[:2]
    pos = torch.arange(S, device=DEV) if positions is None else positions
    pos = (pos + torch.arange(S, device=DEV) if isinstance(pos, int) else pos).reshape(-1, S).expand(B, S)
    leaves = [t.detach().requires_grad_() for t in (q, k, gq, gk)]
    out = rab.qk_norm_rope(*leaves, positions, theta=theta, eps=eps)
    dy = [_rand(*x.shape, dtype=q.dtype, seed=20 + i) for i, x in enumerate((q, k))]
    grads = torch.autograd.grad(out, leaves, dy)
    for i, name in enumerate("qk"):
        want = _plain(leaves[i], leaves[2 + i], pos, theta, eps, dy[i])
        for got, (w, size), what, rel in zip((out[i], grads[i], grads[2 + i]), want, ("out", "dx", "dgain"), (2.0 ** -19, 2.0 ** -18, 2.0 ** -16)):
            _check(got, w, size, f"{name} {what}", rel)
    with torch.no_grad():
        again = rab.qk_norm_rope(q, k, gq, gk, positions, theta=theta, eps=eps)
    assert all(torch.equal(a, b.detach()) for a, b in zip(again, out))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,S,H,G", [(1, 1, 1, 1), (3, 1, 32, 8), (2, 37, 5, 2), (1, 1000, 4, 4), (2, 700, 12, 3)])
@pytest.mark.parametrize("dtype,gain", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
def test_against_64_bits(D, B, S, H, G, dtype, gain):
    _run(_rand(B, S, H, D, dtype=dtype), _rand(B, S, G, D, dtype=dtype, seed=1), *_gains(D, gain), None)


@pytest.mark.parametrize("positions", [0, 77, "one", "each", "far", "int64", "strided"])
def test_positions(positions):
    B, S, D = 3, 50, 128
    at = torch.arange(S, device=DEV)
    pos = {"one": at * 3, "each": torch.randint(0, 5000, (B, S), device=DEV), "far": at + 10 ** 6, "int64": at + 2 ** 33,
           "strided": torch.randint(0, 900, (S, B), device=DEV).t()}.get(positions, positions)
    if isinstance(pos, torch.Tensor) and positions != "int64":
        pos = pos.to(torch.int32) if positions != "strided" else pos
    _run(_rand(B, S, 4, D, dtype=torch.float32), _rand(B, S, 2, D, dtype=torch.float32, seed=1), *_gains(D, torch.float32), pos, theta=500000.0)


def test_positions_of_a_shard():
    from ringattention_b200.ops.flash import Positions

    S, D = 256, 64
    q, k, (gq, gk) = _rand(1, S, 2, D, dtype=torch.bfloat16), _rand(1, S, 2, D, dtype=torch.bfloat16, seed=1), _gains(D, torch.bfloat16)
    pos = Positions(128, 896, 128)
    a = rab.qk_norm_rope(q, k, gq, gk, pos)
    b = rab.qk_norm_rope(q, k, gq, gk, pos.tensor(S, DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_rotation_is_the_librarys():
    from ringattention_b200.ops import kernels as K
    from ringattention_b200.ops.flash import Positions

    x = _rand(2, 60, 4, 128, dtype=torch.bfloat16)
    one = torch.ones(128, device=DEV)
    y, _ = rab.qk_norm_rope(x, x, one, one, 5)
    z = (x.float() * (x.float().square().mean(-1, keepdim=True) + 1e-6).rsqrt()).bfloat16()
    K.rope_(z, Positions(5), 10000.0)
    assert (y.float() - z.float()).abs().max() <= 2.0 ** -7 * 8  # two roundings of numbers below 8


def test_layouts_rows_off_16_bytes_and_broadcast_gradients():
    B, S, H, G, D = 2, 33, 3, 2, 64
    packed = _rand(B, S, H + G, D, dtype=torch.bfloat16)
    _run(packed[:, :, :H], packed[:, :, H:], *_gains(D, torch.float32), 9)
    by_head = _rand(B, H, S, D, dtype=torch.bfloat16).transpose(1, 2)
    _run(by_head, by_head[:, :, :1], *_gains(D, torch.float32), 9)
    odd = _rand(B * S * H * D + 1, dtype=torch.bfloat16)[1:].view(B, S, H, D)
    _run(odd, odd, *_gains(D, torch.bfloat16), None)
    one = _rand(1, 1, 1, D, dtype=torch.bfloat16).expand(B, S, H, D)
    _run(one, one, *_gains(D, torch.bfloat16), None)
    q = _rand(B, S, H, D, dtype=torch.bfloat16).requires_grad_()
    g = torch.ones(D, device=DEV)
    y, _ = rab.qk_norm_rope(q, q.detach(), g, g)
    y.sum().backward()  # an expanded gradient, and none for the keys
    _check(q.grad, *_plain(q, g, torch.arange(S, device=DEV).expand(B, S), 10000.0, 1e-6, torch.ones_like(q))[1], "expanded", 2.0 ** -18)


def test_rows_of_zeros_and_outsized_rows():
    q = _rand(1, 4, 2, 64, dtype=torch.float32)
    q[0, 1] = 0
    q[0, 2] *= 1e18
    q[0, 3] *= 1e-18
    _run(q, q, *_gains(64, torch.float32), None)
    y, _ = rab.qk_norm_rope(q, q, *_gains(64, torch.float32))
    assert bool((y[0, 1] == 0).all())
    q[0, 0, 0, 5] = float("nan")
    y, _ = rab.qk_norm_rope(q, q, *_gains(64, torch.float32))
    assert bool(y[0, 0, 0].isnan().all()) and bool(y[0, 0, 1].isfinite().all()) and bool(y[0, 1:].isfinite().all())


def test_output_views():
    B, S, H, G, D = 2, 1, 4, 2, 128
    q, k, g = _rand(B, S, H, D, dtype=torch.bfloat16), _rand(B, S, G, D, dtype=torch.bfloat16, seed=1), _gains(D, torch.bfloat16)
    want = rab.qk_norm_rope(q, k, *g, 11)
    cache = torch.full((B, 20, G, D), 3.0, device=DEV, dtype=torch.bfloat16)
    y, row = rab.qk_norm_rope(q, k, *g, 11, k_out=cache[:, 11:12])
    assert torch.equal(y, want[0]) and torch.equal(cache[:, 11:12], want[1]) and row.data_ptr() == cache[:, 11:12].data_ptr()
    cache[:, 11] = 3.0
    assert bool((cache == 3.0).all())
    both = rab.qk_norm_rope(q, k, *g, 11, q_out=q, k_out=k)
    assert both[0] is q and both[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_results_do_not_differ_from_call_to_call():
    q, k = (_rand(1, 3000, 8, 128, dtype=torch.bfloat16, seed=i).requires_grad_() for i in range(2))
    g = [t.requires_grad_() for t in _gains(128, torch.float32)]
    dy = [_rand(1, 3000, 8, 128, dtype=torch.bfloat16, seed=5 + i) for i in range(2)]
    a, b = (torch.autograd.grad(rab.qk_norm_rope(q, k, *g), (q, k, *g), dy) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_forward_and_backward_follow_their_inputs():
    B, S, H, D = 1, 300, 4, 64
    g = _gains(D, torch.float32)
    q, k, dy = (torch.zeros(B, S, H, D, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    pos = torch.zeros(S, device=DEV, dtype=torch.int32)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, *g)]
        out = rab.qk_norm_rope(*leaves, pos)
        return (*out, *torch.autograd.grad(out, leaves, (dy, dy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        for i, t in enumerate((q, k, dy)):
            t.copy_(_rand(B, S, H, D, dtype=torch.bfloat16, seed=10 * seed + i))
        pos.copy_(torch.arange(S, device=DEV) * seed)
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_another_stream():
    q, k, g = _rand(2, 500, 8, 128, dtype=torch.bfloat16), _rand(2, 500, 8, 128, dtype=torch.bfloat16, seed=1), _gains(128, torch.bfloat16)
    want = rab.qk_norm_rope(q, k, *g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rab.qk_norm_rope(q, k, *g)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_the_kernels_refuse():
    q, g = torch.zeros(1, 2, 1, 64, device=DEV, dtype=torch.bfloat16), torch.ones(64, device=DEV)
    with pytest.raises(ValueError):
        rab.qk_norm_rope(q.half(), q.half(), g, g)
    with pytest.raises(ValueError):
        rab.qk_norm_rope(q[..., :32], q[..., :32], g[:32], g[:32])
    with pytest.raises(ValueError):
        rab.qk_norm_rope(q, q, g.cpu(), g.cpu())
    with pytest.raises(ValueError):
        rab.qk_norm_rope(q, q, g, g, torch.arange(2))
    with pytest.raises(ValueError):
        rab.qk_norm_rope(q, q, g, g, q_out=torch.zeros(129, device=DEV, dtype=torch.bfloat16)[1:].view(1, 2, 1, 64))
