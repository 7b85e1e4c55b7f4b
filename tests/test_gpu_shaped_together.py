"""Head norms with rotation, shaped attention and distillation as a decoder uses them: one training step whose every link is held against 64 bits
at its own inputs, a prompt and tokens through a cache, captured steps, and a ring's steps with a carry."""
import math

import pytest
import torch
from shaped_plain import attention, check, slopes_for, visible
from test_gpu_distill import _check as check_loss
from test_gpu_distill import _plain as distill_plain
from test_gpu_qknorm import _check as check_norm
from test_gpu_qknorm import _gains, _rand
from test_gpu_qknorm import _plain as norm_plain

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


class Layer:
    """One attention layer and a head: x -> q, k, v -> norms and rotation -> attention -> logits -> distillation."""

    def __init__(self, B, S, H, D, V, K, seed=0):
        self.dims, self.V = (B, S, H, D), V
        E = H * D
        self.x = _rand(B, S, E, dtype=BF, seed=seed, std=1.0)
        self.w_qkv = _rand(3 * E, E, dtype=BF, seed=seed + 1, std=1 / math.sqrt(E))
        self.w_out = _rand(V, E, dtype=BF, seed=seed + 2, std=3 / math.sqrt(E))
        self.gains = [g.to(BF) * 1.5 for g in _gains(D, torch.float32)]
        self.slopes = slopes_for(H, DEV)
        self.prefix = torch.arange(B, device=DEV, dtype=torch.int32) * 9
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.ids = torch.randint(0, V, (B, S, K), device=DEV, generator=g)
        self.ids[:, ::5, 1:] = -1
        self.teacher = _rand(B, S, K, dtype=BF, seed=seed + 3, std=2.0)
        self.cap, self.T = 20.0, 2.0

    def leaves(self):
        return [t.detach().requires_grad_() for t in (self.x, self.w_qkv, self.w_out, *self.gains)]

    def forward(self, x, w_qkv, w_out, gq, gk, keep=None):
        B, S, H, D = self.dims
        qkv = (x @ w_qkv.t()).view(B, S, 3, H, D)
        q, k = rab.qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], gq, gk)
        out = rab.ringattention(q, k, qkv[:, :, 2], blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=self.cap,
                                                                           alibi_slopes=self.slopes, prefix_lens=self.prefix))
        logits = out.reshape(B, S, H * D) @ w_out.t()
        if keep is not None:
            for name, t in (("qkv", qkv), ("q", q), ("k", k), ("out", out), ("logits", logits)):
                t.retain_grad()
                keep[name] = t
        return rab.distillation_loss(logits, self.ids, self.teacher, temperature=self.T)

    def step(self):
        leaves = self.leaves()
        loss = self.forward(*leaves)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]


@pytest.mark.parametrize("B,S,H,D,V,K", [(2, 70, 3, 64, 501, 20), (1, 333, 2, 128, 4000, 64), (3, 1, 2, 64, 33, 4)])
def test_every_link_of_a_training_step(B, S, H, D, V, K):
    layer = Layer(B, S, H, D, V, K)
    leaves, keep = layer.leaves(), {}
    # the retained gradients of qkv are of all three parts together: v's is attention's own
    loss = layer.forward(*leaves, keep=keep)
    loss.backward()
    qkv, at = keep["qkv"], torch.arange(S, device=DEV)
    # norms and rotation
    for i, (name, gain) in enumerate((("q", leaves[3]), ("k", leaves[4]))):
        (y, ys), (dx, dxs), (dg, dgs) = norm_plain(qkv[:, :, i], gain, at.expand(B, S), 10000.0, 1e-6, keep[name].grad)
        check_norm(keep[name], y, ys, name)
        check_norm(qkv.grad[:, :, i], dx, dxs, "d" + name, 2.0 ** -18)
        check_norm(gain.grad, dg, dgs, "dgain " + name, 2.0 ** -16)
    # attention
    want = attention(keep["q"], keep["k"], qkv[:, :, 2], layer.cap, layer.slopes, (at[:, None] - at)[None, None], None,
                     visible(at, at, B, 1, layer.prefix), keep["out"].grad)
    check(keep["out"], want[0], want[1], "out")
    for got, w, b, what in zip((keep["q"].grad, keep["k"].grad, qkv.grad[:, :, 2]), want[2], want[3], ("dq", "dk", "dv")):
        check(got, w, b, what)
    # distillation
    rows = B * S
    each, grad, ls, gs, some = distill_plain(keep["logits"].reshape(rows, V), layer.ids.reshape(rows, K), layer.teacher.reshape(rows, K), layer.T)
    n = max(1, int(some.sum()))
    assert abs(float(loss.detach()) - float(each.sum() / n)) <= float(ls.sum() / n + each.abs().sum() / n) * 2.0 ** -20 + 1e-30
    check_loss(keep["logits"].grad.reshape(rows, V), grad / n, gs / n, "dlogits")


def test_prompt_and_tokens_through_a_cache():
    """Streams of their own lengths: the prompt in one call, then tokens in a captured step whose positions lie on the device. Every output is held
    against 64 bits over the cache, and rows behind a stream's end are never touched."""
    B, H, G, D, S = 3, 4, 4, 128, 96
    gains, slopes, cap = _gains(D, BF), slopes_for(H, DEV), 30.0
    lens = torch.tensor([40, 17, 1], device=DEV)
    P, N = 40, 12
    cache = torch.full((2, B, S, G, D), 9.0, device=DEV, dtype=BF)
    at = torch.arange(S, device=DEV)
    q, k, v = (_rand(B, P, H, D, dtype=BF, seed=i) for i in range(3))
    pos = torch.arange(P, device=DEV).expand(B, P)
    qn, kn = rab.qk_norm_rope(q, k, *gains, pos)
    for b, n in enumerate(lens.tolist()):
        cache[0, b, :n], cache[1, b, :n] = kn[b, :n], v[b, :n]
    mask = ((at <= at[:P, None])[None] & (at < lens[:, None, None]))[:, None]
    first = rab.ringattention_inference(qn, cache[0], cache[1], mask, logit_cap=cap, alibi_slopes=slopes, query_pos=0)

    def held(out, qq, mask, start, what):
        dist = start.reshape(-1, 1, 1, 1) + torch.arange(qq.shape[1], device=DEV)[:, None] - at
        want, bound = attention(qq, cache[0], cache[1], cap, slopes, dist, None, mask)
        check(out, want, bound, what)

    held(first, qn, mask, torch.zeros(B, device=DEV, dtype=torch.int64), "prompt")

    here = lens.clone()  # where each stream's next token goes
    new = [torch.zeros(B, 1, H, D, device=DEV, dtype=BF) for _ in range(3)]
    streams = torch.arange(B, device=DEV)

    def token():
        qn, kn = rab.qk_norm_rope(new[0], new[1], *gains, here[:, None])
        cache[0].index_put_((streams, here), kn[:, 0])
        cache[1].index_put_((streams, here), new[2][:, 0])
        mask = (at <= here[:, None])[:, None, None]
        return qn, mask, rab.ringattention_inference(qn, cache[0], cache[1], mask, logit_cap=cap, alibi_slopes=slopes, query_pos=here)

    kept = cache.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qn, mask, out = token()
    cache.copy_(kept)
    for i in range(N):
        for j, t in enumerate(new):
            t.copy_(_rand(B, 1, H, D, dtype=BF, seed=100 + 10 * i + j))
        here.copy_(lens + i)
        graph.replay()
        held(out, qn, mask, here, f"token {i}")
        got = out.clone()
        assert torch.equal(got, token()[2])
    for b, n in enumerate(lens.tolist()):
        assert bool((cache[:, b, n + N:] == 9.0).all())


def test_two_captured_steps_beside_one_another():
    """Two captured training steps of unequal sizes, replayed in turns and on streams of their own: each gives what the eager step gives."""
    layers = [Layer(1, 300, 2, 64, 700, 10, seed=1), Layer(2, 150, 2, 128, 500, 30, seed=50)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for layer in layers:
            layer.step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    for layer in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(layer.step())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (5, 6):
        for layer in layers:
            layer.x.copy_(_rand(*layer.x.shape, dtype=BF, seed=seed, std=1.0))
        torch.cuda.synchronize()
        for _ in range(2):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for layer, mine in zip(layers, got):
            want = layer.step()
            # the reduction of dq has no fixed order: what depends on it is compared as sums of 32 bits, rounded to bf16 and through a product
            assert torch.equal(mine[0], want[0]) and torch.equal(mine[3], want[3])
            for a, b in zip(mine, want):
                assert a.isfinite().all() and (a.float() - b.float()).norm() <= 2.0 ** -7 * b.float().norm()


def test_on_another_stream():
    layer = Layer(1, 200, 2, 64, 300, 8)
    want = layer.step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = layer.step()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


@pytest.mark.parametrize("cap,sloped,prefix", [(20.0, True, 50), (20.0, False, None), (0.0, True, None), (0.0, False, 300)])
def test_steps_of_a_ring_with_a_carry(cap, sloped, prefix):
    """A rank's queries against three blocks of keys in the ring's order: the carry in fp32, the last step in bf16 with what rounding took."""
    from ringattention_b200.ops import _lib, flash
    from ringattention_b200.ops.flash import MaskSpec, Positions

    B, n, H, D, rank, ranks = 2, 200, 3, 64, 1, 3
    S = n * ranks
    q, dout = _rand(B, n, H, D, dtype=BF, seed=1, std=1.4), _rand(B, n, H, D, dtype=BF, seed=2)
    k, v = _rand(B, S, H, D, dtype=BF, seed=3, std=1.4), _rand(B, S, H, D, dtype=BF, seed=4)
    slopes = slopes_for(H, DEV) if sloped else None
    pre = None if prefix is None else torch.tensor([prefix, prefix + 60], device=DEV, dtype=torch.int32)
    order = [(rank - r) % ranks for r in range(ranks)]
    masks = [MaskSpec(1, Positions(rank * n), Positions(j * n), logit_cap=cap, slopes=slopes, prefix=pre) for j in order]
    o = lse = None
    lo = torch.empty(B, n, H, D, device=DEV, dtype=BF)
    for i, (j, ms) in enumerate(zip(order, masks)):
        last = i == ranks - 1
        o, lse = flash.flash_fwd(q, k[:, j * n:(j + 1) * n], v[:, j * n:(j + 1) * n], ms, o_prev=o, lse_prev=lse, out_fp32=not last, out_lo=lo if last else None)
    dq = torch.empty(B, n, H, D, device=DEV, dtype=torch.float32)
    lse2, delta = flash.flash_bwd_prep(o, dout, lse, dq_acc=dq, out_lo=lo)
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    for j, ms in zip(order, masks):
        cut = slice(j * n, (j + 1) * n)
        flash.flash_bwd(q, k[:, cut], v[:, cut], dout, lse2, delta, ms, dq, dk[:, cut], dv[:, cut])
    _lib.check_status()
    qp, kp = torch.arange(rank * n, (rank + 1) * n, device=DEV), torch.arange(S, device=DEV)
    want, bound, wg, bg = attention(q, k, v, cap, slopes, (qp[:, None] - kp)[None, None], None, visible(qp, kp, B, 1, pre), dout)
    check(o, want, bound, "out")
    for what, a, w, b in zip(("dq", "dk", "dv"), (dq, dk, dv), wg, bg):
        check(a, w, b, what)
