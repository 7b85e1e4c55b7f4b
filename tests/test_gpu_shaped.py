"""Attention with shaped scores (a tanh cap, a slope on the distance, an open prefix) on the kernels, against 64 bits."""
import pytest
import torch
from shaped_plain import attention, check, slopes_for, visible

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _rand(*shape, seed=0, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * std).bfloat16()


def _inputs(B, Sq, Sk, H, D, std=1.4, seed=0):
    q, k = _rand(B, Sq, H, D, seed=seed, std=std), _rand(B, Sk, H, D, seed=seed + 1, std=std)
    return q, k, _rand(B, Sk, H, D, seed=seed + 2), _rand(B, Sq, H, D, seed=seed + 3)


def _train(q, k, v, dout, cap=0.0, slopes=None, prefix=None, cbs=1, bias=None, seg=None, what=""):
    import ringattention_b200 as rab
    from ringattention_b200.ops import _lib

    B, S, H, D = q.shape
    kw = dict(causal_block_size=cbs or None, query_chunk_size=S, key_chunk_size=S, logit_cap=cap or None, alibi_slopes=slopes, prefix_lens=prefix)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = rab.ringattention(*leaves, bias, seg, blockwise_kwargs=kw)
    grads = torch.autograd.grad(out, leaves, dout)
    _lib.check_status()
    at = torch.arange(S, device=DEV)
    want, bound, wg, bg = attention(q, k, v, cap, slopes, (at[:, None] - at)[None, None], bias, visible(at, at, B, cbs, prefix, seg, seg, bias), dout)
    check(out, want, bound, what + " out")
    for n, a, b, c in zip(("dq", "dk", "dv"), grads, wg, bg):
        check(a, b, c, f"{what} {n}")
    with torch.no_grad():
        again = rab.ringattention(q, k, v, bias, seg, blockwise_kwargs=kw)
    assert torch.equal(again, out.detach())


@pytest.mark.parametrize("B,S,H,D", [(1, 1, 1, 64), (2, 17, 3, 64), (1, 128, 2, 128), (3, 129, 2, 64), (1, 300, 5, 128), (2, 1000, 4, 64), (1, 1537, 2, 128)])
@pytest.mark.parametrize("cap,sloped", [(30.0, False), (2.0, False), (0.0, True), (20.0, True), (200.0, False)])
@pytest.mark.parametrize("cbs", [0, 1])
def test_forward_and_backward(B, S, H, D, cap, sloped, cbs):
    """cap 2: nearly all scores in the tanh's far range; 200: the online maximum with a cap."""
    _train(*_inputs(B, S, S, H, D), cap, slopes_for(H, DEV) if sloped else None, cbs=cbs)


@pytest.mark.parametrize("S,D,cbs", [(40, 64, 1), (515, 128, 1), (515, 64, 4), (900, 128, 64)])
@pytest.mark.parametrize("cap,sloped", [(0.0, False), (15.0, False), (0.0, True), (15.0, True)])
def test_prefix_documents_and_padding(S, D, cbs, cap, sloped):
    B, H = 4, 3
    prefix = torch.tensor([0, 5, S // 2 + 3, S + 100], device=DEV, dtype=torch.int32)
    bias = torch.zeros(B, 1, 1, S, device=DEV)
    bias[1, ..., S - 7:] = torch.finfo(torch.float32).min
    bias[2, ..., :9] = float("-inf")
    seg = (torch.arange(S, device=DEV) // max(1, S // 3)).int().expand(B, S).contiguous()
    x = _inputs(B, S, S, H, D, seed=5)
    slopes = slopes_for(H, DEV) if sloped else None
    _train(*x, cap, slopes, prefix, cbs, what="prefix")
    _train(*x, cap, slopes, prefix, cbs, bias=bias, what="prefix, bias")
    _train(*x, cap, slopes, prefix, cbs, bias=bias, seg=seg, what="prefix, bias, documents")
    _train(*x, cap, slopes, 7, cbs, seg=seg, what="prefix as a number")


def test_bias_adds_to_capped_scores():
    B, S, H, D = 2, 333, 4, 64
    bias = (torch.randn(B, H, 1, S, device=DEV) * 3).float()
    _train(*_inputs(B, S, S, H, D, seed=9), 10.0, None, bias=bias)


@pytest.mark.parametrize("form", ["pairs", "halves", "split"])
def test_every_form_of_the_forward(form):
    """Launches of many query tiles, of few, and of few with keys enough to be split."""
    B, Sq, Sk, H, D = {"pairs": (4, 1300, 1300, 32, 64), "halves": (1, 1024, 1024, 8, 64), "split": (1, 140, 9000, 2, 128)}[form]
    from ringattention_b200.ops import _lib, flash
    from ringattention_b200.ops.flash import MaskSpec, Positions

    q, k, v, _ = _inputs(B, Sq, Sk, H, D, seed=3)
    slopes = slopes_for(H, DEV)
    for cap, sl in ((25.0, None), (0.0, slopes), (25.0, slopes)):
        ms = MaskSpec(1, Positions(Sk - Sq), Positions(0), logit_cap=cap, slopes=sl)
        lo = torch.empty(B, Sq, H, D, device=DEV, dtype=torch.bfloat16)
        n = _lib.launches()
        out, lse = flash.flash_fwd(q, k, v, ms, out_lo=lo)
        assert (_lib.launches() - n == 2) == (form == "split")
        _lib.check_status()
        qp, kp = torch.arange(Sk - Sq, Sk, device=DEV), torch.arange(Sk, device=DEV)
        for b in range(B):
            one = slice(b, b + 1)
            want, bound = attention(q[one], k[one], v[one], cap, sl, (qp[:, None] - kp)[None, None], None, visible(qp, kp, 1, 1))
            check(out[one], want, bound, form)
            check((out[one].double() + lo[one].double()), want, bound, form + " with what rounding took")
        assert bool((lo.float().abs() <= out.float().abs() * 2.0 ** -8 + 1e-30).all())


def test_scores_at_the_ends_of_their_range():
    """Products that overflow fp32's squares, and huge caps: the cap holds, and a cap far above all scores changes nothing."""
    import ringattention_b200 as rab

    B, S, H, D = 1, 200, 2, 64
    q, k, v, _ = _inputs(B, S, S, H, D)
    at = torch.arange(S, device=DEV)
    kw = dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S)
    with torch.no_grad():
        far = rab.ringattention(q * 1e18, k * 1e18, v, blockwise_kwargs=dict(kw, logit_cap=5.0))
        want, bound = attention(q * 1e18, k * 1e18, v, 5.0, seen=visible(at, at, B, 1))
        check(far, want, bound, "beyond the range")
        loose = rab.ringattention(q, k, v, blockwise_kwargs=dict(kw, logit_cap=1e30))
        want, bound = attention(q, k, v, seen=visible(at, at, B, 1))
        check(loose, want, bound, "cap 1e30")


@pytest.mark.parametrize("where", ["masked", "seen"])
def test_nan_stays_where_it_is(where):
    import ringattention_b200 as rab

    S, D = 260, 64
    q, k, v, _ = _inputs(1, S, S, 2, D)
    k[0, 130, 0] = float("nan")
    with torch.no_grad():
        out = rab.ringattention(q, k, v, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=30.0))
    bad = out.isnan().any(-1)[0]
    assert not bad[:130].any() and not bad[:, 1].any() and bool(bad[130:, 0].all())


# ------------------------------------------------------------------------------------------------ inference
def _infer(B, Q, S, H, D, cap, sloped, mask=None, pos=None, seed=0, grad=False):
    import ringattention_b200 as rab
    from ringattention_b200.ops import _lib

    q, k, v, dout = _inputs(B, Q, S, H, D, seed=seed)
    slopes = slopes_for(H, DEV) if sloped else None
    leaves = [t.requires_grad_(grad) for t in (q, k, v)]
    with torch.set_grad_enabled(grad):
        out = rab.ringattention_inference(*leaves, mask, logit_cap=cap or None, alibi_slopes=slopes, query_pos=pos)
    first = torch.as_tensor(max(0, S - Q) if pos is None else pos, device=DEV).reshape(-1, 1, 1, 1)
    dist = first + torch.arange(Q, device=DEV)[:, None] - torch.arange(S, device=DEV)
    seen = torch.ones(B, 1, Q, S, dtype=torch.bool, device=DEV) if mask is None else mask.expand(B, -1, Q, S)
    got = attention(q, k, v, cap, slopes, dist, None, seen, dout if grad else None)
    _lib.check_status()
    check(out, got[0], got[1], "out")
    if grad:
        for n, a, b, c in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout), got[2], got[3]):
            check(a, b, c, n)
    return out


@pytest.mark.parametrize("Q", [1, 2, 3, 5, 8, 9, 40])
@pytest.mark.parametrize("S,D", [(1, 64), (33, 128), (700, 64), (5000, 128)])
@pytest.mark.parametrize("cap,sloped", [(30.0, False), (0.0, True), (3.0, True)])
def test_inference(Q, S, D, cap, sloped):
    _infer(2, Q, S, 3, D, cap, sloped, seed=Q)


@pytest.mark.parametrize("Q", [1, 4, 20])
def test_inference_masks_and_positions(Q):
    """Caches filled up to places of their own, a row that sees nothing, a query in the middle of its keys, a mask by head."""
    B, S, H = 3, 900, 4
    n = torch.tensor([900, 300, 20], device=DEV)
    pos = (n - Q).int()
    at = torch.arange(S, device=DEV)
    mask = (at <= pos[:, None, None] + torch.arange(Q, device=DEV)[:, None])[:, None]
    for cap, sloped in ((20.0, True), (0.0, True), (20.0, False)):
        _infer(B, Q, S, H, 128, cap, sloped, mask, pos)
        _infer(B, Q, S, H, 64, cap, sloped, mask, pos.long())
        _infer(B, Q, S, H, 64, cap, sloped, None, 450)
        some = mask.expand(B, H, Q, S).clone()
        some[:, 1] &= at % 3 == 0
        some[1, :, 0] = False
        out = _infer(B, Q, S, H, 128, cap, sloped, some, pos)
        assert bool((out[1, 0] == 0).all())


@pytest.mark.parametrize("Q", [1, 30])
def test_inference_gradients(Q):
    B, S, H = 2, 500, 3
    pos = torch.tensor([470, 100], device=DEV, dtype=torch.int32)
    mask = (torch.arange(S, device=DEV) <= pos[:, None, None] + torch.arange(Q, device=DEV)[:, None])[:, None]
    for cap, sloped in ((20.0, True), (20.0, False), (0.0, True)):
        _infer(B, Q, S, H, 64, cap, sloped, mask, pos, grad=True)


@pytest.mark.parametrize("cap", [15.0, 55.0])
def test_rows_whose_scores_go_from_one_end_of_the_cap_to_the_other(cap):
    """The exponentials of a capped row are taken against its first keys' scores: here those lie at -cap and later ones at +cap, and the reverse."""
    B, S, H, D = 1, 700, 2, 64
    q, k, v, dout = _inputs(B, S, S, H, D, seed=2)
    far = q[:, :1].float().sign() * 100
    q = (q.float().sign() * 0 + far).bfloat16()
    for first in (-1.0, 1.0):
        kk = k.clone()
        kk[:, :300] = (first * far).bfloat16()
        kk[:, 300:600] = (-first * far).bfloat16()
        _train(q, kk, v, dout, cap, cbs=0, what=f"{first}")
        _train(q, kk, v, dout, cap, cbs=1, what=f"{first}, causal")


@pytest.mark.parametrize("cap", [1e-3, 1.0, 1e30])
def test_queries_of_zeros(cap):
    """All scores 0: the mean of the values, whatever the cap."""
    import ringattention_b200 as rab

    S, D = 150, 64
    _, k, v, _ = _inputs(1, S, S, 2, D)
    q = torch.zeros_like(k)
    with torch.no_grad():
        out = rab.ringattention(q, k, v, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=S, key_chunk_size=S, logit_cap=cap))
        one = rab.ringattention_inference(q[:, :1], k, v, logit_cap=cap)
    at = torch.arange(S, device=DEV)
    want, bound = attention(q, k, v, cap, seen=visible(at, at, 1, 1))
    check(out, want, bound, "causal")
    want, bound = attention(q[:, :1], k, v, cap, seen=torch.ones(1, 1, 1, S, dtype=torch.bool, device=DEV))
    check(one, want, bound, "one row")


@pytest.mark.parametrize("Q", [1, 4])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_masked_cache_rows_may_hold_anything(Q, where):
    """Rows behind the end of a stream, not written yet."""
    B, S, H, D = 2, 700, 3, 64
    import ringattention_b200 as rab

    q, k, v, _ = _inputs(B, Q, S, H, D)
    n = torch.tensor([650, 300], device=DEV)
    mask = (torch.arange(S, device=DEV) < n[:, None])[:, None, None]
    kw = dict(logit_cap=20.0, alibi_slopes=slopes_for(H, DEV), query_pos=n - Q)
    with torch.no_grad():
        want = rab.ringattention_inference(q, k, v, mask, **kw)
        bad = k if where == "keys" else v
        bad[0, 650:], bad[1, 300:] = float("nan"), float("inf")
        assert torch.equal(rab.ringattention_inference(q, k, v, mask, **kw), want)


def test_a_cache_index_counts_in_distances_and_prefixes():
    import ringattention_b200 as rab

    B, Q, S, H, D = 2, 5, 1000, 3, 64
    q, k, v, _ = _inputs(B, Q, S, H, D)
    slopes = slopes_for(H, DEV)
    with torch.no_grad():
        out = rab.ringattention(q, k, v, None, None, 700, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=Q, key_chunk_size=S, logit_cap=20.0,
                                                                                alibi_slopes=slopes, prefix_lens=900))
    qp, kp = torch.arange(700, 700 + Q, device=DEV), torch.arange(S, device=DEV)
    want, bound = attention(q, k, v, 20.0, slopes, (qp[:, None] - kp)[None, None], None, visible(qp, kp, B, 1, 900))
    check(out, want, bound)


def test_far_positions_and_one_leaf_for_all():
    import ringattention_b200 as rab

    S, H, D, first = 300, 2, 64, (1 << 24) - 50
    slopes = torch.tensor([1e-6, 3e-5], device=DEV)
    for Q in (1, 2, 20):
        q, k, v, _ = _inputs(1, Q, S, H, D)
        with torch.no_grad():
            out = rab.ringattention_inference(q, k, v, alibi_slopes=slopes, query_pos=first)
        dist = first + torch.arange(Q, device=DEV)[:, None] - torch.arange(S, device=DEV)
        want, bound = attention(q, k, v, 0.0, slopes, dist[None, None], None, torch.ones(1, 1, Q, S, dtype=torch.bool, device=DEV))
        check(out, want, bound, f"{Q} rows")
    x = _rand(1, 200, 2, 64, std=1.4).requires_grad_()
    out = rab.ringattention(x, x, x, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=200, key_chunk_size=200, logit_cap=20.0))
    grad, = torch.autograd.grad(out, x, torch.ones(1, device=DEV, dtype=torch.bfloat16).expand(out.shape))
    at = torch.arange(200, device=DEV)
    _, _, parts, off = attention(x, x, x, 20.0, seen=visible(at, at, 1, 1), dout=torch.ones_like(out))
    # three gradients in bf16, added one by one: two more roundings of sums no larger than the parts' absolute sum
    check(grad, sum(parts), sum(off) + 2 * 2.0 ** -8 * sum(p.abs() for p in parts))
