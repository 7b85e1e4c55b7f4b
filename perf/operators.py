"""The operators of models whose attention scores are shaped, whose queries and keys are normalised, and that learn from a teacher:
their cases, their plain form in elementary torch operations, and what they give in 64 bits.

``attention``  ``ringattention`` on one GPU with scores that are capped by a tanh, lose a slope times their distance, or that see a common
               prefix: forward and backward, or the forward alone;
``inference``  ``ringattention_inference`` with the same scores over a cache: single tokens, a few of them, or a chunk of a prompt;
``norm``       ``qk_norm_rope``: RMS norm of each head's queries and keys and their rotation by position in one pass, forward and backward;
``distil``     ``distillation_loss`` with its backward pass, and ``distillation_loss_and_grad``, which gives both at once.

``own`` picks the library's kernels (true) or the plain form (false) for ``run``.
"""
import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # fine-tuning on short texts, or a test: launches and host work count
        dict(name="capped 512", kind="attention", B=2, S=512, H=8, D=64, cap=30.0, slopes=False, causal=True, prefix=False, docs=0, pad=False, grad=True),
        # a batch of instructions and answers: the instruction is seen from everywhere, lengths differ, no multiple of a tile
        dict(name="prefix padded 1371", kind="attention", B=3, S=1371, H=12, D=64, cap=0.0, slopes=True, causal=True, prefix=True, docs=0, pad=True,
             grad=True),
        # the context of an ordinary pre-training step
        dict(name="capped 4K", kind="attention", B=1, S=4096, H=32, D=128, cap=50.0, slopes=False, causal=True, prefix=False, docs=0, pad=False,
             grad=True),
        # long context out of packed documents
        dict(name="distance packed 8K", kind="attention", B=1, S=8192, H=16, D=128, cap=0.0, slopes=True, causal=True, prefix=False, docs=2048, pad=False,
             grad=True),
        # one GPU's share of a long step, both at once
        dict(name="capped distance 16K", kind="attention", B=1, S=16384, H=8, D=128, cap=20.0, slopes=True, causal=True, prefix=False, docs=0, pad=False,
             grad=True),
        # single tokens at the end of a long document
        dict(name="capped decode 128K", kind="inference", B=1, Q=1, S=131072, H=32, D=128, cap=50.0, slopes=False, mask="none"),
        # four tokens each of a batch of chats of unequal lengths
        dict(name="distance decode batch", kind="inference", B=8, Q=4, S=4000, H=32, D=128, cap=0.0, slopes=True, mask="valid"),
        # a chunk of a prompt against what is cached
        dict(name="capped prompt chunk", kind="inference", B=1, Q=500, S=16384, H=32, D=128, cap=50.0, slopes=False, mask="causal"),
        # the new token of each of a batch of chats
        dict(name="norm one token", kind="norm", B=8, S=1, H=32, G=32, D=128, far=100000, half=True, grad=False),
        # a training step with fewer key heads than query heads
        dict(name="norm 16K", kind="norm", B=1, S=16384, H=32, G=8, D=128, far=0, half=False, grad=True),
        # a short batch with a vocabulary of odd size, logits in 32 bits
        dict(name="distil odd", kind="distil", rows=333, V=10007, K=37, T=2.0, wide=True, form="loss"),
        # a chunk of a training step
        dict(name="distil 4096 x 32000", kind="distil", rows=4096, V=32000, K=64, T=1.0, wide=False, form="both"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["inference"] * 3 + ["norm"] * 2 + ["distil"] * 3)
    if kind == "attention":
        D, H, B, S = rng.choice([64, 128]), rng.choice([1, 3, 4, 8, 16, 32]), rng.choice([1, 1, 2, 3]), _log_int(rng, 1, 16384)
        if S > 256 and rng.random() < 0.5:
            S = S // 128 * 128
        while B * H * S * S > 8 * 16384 * 16384 // 2:
            S = S // 2
        shape = rng.choice(["cap", "cap", "slopes", "both", "prefix"])
        mask = rng.choice(["none", "none", "docs", "pad"])
        return dict(kind=kind, B=B, S=S, H=H, D=D, cap=rng.choice([15.0, 20.0, 30.0, 50.0]) if shape in ("cap", "both") else 0.0,
                    slopes=shape in ("slopes", "both"), causal=shape == "prefix" or rng.random() < 0.8, prefix=shape == "prefix",
                    docs=max(16, S // 8) if mask == "docs" else 0, pad=mask == "pad", grad=rng.random() < 0.75 and S >= 16)
    if kind == "inference":
        D, H = rng.choice([64, 128]), rng.choice([1, 8, 16, 32])
        if rng.random() < 0.65:
            B, Q, S, mask = rng.choice([1, 1, 2, 5, 8]), rng.choice([1, 1, 1, 2, 3, 4, 8]), _log_int(rng, 8, 131072), rng.choice(["none", "valid"])
        else:
            B, Q, S, mask = rng.choice([1, 1, 2]), _log_int(rng, 9, 1000), _log_int(rng, 1000, 32768), "causal"
        while B * H * S * D > 131072 * 32 * 128:
            S = S // 2 + 1
        shape = rng.choice(["cap", "slopes", "both"])
        return dict(kind=kind, B=B, Q=min(Q, S), S=S, H=H, D=D, cap=rng.choice([15.0, 30.0, 50.0]) if shape != "slopes" else 0.0,
                    slopes=shape != "cap", mask=mask)
    if kind == "norm":
        B, S, H = rng.choice([1, 1, 2, 8]), _log_int(rng, 1, 32768), rng.choice([1, 4, 12, 32])
        while B * S * H > 16384 * 32:
            S = S // 2 + 1
        return dict(kind=kind, B=B, S=S, H=H, G=rng.choice([1, max(1, H // 4), H]), D=rng.choice([64, 128, 256]), far=rng.choice([0, 4096, 1000000]),
                    half=rng.random() < 0.7, grad=rng.random() < 0.7)
    rows, V = _log_int(rng, 1, 8192), _log_int(rng, 300, 200000)
    if rng.random() < 0.5:
        V = V // 8 * 8
    while rows * V > 4096 * 32000:
        rows = rows // 2
    return dict(kind=kind, rows=max(1, rows), V=V, K=min(V, _log_int(rng, 1, 256)), T=rng.choice([1.0, 1.0, 2.0, 4.0]), wide=rng.random() < 0.25,
                form=rng.choice(["loss", "mean", "both"]))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device=DEV, generator=g, dtype=torch.float32) * std).to(dtype)


def _slopes(H):
    """Slopes that fall by equal factors from head to head, from 2^(-8/H) to 2^-8."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEV, dtype=torch.float32)


def _segments(case, seed):
    """Packed documents with a mean length of ``docs`` tokens: ids that grow along the sequence."""
    if not case["docs"]:
        return None
    g = torch.Generator()
    g.manual_seed(int(seed) + 7)
    new = torch.rand(case["B"], case["S"], generator=g) < 1.0 / case["docs"]
    new[:, 0] = False
    return new.int().cumsum(1).int().to(DEV)


def prepare(case, seed):
    return {"attention": _prepare_attention, "inference": _prepare_inference, "norm": _prepare_norm, "distil": _prepare_distil}[case["kind"]](case, seed)


def _prepare_attention(case, seed):
    """Scores with a deviation of about two, as those of trained heads."""
    B, S, H, D = case["B"], case["S"], case["H"], case["D"]
    g = _gen(seed)
    q, k = _randn(g, B, S, H, D, std=1.4), _randn(g, B, S, H, D, std=1.4)
    v, dout = _randn(g, B, S, H, D), _randn(g, B, S, H, D)
    bias = prefix = None
    if case["pad"]:  # rows of the batch end at lengths of their own
        n = torch.randint((S + 1) // 2, S + 1, (B,), device=DEV, generator=g)
        bias = torch.zeros(B, 1, 1, S, device=DEV).masked_fill_(torch.arange(S, device=DEV)[None, None, None] >= n[:, None, None, None],
                                                              torch.finfo(torch.float32).min)
    if case["prefix"]:
        prefix = torch.randint(0, S // 2 + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    kw = dict(causal_block_size=1 if case["causal"] else None, query_chunk_size=S, key_chunk_size=S, deterministic=True, dropout_rng=None,
              attn_pdrop=0.0, dtype=torch.float32, policy="nothing_saveable", precision=None, prevent_cse=True,
              logit_cap=case["cap"] or None, alibi_slopes=_slopes(H) if case["slopes"] else None, prefix_lens=prefix)
    return dict(case=case, q=q.requires_grad_(case["grad"]), k=k.requires_grad_(case["grad"]), v=v.requires_grad_(case["grad"]), dout=dout,
                bias=bias, seg=_segments(case, seed), kw=kw)


def _prepare_inference(case, seed):
    B, Q, S, H, D = case["B"], case["Q"], case["S"], case["H"], case["D"]
    g = _gen(seed)
    q, k, v = _randn(g, B, Q, H, D, std=1.4), _randn(g, B, S, H, D, std=1.4), _randn(g, B, S, H, D)
    at, mask, pos = torch.arange(S, device=DEV), None, S - Q
    if case["mask"] == "valid":  # each row of the batch has filled its cache up to a place of its own, the new tokens at its end
        n = torch.randint((S + 1) // 2, S + 1, (B,), device=DEV, generator=g).clamp_min_(Q)
        pos = (n - Q).to(torch.int32)
        mask = (at[None, None] <= pos[:, None, None] + torch.arange(Q, device=DEV)[None, :, None])[:, None]
    elif case["mask"] == "causal":  # the chunk's rows are the last Q of the S cached ones; some of them are padding and see nothing
        mask = at[None] <= torch.arange(S - Q, S, device=DEV)[:, None]
        mask = (mask & (torch.rand(Q, 1, device=DEV, generator=g) > 0.02))[None, None]
    return dict(case=case, q=q, k=k, v=v, mask=mask, pos=pos, slopes=_slopes(H) if case["slopes"] else None)


def _prepare_norm(case, seed):
    B, S, H, G, D = case["B"], case["S"], case["H"], case["G"], case["D"]
    g = _gen(seed)
    dt = torch.bfloat16 if case["half"] else torch.float32  # of the gains
    packed = _randn(g, B, S, H + G, D, std=1.7)             # queries and keys come out of one projection
    q, k = packed[:, :, :H], packed[:, :, H:]
    gq, gk = (1 + 0.1 * _randn(g, 2, D, dtype=torch.float32)).to(dt).unbind()
    pos = torch.randint(0, case["far"] + 1, (B, 1), device=DEV, generator=g) + torch.arange(S, device=DEV)
    s = dict(case=case, q=q, k=k, gq=gq.clone(), gk=gk.clone(), pos=pos.to(torch.int32), dq=_randn(g, B, S, H, D), dk=_randn(g, B, S, G, D))
    if case["grad"]:
        for n in ("q", "k", "gq", "gk"):
            s[n] = s[n].detach().requires_grad_()
    return s


def _prepare_distil(case, seed):
    """A teacher that agrees with the student up to some noise; fewer than ``K`` entries in some rows, none in a few (padding)."""
    rows, V, K = case["rows"], case["V"], case["K"]
    g = _gen(seed)
    logits = _randn(g, rows, V, std=2.5, dtype=torch.float32 if case["wide"] else torch.bfloat16)
    first = torch.randint(0, V, (rows, 1), device=DEV, generator=g)
    ids = (first + torch.arange(K, device=DEV) * (V // K)) % V
    teacher = (logits.gather(1, ids).float() + _randn(g, rows, K, dtype=torch.float32) + 2.0).to(logits.dtype)
    n = torch.randint(1, K + 1, (rows, 1), device=DEV, generator=g)
    n = torch.where(torch.rand(rows, 1, device=DEV, generator=g) < 0.05, 0, n)
    ids = torch.where(torch.arange(K, device=DEV) < n, ids, -1).to(torch.int32)
    dloss = torch.rand(rows, device=DEV, generator=g, dtype=torch.float32) + 0.5
    return dict(case=case, logits=logits.requires_grad_(case["form"] != "both"), ids=ids, teacher=teacher, dloss=dloss)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"attention": _run_attention, "inference": _run_inference, "norm": _run_norm, "distil": _run_distil}[s["case"]["kind"]](s)


def _hidden(q_pos, k_pos, causal, prefix, seg, bias):
    """Hidden pairs ``(B | 1, 1, Sq, Sk)``, or None."""
    m = None
    if causal:
        m = (k_pos[None] > q_pos[:, None])[None, None]
        if prefix is not None:
            m = m & (k_pos[None, None, None] >= prefix[:, None, None, None])
    if seg is not None:
        d = (seg[:, :, None] != seg[:, None, :])[:, None]
        m = d if m is None else m | d
    if bias is not None:
        m = bias < -1e30 if m is None else m | (bias < -1e30)
    return m


def _plain_scores(q, k, cap, slopes, distance, hidden):
    """Shaped scores ``(B, H, Sq, Sk)`` and the tanh in them (or None); ``q, k (B, H, S, D)`` in 32 bits."""
    x, t = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(q.shape[3])), None
    if cap:
        t = x.div_(cap).tanh_()
        x = t * cap
    if slopes is not None:
        x = x.sub_(slopes[:, None, None] * distance)
    if hidden is not None:
        x = x.masked_fill_(hidden, -math.inf)
    return x, t


def _plain_softmax(x):
    """Probabilities of each row; all 0 in a row that sees nothing."""
    x = x.sub_(x.amax(3, keepdim=True).clamp_min(-3e38)).exp_()
    return x.div_(x.sum(3, keepdim=True).clamp_min(1e-30))


def _run_attention(s):
    case, kw = s["case"], s["kw"]
    if own:
        import ringattention_b200 as rab

        if not case["grad"]:
            with torch.no_grad():
                return rab.ringattention(s["q"], s["k"], s["v"], s["bias"], s["seg"], blockwise_kwargs=kw)
        out = rab.ringattention(s["q"], s["k"], s["v"], s["bias"], s["seg"], blockwise_kwargs=kw)
        return dict(out=out, grads=torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    with torch.no_grad():
        q, k, v, g = (t.float().transpose(1, 2) for t in (s["q"], s["k"], s["v"], s["dout"]))
        at = torch.arange(case["S"], device=DEV)
        x, t = _plain_scores(q, k, case["cap"], kw["alibi_slopes"], (at[:, None] - at[None]).abs().float() if case["slopes"] else None,
                             _hidden(at, at, case["causal"], kw["prefix_lens"], s["seg"], s["bias"]))
        p = _plain_softmax(x)
        out = (p @ v).transpose(1, 2).to(torch.bfloat16)
        if not case["grad"]:
            return out
        dv = p.transpose(2, 3) @ g
        dp = g @ v.transpose(2, 3)
        ds = dp.sub_((dp * p).sum(3, keepdim=True)).mul_(p)
        if t is not None:
            ds = ds.mul_(1 - t * t)
        ds = ds.mul_(1.0 / math.sqrt(case["D"]))
        grads = ds @ k, ds.transpose(2, 3) @ q, dv
        return dict(out=out, grads=tuple(x.transpose(1, 2).to(torch.bfloat16) for x in grads))


def _run_inference(s):
    case = s["case"]
    if own:
        import ringattention_b200 as rab

        with torch.no_grad():
            return rab.ringattention_inference(s["q"], s["k"], s["v"], s["mask"], logit_cap=case["cap"] or None, alibi_slopes=s["slopes"],
                                               query_pos=s["pos"])
    q, k, v = (t.float().transpose(1, 2) for t in (s["q"], s["k"], s["v"]))
    distance = None
    if case["slopes"]:
        pos = torch.as_tensor(s["pos"], device=DEV).reshape(-1, 1, 1, 1) + torch.arange(case["Q"], device=DEV)[None, None, :, None]
        distance = (pos - torch.arange(case["S"], device=DEV)).abs().float()
    x, _ = _plain_scores(q, k, case["cap"], s["slopes"], distance, None if s["mask"] is None else ~s["mask"])
    return (_plain_softmax(x) @ v).transpose(1, 2).to(torch.bfloat16)


def _plain_turn(x, cos, sin):
    """Pairs (i, i + D/2) turned by the angle of their position."""
    n = x.shape[-1] // 2
    a, b = x[..., :n], x[..., n:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_norm(x, gain, cos, sin):
    n = x.float()
    n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + 1e-6)
    return _plain_turn(n * gain.float(), cos, sin).to(torch.bfloat16)


def _plain_norm_grads(x, gain, dy, cos, sin):
    """The rotation's inverse, then ``dx = r (w - n mean(w n))`` with ``r = 1/rms``, ``n = r x`` and ``w = gain dn``."""
    g, n = _plain_turn(dy.float(), cos, -sin), x.float()
    r = torch.rsqrt(n.square().mean(-1, keepdim=True) + 1e-6)
    n = n * r
    w = g * gain.float()
    return (r * (w - n * (w * n).mean(-1, keepdim=True))).to(torch.bfloat16), (g * n).double().sum((0, 1, 2)).to(gain.dtype)


def _run_norm(s):
    case = s["case"]
    if own:
        import ringattention_b200 as rab

        if not case["grad"]:
            with torch.no_grad():
                return rab.qk_norm_rope(s["q"], s["k"], s["gq"], s["gk"], s["pos"], theta=500000.0)
        out = rab.qk_norm_rope(s["q"], s["k"], s["gq"], s["gk"], s["pos"], theta=500000.0)
        return dict(out=out, grads=torch.autograd.grad(out, (s["q"], s["k"], s["gq"], s["gk"]), (s["dq"], s["dk"])))
    with torch.no_grad():
        D = case["D"]
        angle = s["pos"].double()[:, :, None, None] * 500000.0 ** (-2.0 * torch.arange(D // 2, device=DEV, dtype=torch.float64) / D)
        cos, sin = angle.cos().float(), angle.sin().float()
        out = _plain_norm(s["q"], s["gq"], cos, sin), _plain_norm(s["k"], s["gk"], cos, sin)
        if not case["grad"]:
            return out
        (dq, dgq), (dk, dgk) = _plain_norm_grads(s["q"], s["gq"], s["dq"], cos, sin), _plain_norm_grads(s["k"], s["gk"], s["dk"], cos, sin)
        return dict(out=out, grads=(dq, dk, dgq, dgk))


def _run_distil(s):
    case = s["case"]
    rows, T = case["rows"], case["T"]
    if own:
        import ringattention_b200 as rab

        if case["form"] == "both":
            loss, grad = rab.distillation_loss_and_grad(s["logits"], s["ids"], s["teacher"], temperature=T, grad_scale=1.0 / rows)
            return dict(loss=loss, grad=grad)
        if case["form"] == "mean":
            loss = rab.distillation_loss(s["logits"], s["ids"], s["teacher"], temperature=T)
            return dict(loss=loss, grad=torch.autograd.grad(loss, s["logits"])[0])
        loss = rab.distillation_loss(s["logits"], s["ids"], s["teacher"], temperature=T, reduction="none")
        return dict(loss=loss, grad=torch.autograd.grad(loss, s["logits"], s["dloss"])[0])
    with torch.no_grad():
        there = s["ids"] >= 0
        ids = s["ids"].long().clamp_min(0)
        some = there.any(1)
        x = s["logits"].float() / T
        x = x - x.amax(1, keepdim=True)
        e = x.exp()
        z = e.sum(1, keepdim=True)
        u = (s["teacher"].float() / T).masked_fill(~there, -math.inf)
        u = u - u.amax(1, keepdim=True).clamp_min(-3e38)
        p = u.exp()
        w = p.sum(1, keepdim=True).clamp_min(1e-30)
        p = p / w
        # log p - log q at the teacher's entries
        d = (u - x.gather(1, ids)) - (w / z).log()
        loss = torch.where(some, T * T * (p * d.masked_fill(~there, 0.0)).sum(1), 0.0)
        scale = {"both": torch.full((rows,), 1.0 / rows, device=DEV), "mean": (1.0 / some.sum().clamp_min(1)).expand(rows), "loss": s["dloss"]}[case["form"]]
        scale = torch.where(some, scale * T, 0.0)[:, None]
        grad = (e / z * scale).scatter_add_(1, ids, -p * scale).to(s["logits"].dtype)
        return dict(loss=loss.sum() / some.sum().clamp_min(1) if case["form"] == "mean" else loss, grad=grad)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "attention":
        B, S, H, D = case["B"], case["S"], case["H"], case["D"]
        if case["docs"]:
            pairs = B * S * min(min(S, case["docs"]), (S + 1) / 2)  # documents of geometric length: mean n, mean square about 2 n^2
        else:
            pairs = B * S * (S + 1) / 2 if case["causal"] else B * S * S
        rows = B * S * H * D * 2
        return dict(bytes=(8 if case["grad"] else 4) * rows, flops=(14 if case["grad"] else 4) * pairs * H * D)
    if case["kind"] == "inference":
        B, Q, S, H, D = case["B"], case["Q"], case["S"], case["H"], case["D"]
        pairs = {"none": B * Q * S, "valid": B * Q * S * 0.75, "causal": B * Q * (S - (Q - 1) / 2)}[case["mask"]]
        keys = B * S * (0.75 if case["mask"] == "valid" else 1.0)
        return dict(bytes=4 * keys * H * D + 4 * B * Q * H * D, flops=4 * pairs * H * D)
    if case["kind"] == "norm":
        n = case["B"] * case["S"] * (case["H"] + case["G"]) * case["D"]
        return dict(bytes=(8 if case["grad"] else 4) * n, flops=(20 if case["grad"] else 8) * n)
    n, size = case["rows"] * case["V"], 4 if case["wide"] else 2
    return dict(bytes=2 * size * n + case["rows"] * (case["K"] * (4 + size) + 8), flops=6 * n)


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "inference": _exact_inference, "norm": _exact_norm, "distil": _exact_distil}[case["kind"]](case, s)


def _one_head(q, k, v, cap, slope, q_pos, seen, dout=None, rows=2048):
    """One head of one batch row in 64 bits: ``seen(r0, r1)`` tells which keys these query rows see. With ``dout`` the gradients too."""
    scale, k_pos = 1.0 / math.sqrt(q.shape[1]), torch.arange(k.shape[0], device=DEV)
    out, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for r0 in range(0, q.shape[0], rows):
        r1 = min(q.shape[0], r0 + rows)
        x = torch.mm(q[r0:r1], k.t()) * scale
        steep = torch.ones_like(x)  # what a score changes by with the product below it
        if cap:
            steep = torch.cosh(x / cap).pow(-2)
            x = cap * torch.tanh(x / cap)
        if slope:
            x = x - slope * (q_pos[r0:r1, None] - k_pos).abs()
        x = torch.where(seen(r0, r1), x, -math.inf)
        p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)).nan_to_num(nan=0.0)
        out[r0:r1] = p @ v
        if dout is not None:
            g = dout[r0:r1]
            dv.addmm_(p.t(), g)
            ds = p * steep * (g @ v.t() - (g * out[r0:r1]).sum(1, keepdim=True)) * scale
            dq[r0:r1] = ds @ k
            dk.addmm_(ds.t(), q[r0:r1])
    return out, dq, dk, dv


def _exact_attention(case, s):
    B, S, H, D = case["B"], case["S"], case["H"], case["D"]
    got = torch.empty(4, B, S, H, D, device=DEV, dtype=torch.float64)
    at, kw = torch.arange(S, device=DEV), s["kw"]
    for b in range(B):
        def seen(r0, r1):
            m = torch.ones(r1 - r0, S, dtype=torch.bool, device=DEV)
            if case["causal"]:
                m = at <= at[r0:r1, None]
                if case["prefix"]:
                    m = m | (at < kw["prefix_lens"][b])
            if s["seg"] is not None:
                m = m & (s["seg"][b] == s["seg"][b, r0:r1, None])
            if s["bias"] is not None:
                m = m & (s["bias"][b, 0, 0] == 0)
            return m
        for h in range(H):
            slope = float(kw["alibi_slopes"][h]) if case["slopes"] else 0.0
            r = _one_head(*(t[b, :, h].double() for t in (s["q"], s["k"], s["v"])), case["cap"], slope, at, seen,
                          s["dout"][b, :, h].double() if case["grad"] else None)
            for i in range(4 if case["grad"] else 1):
                got[i, b, :, h] = r[i]
    return dict(out=got[0], grads=(got[1], got[2], got[3])) if case["grad"] else got[0]


def _exact_inference(case, s):
    B, Q, S, H, D = case["B"], case["Q"], case["S"], case["H"], case["D"]
    got = torch.empty(B, Q, H, D, device=DEV, dtype=torch.float64)
    for b in range(B):
        first = s["pos"] if isinstance(s["pos"], int) else int(s["pos"][b])
        m = torch.ones(Q, S, dtype=torch.bool, device=DEV) if s["mask"] is None else s["mask"][b if s["mask"].shape[0] > 1 else 0, 0]
        for h in range(H):
            slope = float(s["slopes"][h]) if case["slopes"] else 0.0
            got[b, :, h] = _one_head(*(t[b, :, h].double() for t in (s["q"], s["k"], s["v"])), case["cap"], slope,
                                     first + torch.arange(Q, device=DEV), lambda r0, r1: m[r0:r1])[0]
    return got


def _exact_norm(case, s):
    """Turned as complex numbers; the gradients by torch's autograd in 64 bits."""
    n = case["D"] // 2
    freq = torch.exp(torch.arange(n, device=DEV, dtype=torch.float64) * (-math.log(500000.0) / n))
    turn = torch.polar(torch.ones(1, device=DEV, dtype=torch.float64), s["pos"].double()[:, :, None, None] * freq)
    leaves = [s[name].detach().double().requires_grad_(case["grad"]) for name in ("q", "k", "gq", "gk")]

    def one(x, gain):
        y = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * gain
        z = torch.complex(*y.split(n, -1)) * turn
        return torch.cat([z.real, z.imag], -1)

    with torch.set_grad_enabled(case["grad"]):
        out = one(leaves[0], leaves[2]), one(leaves[1], leaves[3])
        if not case["grad"]:
            return out
        grads = torch.autograd.grad(out, leaves, (s["dq"].double(), s["dk"].double()))
    return dict(out=tuple(x.detach() for x in out), grads=grads)


def _exact_distil(case, s):
    rows, V, T = case["rows"], case["V"], case["T"]
    loss, grad = torch.zeros(rows, device=DEV, dtype=torch.float64), torch.zeros(rows, V, device=DEV, dtype=torch.float64)
    there = (s["ids"] >= 0).any(1)
    for r0 in range(0, rows, 512):
        at = slice(r0, min(rows, r0 + 512))
        ids, used = s["ids"][at].long(), s["ids"][at] >= 0
        log_q = torch.log_softmax(s["logits"][at].detach().double() / T, 1)
        log_p = torch.log_softmax(torch.where(used, s["teacher"][at].double() / T, -math.inf), 1)
        p = torch.where(used, log_p.exp(), 0.0)
        parts = torch.where(used, p * (log_p - log_q.gather(1, ids.clamp_min(0))), 0.0)
        loss[at] = torch.where(there[at], parts.sum(1) * T * T, 0.0)
        target = torch.zeros_like(log_q).scatter_add_(1, ids.clamp_min(0), p)
        grad[at] = torch.where(there[at, None], (log_q.exp() - target) * T, 0.0)
    n = max(1, int(there.sum()))
    if case["form"] == "mean":
        return dict(loss=loss.sum() / n, grad=grad / n)
    return dict(loss=loss, grad=grad * s["dloss"].double()[:, None] if case["form"] == "loss" else grad / rows)
