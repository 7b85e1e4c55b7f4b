"""``qk_norm_rope`` and the distillation loss on the CPU, what they refuse, and the layout of their launchers' arguments."""
import re
import struct

import pytest
import torch

import ringattention_b200 as rab


def _qk(B=2, S=5, H=3, G=2, D=8, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    return r(B, S, H, D), r(B, S, G, D), 1 + 0.2 * r(D), 1 + 0.2 * r(D)


def _turned(x, gain, pos, theta=10000.0, eps=1e-6):
    n = x.shape[-1] // 2
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain
    z = torch.complex(y[..., :n], y[..., n:])
    a = pos[..., None, None] * torch.tensor([theta ** (-i / n) for i in range(n)], dtype=torch.float64)
    z = z * torch.exp(1j * a)
    return torch.cat([z.real, z.imag], -1)


def test_norm_and_rotation_in_64_bits():
    q, k, gq, gk = _qk()
    for positions, pos in ((None, torch.arange(5.0)), (9, 9 + torch.arange(5.0)), (torch.arange(5) * 7, torch.arange(5.0) * 7),
                           (torch.arange(10).view(2, 5), torch.arange(10.0).view(2, 5))):
        a, b = rab.qk_norm_rope(q, k, gq, gk, positions)
        assert torch.allclose(a, _turned(q, gq, pos.double()), atol=1e-12) and torch.allclose(b, _turned(k, gk, pos.double()), atol=1e-12)
    leaves = [t[:1, :3].clone().requires_grad_() for t in (q, k)] + [t.clone().requires_grad_() for t in (gq, gk)]
    assert torch.autograd.gradcheck(lambda *x: rab.qk_norm_rope(*x, 3), leaves)


def test_norm_into_given_tensors():
    q, k, gq, gk = _qk(dtype=torch.float32)
    want = rab.qk_norm_rope(q, k, gq, gk)
    cache = torch.zeros(2, 9, 2, 8)
    _, kk = rab.qk_norm_rope(q, k, gq, gk, k_out=cache[:, 2:7])
    assert torch.equal(cache[:, 2:7], want[1]) and kk.data_ptr() == cache[:, 2:7].data_ptr()


@pytest.mark.parametrize("change", [dict(q=torch.zeros(5, 3, 8)), dict(k=torch.zeros(2, 4, 2, 8)), dict(k=torch.zeros(2, 5, 2, 6)), dict(k=torch.zeros(2, 5, 0, 8)),
                                    dict(q=torch.zeros(2, 5, 3, 8, dtype=torch.float64)), dict(q_gain=torch.zeros(7)), dict(k_gain=torch.zeros(8, dtype=torch.float64)),
                                    dict(positions=torch.arange(4)), dict(positions=torch.arange(5.0)), dict(positions=torch.zeros(3, 5, dtype=torch.int32)),
                                    dict(positions=-1), dict(positions=2 ** 31), dict(positions=True), dict(positions="0"), dict(theta=0.0),
                                    dict(theta=float("inf")), dict(eps=-1.0), dict(eps="x"), dict(q_out=torch.zeros(2, 5, 2, 8)),
                                    dict(q_out=torch.zeros(2, 5, 3, 8, dtype=torch.float64))])
def test_what_norm_refuses(change):
    q, k, gq, gk = _qk(dtype=torch.float32)
    with pytest.raises(ValueError):
        rab.qk_norm_rope(**{**dict(q=q, k=k, q_gain=gq, k_gain=gk), **change})


def test_output_views_do_not_go_with_gradients():
    q, k, gq, gk = _qk(dtype=torch.float32)
    with pytest.raises(ValueError):
        rab.qk_norm_rope(q.requires_grad_(), k, gq, gk, q_out=torch.empty_like(q))
    with torch.no_grad():
        rab.qk_norm_rope(q, k, gq, gk, q_out=torch.empty_like(q))


def _logits(rows=4, V=9, K=3, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g, dtype=torch.float64).to(dtype), torch.randint(0, V, (rows, K), generator=g),
            torch.randn(rows, K, generator=g, dtype=torch.float64).to(dtype))


def test_loss_in_64_bits():
    x, ids, t = _logits()
    ids[1, 1], ids[2], ids[3, 0] = -1, -1, 9
    T = 1.7
    want = []
    for r in range(4):
        used = [k for k in range(3) if 0 <= ids[r, k] < 9]
        p = torch.softmax(t[r, used] / T, 0)
        q = torch.softmax(x[r] / T, 0)[ids[r, used]]
        want.append(T * T * (p * (p / q).log()).sum() if used else torch.tensor(0.0))
    want = torch.stack([w.double() for w in want])
    assert torch.allclose(rab.distillation_loss(x, ids, t, temperature=T, reduction="none"), want)
    assert torch.allclose(rab.distillation_loss(x, ids, t, temperature=T), want.sum() / 3)
    assert torch.allclose(rab.distillation_loss(x, ids, t, temperature=T, reduction="sum"), want.sum())
    leaf = x.clone().requires_grad_()
    assert torch.autograd.gradcheck(lambda z: rab.distillation_loss(z, ids, t, temperature=T), (leaf,))
    loss, grad = rab.distillation_loss_and_grad(x, ids, t, temperature=T, grad_scale=0.5)
    g, = torch.autograd.grad(rab.distillation_loss(leaf, ids, t, temperature=T, reduction="sum"), leaf)
    assert torch.allclose(loss, want) and torch.allclose(grad, g * 0.5)
    out = x.clone()
    assert rab.distillation_loss_and_grad(out, ids, t, temperature=T, grad_scale=0.5, out=out)[1] is out and torch.allclose(out, grad)


def test_rows_without_entries_in_plain_pytorch():
    x, ids, t = _logits()
    ids[0], x[0] = -1, float("nan")
    t[1], x[1] = float("-inf"), float("inf")
    leaf = x.clone().requires_grad_()
    loss = rab.distillation_loss(leaf, ids, t, reduction="none")
    g, = torch.autograd.grad(loss.sum(), leaf)
    assert bool((loss[:2] == 0).all()) and bool((g[:2] == 0).all()) and bool(g.isfinite().all())


@pytest.mark.parametrize("change", [dict(teacher_ids=torch.zeros(4, 2, dtype=torch.int64)), dict(teacher_ids=torch.zeros(4, 3)), dict(teacher_ids=torch.zeros(3, 3, dtype=torch.int64)),
                                    dict(logits=torch.zeros(4, 9, dtype=torch.int32)), dict(logits=torch.zeros(5, 9)), dict(temperature=0.0), dict(temperature=-1),
                                    dict(temperature=float("nan")), dict(temperature=True), dict(temperature=float("inf")), dict(logits=torch.zeros(4, 0)),
                                    dict(teacher_logits=torch.zeros(4, 3, requires_grad=True)), dict(reduction="max"),
                                    dict(teacher_ids=torch.zeros(4, 1025, dtype=torch.int32), teacher_logits=torch.zeros(4, 1025)),
                                    dict(logits=torch.zeros(0, 9), teacher_ids=torch.zeros(0, 3, dtype=torch.int32), teacher_logits=torch.zeros(0, 3))])
def test_what_the_loss_refuses(change):
    x, ids, t = _logits(dtype=torch.float32)
    args = {**dict(logits=x, teacher_ids=ids, teacher_logits=t), **change}
    with pytest.raises(ValueError):
        rab.distillation_loss(**args)
    if "reduction" not in args:
        with pytest.raises(ValueError):
            rab.distillation_loss_and_grad(**args)


@pytest.mark.parametrize("module,source,name", [("qknorm", "qk_norm_rope.cu", "RaQkNormArgs"), ("distill", "distill.cu", "RaDistillArgs")])
def test_packed_structures_are_laid_out_as_declared(module, source, name):
    """One code for each field of the C structure, in its order, at offsets that natural alignment gives (nested structures end on 8 bytes)."""
    import importlib

    from ringattention_b200 import _build

    text = re.sub(r"//[^\n]*", "", (_build.CSRC / source).read_text())
    code = {"int": "i", "long long": "q", "float": "f", "double": "d"}

    def fields(struct_name):
        body, out = re.search(r"struct " + struct_name + r"\s*\{(.*?)\};", text, re.S).group(1), ""
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            kind = re.match(r"(?:const\s+)?(long long|\w+)", decl).group(1)
            out += fields(kind) + "0P" if kind.startswith("Ra") else "".join("P" if "*" in one else code[kind] for one in decl.split(","))
        return out

    have = getattr(importlib.import_module(f"ringattention_b200.ops.{module}"), "_ARGS")
    spell = lambda fmt: "".join(c * int(n) if n and n != "0" else (n + c) for n, c in re.findall(r"(\d*)([a-zA-Z])", fmt))
    assert spell(have.format) == fields(name)
    assert have.size == struct.calcsize("@" + fields(name) + "0P")


def test_memory_that_outputs_may_have():
    from ringattention_b200.ops import _lib

    buf = torch.zeros(2, 5, 7, 8)  # queries, keys and values of one projection
    q, k = buf[:, :, :3], buf[:, :, 3:5]
    assert _lib.apart(q, k) and _lib.apart(k, q) and _lib.apart(q[:, 1:2], k[:, 1:2]) and _lib.apart(q, torch.zeros(2, 5, 2, 8))
    assert not _lib.apart(q, buf[:, :, 2:4]) and not _lib.apart(q, q) and not _lib.apart(buf[:, 1:], buf[:, :4]) and not _lib.apart(q, buf.flatten()[40:200])
    cache = torch.zeros(2, 2, 3, 9, 8)  # keys and values, heads before rows
    assert _lib.apart(cache[:, 0].permute(0, 2, 1, 3)[:, 3:4], cache[:, 0].permute(0, 2, 1, 3)[:, 4:5])
    assert _lib.apart(buf[0, 0, :, :4], buf[0, 0, :, 4:]) and not _lib.apart(buf[0, 0, :, :5], buf[0, 0, :, 4:])
    assert _lib.writable(q) and _lib.writable(cache.permute(0, 3, 2, 1, 4)) and not _lib.writable(q[:, :1].expand(2, 5, 3, 8))
    assert not _lib.writable(torch.zeros(20).as_strided((4, 8), (4, 1))) and _lib.writable(torch.zeros(1).expand(1))


def test_outputs_that_overlap_are_refused():
    buf = torch.randn(2, 5, 9, 8)
    q, k, g = buf[:, :, :3], buf[:, :, 3:5], torch.ones(8)
    for bad in (dict(q_out=k[:, :, :1].expand_as(q)), dict(q_out=buf[:, :, 2:5]), dict(k_out=buf[:, :, 2:4]), dict(q_out=buf[:, :, 6:], k_out=buf[:, :, 5:7])):
        with pytest.raises(ValueError, match="overlaps"):
            rab.qk_norm_rope(q, k, g, g, **bad)
    with pytest.raises(ValueError, match="overlaps"):
        rab.qk_norm_rope(q, q, g, g, q_out=q)
    want = rab.qk_norm_rope(q, k, g, g)
    rab.qk_norm_rope(q, k, g, g, q_out=q, k_out=buf[:, :, 5:7])
    assert torch.equal(q, want[0]) and torch.equal(buf[:, :, 5:7], want[1])


def test_calls_run_on_their_tensors_device(monkeypatch):
    """With the tensors on another device than the current one, every entry point makes theirs the current one, once."""
    from ringattention_b200 import api

    entered = []

    class Device:
        def __init__(self, device):
            entered.append(device)

        def __enter__(self):
            monkeypatch.setattr(api, "_elsewhere", lambda x: False)

        def __exit__(self, *a):
            monkeypatch.setattr(api, "_elsewhere", lambda x: True)

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(api, "_elsewhere", lambda x: True)
    q, k, gq, gk = _qk(dtype=torch.float32)
    x, ids, t = _logits(dtype=torch.float32)
    buf, kb, y = q.clone(), k.clone(), x.clone()
    calls = [lambda: rab.qk_norm_rope(q, k, gq, gk, 3, theta=100.0, eps=1e-3, q_out=buf, k_out=kb), lambda: rab.distillation_loss(x, ids, t, temperature=2.0, reduction="sum"),
             lambda: rab.distillation_loss_and_grad(x, ids, t, temperature=2.0, grad_scale=0.5, out=y),
             lambda: rab.ringattention(q, q, q, blockwise_kwargs=dict(causal_block_size=1, query_chunk_size=5, key_chunk_size=5, logit_cap=2.0)),
             lambda: rab.ringattention_inference(q, q, q, torch.ones(2, 1, 5, 5, dtype=torch.bool), logit_cap=3.0, alibi_slopes=torch.ones(3), query_pos=7)]
    got = [f() for f in calls]
    assert len(entered) == len(calls)
    monkeypatch.setattr(api, "_elsewhere", lambda x: False)
    for f, a in zip(calls, got):
        b = f()
        assert all(torch.equal(u, v) for u, v in zip(a, b)) if isinstance(a, tuple) else torch.equal(a, b)
