"""``qk_norm_rope`` at its edges without a GPU: position maps and outputs that are refused."""
import pytest
import torch

import ringattention_b200 as rab
from ringattention_b200.ops.flash import Positions


def _args(S=5):
    return torch.randn(2, S, 3, 8), torch.randn(2, S, 2, 8), torch.ones(8), torch.ones(8)


@pytest.mark.parametrize("bad", [Positions(2 ** 31 - 4), Positions(0, 2 ** 31 - 1, 3), Positions(0, 0, -1), Positions(-(2 ** 31) - 1), Positions(2 ** 40),
                                 Positions(0, 2 ** 40)])
def test_position_maps_beyond_32_bits_are_refused(bad):
    with pytest.raises(ValueError):
        rab.qk_norm_rope(*_args(), bad)


@pytest.mark.parametrize("good", [Positions(2 ** 31 - 5), Positions(0, 2 ** 31 - 2, 3), Positions(7, 90, 0), Positions(-3)])
def test_position_maps_within_32_bits(good):
    x = _args()
    got, want = rab.qk_norm_rope(*x, good), rab.qk_norm_rope(*x, good.tensor(5, "cpu"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_outputs_over_the_gains_or_the_positions_are_refused():
    q, k, gq, gk = _args()
    buf = torch.zeros(q.numel() + 64)
    q_out, k_out = buf[:q.numel()].view(q.shape), buf[:k.numel()].view(k.shape)
    inside, behind = buf[40:48], buf[q.numel():q.numel() + 8]
    for name, out in (("q_out", q_out), ("k_out", k_out)):
        for bad in (dict(q_gain=inside), dict(k_gain=inside), dict(positions=buf.view(torch.int32)[3:8]), dict(positions=buf.view(torch.int64)[3:13].view(2, 5))):
            with pytest.raises(ValueError, match="overlaps"):
                rab.qk_norm_rope(**{**dict(q=q, k=k, q_gain=gq, k_gain=gk), **bad, name: out})
    want = rab.qk_norm_rope(q, k, behind + 1, gk)
    behind += 1
    got = rab.qk_norm_rope(q, k, behind, gk, q_out=q_out)
    assert got[0] is q_out and torch.equal(q_out, want[0])
