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
