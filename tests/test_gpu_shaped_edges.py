"""Shaped attention at its edges on the kernels: prefixes and query positions at the ends of their types, constants that change before the backward
pass, what rounding takes from the output, dropout, shards of two runs and sharded caches."""
import math

import pytest
import torch
from shaped_plain import HALF, SLACK, attention, check, slopes_for, visible
from test_gpu_shaped import _inputs, _rand, _train

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ prefixes
@pytest.mark.parametrize("cbs", [1, 4])
@pytest.mark.parametrize("prefix", [-(2 ** 31), -(2 ** 31) + 130, -1, torch.tensor([torch.iinfo(torch.int64).min, 2 ** 62]),
                                    torch.tensor([-(2 ** 31), 2 ** 31 - 1], dtype=torch.int32)])
def test_prefixes_at_the_ends_of_their_type(cbs, prefix):
    """Far below zero nothing is open, far behind the end everything: over several key tiles, forward and backward."""
    B, S, H, D = 2, 400, 2, 64
    prefix = prefix.to(DEV) if isinstance(prefix, torch.Tensor) else prefix
    for cap in (0.0, 20.0):
        _train(*_inputs(B, S, S, H, D, seed=4), cap, None, prefix, cbs, what=f"cap {cap}")
