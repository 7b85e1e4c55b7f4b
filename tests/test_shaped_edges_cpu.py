"""Shaped attention at its edges without a GPU: query positions far away, plans and what they refuse, rings of the PyTorch path."""
import pytest
import torch
from shaped_plain import attention

import ringattention_b200 as rab


def _rand(B, S, H, D, n=3, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, S, H, D, generator=g, dtype=torch.float64).to(dtype) for _ in range(n)]


@pytest.mark.parametrize("pos", [2 ** 29, 2 ** 30 - 1, torch.tensor([2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32), torch.tensor([2 ** 62, -(2 ** 62)])])
def test_queries_beyond_either_end_of_the_cache(pos):
    """In 32 bits as in 64 bits from the end of the cache on: 50 keys, slopes up to 0.5, so 2^-24 of scores up to 25 and a few roundings of sums."""
    B, Q, S, H, D = 2, 3, 50, 2, 8
    q, k, v = _rand(B, S, H, D)
    q, slopes = q[:, :Q], torch.tensor([0.5, 0.1])
    got = rab.ringattention_inference(q, k, v, logit_cap=5.0, alibi_slopes=slopes, query_pos=pos)
    rows = torch.as_tensor(pos).long().reshape(-1, 1) + torch.arange(Q)
    dist = rows.clamp(0, S - 1)[:, None, :, None] - torch.arange(S)
    want, _ = attention(q, k, v, 5.0, slopes, dist, None, torch.ones(B, 1, Q, S, dtype=torch.bool))
    assert torch.allclose(got.double(), want, atol=2e-5)
