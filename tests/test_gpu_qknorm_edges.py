"""``qk_norm_rope`` at its edges on the kernels."""
import pytest
import torch
from test_gpu_qknorm import _gains, _rand

import ringattention_b200 as rab

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_derivatives_are_refused(which):
    from torch.autograd import forward_ad

    q, g = _rand(1, 3, 2, 64, dtype=torch.bfloat16), _gains(64, torch.float32)
    x = [q, q.clone(), *g]
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="forward mode"):
            rab.qk_norm_rope(*x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            rab.qk_norm_rope(*x)
        with pytest.raises(ValueError):
            rab.qk_norm_rope(*x, q_out=torch.empty_like(q))
        rab.qk_norm_rope(q, q, *g)  # (no tangent here)
