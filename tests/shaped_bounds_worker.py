"""Run under RINGATTN_B200_BOUNDS_CHECK=1 by test_gpu_shaped_bounds.py: shaped attention, head norms and distillation at ragged shapes, outputs inside
canary-padded buffers; prints one line ``BOUNDS {...}`` with what was found."""
import json
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from bounds_worker import canaries_intact, canary  # noqa: E402
from ringattention_b200.ops import _lib, decode as Dk, distill, flash, inference as I, qknorm  # noqa: E402


def main():
    torch.manual_seed(0)
    dev, bf = "cuda", torch.bfloat16
    rnd = lambda *s: torch.randn(*s, device=dev).to(bf)
    B, H = 2, 3
    slopes = torch.tensor([0.5, 0.25, 0.125], device=dev)
    prefix = torch.tensor([0, 77], device=dev, dtype=torch.int32)
    for D, Sq, Sk in ((128, 300, 777), (64, 129, 255), (64, 1, 1), (128, 130, 5000)):
        q, k, v, do = rnd(B, Sq, H, D), rnd(B, Sk, H, D), rnd(B, Sk, H, D), rnd(B, Sq, H, D)
        keep = torch.rand(B, 1, Sq, Sk, device=dev) < 0.9
        for cap, sl, pre in ((20.0, None, None), (0.0, slopes, prefix), (20.0, slopes, prefix), (0.0, None, prefix)):
            ms = flash.MaskSpec(causal_block_size=1, q_pos=flash.Positions(Sk - Sq), k_pos=flash.Positions(0), logit_cap=cap, slopes=sl, prefix=pre)
            ms.keep_q, ms.keep_k = flash.pack_mask(keep)
            out, lo = canary((B, Sq, H, D), bf), canary((B, Sq, H, D), bf)
            out, lse = flash.flash_fwd(q, k, v, ms, out=out, lse_out=canary((B, H, Sq), torch.float32), out_lo=lo)
            dq_acc = canary((B, Sq, H, D), torch.float32, fill=0.0)
            lse2, delta = flash.flash_bwd_prep(out, do, lse, dq_acc=dq_acc, out_lo=lo)
            flash.flash_bwd(q, k, v, do, lse2, delta, ms, dq_acc, canary((B, Sk, H, D), bf), canary((B, Sk, H, D), bf))
            flash.flash_bwd_run(q, k, v, out, lse, do, ms, canary((B, Sq, H, D), bf), canary((B, Sk, H, D), bf), canary((B, Sk, H, D), bf), out_lo=lo)
        for Q in (1, 2, 4, 8):
            qd, pos = rnd(B, Q, H, D), torch.tensor([Sk - 1, 0], device=dev)
            for cap, sl in ((20.0, None), (None, slopes), (20.0, slopes)):
                for mask in (None, torch.rand(B, 1, Q, Sk, device=dev) < 0.9):
                    shape = I.inference_shape(qd, k, 1, cap, sl, pos)
                    o, l = Dk.decode_partial(qd, k, v, mask=None if mask is None else mask.view(torch.uint8), shape=shape)
                    Dk.merge_partials(o, l, H, Q, out=canary((B, Q, H, D), bf))
    for D, dt in ((64, bf), (128, torch.float32), (256, bf)):
        for B, S, H, G in ((1, 1, 1, 1), (3, 37, 5, 2), (2, 700, 12, 3)):
            q, k, dy, dk = (torch.randn(B, S, n, D, device=dev).to(dt) for n in (H, G, H, G))
            gains = [torch.ones(D, device=dev) for _ in range(2)]
            pos = torch.randint(0, 1 << 20, (B, S), device=dev)
            qknorm.norm_rope_fwd(q, k, *gains, pos, 1e4, 1e-6, canary((B, S, H, D), dt), canary((B, S, G, D), dt))
            got = qknorm.norm_rope_bwd(q, k, *gains, dy, dk, pos, 1e4, 1e-6)
            assert all(t.isfinite().all() for t in got)
    for rows, V, K, dt in ((1, 1, 1, bf), (5, 301, 40, bf), (17, 4097, 1024, torch.float32), (2, 70001, 64, bf)):
        x, t = torch.randn(rows, V, device=dev).to(dt), torch.randn(rows, K, device=dev)
        ids = torch.randint(-2, V + 2, (rows, K), device=dev)
        stats = canary((rows, 2), torch.float32)
        distill.distill_rows(x, ids, t, 2.0, stats=stats, loss=canary((rows,), torch.float32))
        distill.distill_rows(x, ids, t, 2.0, grad=canary((rows, V), dt), loss=canary((rows,), torch.float32))
        distill.distill_rows_bwd(x, ids, t, 2.0, stats, torch.ones(rows, device=dev))
    torch.cuda.synchronize()
    _lib.check_status()
    print("BOUNDS " + json.dumps({"clean": _lib.bounds_report(reset=True), "canaries_intact": canaries_intact()}), flush=True)


if __name__ == "__main__":
    main()
