"""Run by test_gpu_distill_edges.py under RINGATTN_B200_BOUNDS_CHECK: distillation at a high temperature with outputs inside canary-padded buffers; prints
one line ``BOUNDS {...}`` with what was found."""
import json
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from bounds_worker import canaries_intact, canary  # noqa: E402
from ringattention_b200.ops import _lib, distill  # noqa: E402


def main():
    dev = "cuda"
    for rows, V, K, dt in ((1, 1, 1, torch.bfloat16), (5, 301, 200, torch.bfloat16), (17, 2047, 1024, torch.float32), (300, 1024, 1024, torch.bfloat16)):
        x, t = torch.randn(rows, V, device=dev).to(dt), torch.randn(rows, K, device=dev)
        ids = torch.randint(-2, V + 2, (rows, K), device=dev)
        stats = canary((rows, 2), torch.float32)
        distill.distill_rows(x, ids, t, 20.0, stats=stats, loss=canary((rows,), torch.float32))
        distill.distill_rows(x, ids, t, 20.0, grad=canary((rows, V), dt), loss=canary((rows,), torch.float32))
        distill.distill_rows_bwd(x, ids, t, 20.0, stats, torch.ones(rows, device=dev))
    torch.cuda.synchronize()
    _lib.check_status()
    print("BOUNDS " + json.dumps({"clean": _lib.bounds_report(reset=True), "canaries_intact": canaries_intact()}), flush=True)


if __name__ == "__main__":
    main()
