"""Shaped attention, head norms and distillation in the checked build of the kernel library (in a child process), outputs between canaries."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("checked", [True, False])
def test_no_access_out_of_range_and_canaries_survive(checked):
    p = subprocess.run([sys.executable, os.path.join(HERE, "shaped_bounds_worker.py")], capture_output=True, text=True, timeout=900,
                       env=dict(os.environ, RINGATTN_B200_BOUNDS_CHECK="1" if checked else "0"))
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-3000:]
    rep = json.loads([ln for ln in p.stdout.splitlines() if ln.startswith("BOUNDS ")][-1][len("BOUNDS "):])
    assert rep["clean"]["checked"] is checked and rep["clean"]["violations"] == 0, rep["clean"]
    assert rep["canaries_intact"] is True
