"""``GCORE_PDL=0`` switches every overlapped launch off, those outside of a decode chain too."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("env,want", [({}, 1), ({"GCORE_PDL": "1"}, 1), ({"GCORE_PDL": "0"}, 0)])
def test_switch(env, want):
    if not (ROOT / "gcore_b200" / "ops" / "_gk_kernels.so").exists():
        pytest.skip("the kernel library is not built")
    base = {k: v for k, v in os.environ.items() if k != "GCORE_PDL"}
    out = subprocess.run([sys.executable, "-c", "from gcore_b200.ops import _lib; print(_lib.kernels().gk_set_overlap(1))"], cwd=ROOT,
                         env={**base, **env}, check=True, capture_output=True, text=True).stdout
    assert int(out.split()[-1]) == want
