"""The timing tool's table of low-precision serving runs and reports what it is asked for."""
import json

import pytest

from gcore_b200.tools import kernel_bench

pytestmark = pytest.mark.gpu


def test_low_precision_table(capsys):
    kernel_bench.main(["low_precision", "--only", "rows 64"])
    row, = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    assert row["name"].startswith("rows 64") and 0 < row["us"] < 1000 and 0 < row["fp32_scales"] < 1000
