"""The serving example runs, gives every page back to somebody, and differs from a BF16 cache by the 8 bits only."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.mark.parametrize("dtype,page_len", [("int8", 16), ("e4m3", 64)])
def test_serving_example(dtype, page_len):
    import paged_serving
    got = paged_serving.main(["--requests", "12", "--steps", "24", "--prompt", "300", "--page-len", str(page_len),
                              "--dtype", dtype, "--check"])
    assert got["finite"] and got["device_status"] == 0
    assert got["pages_used"] + got["pages_free"] == got["pages"]
    # A value is off by half a step, and by as much again when its block's scale grew under it.  With N(0,1) rows the
    # step is about amax / 127 = 0.03 (int8) or a sixteenth of the value (e4m3); the outputs average the values, so
    # the largest of a few thousand differences stays below the largest single value's two half steps over the
    # outputs' RMS, which is about 1 / sqrt(300) of a value's or more: 4 * 0.0625 / (1 / 17) = 4.
    assert got["difference"] < 4.0
