"""examples/paged_budget.py runs as written, and its keys and pages are accounted for."""
from __future__ import annotations

import importlib.util

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("args", [[], ["--differential", "--dtype", "e4m3", "--page-len", "16", "--budget", "100", "--slack", "1"]])
def test_example(args):
    spec = importlib.util.spec_from_file_location("paged_budget", ROOT / "examples" / "paged_budget.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(["--requests", "9", "--steps", "25", "--prompt", "700", *args])
    assert got["finite"] and got["device_status"] == 0 and got["accounted"]
    assert got["pages_used"] == got["pages_needed"]
    budget, slack = (100, 1) if args else (256, 16)
    assert got["longest"] < budget + slack
