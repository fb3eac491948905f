"""GPU tests of the paged 8-bit cache at the ends of its accepted arguments, each through every kernel that takes the
call: one token a sequence, a few queries a sequence (at most 6 rows of one on average, 12 in all) and chunks."""
from __future__ import annotations

import pytest
import torch

import attention_accelerator_b200 as gqa
from test_paged_gpu import ints

pytestmark = pytest.mark.gpu


def test_the_longest_slot_list():
    """As many entries as an int32 counts: the list is filled to its end, and nothing before its start."""
    n = 0x7FFFFFFF
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    table, free = ints([[0, -1]]), ints([5, 6, 7])
    plan = gqa.plan_pages(ints([30]), ints([2]), table, free, ints([0]), page_len=64, max_tokens=n)
    assert plan.counts.tolist() == [2, 0, 0, 0] and plan.slots[:3].tolist() == [30, 31, -1]
    assert plan.positions[:3].tolist() == [30, 31, -1]
    for at in range(0, n, 1 << 28):
        assert int((plan.slots[max(2, at):at + (1 << 28)] != -1).sum()) == 0
        assert int((plan.positions[max(2, at):at + (1 << 28)] != -1).sum()) == 0
    del plan
    torch.cuda.empty_cache()
