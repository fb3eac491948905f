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


def test_an_append_of_as_many_rows_as_an_int32_counts():
    """Rows that are all one row; only the last two are stored, at the list's very end."""
    n = 0x7FFFFFFF
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    cache = gqa.paged_cache(1, 64, dtype=torch.int8, kv_heads=1)
    row = torch.full((1, 1, 128), 3.0, dtype=torch.bfloat16, device="cuda").expand(n, 1, 128)
    slots = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    slots[n - 2], slots[n - 1] = 8, 9
    gqa.append_paged(cache, row, row, slots)
    k, _ = gqa.read_paged(cache, ints([7, 8, 9, 10], torch.int64))
    assert k[:, 0, 0].tolist() == [0.0, 3.0, 3.0, 0.0]
    del slots, row
    torch.cuda.empty_cache()
