"""GPU tests of differential attention's rows that see nothing: 0, whatever their lambda or the norm's weight is."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from test_paged_gpu import Setup, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,lens", [([70, 3, 130], [300, 9000, 130]), ([5, 4, 6], [3000, 20000, 20]), ([2], [30])])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("norm", [False, True])
def test_rows_that_see_nothing_are_0_whatever_their_lambda(counts, lens, value, norm):
    s = Setup(lens, seed=len(lens), page_len=64, code="e4m3")
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    rows = first[-1]
    q = s.queries(rows)
    starts = torch.zeros(rows, dtype=torch.int32, device="cuda")
    empty = torch.arange(rows, device="cuda") % 3 == 1
    starts[empty] = 1 << 30
    lam = torch.rand(rows, 16, generator=s.gen, device="cuda")
    gain = torch.ones(128, device="cuda") if norm else None
    args = (q, s.cache, ints(s.table), ints(lens), ints(first))
    want = gqa.decode_paged_diff_chunked(*args, lam, norm_weight=gain, doc_starts=starts)
    assert not want[empty].any() and bool(want[~empty].isfinite().all())
    lam[empty] = value
    got = gqa.decode_paged_diff_chunked(*args, lam, norm_weight=gain, doc_starts=starts)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    if norm:
        got = gqa.decode_paged_diff_chunked(*args, lam, norm_weight=torch.full_like(gain, value), doc_starts=starts)
        assert not got[empty].any() and not bool(got[~empty].isfinite().any())


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_sequences_without_keys_are_0_whatever_their_lambda(value):
    lens = [0, 40, 0, 5]
    s = Setup(lens, seed=4, page_len=16, code="int8")
    lam = torch.full((4, 16), value, device="cuda")
    lam[1], lam[3] = 0.5, 0.25
    got = gqa.decode_paged_diff(s.queries(4), s.cache, ints(s.table), ints(lens), lam, norm_weight=torch.ones(128, device="cuda"))
    assert not got[0].any() and not got[2].any() and bool(got[1].isfinite().all()) and bool(got[3].isfinite().all())
