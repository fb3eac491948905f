"""GPU tests of differential attention where its two maps nearly cancel, in all three kernels."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from test_paged_diff_gpu import check_diff
from test_paged_gpu import CHUNK_UNIT, DECODE_UNIT, Setup, ints

pytestmark = pytest.mark.gpu

#: one token a sequence, a few, whole prompts: the one-token, the few-query and the chunked kernel; long ones cross shares
CALLS = [(None, [700, 1, 65, 9000]), ([5, 1, 6, 3], [900, 1, 64, 20000]), ([300, 64, 1], [9000, 64, 20])]


def call(counts, lens, seed, code):
    """Setup, queries, owner and position of each, and the function that makes the call."""
    s = Setup(lens, seed=seed, page_len=64, code=code)
    n = counts or [1] * len(lens)
    first = np.concatenate([[0], np.cumsum(n)]).tolist()
    owner = [b for b, c in enumerate(n) for _ in range(c)]
    pos = [lens[b] - c + i for b, c in enumerate(n) for i in range(c)]

    def run(q, lambdas, **more):
        args = (q, s.cache, ints(s.table), ints(lens))
        if counts is None:
            return gqa.decode_paged_diff(*args, lambdas, **more)
        return gqa.decode_paged_diff_chunked(*args, ints(first), lambdas, **more)

    return s, s.queries(first[-1]), owner, pos, run


@pytest.mark.parametrize("counts,lens", CALLS)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_equal_maps_leave_nothing(counts, lens, code):
    s, q, owner, pos, run = call(counts, lens, 9, code)
    q[:, 1::2] = q[:, 0::2]
    one = torch.ones(16, device="cuda")
    assert not run(q, one).any()
    assert not run(q, one, norm_weight=torch.ones(128, device="cuda")).any()


@pytest.mark.parametrize("counts,lens", CALLS)
@pytest.mark.parametrize("correlation,lam,norm", [(0.98, 0.8, True), (0.999, 0.8, False), (0.999, 1.0, True)])
def test_maps_that_nearly_cancel(counts, lens, correlation, lam, norm):
    """Second maps whose queries are the first ones' but for a little: what is left is off by the maps' own errors -- 22
    bits of their operands in the one-token kernel, an FP16 rounding in the others -- and no more."""
    s, q, owner, pos, run = call(counts, lens, 10, "int8")
    noise = torch.randn(q[:, 0::2].shape, generator=s.gen, device="cuda")
    q[:, 1::2] = (correlation * q[:, 0::2].float() + (1 - correlation ** 2) ** 0.5 * noise).to(torch.bfloat16)
    lambdas = torch.full((16,), lam, device="cuda")
    weight = torch.ones(128, device="cuda") if norm else None
    got = run(q, lambdas, norm_weight=weight)
    pick = sorted(set(range(0, len(owner), max(1, len(owner) // 40))) | {len(owner) - 1})
    check_diff(got[pick], q[pick], s, [owner[i] for i in pick], [pos[i] for i in pick], lambdas,
               unit=DECODE_UNIT if counts is None else CHUNK_UNIT, weight=weight)
