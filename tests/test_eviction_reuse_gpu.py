"""GPU tests of a budget of keys over the life of a server: rows of the batch that are used again, parts of a batch."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import _lib
from oracle import paged as ref
from test_eviction_gpu import random_state
from test_paged_gpu import THETA, ints, rows_of

pytestmark = pytest.mark.gpu


# ---- a row's next request -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("scale", [1, 700])
def test_planning_forgets_what_was_evicted_from_ended_and_new_requests(scale, in_place):
    lens, new = [0, 5, 30, 7, 0, 0], [3 * scale, -1, 2 * scale, 0, 0, -1]
    requests, width = len(lens), 150
    w = gqa.key_weights(requests, width * 16, kv_heads=1)
    table = torch.arange(requests * width, dtype=torch.int32, device="cuda").view(requests, width)
    free, n_free = torch.arange(2000, 3000, dtype=torch.int32, device="cuda"), ints([900])
    for room, status in ((5 * scale - 1, _lib.GQA_ERR_PAGES), (5 * scale, _lib.GQA_OK)):
        w.evicted.copy_(ints([9] * requests))
        ln = ints(lens)
        out = dict(lens_out=ln, n_free_out=n_free) if in_place else {}
        plan = gqa.plan_pages(ln, ints(new), table.clone(), free.clone(), n_free, page_len=16, max_tokens=room, weights=w, **out)
        assert int(plan.counts[3]) == status
        if status:
            assert plan.lens.tolist() == lens and w.evicted.tolist() == [9] * requests
        else:
            assert plan.lens.tolist() == [3 * scale, 0, 30 + 2 * scale, 7, 0, 0]
            assert w.evicted.tolist() == [0, 0, 9, 9, 0, 0]


def test_planning_refuses_other_weights():
    table, free = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.arange(8, dtype=torch.int32, device="cuda")
    for w in (gqa.key_weights(3, 64), gqa.key_weights(2, 64, device=torch.device("cpu"))):
        with pytest.raises(ValueError, match="weights.evicted"):
            gqa.plan_pages(ints([0, 0]), ints([1, 1]), table, free, ints([8]), page_len=16, max_tokens=2, weights=w)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_the_next_request_in_a_row_that_was_cut(code):
    """A request is cut and ends; the next one in its row is stored at its own positions and answered as in a cache of its
    own, and as 64-bit attention over the rows that it was given."""
    gen = torch.Generator("cuda").manual_seed(3)
    page_len, width, budget = 16, 24, 48
    top = ref.CODE_MAX[code]

    def rows(n, heads):
        return torch.randn(n, heads, 128, generator=gen, device="cuda").to(torch.bfloat16)

    class Server:
        def __init__(self):
            self.cache = gqa.paged_cache(2 * width, page_len, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn)
            self.weights = gqa.key_weights(2, width * page_len)
            self.table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
            self.free, self.n_free = torch.arange(2 * width, dtype=torch.int32, device="cuda"), ints([2 * width])
            self.lens = ints([0, 0])

        def append(self, new, k, v):
            total = sum(max(0, n) for n in new)
            plan = gqa.plan_pages(self.lens, ints(new), self.table, self.free, self.n_free, page_len=page_len, max_tokens=total,
                                  lens_out=self.lens, n_free_out=self.n_free, weights=self.weights)
            owner = torch.searchsorted(plan.first_token[1:], torch.arange(total, dtype=torch.int32, device="cuda"), right=True)
            gqa.append_paged(self.cache, k, v, plan.slots, positions=plan.positions + self.weights.evicted[owner])

    used, fresh = Server(), Server()
    prompt = [rows(300, h) for h in (8, 8, 32)]
    used.append([200, 100], *prompt[:2])
    gqa.add_key_weights(torch.cat([prompt[2][184:200], prompt[2][284:300]]), used.cache, used.table, used.lens,
                        ints([0, 16, 32]), used.weights, known=ints([0, 0]))
    plan = gqa.plan_eviction(used.weights, used.lens, ints([budget, budget]), used.table, used.free, used.n_free,
                             page_len=page_len, max_keep=budget, lens_out=used.lens, n_free_out=used.n_free)
    gqa.evict_paged(used.cache, used.table, used.weights, plan)
    assert used.weights.evicted.tolist() == [152, 52]
    used.append([-1, 1], rows(1, 8), rows(1, 8))
    assert used.weights.evicted.tolist() == [0, 52]

    k, v, q = rows(100, 8), rows(100, 8), rows(100, 32)
    k1, v1, q1 = rows(1, 8), rows(1, 8), rows(1, 32)
    other = rows(1, 8)
    got = []
    for server, at in ((used, 0), (fresh, 0)):
        server.append([100, 0], k, v)
        gqa.add_key_weights(q[84:], server.cache, server.table[:1], server.lens[:1], ints([0, 16]), server.weights[:1],
                            known=ints([0]))
        server.append([1, 1], torch.cat([k1, other]), torch.cat([v1, other]))
        out = gqa.decode_paged_weights(q1, server.cache, server.table[:1], server.lens[:1], server.weights[:1])
        got.append((out, server.weights.weight[0, :, :101].clone(), server.weights.position[0, :, :101].clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)

    # The rows as they are held: half a code of what was given, a whole one where a page's scale grew behind them.
    p = np.arange(101)
    page = used.table[0].cpu().numpy()[p // page_len]
    held = []
    for c, s, given, new in ((used.cache.k, used.cache.k_scale, k, k1), (used.cache.v, used.cache.v_scale, v, v1)):
        scale = s.cpu().numpy().astype(np.float64)[page][..., None]
        held.append(ref.code_values(rows_of(used.cache, c)[page, p % page_len], code) * scale)
        want = torch.cat([given, new]).double().cpu().numpy()
        if given is k:
            want = ref.rope(want, p, THETA)
        step = scale if code == "int8" else np.maximum(2.0 ** -3 * np.abs(want), 2.0 ** -9 * scale)
        assert np.all(np.abs(held[-1] - want) <= 1.1 * step + 2.0 ** -18 * scale * top)
    x = ref.rope(q1.double().cpu().numpy(), np.array([100]), THETA)[0]
    want, size, most = ref.attend(x, *held, 0, np.ones(101, bool), scale=1 / math.sqrt(128))
    out = got[0][0][0].float().cpu().numpy()
    assert np.all(np.abs(out - want) <= 2.0 ** -8 * np.abs(want) + (math.expm1(2 * 2.0 ** -18 * most) + 2.0 ** -17) * size)
    assert bool((got[0][2] == torch.arange(101, device="cuda", dtype=torch.int32)).all())


# ---- parts of a batch ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lo,hi", [(0, 4), (1, 3)])
def test_lens_out_of_the_same_memory(lo, hi):
    """``lens_out`` that is ``lens`` by its memory, as slices of one tensor are: the tokens evicted join the weights' own."""
    lens, keep = [50, 60, 70, 80], [20, 30, 0, 25]
    weight, position, evicted = random_state(0, lens, 2, 96)
    w = gqa.KeyWeights(torch.from_numpy(weight).cuda(), torch.from_numpy(position).cuda(), ints(evicted))
    ln, table = ints(lens), torch.arange(24, dtype=torch.int32, device="cuda").view(4, 6)
    stack, n_free = torch.zeros(24, dtype=torch.int32, device="cuda"), ints([0])
    plan = gqa.plan_eviction(w[lo:hi], ln[lo:hi], ints(keep[lo:hi]), table[lo:hi], stack, n_free, page_len=16, max_keep=32,
                             lens_out=ln[lo:hi], n_free_out=n_free)
    plan.check()
    after = [min(n, k) if k and lo <= r < hi else n for r, (n, k) in enumerate(zip(lens, keep))]
    assert ln.tolist() == after
    assert w.evicted.tolist() == [e + n - a for e, n, a in zip(evicted, lens, after)]
