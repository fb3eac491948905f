"""GPU tests of eviction from the paged 8-bit cache -- keys' weights, the choice, the move -- against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import _lib
from oracle import paged as ref
from test_paged_gpu import DECODE_UNIT, ODD_LENS, THETA, Setup, check, ints, random_cache, rows_of

pytestmark = pytest.mark.gpu


# ---- the keys' weights -------------------------------------------------------------------------------------------
def some_weights(s, evicted=None, capacity=None):
    """Weights that a program already has: any values, NaN where no row is."""
    n, room = len(s.lens), capacity or len(s.table[0]) * s.page_len
    w = gqa.key_weights(n, room, kv_heads=s.heads)
    w.weight.copy_(torch.rand(w.weight.shape, generator=s.gen, device="cuda"))
    w.position.copy_(torch.randint(0, 1 << 20, w.position.shape, generator=s.gen, device="cuda"))
    for b, length in enumerate(s.lens):
        w.weight[b, :, length:] = math.nan
    if evicted:
        w.evicted.copy_(ints(evicted))
    return w


def exact_weights(s, q, counts, evicted, cap=0.0, scale=1 / math.sqrt(128), q_rotated=False):
    """[batch][heads, length] sums of softmax weights in 64 bits, and bounds of their errors: a weight by e to twice a
    score's, 2^-18 of the sum of the largest |q| times |k| (the 22 bits of Q's two parts, FP32's sums, rotation and
    scale) and 2^-20 of the cap, plus 2^-20 for FP32's exponential, row sum and total."""
    out, at = [], 0
    x = q.double()
    for b, (length, n) in enumerate(zip(s.lens, counts)):
        k = torch.from_numpy(s.values(b)[0]).cuda() if length else torch.zeros(0, s.heads, 128, dtype=torch.float64, device="cuda")
        rows = torch.arange(length - n, length, device="cuda")
        xb = x[at:at + n]
        at += n
        if not q_rotated and n:
            pos = (rows + evicted[b]).cpu().numpy()
            xb = torch.from_numpy(ref.rope(xb.cpu().numpy(), pos, THETA)).cuda()
        total = torch.zeros(s.heads, length, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(total)
        for h in range(s.heads if n and length else 0):
            for g in range(4):
                qh = xb[:, 4 * h + g]
                z = scale * (qh @ k[:, h].T)
                most = abs(scale) * float(qh.abs().max()) * float(k[:, h].abs().sum(-1).max())
                if cap:
                    z = cap * torch.tanh(z / cap)
                z.masked_fill_(torch.arange(length, device="cuda")[None] > rows[:, None], -math.inf)
                w = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)).nan_to_num_(nan=0.0).sum(0)
                total[h] += w
                bound[h] += w * (math.expm1(2 * (2.0 ** -18 * most + 2.0 ** -20 * cap)) + 2.0 ** -20)
        out.append((total, bound))
    return out


def check_weights(s, w, before, want, known, evicted):
    """Every row's weight and position after a call; rows past the lengths as they were."""
    old_weight, old_position = before
    for b, (length, (total, bound)) in enumerate(zip(s.lens, want)):
        row = torch.arange(length, device="cuda")
        start = torch.where(row < known[b], old_weight[b, :, :length].double(), 0.0)
        got = w.weight[b, :, :length].double()
        tol = bound + 2.0 ** -23 * (start + total) + 1e-30
        bad = ~((got - start - total).abs() <= tol)
        assert not bool(bad.any()), (b, int(bad.sum()), float(((got - start - total).abs() / tol).max()))
        assert torch.equal(w.position[b, :, :length], torch.where(row < known[b], old_position[b, :, :length],
                                                                   row + evicted[b]).int())
        assert torch.equal(w.weight[b, :, length:].isnan(), old_weight[b, :, length:].isnan())
        assert torch.equal(w.position[b, :, length:], old_position[b, :, length:])


@pytest.mark.parametrize("page_len", [16, 32, 64, 128])
@pytest.mark.parametrize("code,layout,cap", [("int8", "head_major", 0.0), ("e4m3", "position_major", 5.0),
                                             ("e4m3", "head_major", 0.0)])
def test_decode_weights(page_len, code, layout, cap):
    lens = ODD_LENS
    s = Setup(lens, seed=page_len, page_len=page_len, code=code, layout=layout)
    evicted = [7 * b for b in range(len(lens))]
    w, q = some_weights(s, evicted), s.queries(len(lens))
    s.poison(lambda b, p: False)
    before = w.weight.clone(), w.position.clone()
    got = gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), w, score_cap=cap or None)
    now = [0 if n == 1 else e for n, e in zip(lens, evicted)]
    assert w.evicted.tolist() == now
    check(got, q, s, list(range(len(lens))), [max(0, n - 1) + e if n else -1 for n, e in zip(lens, now)], unit=DECODE_UNIT, cap=cap)
    want = exact_weights(s, q, [1] * len(lens), now, cap)
    check_weights(s, w, before, want, [n - 1 for n in lens], now)
    plain = gqa.decode_paged(q, s.cache, ints(s.table), ints(lens), score_cap=cap or None,
                             query_positions=ints([n - 1 + e for n, e in zip(lens, now)]))
    assert bool(((got.float() - plain.float()).abs() <= 2.0 ** -7 * plain.float().abs() + 2.0 ** -12).all())
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("lens", [[30], [1], [20000], [5000, 1, 700], [90] * 700])
def test_decode_weights_of_few_and_many(lens):
    s = Setup(lens, seed=sum(lens), page_len=64, code="int8", heads=3 if len(lens) > 3 else 8)
    w, q = some_weights(s), s.queries(len(lens))
    before = w.weight.clone(), w.position.clone()
    gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), w)
    check_weights(s, w, before, exact_weights(s, q, [1] * len(lens), [0] * len(lens)), [n - 1 for n in lens], [0] * len(lens))
    again = some_weights(s)
    again.weight.copy_(before[0])
    gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), again)
    for b, n in enumerate(lens):
        assert torch.equal(again.weight[b, :, :n], w.weight[b, :, :n])


COUNTS = [([1], [1]), ([1], [300]), ([64], [8192]), ([5], [5]), ([33, 0, 1, 64, 65], [33, 10, 400, 64, 700]),
          ([257], [257]), ([31, 32, 33, 127, 129], [1000, 32, 500, 127, 200]), ([300, 1, 64], [2000, 1, 64]),
          ([2] * 60, [2 + 17 * i for i in range(60)]), ([700], [5000])]


@pytest.mark.parametrize("counts,lens", COUNTS)
@pytest.mark.parametrize("code,page_len,layout,cap", [("int8", 16, "position_major", 0.0), ("e4m3", 64, "head_major", 0.0),
                                                      ("int8", 128, "head_major", 5.0), ("e4m3", 32, "position_major", 3.0)])
def test_add_key_weights(counts, lens, code, page_len, layout, cap):
    s = Setup(lens, seed=sum(lens), page_len=page_len, code=code, layout=layout)
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    evicted = [3 + b for b in range(len(lens))]
    w, q = some_weights(s, evicted), s.queries(first[-1] + 2)
    s.poison(lambda b, p: False)
    before = w.weight.clone(), w.position.clone()
    known = [n - c for n, c in zip(lens, counts)]
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints(first), w, score_cap=cap or None)
    now = [0 if c and k == 0 else e for c, k, e in zip(counts, known, evicted)]
    assert w.evicted.tolist() == now
    check_weights(s, w, before, exact_weights(s, q, counts, now, cap), known, now)
    again = some_weights(s, evicted)
    for t, x in zip((again.weight, again.position), before):
        t.copy_(x)
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints(first), again, score_cap=cap or None)
    assert torch.equal(again.weight.nan_to_num(), w.weight.nan_to_num())
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("heads", [1, 2, 5])
@pytest.mark.parametrize("known", ["zeros", "some", "all"])
def test_known_rows_and_head_shards(heads, known):
    """Rows that are new although no query is theirs (a prompt of which only the end is looked at), and none that are."""
    lens, counts = [500, 129, 64, 700], [16, 40, 64, 0]
    s = Setup(lens, seed=heads, page_len=32, code="e4m3", heads=heads)
    k = {"zeros": [0, -3, 0, 0], "some": [100, 60, 10, 5], "all": [500, 200, 64, 700]}[known]
    w, q = some_weights(s, [9, 9, 9, 9]), s.queries(120)
    before = w.weight.clone(), w.position.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints([0, 16, 56, 120, 120]), w, known=ints(k), q_rotated=True,
                        scale=-0.05)
    now = [0 if n and x <= 0 else 9 for n, x in zip(counts, k)]
    assert w.evicted.tolist() == now
    want = exact_weights(s, q, counts, now, scale=-0.05, q_rotated=True)
    check_weights(s, w, before, want, [x if n else 10000 for n, x in zip(counts, k)], now)


def test_one_query_a_sequence_agrees_with_decode():
    lens = [700, 65, 1, 130]
    s = Setup(lens, seed=12, page_len=32, code="e4m3")
    q = s.queries(4)
    a, b = some_weights(s), some_weights(s)
    b.weight.copy_(a.weight), b.position.copy_(a.position)
    gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), a)
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints([0, 1, 2, 3, 4]), b)
    assert torch.equal(a.position, b.position)
    assert torch.allclose(a.weight.nan_to_num(), b.weight.nan_to_num(), rtol=2.0 ** -15, atol=0)


def test_a_page_scale_or_query_that_is_no_number_stays_with_its_own():
    """NaN reaches the weights of its sequence and head (a page's scale) or of its row's keys, and no others."""
    lens, counts = [300, 200], [40, 3]
    s = Setup(lens, seed=3, page_len=64, code="int8")
    q = s.queries(43)
    args = (q, s.cache, ints(s.table), ints(lens), ints([0, 40, 43]))
    clean = some_weights(s)
    before = clean.weight.clone()
    gqa.add_key_weights(*args, clean)
    s.cache.k_scale[s.table[0][1], 2] = math.nan
    q[41, 4 * 5 + 1, 7] = math.inf
    w = some_weights(s)
    w.weight.copy_(before)
    gqa.add_key_weights(*args, w)
    for b, n in enumerate(lens):
        for h in range(8):
            same = torch.equal(w.weight[b, h, :n], clean.weight[b, h, :n])
            nan = bool(w.weight[b, h, :n].isnan().any())
            assert nan == ((b, h) in ((0, 2), (1, 5))) and same == (not nan), (b, h)
    assert bool(w.weight[1, 5, 199].isfinite()) and bool(w.weight[1, 5, :199].isnan().all())


@pytest.mark.parametrize("which", ["k_scale", "v_scale", "query"])
def test_a_decode_step_of_what_is_no_number(which):
    """Every key of that sequence and head has a weight of NaN, no other one has; the plan takes them in order."""
    lens = [300, 200, 7]
    s = Setup(lens, seed=3, page_len=64, code="e4m3")
    q = s.queries(3)
    clean, w = some_weights(s), some_weights(s)
    w.weight.copy_(clean.weight)
    gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), clean)
    if which == "query":
        q[0, 4 * 2 + 3, 70] = math.nan
    else:
        getattr(s.cache, which)[s.table[0][1], 2] = math.nan
    gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), w)
    for b, n in enumerate(lens):
        for h in range(8):
            if (b, h) == (0, 2):
                assert bool(w.weight[b, h, :n].isnan().all())
            else:
                assert torch.equal(w.weight[b, h, :n], clean.weight[b, h, :n]), (b, h)
    free = torch.zeros(64, dtype=torch.int32, device="cuda")
    plan = gqa.plan_eviction(w, ints(lens), ints([50, 0, 0]), ints(s.table), free, ints([0]), page_len=64, max_keep=50, sinks=0,
                             recent=0)
    plan.check()
    take = ref.plan_eviction(w.weight.cpu().numpy(), w.position.cpu().numpy(), lens, [0, 0, 0], [50, 0, 0], s.table, [], 64, 64,
                             max_keep=50, sinks=0, recent=0)[1]
    assert np.array_equal(plan.take.cpu().numpy(), take) and plan.lens.tolist() == [50, 200, 7]


def test_a_huge_query_costs_its_neighbours_nothing():
    """Rows of one unit have factors of their own: one of 2^60 beside ordinary ones."""
    lens = [200]
    s = Setup(lens, seed=5, page_len=64, code="e4m3")
    q = s.queries(10)
    w = some_weights(s)
    before = w.weight.clone(), w.position.clone()
    q[3] *= 2.0 ** -60
    q[5, :16] = 0.0
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints([0, 10]), w)
    check_weights(s, w, before, exact_weights(s, q, [10], [0]), [190], [0])


# ---- the choice --------------------------------------------------------------------------------------------------
def random_state(seed, lens, heads, room, *, ties=True):
    rng = np.random.RandomState(seed)
    n = len(lens)
    weight = np.exp(2 * rng.randn(n, heads, room)).astype(np.float32)
    if ties:
        weight = np.where(rng.rand(*weight.shape) < 0.5, np.round(weight), weight).astype(np.float32)
    evicted = rng.randint(0, 50, n)
    position = np.argsort(rng.rand(n, heads, room + 50), -1)[..., :room].astype(np.int32)
    return weight, position, evicted.tolist()


def run_eviction(weight, position, lens, evicted, keep, table, free, capacity, page_len, max_keep, sinks, recent,
                 in_place=False):
    w = gqa.KeyWeights(torch.from_numpy(weight).cuda(), torch.from_numpy(position).cuda(), ints(evicted))
    stack = ints(free + [-7] * (capacity - len(free)))
    ln, n_free = ints(lens), ints([len(free)])
    more = {"lens_out": ln, "n_free_out": n_free} if in_place else {}
    plan = gqa.plan_eviction(w, ln, ints(keep), ints(table), stack, n_free, page_len=page_len, max_keep=max_keep,
                             sinks=sinks, recent=recent, **more)
    if in_place:
        assert plan.lens is ln and plan.evicted is w.evicted and plan.n_free is n_free
    else:
        assert ln.tolist() == lens and w.evicted.tolist() == evicted and n_free.tolist() == [len(free)]
    return plan, stack


@pytest.mark.parametrize("requests,heads,longest,keep,page_len,sinks,recent", [
    (1, 8, 40, 16, 16, 4, 8), (1, 1, 2, 1, 128, 0, 0), (3, 2, 70, 33, 32, 0, 0), (5, 8, 513, 100, 16, 4, 32),
    (64, 3, 300, 257, 64, 2, 16), (2, 2, 9001, 2000, 64, 4, 64), (2, 1, 5000, 4990, 128, 4, 5000), (700, 1, 50, 20, 16, 1, 3)])
def test_plan_matches_the_definition(requests, heads, longest, keep, page_len, sinks, recent):
    rng = np.random.RandomState(requests + keep)
    width = -(-longest // page_len)
    for step in range(2):
        lens = [longest] + [int(rng.randint(0, longest + 1)) for _ in range(requests - 1)]
        weight, position, evicted = random_state(step, lens, heads, width * page_len + step)
        keeps = [keep] + [int(rng.choice([keep, keep // 2, 0, -1, keep * 3])) for _ in range(requests - 1)]
        table = np.arange(requests * width).reshape(requests, width).tolist()
        free, capacity = [requests * width + i for i in range(5)], requests * width + 5
        plan, stack = run_eviction(weight, position, lens, evicted, keeps, table, free, capacity, page_len, keep, sinks, recent,
                                   in_place=step == 1)
        ok, take, after, gone, cuts, rows, given = ref.plan_eviction(
            weight, position, lens, evicted, keeps, table, free, page_len, capacity, max_keep=keep, sinks=sinks, recent=recent)
        assert ok and plan.counts.tolist() == [cuts, rows, given, 0]
        assert plan.lens.tolist() == after and plan.evicted.tolist() == gone and plan.n_free.tolist() == [len(free)]
        assert stack.tolist()[:len(free)] == free
        assert np.array_equal(plan.take.cpu().numpy(), take)
        plan.check()


def test_plan_orders_what_is_no_ordinary_weight():
    """Infinity above all numbers, NaN above it; zeros of either sign and what is negative alike: the lower rows."""
    row = np.array([0.0, -0.0, -3.0, np.nan, 1.0, np.inf, 1e-45, 2.0, 0.0, np.nan, 1.0, 3e38], np.float32)
    for keep in range(1, 12):
        weight = np.tile(row, (1, 2, 2))[:, :, :16].copy()
        position = np.tile(np.arange(100, 116, dtype=np.int32), (1, 2, 1))
        args = ([12], [200], [keep], [[3]])
        plan, _ = run_eviction(weight, position, *args, [], 4, 16, 16, 0, 0)
        take = ref.plan_eviction(weight, position, *args, [], 16, 4, max_keep=16, sinks=0, recent=0)[1]
        assert np.array_equal(plan.take.cpu().numpy(), take), keep
    equal = np.ones((1, 1, 16), np.float32)
    plan, _ = run_eviction(equal, np.arange(16, dtype=np.int32)[None, None].copy(), [16], [0], [5], [[0]], [], 1, 16, 5, 0, 3)
    assert plan.take.tolist() == [[[-1, -1, 13, 14, 15]]]


@pytest.mark.parametrize("why", ["negative", "width", "capacity", "stack"])
def test_plan_refuses_and_changes_nothing(why):
    lens, width, capacity, room = [40, 33, 48], 3, 9, 48
    free = [100, 101]
    if why == "negative":
        lens[1] = -1
    elif why == "width":
        lens[1] = 49
    elif why == "capacity":
        room = 40
    else:
        capacity = 3
    weight, position, evicted = random_state(0, lens, 2, room)
    table = np.arange(9).reshape(3, 3).tolist()
    plan, stack = run_eviction(weight, position, lens, evicted, [10, 10, 10], table, free, capacity, 16, 16, 2, 4)
    assert plan.counts.tolist() == [0, 0, 0, _lib.GQA_ERR_PAGES]
    assert plan.lens.tolist() == lens and plan.evicted.tolist() == evicted and plan.n_free.tolist() == [2]
    assert stack.tolist()[:2] == free and set(stack.tolist()[2:]) <= {-7} and set(plan.take.flatten().tolist()) == {-1}
    with pytest.raises(gqa.GqaError, match="refused"):
        plan.check()


# ---- the move ----------------------------------------------------------------------------------------------------
def move_setup(seed, lens, keep, page_len, code, layout, heads=8, spread=0.5):
    gen = torch.Generator("cuda").manual_seed(seed)
    need = [-(-n // page_len) for n in lens]
    pages, width = sum(need) + 2, max(1, max(need))
    cache = random_cache(gen, pages, page_len, code, layout, heads)
    for s in (cache.k_scale, cache.v_scale):
        s.mul_(torch.exp(spread * torch.randn(s.shape, generator=gen, device="cuda")))
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table = [[-1] * width for _ in lens]
    for b, n in enumerate(need):
        table[b][:n] = [order.pop() for _ in range(n)]
    room = width * page_len
    weight, position, evicted = random_state(seed, lens, heads, room)
    w = gqa.KeyWeights(torch.from_numpy(weight).cuda(), torch.from_numpy(position).cuda(), ints(evicted))
    return cache, table, w


def values64(cache, code):
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        out.append((ref.code_values(rows_of(cache, c).transpose(0, 2, 1, 3), code), s.cpu().numpy().astype(np.float64)))
    return out


@pytest.mark.parametrize("lens,keep,page_len", [([40], 16, 16), ([2], 1, 16), ([300, 17, 16, 200], 100, 16), ([513, 512], 129, 64),
                                                ([700], 65, 128), ([260] * 9, 250, 32), ([1000], 31, 32), ([400], 256, 128)])
@pytest.mark.parametrize("code,layout", [("int8", "head_major"), ("e4m3", "position_major")])
def test_move(lens, keep, page_len, code, layout):
    cache, table, w = move_setup(len(lens) + keep, lens, keep, page_len, code, layout)
    before = values64(cache, code)
    weight, position = w.weight.clone(), w.position.clone()
    free, n_free = torch.full((cache.pages + 4,), -1, dtype=torch.int32, device="cuda"), ints([0])
    plan = gqa.plan_eviction(w, ints(lens), ints([keep] * len(lens)), ints(table), free, n_free, page_len=page_len,
                             max_keep=keep, sinks=1, recent=4)
    gqa.evict_paged(cache, ints(table), w, plan)
    take, after = plan.take.cpu().numpy(), plan.lens.tolist()
    assert after == [min(n, keep) for n in lens]
    for name, (codes, scale), (got, got_scale) in zip("kv", before, values64(cache, code)):
        want, want_scale = codes.copy(), scale.copy()
        ref.evict(want, want_scale, take, after, table, page_len, code)
        # The scale is rounded once more than in 64 bits; codes may go to either side where that moves a half.
        assert np.all(np.abs(got_scale - want_scale) <= 2.0 ** -22 * want_scale), name
        far = got != want
        step = np.maximum(np.abs(got - want), 1e-300)
        near = np.maximum(np.abs(want), 2.0 ** -6) * 2.0 ** -3 if code == "e4m3" else np.ones_like(want)
        assert np.all(step[far] <= near[far] * 1.001), name
        assert far.sum() <= 0.002 * far.size + 2, (name, int(far.sum()), far.size)
    for r in range(len(lens)):
        for h in range(8):
            i = np.flatnonzero(take[r, h] >= 0)
            weight[r, h, i] = weight[r, h, torch.from_numpy(take[r, h, i]).cuda().long()]
            position[r, h, i] = position[r, h, torch.from_numpy(take[r, h, i]).cuda().long()]
    assert torch.equal(w.weight, weight) and torch.equal(w.position, position)


def test_a_move_within_equal_scales_changes_no_code():
    """Rows from blocks of a scale no larger than the new block's: those of the same scale keep their codes, the others of
    the block all of them."""
    cache, table, w = move_setup(3, [64], 32, 16, "int8", "head_major")
    cache.k_scale.fill_(0.5), cache.v_scale.fill_(0.25)
    before = values64(cache, "int8")
    plan = gqa.plan_eviction(w, ints([64]), ints([32]), ints(table), ints([0] * 8), ints([0]), page_len=16, max_keep=32)
    gqa.evict_paged(cache, ints(table), w, plan)
    take = plan.take.cpu().numpy()[0]
    for (codes, scale), (got, got_scale) in zip(before, values64(cache, "int8")):
        assert np.array_equal(scale, got_scale)
        for h in range(8):
            for i in range(32):
                s = take[h, i] if take[h, i] >= 0 else i
                assert np.array_equal(got[table[0][i // 16], h, i % 16], codes[table[0][s // 16], h, s % 16])


def test_move_of_scales_that_are_no_numbers():
    """A NaN block's row makes its new block NaN (codes 0 for it); a block of zeros moves as zeros; the rest is untouched."""
    cache, table, w = move_setup(4, [64], 16, 16, "e4m3", "head_major", heads=2)
    w.weight.zero_()
    w.position.copy_(torch.arange(64, device="cuda").expand(1, 2, 64))
    w.weight[0, :, :13] = 5.0
    w.weight[0, :, 20] = w.weight[0, :, 40] = w.weight[0, :, 63] = 9.0   # rows of three other pages
    cache.k_scale[table[0][1], 0] = math.nan
    cache.v_scale[table[0][2], :] = 2.0 ** -100
    cache.v.view(torch.uint8)[table[0][2]] = 0
    before = values64(cache, "e4m3")
    plan = gqa.plan_eviction(w, ints([64]), ints([16]), ints(table), ints([0] * 8), ints([0]), page_len=16, max_keep=16,
                             sinks=0, recent=0)
    assert plan.take.tolist() == [[[-1] * 13 + [20, 40, 63]] * 2]
    gqa.evict_paged(cache, ints(table), w, plan)
    (k, ks), (v, vs) = values64(cache, "e4m3")
    page = table[0][0]
    assert math.isnan(ks[page, 0]) and not k[page, 0, 13:].any() and np.isfinite(ks[page, 1]) and np.isfinite(vs[page]).all()
    assert np.array_equal(k[page, 0, :13], before[0][0][page, 0, :13])
    assert not v[page, :, 14].any() and v[page, :, 15].any()


# ---- together ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_a_serving_run(code):
    """Prompts, their last tokens' weights, a cut to the budget, then steps that append, attend, add up and cut: every
    output against 64-bit attention over the rows that are held, pages accounted for."""
    gen = torch.Generator("cuda").manual_seed(11)
    requests, page_len, budget, width = 3, 16, 48, 12
    prompts = [150, 40, 97]
    cache = gqa.paged_cache(requests * width, page_len, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn)
    weights = gqa.key_weights(requests, width * page_len)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    free, n_free = torch.arange(requests * width, dtype=torch.int32, device="cuda"), ints([requests * width])
    lens, keep = ints([0] * requests), ints([budget] * requests)

    def rows(n, heads):
        return torch.randn(n, heads, 128, generator=gen, device="cuda").to(torch.bfloat16)

    def append(new):
        total = sum(new)
        plan = gqa.plan_pages(lens, ints(new), table, free, n_free, page_len=page_len, max_tokens=total, lens_out=lens,
                              n_free_out=n_free)
        owner = torch.searchsorted(plan.first_token[1:], torch.arange(total, dtype=torch.int32, device="cuda"), right=True)
        gqa.append_paged(cache, rows(total, 8), rows(total, 8), plan.slots,
                         positions=plan.positions + weights.evicted[owner])
        return plan, rows(total, 32)

    def cut():
        plan = gqa.plan_eviction(weights, lens, keep, table, free, n_free, page_len=page_len, max_keep=budget, sinks=2,
                                 recent=8, lens_out=lens, n_free_out=n_free)
        gqa.evict_paged(cache, table, weights, plan)
        plan.check()
        return plan

    def held():
        """[request] (K, V) values of the rows that are held, from the cache."""
        out = []
        for r, n in enumerate(lens.tolist()):
            p = np.arange(n)
            page = table[r].cpu().numpy()[p // page_len]
            out.append([ref.code_values(rows_of(cache, c)[page, p % page_len], code) *
                        s.cpu().numpy().astype(np.float64)[page][..., None]
                        for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))])
        return out

    plan, q = append(prompts)
    last = torch.cat([q[plan.first_token[r + 1] - 16:plan.first_token[r + 1]] for r in range(requests)])
    gqa.add_key_weights(last, cache, table, lens, ints([0, 16, 32, 48]), weights, known=ints([0] * requests))
    assert torch.allclose(weights.weight.sum(-1), torch.full((requests, 8), 64.0, device="cuda"), rtol=1e-5)
    cut()
    assert lens.tolist() == [48, 40, 48] and weights.evicted.tolist() == [102, 0, 49]
    tokens = list(prompts)
    for step in range(20):
        _, q = append([1] * requests)
        tokens = [n + 1 for n in tokens]
        before = weights.weight.clone()
        length = lens.tolist()
        out = gqa.decode_paged_weights(q, cache, table, lens, weights).float().cpu().numpy()
        kv = held()
        x = ref.rope(q.double().cpu().numpy(), np.array([n - 1 for n in tokens]), THETA)
        for r in range(requests):
            want, size, most = ref.attend(x[r], *kv[r], 0, np.ones(length[r], bool), scale=1 / math.sqrt(128))
            z = 2.0 ** -18 * most
            assert np.all(np.abs(out[r] - want) <= 2.0 ** -8 * np.abs(want) + (math.expm1(2 * z) + 2.0 ** -17) * size)
            gain = weights.weight[r, :, :length[r]].clone()
            gain[:, :length[r] - 1] -= before[r, :, :length[r] - 1]
            assert torch.allclose(gain.sum(-1), torch.full((8,), 4.0, device="cuda"), rtol=1e-4)
            pos = weights.position[r, :, :length[r]]
            assert bool((pos[:, length[r] - 1] == tokens[r] - 1).all())
            for h in range(8):
                p = pos[h].tolist()
                assert len(set(p)) == len(p) and max(p) == tokens[r] - 1
                assert {0, 1} <= set(p) and set(range(tokens[r] - 8, tokens[r])) <= set(p)
        cut()
        now = lens.tolist()
        assert now == [min(n, budget) for n in length]
        assert [n + e for n, e in zip(now, weights.evicted.tolist())] == tokens
        used = sum(-(-n // page_len) for n in now)
        assert n_free.tolist() == [requests * width - used]
        pages = [table[r, i].item() for r in range(requests) for i in range(-(-now[r] // page_len))]
        assert len(set(pages) | set(free[:n_free.item()].tolist())) == requests * width
    assert gqa.read_device_status() == 0


def test_a_captured_step_follows_its_lengths():
    """Decode with weights, plan and move in one graph: replays with other lengths equal the calls one by one, and the
    stream's plain calls in between share nothing that matters."""
    lens, keep, page_len = [300, 200, 129], 128, 64
    cache, table, w = move_setup(9, lens, keep, page_len, "int8", "head_major")
    table, ln, kp = ints(table), ints(lens), ints([keep] * 3)
    q = torch.randn(3, 32, 128, device="cuda").to(torch.bfloat16)
    state = [cache.k, cache.v, cache.k_scale, cache.v_scale, w.weight, w.position, w.evicted, ln]
    start = [t.clone() for t in state]
    free, n_free = torch.zeros(40, dtype=torch.int32, device="cuda"), ints([0])

    def step():
        out = gqa.decode_paged_weights(q, cache, table, ln, w)
        gqa.add_key_weights(q, cache, table, ln, ints_first, w)
        plan = gqa.plan_eviction(w, ln, kp, table, free, n_free, page_len=page_len, max_keep=keep, lens_out=ln)
        gqa.evict_paged(cache, table, w, plan)
        return out, plan.take

    ints_first = ints([0, 1, 2, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, take = step()
        for now in (lens, [200, 128, 1], [0, 300, 64]):
            results = []
            for replay in (True, False):
                for t, x in zip(state, start):
                    t.copy_(x)
                ln.copy_(ints(now))
                if replay:
                    graph.replay()
                    got = out, take
                else:
                    got = step()
                gqa.decode_paged(q, cache, table, ln)
                results.append([x.clone() for x in got] + [t.clone() for t in state])
            for a, b in zip(*results):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    side.synchronize()
    assert gqa.read_device_status() == 0


def test_refusals():
    lens = [40, 30]
    s = Setup(lens, seed=1, page_len=16)
    w, q = some_weights(s), s.queries(2)
    table, ln = ints(s.table), ints(lens)
    small = gqa.key_weights(2, 47)
    for bad, match in [(small, "hold 47 rows"), (gqa.key_weights(3, 48), "3 requests"), (gqa.key_weights(2, 48, kv_heads=4), "4 heads"),
                       (gqa.key_weights(2, 48, device=torch.device("cpu")), "are on cpu")]:
        with pytest.raises(ValueError, match=match):
            gqa.decode_paged_weights(q, s.cache, table, ln, bad)
        with pytest.raises(ValueError, match=match):
            gqa.add_key_weights(q, s.cache, table, ln, ints([0, 1, 2]), bad)
    with pytest.raises(ValueError, match="known"):
        gqa.add_key_weights(q, s.cache, table, ln, ints([0, 1, 2]), w, known=ints([0]))
    with pytest.raises(ValueError, match="first_query"):
        gqa.add_key_weights(q, s.cache, table, ln, None, w)
    with pytest.raises(ValueError, match="first_query"):
        gqa.add_key_weights(q, s.cache, table, ln, ints([0, 2]), w)
    free, n_free, keep = ints([0] * 8), ints([0]), ints([8, 8])
    good = dict(page_len=16, max_keep=8)
    for change, match in [(dict(page_len=24), "page_len"), (dict(max_keep=0), "max_keep"), (dict(sinks=-1), "negative"),
                          (dict(recent=1 << 31), "negative"), (dict(lens_out=ints([0])), "lens_out"),
                          (dict(evicted_out=ints([0, 0], torch.int64)), "evicted_out")]:
        with pytest.raises(ValueError, match=match):
            gqa.plan_eviction(w, ln, keep, table, free, n_free, **{**good, **change})
    with pytest.raises(ValueError, match="keep"):
        gqa.plan_eviction(w, ln, keep[:1], table, free, n_free, **good)
    with pytest.raises(ValueError, match="weights are of"):
        gqa.plan_eviction(gqa.key_weights(3, 48), ln, keep, table, free, n_free, **good)
    plan = gqa.plan_eviction(w, ln, keep, table, free, n_free, **good)
    with pytest.raises(ValueError, match="take"):
        gqa.evict_paged(s.cache, table, w, gqa.EvictionPlan(plan.take[:, :4], plan.lens, None, None, None))
    with pytest.raises(ValueError, match="hold 47 rows"):
        gqa.evict_paged(s.cache, table, small, plan)


@pytest.mark.parametrize("requests,heads,longest,keep", [(1, 8, 131072, 4000), (1, 1, 40000, 39000), (3, 8, 20000, 1),
                                                         (40, 8, 50500, 700), (70, 8, 8200, 4096)])
@pytest.mark.parametrize("kind", ["spread", "equal", "two"])
def test_plan_of_long_requests(requests, heads, longest, keep, kind):
    """Requests whose rows several thread blocks share, and more rows than one keeps on chip, against a stable sort."""
    gen = torch.Generator("cuda").manual_seed(longest)
    page_len = 64
    width = -(-longest // page_len)
    w = gqa.key_weights(requests, width * page_len, kv_heads=heads)
    if kind == "spread":
        w.weight.copy_(torch.exp(3 * torch.randn(w.weight.shape, generator=gen, device="cuda")))
        w.weight[..., ::3] = 1.0
    elif kind == "two":
        w.weight.copy_(torch.randint(0, 2, w.weight.shape, generator=gen, device="cuda"))
    w.position.copy_(torch.arange(width * page_len, device="cuda").flip(0).expand_as(w.position))
    lens = [longest - (r * 977) % (longest // 2) for r in range(requests)]
    free, n_free = torch.full((requests * width,), -1, dtype=torch.int32, device="cuda"), ints([0])
    table = torch.arange(requests * width, dtype=torch.int32, device="cuda").view(requests, width)
    ln = ints(lens)
    plan = gqa.plan_eviction(w, ln, ints([keep] * requests), table, free, n_free, page_len=page_len, max_keep=keep, sinks=3,
                             recent=5)
    plan.check()
    row = torch.arange(width * page_len, device="cuda")
    safe = (w.position < 3) | (w.position >= (ln - 5)[:, None, None])
    mark = w.weight.view(torch.int32).long() + (safe.long() << 32)
    mark = torch.where(row < ln[:, None, None], mark, -1)
    order = torch.sort(mark, dim=-1, descending=True, stable=True).indices[..., :keep]
    stays = torch.zeros_like(mark, dtype=torch.bool).scatter_(-1, order, True)
    stays &= (ln > keep)[:, None, None] | (row < ln[:, None, None])
    for r in range(requests):
        for h in range(0, heads, 3):
            if lens[r] <= keep:
                assert bool((plan.take[r, h] == -1).all())
                continue
            holes, fills = torch.nonzero(~stays[r, h, :keep])[:, 0], torch.nonzero(stays[r, h, keep:])[:, 0] + keep
            want = torch.full((keep,), -1, dtype=torch.int32, device="cuda")
            want[holes] = fills.int()
            assert torch.equal(plan.take[r, h], want), (r, h)


# ---- edges -------------------------------------------------------------------------------------------------------
def test_rows_far_into_large_tensors():
    """Weights and positions past 2^31 elements and 4 GB: the last request and head of a wide state."""
    lens = [70, 130]
    s = Setup(lens, seed=2, page_len=64, code="int8")
    room = 1 << 28
    w = gqa.KeyWeights(torch.empty(2, 8, room, device="cuda"), torch.empty(2, 8, room, dtype=torch.int32, device="cuda"),
                       ints([0, 5]))
    for b, n in enumerate(lens):
        w.weight[b, :, :n] = torch.rand(8, n, generator=s.gen, device="cuda")
        w.position[b, :, :n] = torch.arange(n, device="cuda")
    near = gqa.key_weights(2, 192)
    near.weight[:, :, :130], near.position[:, :, :130] = w.weight[:, :, :130], w.position[:, :, :130]
    near.evicted.copy_(w.evicted)
    q, table, ln = s.queries(6), ints(s.table), ints(lens)
    state = [t.clone() for t in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)]
    results = []
    for x in (w, near):
        for t, before in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), state):
            t.copy_(before)
        out = gqa.decode_paged_weights(q[:2], s.cache, table, ln, x)
        gqa.add_key_weights(q, s.cache, table, ln, ints([0, 4, 6]), x)
        plan = gqa.plan_eviction(x, ln, ints([40, 100]), table, torch.zeros(9, dtype=torch.int32, device="cuda"), ints([0]),
                                 page_len=64, max_keep=100)
        gqa.evict_paged(s.cache, table, x, plan)
        results.append([out, plan.take, x.evicted.clone(), s.cache.k.clone(), s.cache.v_scale.clone()] +
                       [t[b, :, :n].clone() for t in (x.weight, x.position) for b, n in enumerate(lens)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_scores_past_4_gb():
    """A table that could name 2^26 keys: the scores of a step's last heads lie past 4 GB of its workspace."""
    lens = [300]
    s = Setup(lens, seed=6, page_len=128, code="e4m3")
    wide = torch.full((1, (1 << 26) // 128), -1, dtype=torch.int32, device="cuda")
    wide[0, :3] = ints(s.table)[0]
    q = s.queries(1)
    with torch.cuda.stream(torch.cuda.Stream()):
        big = gqa.key_weights(1, 1 << 26)
        a = gqa.decode_paged_weights(q, s.cache, wide, ints(lens), big)
        small = gqa.key_weights(1, 384)
        b = gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), small)
        assert torch.equal(a, b) and torch.equal(big.weight[:, :, :384], small.weight)
        torch.cuda.current_stream().synchronize()


def test_calls_without_queries_or_keys():
    lens = [0, 40, 0]
    s = Setup(lens, seed=2, page_len=16)
    w, q = some_weights(s, [4, 4, 4]), s.queries(3)
    before = [t.clone() for t in (w.weight, w.position, w.evicted)]
    table, ln = ints(s.table), ints(lens)
    gqa.add_key_weights(q, s.cache, table, ln, ints([0, 0, 0, 0]), w)
    gqa.add_key_weights(q[:0], s.cache, table, ln, ints([0, 0, 0, 0]), w)
    gqa.add_key_weights(q, s.cache, table, ln, ints([0, 2, 2, 3]), w)  # queries of sequences without keys
    for t, x in zip((w.weight, w.position, w.evicted), before):
        assert torch.equal(t.nan_to_num(), x.nan_to_num())
    none = ints([0, 0, 0])
    assert not gqa.decode_paged_weights(q, s.cache, table, none, w).any()
    for t, x in zip((w.weight, w.position, w.evicted), before):
        assert torch.equal(t.nan_to_num(), x.nan_to_num())
    plan = gqa.plan_eviction(w, none, ints([8, 8, 8]), table, ints([0] * 8), ints([0]), page_len=16, max_keep=8)
    assert plan.counts.tolist() == [0, 0, 0, 0] and bool((plan.take == -1).all())
    gqa.evict_paged(s.cache, table, w, plan)


def test_lengths_and_queries_that_are_out_of_range():
    """More queries than keys, a length past what the table names, rows of first_query out of order: nothing outside is
    read or written, and what is in range is right."""
    lens = [40, 48, 5]
    s = Setup(lens, seed=8, page_len=16)
    w, q = some_weights(s), s.queries(60)
    before = w.weight.clone(), w.position.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints([0, 3, 5, 60]), w)   # 55 queries of 5 keys
    want = exact_weights(s, torch.cat([q[:5], q[55:60]]), [3, 2, 5], [0, 0, 0])
    check_weights(s, w, before, want, [37, 46, 0], [0, 0, 0])
    marked = w.weight.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints([1000, 48, -7]), ints([0, 3, 5, 9]), w)
    assert torch.equal(w.weight[2].nan_to_num(), marked[2].nan_to_num()) and bool((w.weight[0, :, :40] >= marked[0, :, :40]).all())
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints([70, -4, 50, 20]), w)
    assert gqa.read_device_status() == 0


def test_the_largest_batch():
    lens = [1 + (b * 7) % 40 for b in range(8192)]
    s = Setup(lens, seed=1, page_len=32, code="e4m3", heads=1)
    w, q = some_weights(s), s.queries(8192)
    before = w.weight.clone(), w.position.clone()
    table, ln = ints(s.table), ints(lens)
    gqa.decode_paged_weights(q, s.cache, table, ln, w)
    other = some_weights(s)
    other.weight.copy_(before[0]), other.position.copy_(before[1])
    gqa.add_key_weights(q, s.cache, table, ln, ints(list(range(8193))), other)
    assert torch.allclose(w.weight.nan_to_num(), other.weight.nan_to_num(), rtol=2.0 ** -14, atol=0)
    pick = [0, 1, 4095, 8190, 8191]
    for b in pick:
        assert torch.allclose((w.weight[b, 0, :lens[b]] - torch.where(torch.arange(lens[b], device="cuda") < lens[b] - 1,
                                                                       before[0][b, 0, :lens[b]], 0.0)).sum(),
                              torch.tensor(4.0, device="cuda"), rtol=1e-4)
    free = torch.zeros(20000, dtype=torch.int32, device="cuda")
    plan = gqa.plan_eviction(w, ln, ints([8] * 8192), table, free, ints([0]), page_len=32, max_keep=8, sinks=1, recent=2)
    plan.check()
    assert plan.lens.tolist() == [min(n, 8) for n in lens]
    assert plan.counts.tolist() == [sum(n > 8 for n in lens), sum(max(0, n - 8) for n in lens), sum(n > 32 for n in lens), 0]
    gave = [s.table[b][1] for b in range(8192) if lens[b] > 32]
    assert free[:len(gave)].tolist() == gave
    gqa.evict_paged(s.cache, table, w, plan)
    assert gqa.read_device_status() == 0


def test_some_of_the_requests():
    """Rows 1 and 2 of a state of 4 requests: a slice of it, of the table and of the lengths."""
    lens = [50, 60, 70, 80]
    s = Setup(lens, seed=7, page_len=16)
    w, q = some_weights(s, [1, 2, 3, 4]), s.queries(2)
    before = w.weight.clone(), w.position.clone()
    gqa.decode_paged_weights(q, s.cache, ints(s.table)[1:3], ints(lens)[1:3], w[1:3])
    for b in (0, 3):
        assert torch.equal(w.weight[b].nan_to_num(), before[0][b].nan_to_num()) and torch.equal(w.position[b], before[1][b])
    alone = gqa.KeyWeights(before[0][1:3].contiguous(), before[1][1:3].contiguous(), ints([2, 3]))
    gqa.decode_paged_weights(q, s.cache, ints(s.table)[1:3], ints(lens)[1:3], alone)
    assert torch.equal(alone.weight.nan_to_num(), w.weight[1:3].nan_to_num()) and torch.equal(alone.position, w.position[1:3])


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    setups = [Setup([3000, 200], seed=i, page_len=64, code="int8") for i in (1, 2)]
    states = [(s, some_weights(s), s.queries(80)) for s in setups]
    want = []
    for s, w, q in states:
        copy = gqa.KeyWeights(w.weight.clone(), w.position.clone(), w.evicted.clone())
        table, ln = ints(s.table), ints(s.lens)
        for _ in range(5):
            gqa.add_key_weights(q, s.cache, table, ln, ints([0, 64, 80]), copy)
            out = gqa.decode_paged_weights(q[:2], s.cache, table, ln, copy)
            plan = gqa.plan_eviction(copy, ln, ints([1000, 100]), table, torch.zeros(99, dtype=torch.int32, device="cuda"),
                                     ints([0]), page_len=64, max_keep=1000)
        want.append((copy.weight, out, plan.take))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [None, None]
    for step in range(5):
        for i, ((s, w, q), st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                table, ln = ints(s.table), ints(s.lens)
                gqa.add_key_weights(q, s.cache, table, ln, ints([0, 64, 80]), w)
                out = gqa.decode_paged_weights(q[:2], s.cache, table, ln, w)
                plan = gqa.plan_eviction(w, ln, ints([1000, 100]), table, torch.zeros(99, dtype=torch.int32, device="cuda"),
                                         ints([0]), page_len=64, max_keep=1000)
                got[i] = (w.weight, out, plan.take)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x.nan_to_num(), y.nan_to_num())


def test_c_refuses_masks_and_small_workspaces():
    """What the Python calls do not offer: bias, documents, prefixes and positions with the keys' weights."""
    import ctypes
    lens = [20, 30]
    s = Setup(lens, seed=1, page_len=16)
    w, q = some_weights(s), s.queries(2)
    lib, table, ln, out, first = _lib.load(), ints(s.table), ints(lens), torch.empty_like(q), ints([0, 1, 2])
    base = dict(batch=2, rows=2, block_table=table.data_ptr(), table_stride=2, table_width=2, seq_lens=ln.data_ptr(),
                scale=0.1, rope_theta=5e5, q_row_stride=4096, q_head_stride=128, out_row_stride=4096, out_head_stride=128)

    def status(name, **change):
        p = _lib.GqaPagedParams(**{**base, "first_query": first.data_ptr() if name == "add" else None, **change})
        args = (q.data_ptr(), ctypes.byref(s.cache.c), ctypes.byref(p), ctypes.byref(w.c), None, None, 0, None)
        if name == "add":
            return lib.gqa_add_key_weights(*args)
        return lib.gqa_decode_paged_weights(q.data_ptr(), out.data_ptr(), *args[1:4], None, 0, None)

    zeros = ints([0, 0])
    for name in ("add", "decode"):
        for field in ("doc_starts", "prefix_ends", "slopes"):
            assert status(name, **{field: torch.zeros(64, device="cuda").data_ptr() if field == "slopes" else zeros.data_ptr()}) \
                == _lib.GQA_ERR_FLAGS
        assert status(name) == _lib.GQA_ERR_WORKSPACE
        assert status(name, table_width=3, table_stride=3) == _lib.GQA_ERR_KV_RANGE  # more keys than weights
    assert status("decode", query_positions=zeros.data_ptr()) == _lib.GQA_ERR_FLAGS


@pytest.mark.parametrize("counts,lens,known", [([200, 130, 70], [500, 130, 300], [0, 0, 0]), ([200, 130, 70], [500, 130, 300], [100, 60, 300])])
def test_known_rows_of_many_units(counts, lens, known):
    s = Setup(lens, seed=4, page_len=16, code="e4m3")
    w, q = some_weights(s, [9, 9, 9]), s.queries(sum(counts))
    before = w.weight.clone(), w.position.clone()
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints(first), w, known=ints(known))
    now = [0 if k <= 0 else 9 for k in known]
    assert w.evicted.tolist() == now
    check_weights(s, w, before, exact_weights(s, q, counts, now), known, now)


@pytest.mark.parametrize("lens,counts,heads", [([2600, 700, 64, 1, 129], [2600, 700, 64, 1, 129], 8),
                                               ([3000, 40000], [65, 70], 1), ([300] * 40, [300] * 40, 2)])
def test_units_of_many_shares(lens, counts, heads):
    """Sums of several units share by share, in both of their layouts, beside sequences of one unit."""
    s = Setup(lens, seed=6, page_len=64, code="int8", heads=heads)
    w, q = some_weights(s), s.queries(sum(counts))
    before = w.weight.clone(), w.position.clone()
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    for turn in range(2):   # the second finds the first's sums in the workspace
        for t, x in zip((w.weight, w.position), before):
            t.copy_(x)
        gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints(first), w)
        check_weights(s, w, before, exact_weights(s, q, counts, [0] * len(lens)), [n - c for n, c in zip(lens, counts)],
                      [0] * len(lens))


def test_queries_that_several_sequences_claim():
    """Numbers of first queries that fall: the weights are anything, the call ends, and the next one is right."""
    lens = [700, 800, 900, 700, 800, 900]
    s = Setup(lens, seed=8, page_len=16, code="e4m3")
    w, q = some_weights(s), s.queries(600)
    guard = w.weight.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints([0, 600, 0, 600, -5, 700, 600]), w)
    assert gqa.read_device_status() == 0
    for b, n in enumerate(lens):
        assert torch.equal(w.weight[b, :, n:].nan_to_num(), guard[b, :, n:].nan_to_num())
    counts = [100] * 6
    w = some_weights(s)
    before = w.weight.clone(), w.position.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints(lens), ints(range(0, 601, 100)), w)
    check_weights(s, w, before, exact_weights(s, q, counts, [0] * 6), [n - 100 for n in lens], [0] * 6)


@pytest.mark.parametrize("cap", [1e-38, 1e-3, 30.0, 1e5, 3e38])
@pytest.mark.parametrize("rotated", [False, True])
def test_caps_of_any_size(cap, rotated):
    """Far below the scores every visible key weighs the same; far above them the cap changes nothing."""
    lens, counts = [130, 64], [70, 1]
    s = Setup(lens, seed=4, page_len=64, code="int8")
    q = s.queries(71)
    # (Of a cap of 1e5 and more the scores' own rounding is all there is: the bound's cap is what is left of it.)
    near = cap if 1e-3 < cap < 1e4 else 0.0
    for call in ("add", "decode"):
        w = some_weights(s)
        before = w.weight.clone(), w.position.clone()
        rows, n = (q, counts) if call == "add" else (q[:2], [1, 1])
        more = dict(score_cap=cap, q_rotated=rotated)
        if call == "add":
            gqa.add_key_weights(rows, s.cache, ints(s.table), ints(lens), ints([0, 70, 71]), w, **more)
        else:
            gqa.decode_paged_weights(rows, s.cache, ints(s.table), ints(lens), w, **more)
        if cap <= 1e-3:   # tanh is 1 or -1 for all scores but the smallest; all weights within 2 cap of one another
            for b, (length, c) in enumerate(zip(lens, n)):
                vis = (torch.arange(length - c, length)[:, None] >= torch.arange(length)[None]).double()
                want = 4 * (vis / vis.sum(-1, keepdim=True)).sum(0).cuda()
                start = torch.where(torch.arange(length, device="cuda") < length - c, before[0][b, :, :length].double(), 0.0)
                assert bool(((w.weight[b, :, :length].double() - start - want).abs() <= (math.expm1(2 * cap) + 2.0 ** -18) * want
                             + 2.0 ** -23 * (start + want)).all())
        else:
            check_weights(s, w, before, exact_weights(s, rows, n, [0, 0], near, q_rotated=rotated),
                          [x - c for x, c in zip(lens, n)], [0, 0])


FRESH = """
import torch, attention_accelerator_b200 as gqa
dev = torch.device("cuda", 0)
i32 = dict(dtype=torch.int32, device=dev)
cache = gqa.paged_cache(20, 32, dtype=torch.int8)
cache.k.random_(-127, 127), cache.v.random_(-127, 127), cache.k_scale.fill_(0.01), cache.v_scale.fill_(0.01)
table, lens = torch.arange(20, **i32).view(2, 10), torch.tensor([300, 200], **i32)
w = gqa.key_weights(2, 320)
q, first, keep = torch.randn(40, 32, 128, device=dev).bfloat16(), torch.tensor([0, 30, 40], **i32), torch.tensor([100, 150], **i32)
free, n_free, lam = torch.zeros(20, **i32), torch.zeros(1, **i32), torch.rand(16, device=dev)
def step():
    gqa.add_key_weights(q, cache, table, lens, first, w)
    out = gqa.decode_paged_weights(q[:2], cache, table, lens, w)
    d = gqa.decode_paged_diff(q[:2], cache, table, lens, lam)
    c = gqa.decode_paged_diff_chunked(q, cache, table, lens, first, lam)
    plan = gqa.plan_eviction(w, lens, keep, table, free, n_free, page_len=32, max_keep=150)
    gqa.evict_paged(cache, table, w, plan)
    return out, d, c, plan.take
state = [cache.k, cache.v, cache.k_scale, cache.v_scale, w.weight, w.position, w.evicted]
start = [t.clone() for t in state]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
for t, x in zip(state, start):
    t.copy_(x)
for a, b in zip(got, step()):
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
print("equal")
"""


def test_a_fresh_process_captures_without_a_warm_up():
    """Every kernel's first launch is a capture's."""
    import subprocess
    import sys
    from conftest import ROOT
    res = subprocess.run([sys.executable, "-c", FRESH], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "equal" in res.stdout, res.stdout + res.stderr
