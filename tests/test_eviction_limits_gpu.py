"""GPU tests of the keys' weights and of eviction where numbers are largest: tables, lengths, positions, scores."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import _lib
from test_eviction_gpu import exact_weights, some_weights
from test_paged_cpu import c_cache, c_params
from test_paged_gpu import Setup, ints

pytestmark = pytest.mark.gpu


def test_a_request_that_gives_back_millions_of_pages():
    """4.3 million pages of one request: refused by a stack that lacks room for a few of them, else all given back."""
    page_len, pages, keep = 16, 4_300_000, 40
    length = pages * page_len - 5
    w = gqa.key_weights(1, pages * page_len, kv_heads=1)
    w.weight[0, 0, length - keep:length] = 1.0
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    given = table[0, -(-keep // page_len):]
    for room in (given.numel() - 1, given.numel()):
        stack = torch.full((given.numel() + 8,), -7, dtype=torch.int32, device="cuda")
        plan = gqa.plan_eviction(w, ints([length]), ints([keep]), table, stack[:room], ints([0]), page_len=page_len,
                                 max_keep=keep, sinks=0, recent=0)
        if room < given.numel():
            assert plan.counts.tolist() == [0, 0, 0, _lib.GQA_ERR_PAGES] and plan.n_free.tolist() == [0]
            assert plan.lens.tolist() == [length] and bool((stack == -7).all()) and bool((plan.take == -1).all())
        else:
            assert plan.counts.tolist() == [1, length - keep, room, 0] and plan.n_free.tolist() == [room]
            assert torch.equal(stack[:room], given) and bool((stack[room:] == -7).all())
            assert plan.take.flatten().tolist() == list(range(length - keep, length))
            assert plan.lens.tolist() == [keep] and plan.evicted.tolist() == [length - keep]


def test_requests_that_lose_more_than_2_31_rows():
    """The count of evicted rows stops at 2^31 - 1; lengths, tokens evicted and pages are whole."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    requests, length, page_len = 2100, 1 << 20, 128
    w = gqa.key_weights(requests, length, kv_heads=1)
    width = length // page_len
    table = torch.arange(requests * width, dtype=torch.int32, device="cuda").view(requests, width)
    stack = torch.full((requests * width,), -7, dtype=torch.int32, device="cuda")
    plan = gqa.plan_eviction(w, ints([length] * requests), ints([8] * requests), table, stack, ints([0]), page_len=page_len,
                             max_keep=8, sinks=0, recent=0)
    given = requests * (width - 1)
    assert plan.counts.tolist() == [requests, 0x7FFFFFFF, given, 0] and plan.n_free.tolist() == [given]
    assert torch.equal(stack[:given], table[:, 1:].flatten()) and bool((stack[given:] == -7).all())
    assert plan.lens.tolist() == [8] * requests and plan.evicted.tolist() == [length - 8] * requests
    assert bool((plan.take == -1).all())  # equal weights: the lower rows stay


@pytest.mark.parametrize("length", [(1 << 29) + 50, 1 << 30, 0x7FFFFFFF])
@pytest.mark.parametrize("counts", [[3, 64], [200, 1]])
def test_queries_far_behind_the_keys(length, counts):
    """Lengths past what the table names: the queries stand up to 2^31 rows behind its keys and see them all.  Bounds as
    in :func:`test_eviction_gpu.exact_weights`."""
    held = 320
    s = Setup([held] * 2, seed=counts[0], page_len=64, code="int8", heads=2)
    w, q = some_weights(s), s.queries(sum(counts))
    before = w.weight.double(), w.position.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints([length] * 2), ints([0, counts[0], sum(counts)]), w, q_rotated=True)
    assert torch.equal(w.position, before[1]) and gqa.read_device_status() == 0
    for b, n in enumerate(counts):
        rows = q[sum(counts[:b]):][:n].double()
        k = torch.from_numpy(s.values(b)[0]).cuda()
        for h in range(2):
            want, bound = before[0][b, h].clone(), 0.0
            for g in range(4):
                x = rows[:, 4 * h + g]
                weight = torch.softmax(x @ k[:, h].T / math.sqrt(128), -1).sum(0)
                most = float(x.abs().max()) * float(k[:, h].abs().sum(-1).max()) / math.sqrt(128)
                want += weight
                bound = bound + weight * (math.expm1(2 * 2.0 ** -18 * most) + 2.0 ** -20)
            error = (w.weight[b, h].double() - want).abs()
            assert bool((error <= bound + 2.0 ** -23 * want).all()), (b, h, float((error / want).max()))


@pytest.mark.parametrize("power,cap", [(4, 0.0), (14, 0.0), (18, 0.0), (24, 0.0), (28, 0.0), (32, 0.0), (40, 0.0), (60, 0.0),
                                       (118, 0.0), (126, 0.0), (60, 1e6), (126, 1e30)])
@pytest.mark.parametrize("n", [1, 40, 100])
def test_queries_of_any_size_beside_ordinary_ones(power, cap, n):
    """Rows of up to BF16's largest numbers, each the value of one key: it gets their whole weight (with a cap that they
    pass, all keys of a positive score share it; one beyond 2^96 is none, as the call's arguments say), and the other rows
    of their unit give what they give without them."""
    exact_cap = cap if cap <= 2.0 ** 96 else 0.0
    length = 700
    s = Setup([length], seed=power, page_len=64, code="int8", heads=2)
    s.cache.k_scale.fill_(2.0 ** -17)  # scores of 2^126 times a key stay within FP32
    q = (s.queries(n).float() * 2.0 ** 10).to(torch.bfloat16)
    plain, k = q.clone(), torch.from_numpy(s.values(0)[0]).cuda()
    picks = [(row, head, 17 * row % (length - n + row + 1)) for row in {n // 10, n - 1} for head in (1, 6)]
    for row, head, key in picks:
        x = k[key, head // 4]
        q[row, head] = (x / x.abs().max() * 2.0 ** power).to(torch.bfloat16)
        plain[row, head] = 0.0
    w = some_weights(s)
    before = w.weight.clone()
    gqa.add_key_weights(q, s.cache, ints(s.table), ints([length]), ints([0, n]), w, q_rotated=True, score_cap=cap or None)
    total, bound = exact_weights(s, plain, [n], [0], cap=exact_cap, q_rotated=True)[0]
    for row, head, key in picks:
        seen = length - n + row + 1
        total[head // 4, :seen] -= 1.0 / seen  # a row of zeros gives every key as much
        x = q[row, head].double()
        z = k[:seen, head // 4] @ x / math.sqrt(128)
        if exact_cap:
            z = exact_cap * torch.tanh(z / exact_cap)
        p = torch.softmax(z, -1)
        total[head // 4, :seen] += p
        if power >= 24:  # no two scores are near each other but those at the cap, which are the same
            assert float(p.max() - p[p > 0].min()) < 1e-12 and abs(float((p > 0).sum() * p.max()) - 1) < 1e-12
            bound[head // 4, :seen] += 2.0 ** -20 * p
        else:
            most = float(x.abs().max()) * float(k[:, head // 4].abs().sum(-1).max()) / math.sqrt(128)
            bound[head // 4, :seen] += p * (math.expm1(2 * 2.0 ** -18 * most) + 2.0 ** -20)
    start = before[0, :, :length].double()
    start[:, length - n:] = 0.0
    error = (w.weight[0, :, :length].double() - start - total).abs()
    # (2^-40: the rows of zeros that were taken out again.)
    assert bool((error <= bound + 2.0 ** -23 * (start + total) + 2.0 ** -40).all()), float(error.max())


@pytest.mark.parametrize("v_scale", [1 / 127, 2.0 ** -4, 2.0 ** -40, 2.0 ** 30])
@pytest.mark.parametrize("power", [8, 20, 24, 28, 30, 31, 32, 33, 34, 35, 36, 37, 38, 60, 118])
def test_decode_steps_of_queries_of_any_size(power, v_scale):
    """One token a sequence: the scores' rounding takes no part in the sums, whatever V's scales add to the exponents."""
    lens = [300] * 15 + [5000]
    s = Setup(lens, seed=power, page_len=64, code="int8", heads=2)
    s.cache.k_scale.fill_(2.0 ** -17)
    s.cache.v_scale.fill_(v_scale)
    k = [torch.from_numpy(s.values(b)[0]).cuda() for b in range(len(lens))]
    q = torch.zeros(len(lens), 8, 128, dtype=torch.bfloat16, device="cuda")
    for b in range(len(lens)):
        for head in range(8):
            x = k[b][(7 * b + head) % 300, head // 4]
            q[b, head] = (x / x.abs().max() * 2.0 ** (power + (b % 8) / 8)).to(torch.bfloat16)
    w = some_weights(s)
    before = w.weight.double()
    gqa.decode_paged_weights(q, s.cache, ints(s.table), ints(lens), w, q_rotated=True)
    for b, n in enumerate(lens):
        for h in range(2):
            want, bound = before[b, h, :n].clone(), 0.0
            want[n - 1] = 0.0
            for g in range(4):
                x = q[b, 4 * h + g].double()
                p = torch.softmax(k[b][:, h] @ x / math.sqrt(128), -1)
                want += p
                if power >= 24:  # one key stands out
                    assert float(p.max()) > 1 - 1e-12
                    bound = bound + 2.0 ** -20 * p
                else:
                    most = float(x.abs().max()) * float(k[b][:, h].abs().sum(-1).max()) / math.sqrt(128)
                    bound = bound + p * (math.expm1(2 * 2.0 ** -18 * most) + 2.0 ** -20)
            error = (w.weight[b, h, :n].double() - want).abs()
            assert bool((error <= bound + 2.0 ** -23 * want).all()), (b, h, float(error.max()))


@pytest.mark.parametrize("batch,rows,heads,width", [(1, 1, 1, 1), (64, 64, 8, 512), (8192, 8192, 8, 4), (8192, 8192, 1, 512),
                                                    (8, 512, 8, 256), (6, 9000, 8, 129), (48, 4096, 3, 2048), (1, 100000, 8, 1 << 14)])
def test_workspaces_are_of_the_stated_size(batch, rows, heads, width):
    """As the header states it: 132 KB a unit and head, 16 bytes a key, sequence and head, and what thread blocks leave."""
    lib, page_len = _lib.load(), 64
    c = c_cache(kv_heads=heads, page_len=page_len)
    keys = width * page_len
    many = lib.gqa_key_weights_workspace_bytes(ctypes.byref(c), ctypes.byref(c_params(
        batch=batch, rows=rows, table_width=width, table_stride=width, first_query=4096)))
    sums = keys * (8 * heads * batch + 1200) if rows > 64 else 0
    assert 0 < many <= 132 * 1024 * heads * (rows // 64 + batch + 1) + sums * 1.01 + 128 * 8 * heads * batch + (4 << 20)
    one = lib.gqa_key_weights_workspace_bytes(ctypes.byref(c), ctypes.byref(c_params(
        batch=batch, rows=batch, table_width=width, table_stride=width, first_query=None)))
    assert 16 * keys * batch * heads < one <= 16 * keys * batch * heads + (4 << 20)
