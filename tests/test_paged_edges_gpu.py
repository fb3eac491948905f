"""GPU tests of the paged 8-bit cache at the ends of its accepted arguments, each through every kernel that takes the
call: one token a sequence, a few queries a sequence (at most 6 rows of one on average, 12 in all) and chunks."""
from __future__ import annotations

import math
import threading

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import api
from oracle import paged as ref
from test_paged_gpu import CHUNK_UNIT, DECODE_UNIT, THETA, Setup, ints, rows_of

pytestmark = pytest.mark.gpu

#: name -> queries of each of the two sequences of a call that the kernel of that name takes
KERNELS = {"decode": [1, 1], "few": [5, 2], "chunk": [70, 65]}


def unit_of(kernel):
    return DECODE_UNIT if kernel == "decode" else CHUNK_UNIT


def placed(kernel, lens):
    """(first_query, owner, position) of a call's rows: the last tokens of each sequence."""
    counts = KERNELS[kernel]
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    return first, owner, [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]


def attend(kernel, q, cache, table, lens, first, **more):
    if kernel == "decode":
        return gqa.decode_paged(q, cache, table, lens, **more)
    return gqa.decode_paged_chunked(q, cache, table, lens, ints(first), **more)


def close(got, q, setup, owner, positions, *, unit, theta=THETA, q_rotated=False, cap=0.0, slopes=None, starts=None,
          scale=1 / math.sqrt(128), floor=2.0 ** -22):
    """Outputs (27 rows of a chunk, every row of less) against 64 bits.  A score is off by 2 units of the sum of its
    terms' sizes (Q, and K's or the cap's rounding), FP32's 2^-19 of that and 2^-22 of the bias -- nothing that grows
    with the cap alone; a weight by e to twice that, 3 units and 2^-20; the output by its BF16 rounding, and by
    ``floor`` of its row's largest sum of |weight * value|: weights below FP16's range (2^-31 of the largest weight
    times scale, a few hundred of them)."""
    got = got.float().cpu().numpy().astype(np.float64)
    x = q.float().cpu().numpy().astype(np.float64)
    if not q_rotated:
        x = ref.rope(x, np.array(positions), theta)
    slopes = slopes.cpu().numpy().astype(np.float64) if slopes is not None else None
    kv = {b: setup.values(b) for b in set(owner)}
    rows = len(owner)
    for i in sorted(set(range(0, rows, max(1, rows // 27))) | {rows - 1}):
        b, m = owner[i], positions[i]
        p = np.arange(setup.lens[b])
        seen = (p >= (starts[i] if starts is not None else 0)) & (p <= m)
        k, v = kv[b]
        out, size, most = ref.attend(x[i], k, v, m, seen, scale=scale, cap=cap, slopes=slopes)
        far = np.abs(m - p).max() * slopes.max() if slopes is not None and len(p) else 0.0
        z = (2 * unit + 2.0 ** -19) * most + 2.0 ** -22 * far
        tol = (2.0 ** -8 * np.abs(out) + (math.expm1(2 * z) + 3 * unit + 2.0 ** -20) * size * 1.01
               + floor * size.max(-1, keepdims=True) + 1e-37)
        bad = ~(np.abs(got[i] - out) <= tol)
        assert not bad.any(), (i, b, m, int(bad.sum()), got[i][bad][:4], out[bad][:4])


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


def test_graphs_captured_without_a_warm_up(monkeypatch):
    """Two steps captured on a stream that has run nothing: each replays first, in any order, whatever the memory
    behind their workspaces held, and the stream's own calls beside them."""
    page_len, lens = 64, [5000, 3]
    side = torch.cuda.Stream()
    graphs, steps = [], []
    for seed in (81, 82):
        s = Setup(lens, seed=seed, page_len=page_len, width=120, spare=40)
        q, qc = s.queries(2), s.queries(70)
        held, new, spare = ints(lens), ints([1500, 1]), ints(s.unused + [-1] * 100)
        table, n_free = ints(s.table), ints([0])
        state = dict(table=table, spare=spare, held=held)
        start = {k: v.clone() for k, v in state.items()}
        n_free.fill_(len(s.unused))
        count = n_free.clone()

        def step(s=s, q=q, qc=qc, state=state, new=new, n_free=n_free):
            a = gqa.decode_paged(q, s.cache, state["table"], state["held"])
            b = gqa.decode_paged_chunked(qc, s.cache, state["table"], state["held"], first)
            plan = gqa.plan_pages(state["held"], new, state["table"], state["spare"], n_free, page_len=page_len,
                                  max_tokens=1600)
            return a, b, plan.lens, plan.n_free, plan.slots

        first = ints([0, 67, 70])
        steps.append((step, state, start, n_free, count))
    torch.cuda.synchronize()

    def restore(i):
        _, state, start, n_free, count = steps[i]
        for name, t in state.items():
            t.copy_(start[name])
        n_free.copy_(count)

    want = []
    for i in range(2):
        want.append([t.clone() for t in steps[i][0]()])
        restore(i)
    zeros, nodes = torch.zeros, []

    def spy(*args, **kw):
        nodes.append(torch.cuda.is_current_stream_capturing())
        return zeros(*args, **kw)

    monkeypatch.setattr(torch, "zeros", spy)
    torch.cuda.synchronize()
    for key in [k for k in api._ws if k[1] in (side.cuda_stream, ("paged", side.cuda_stream))]:
        api._ws_retired.append(api._ws.pop(key))  # (streams come round: another test's workspace is not this one's)
    known = set(api._ws)
    for step, *_ in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    made = set(api._ws) - known
    assert nodes and not any(nodes)  # none is zeroed by a node of a graph
    assert made and not any(bool(api._ws[key].any()) for key in made)  # zero before either graph has run
    for i in (1, 0, 0, 1):
        graphs[i][0].replay()
        torch.cuda.synchronize()
        for a, b in zip(graphs[i][1], want[i]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        restore(i)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = steps[0][0]()
    side.synchronize()
    for a, b in zip(got, want[0]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_plans_of_different_sizes_from_two_threads():
    """Each thread plans for its own number of requests on its own stream: none is refused for the other's sake."""
    failed = []

    def work(requests):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                zeros = torch.zeros(requests, dtype=torch.int32, device="cuda")
                table = torch.zeros(requests, 1, dtype=torch.int32, device="cuda")
                for _ in range(2000):
                    plan = gqa.plan_pages(zeros, zeros, table, zeros, zeros[:1], page_len=16, max_tokens=1)
                plan.check()
        except Exception as e:  # noqa: BLE001 -- whatever it is, the test shows it
            failed.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in (3500, 8192, 5000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("scale,loud", [(-0.1, 1), (-0.3, 8), (0.3, 8)])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_scores_of_either_sign_of_the_scale(kernel, scale, loud, code):
    """Softmax of -z is as good as that of z: over several whole tiles, with queries large enough for weights far apart."""
    lens = [700, 641]
    s = Setup(lens, seed=71, page_len=32, code=code)
    first, owner, pos = placed(kernel, lens)
    q = s.queries(first[-1]) * loud
    got = attend(kernel, q, s.cache, ints(s.table), ints(lens), first, scale=scale)
    close(got, q, s, owner, pos, unit=unit_of(kernel), scale=scale)
    got = attend(kernel, q, s.cache, ints(s.table), ints(lens), first, scale=scale, score_cap=5.0)
    close(got, q, s, owner, pos, unit=unit_of(kernel), scale=scale, cap=5.0)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("cap", [1e-38, 1e-30, 1.0, 50.0, 1e4, 1e6, 1e8, 1e20, 1e30, 3e38])
def test_caps_of_every_size(kernel, cap):
    """A cap far above the scores changes nothing, one far below them makes the weights equal."""
    lens = [700, 150]
    s = Setup(lens, seed=72, page_len=16, code="e4m3")
    first, owner, pos = placed(kernel, lens)
    q = s.queries(first[-1]) * 4
    got = attend(kernel, q, s.cache, ints(s.table), ints(lens), first, score_cap=cap)
    close(got, q, s, owner, pos, unit=unit_of(kernel), cap=float(np.float32(cap)))


def spread(s, scales, owner=0):
    """V scales of a sequence's pages, first to last (a list, or a function of the page's number)."""
    for col in range(-(-s.lens[owner] // s.page_len)):
        s.cache.v_scale[s.table[owner][col]] = scales(col) / (127 if s.code == "int8" else 448)


RATIOS = [2.0 ** -10, 2.0 ** -20, 2.0 ** -24, 2.0 ** -30, 2.0 ** -60]


@pytest.mark.parametrize("kernel", ["few", "chunk"])
@pytest.mark.parametrize("ratio", RATIOS)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("loud_first", [True, False])
def test_quiet_pages_beside_loud_ones_that_a_row_does_not_see(kernel, ratio, code, loud_first):
    """Every second row sees none of the loud pages: its output is the quiet pages' to full precision."""
    lens = [700, 640]
    s = Setup(lens, seed=73, page_len=16, code=code)
    first, owner, pos = placed(kernel, lens)
    cut = 320
    for b in (0, 1):
        spread(s, lambda col: (1.0 if (col * 16 < cut) == loud_first else ratio), b)
    q = s.queries(first[-1])
    starts = [cut if i % 2 else 0 for i in range(first[-1])]
    got = attend(kernel, q, s.cache, ints(s.table), ints(lens), first, doc_starts=ints(starts))
    close(got, q, s, owner, pos, unit=unit_of(kernel), starts=starts)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("ratio", RATIOS)
def test_quiet_pages_beside_loud_ones_of_no_weight(kernel, ratio):
    """The bias takes the weight of the loud pages, 400 keys away, below 2^-144: what is left is the quiet pages'."""
    lens = [700, 640]
    # (One token: among others, so that a warp has several tiles of a sequence.)
    s = Setup(lens + ([700] * 30 if kernel == "decode" else []), seed=74, page_len=64, code="int8")
    first, owner, pos = placed(kernel, lens)
    for b in (0, 1):
        spread(s, lambda col: 1.0 if col < 3 else ratio, b)
    q = s.queries(first[-1] if kernel != "decode" else len(s.lens))
    slopes = torch.full((32,), 0.25, device="cuda")
    got = attend(kernel, q, s.cache, ints(s.table), ints(s.lens), first, distance_slopes=slopes, q_rotated=True)
    close(got, q, s, owner, pos, unit=unit_of(kernel), slopes=slopes, q_rotated=True)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("size", [1e18, 1.0, 1e-18])
@pytest.mark.parametrize("quiet", [0.0, 2.0 ** -100])
def test_pages_of_zeros_beside_others(kernel, size, quiet):
    """Blocks of zeros have the smallest scale that an append writes, pages never written one of 0: their keys keep
    their weights, and the others their values, wherever in the sequence they are."""
    lens = [700, 640]
    for places in (lambda col: col == 0, lambda col: col < 9, lambda col: col % 3 == 1, lambda col: col > 5):
        s = Setup(lens, seed=75, page_len=64, code="e4m3")
        first, owner, pos = placed(kernel, lens)
        v = s.cache.v.view(torch.uint8)
        for b in (0, 1):
            spread(s, lambda col: quiet * 448 if places(col) else size, b)
            for col, page in enumerate(s.table[b]):
                if places(col) and page >= 0:
                    v[page] = 0
        q = s.queries(first[-1])
        got = attend(kernel, q, s.cache, ints(s.table), ints(lens), first)
        close(got, q, s, owner, pos, unit=unit_of(kernel))


@pytest.mark.parametrize("theta", [0.05, 0.3, 1.0, 10.0])
def test_small_rope_bases(theta):
    """Bases below 1 turn a pair by more than a radian a position, up to several turns: only their fraction counts."""
    lens = [300, 200]
    s = Setup(lens, seed=76, page_len=32, code="int8")
    for kernel in KERNELS:
        first, owner, pos = placed(kernel, lens)
        q = s.queries(first[-1])
        got = attend(kernel, q, s.cache, ints(s.table), ints(lens), first, rope_theta=theta)
        close(got, q, s, owner, pos, unit=unit_of(kernel), theta=float(np.float32(theta)))
    cache = gqa.paged_cache(2, 64, dtype=torch.int8)
    k = torch.randn(70, 8, 128, generator=s.gen, device="cuda").to(torch.bfloat16)
    at = torch.arange(70, device="cuda")
    gqa.append_paged(cache, k, k, at, positions=at.int() * 3, rope_theta=theta)
    want = ref.rope(k.float().cpu().numpy(), np.arange(70) * 3, float(np.float32(theta)))
    scale = cache.k_scale.cpu().numpy().astype(np.float64)[np.arange(70) // 64][..., None]
    got = ref.code_values(rows_of(cache, cache.k).reshape(128, 8, 128)[:70], "int8") * scale
    assert (np.abs(got - want) <= scale * (0.5 + 2.0 ** -6)).all()
    # The BF16 cache's rotation, by the same table: one BF16 rounding, and FP32's.
    got = gqa.rope_k_cache(k, at.int() * 3, rope_theta=theta).float().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -18).all()


@pytest.mark.parametrize("order", ["paged first", "others first", "captured first"])
def test_the_first_call_of_a_process(order):
    """Kernels are prepared by the first call that needs them, whichever call of the library that is."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys, torch
import attention_accelerator_b200 as gqa
q = torch.randn(1, 32, 128, device="cuda").bfloat16()
k = torch.randn(64, 8, 128, device="cuda").bfloat16()
table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda")
cache = gqa.paged_cache(1, 64, dtype=torch.int8)
gqa.append_paged(cache, k, k, torch.arange(64, device="cuda"), positions=torch.arange(64, device="cuda").int())
def paged(): return gqa.decode_paged(q, cache, table, lens)
def others(): return gqa.decode(q[0], k, k, seq_len=64, query_position=63, kv_block_len=16, layout="position_major")
if sys.argv[1] == "captured first":
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        a = paged()
    graph.replay()
    torch.cuda.synchronize()
    b = others()
elif sys.argv[1] == "paged first":
    a, b = paged(), others()
else:
    b, a = others(), paged()
assert float((a[0].float() - b.float()).abs().max()) < 0.1, (a, b)
"""
    run = subprocess.run([sys.executable, "-c", code, order], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0, run.stderr[-2000:]


def test_chunks_of_pages_outside_the_cache():
    """Table entries that name no page read as zeros, in a chunk as in the other calls."""
    lens = [200, 640]
    s = Setup(lens, seed=77, page_len=32, code="e4m3")
    first, owner, pos = placed("chunk", lens)
    q = s.queries(first[-1])
    s.poison(lambda b, p: False)
    v, k = s.cache.v.view(torch.uint8), s.cache.k.view(torch.uint8)
    for page in (-5, s.cache.pages, 1 << 30, -(1 << 31)):
        table = [list(row) for row in s.table]
        table[0][2], table[1][0] = page, page
        got = gqa.decode_paged_chunked(q, s.cache, ints(table), ints(lens), ints(first))
        zero = Setup(lens, seed=77, page_len=32, code="e4m3")
        for b, col in ((0, 2), (1, 0)):
            zero.cache.k.view(torch.uint8)[zero.table[b][col]] = 0
            zero.cache.v.view(torch.uint8)[zero.table[b][col]] = 0
        close(got, q, zero, owner, pos, unit=CHUNK_UNIT)
    table = [[-1 if c % 2 else 1 << 30 for c in range(len(row))] for row in s.table]
    assert not gqa.decode_paged_chunked(q, s.cache, ints(table), ints(lens), ints(first)).any()
    assert k.shape == v.shape and gqa.read_device_status() == 0


def test_chunks_of_pages_past_32_bits():
    pages = 36000
    k, v = (torch.empty(pages, 8, 128, 128, dtype=torch.uint8, device="cuda").view(torch.int8) for _ in range(2))
    ks, vs = (torch.empty(pages, 8, dtype=torch.float32, device="cuda") for _ in range(2))
    cache = gqa.PagedCache(k, v, ks, vs)
    lens = [300, 140]
    s = Setup(lens, seed=78, page_len=128, spare=0)
    table, far = [[-1] * 3 for _ in lens], [35999, 17, 35000, 34000, 33000]
    for b, n in enumerate((3, 2)):
        for col in range(n):
            src, dst = s.table[b][col], far.pop()
            k[dst], v[dst], ks[dst], vs[dst] = s.cache.k[src], s.cache.v[src], s.cache.k_scale[src], s.cache.v_scale[src]
            table[b][col] = dst
    first, owner, pos = placed("chunk", lens)
    q = s.queries(first[-1])
    close(gqa.decode_paged_chunked(q, cache, ints(table), ints(lens), ints(first)), q, s, owner, pos, unit=CHUNK_UNIT)


def test_a_visible_nan_in_a_chunk_reaches_its_rows_only():
    lens = [200, 300]
    s = Setup(lens, seed=79, page_len=16, code="int8")
    first, owner, pos = placed("chunk", lens)
    q = s.queries(first[-1])
    s.cache.v_scale[s.table[0][10], 2] = math.nan   # keys 160 to 175
    s.cache.k_scale[s.table[1][16], 5] = math.nan   # keys 256 to 271
    nan = torch.isnan(gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first))).any(-1)
    want = torch.zeros_like(nan)
    for i, (b, m) in enumerate(zip(owner, pos)):
        if b == 0 and m >= 160:
            want[i, 8:12] = True
        if b == 1 and m >= 256:
            want[i, 20:24] = True
    assert torch.equal(nan, want)


def test_first_query_of_a_chunk_is_kept_within_the_rows():
    lens = [300, 300, 300]
    s = Setup(lens, seed=80, page_len=32)
    q = s.queries(100)
    guard = torch.full((300, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    for first in ([0, 70, 100, 1 << 30], [-7, 70, 90, 100], [0, 120, 90, 100], [90, 70, 0, 100], [-(1 << 31), 0, 99, 100]):
        gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), out=guard[100:200])
        assert bool((guard[:100] == 5.0).all()) and bool((guard[200:] == 5.0).all())
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("kernel", KERNELS)
def test_strided_rows_of_each_kernel(kernel):
    lens = [90, 200]
    s = Setup(lens, seed=83, page_len=16)
    first, owner, pos = placed(kernel, lens)
    n = first[-1]
    wide = torch.zeros(n, 40, 256, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 3:35, 64:192]
    q.copy_(s.queries(n))
    out = torch.zeros(n, 34, 136, dtype=torch.bfloat16, device="cuda")
    table = torch.full((2, 50), 9999, dtype=torch.int32, device="cuda")
    table[:, :len(s.table[0])] = ints(s.table)
    got = attend(kernel, q, s.cache, table[:, :len(s.table[0])], ints(lens), first, out=out[:, 1:33, :128], scale=0.3)
    close(got, q, s, owner, pos, unit=unit_of(kernel), scale=0.3)
    assert not out[:, 0].any() and not out[:, 33].any() and not out[..., 128:].any()


@pytest.mark.parametrize("kernel", ["few", "chunk"])
def test_chunked_calls_in_a_graph_follow_the_lengths(kernel):
    lens, counts = [700, 640], KERNELS[kernel]
    s = Setup(lens, seed=84, page_len=64, code="e4m3")
    first, owner, _ = placed(kernel, lens)
    q, table, held = s.queries(first[-1]), ints(s.table), ints(lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    at = ints(first)
    with torch.cuda.stream(side):
        gqa.decode_paged_chunked(q, s.cache, table, held, at)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = gqa.decode_paged_chunked(q, s.cache, table, held, at)
    for now in ([700, 640], [counts[0], 333], [512, 640]):
        held.copy_(ints(now))
        graph.replay()
        torch.cuda.synchronize()
        s.lens = now
        pos = [now[b] - n + i for b, n in enumerate(counts) for i in range(n)]
        close(out, q, s, owner, pos, unit=CHUNK_UNIT)
