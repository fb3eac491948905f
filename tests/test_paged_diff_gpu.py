"""GPU tests of differential attention over the paged 8-bit cache against its definition in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from oracle import paged as ref
from test_paged_gpu import CHUNK_UNIT, DECODE_UNIT, MODS, ODD_LENS, THETA, Setup, ints, modifiers

pytestmark = pytest.mark.gpu


def learned(s, rows, by_row, norm):
    """Lambdas of a call's heads or rows, and its norm's weight."""
    heads = 2 * s.heads
    lam = 0.1 + 0.8 * torch.rand(rows if by_row else 1, heads, generator=s.gen, device="cuda")
    weight = 1.0 + 0.2 * torch.randn(128, generator=s.gen, device="cuda") if norm else None
    return lam if by_row else lam[0], weight


def check_diff(got, q, setup, owner, positions, lambdas, *, unit, weight=None, eps=1e-5, out_scale=1.0, q_rotated=False,
               cap=0.0, slopes=None, starts=None, ends=None):
    """Every output against 64 bits.  The maps' products are off by what attention's outputs are before their rounding
    (a score by z, a weight by e^2z - 1, three units for the roundings of weights and V), the difference by the sum of
    both and FP32's 2^-20; the norm passes that on (:func:`oracle.paged.attend_diff`) and adds FP32's 2^-20 of the
    result, which is rounded to BF16 (2^-8 of it at most)."""
    got = got.float().cpu().numpy().astype(np.float64)
    x = q.float().cpu().numpy().astype(np.float64)
    if not q_rotated:
        x = ref.rope(x, np.array(positions), THETA)
    slopes = slopes.cpu().numpy().astype(np.float64) if slopes is not None else None
    lam = lambdas.cpu().numpy()
    kv = {b: setup.values(b) for b in set(owner)}
    w = weight.cpu().numpy().astype(np.float64) if weight is not None else None
    for i, (b, m) in enumerate(zip(owner, positions)):
        p = np.arange(setup.lens[b])
        end = max(m + 1, ends[i] if ends is not None else 0)
        seen = (p >= (starts[i] if starts is not None else 0)) & (p < end)
        k, v = kv[b]
        out, size, most = ref.attend_diff(x[i], k, v, m, seen, lam[i] if lam.ndim == 2 else lam, norm_weight=w, eps=eps,
                                          out_scale=out_scale, scale=1 / math.sqrt(128), cap=cap, slopes=slopes)
        far = np.abs(m - p).max() * slopes.max() if slopes is not None and len(p) else 0.0
        z = (2 * unit + 2.0 ** -20) * most + 2.0 ** -20 * cap + 2.0 ** -22 * far
        tol = (2.0 ** -8 + 2.0 ** -20) * np.abs(out) + (math.expm1(2 * z) + 3 * unit + 2.0 ** -19) * size * 1.05 + 1e-30
        bad = ~(np.abs(got[i] - out) <= tol)
        assert not bad.any(), (i, b, m, int(bad.sum()), float((np.abs(got[i] - out) / tol)[~np.isnan(got[i])].max()))


@pytest.mark.parametrize("page_len", [16, 32, 64, 128])
@pytest.mark.parametrize("code,layout,by_row,norm", [("int8", "head_major", False, True), ("e4m3", "position_major", True, False),
                                                     ("e4m3", "head_major", True, True)])
def test_decode_lengths(page_len, code, layout, by_row, norm):
    s = Setup(ODD_LENS, seed=page_len, page_len=page_len, code=code, layout=layout)
    n = len(ODD_LENS)
    q = s.queries(n)
    s.poison(lambda b, p: False)
    lam, weight = learned(s, n, by_row, norm)
    args = (q, s.cache, ints(s.table), ints(ODD_LENS), lam)
    got = gqa.decode_paged_diff(*args, norm_weight=weight, out_scale=0.4)
    assert got.shape == (n, 16, 128) and got.dtype == torch.bfloat16
    check_diff(got, q, s, list(range(n)), [m - 1 for m in ODD_LENS], lam, unit=DECODE_UNIT, weight=weight, out_scale=0.4)
    assert not got[1].any()  # a sequence without keys
    again = gqa.decode_paged_diff(*args, norm_weight=weight, out_scale=0.4)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("lens", [[30], [1], [4096], [20000], [5000, 1, 700], [90] * 700])
@pytest.mark.parametrize("norm", [True, False])
def test_decode_few_and_many_sequences(lens, norm):
    s = Setup(lens, seed=sum(lens), page_len=16 if lens == [30] else 64, code="int8")
    q = s.queries(len(lens))
    lam, weight = learned(s, len(lens), norm, norm)
    got = gqa.decode_paged_diff(q, s.cache, ints(s.table), ints(lens), lam, norm_weight=weight)
    pick = list(range(0, len(lens), max(1, len(lens) // 25)))
    check_diff(got[pick], q[pick], s, pick, [lens[b] - 1 for b in pick], lam[pick] if norm else lam, unit=DECODE_UNIT,
               weight=weight)


@pytest.mark.parametrize("heads", [1, 2, 3, 5])
def test_head_shards(heads):
    lens = [200, 1, 77]
    s = Setup(lens, seed=heads, page_len=32, code="e4m3", heads=heads, layout="position_major")
    q = s.queries(3)
    lam, weight = learned(s, 3, True, True)
    got = gqa.decode_paged_diff(q, s.cache, ints(s.table), ints(lens), lam, norm_weight=weight)
    check_diff(got, q, s, [0, 1, 2], [199, 0, 76], lam, unit=DECODE_UNIT, weight=weight)
    first = [0, 100, 101, 150]
    q = s.queries(150)
    owner = [0] * 100 + [1] + [2] * 49
    pos = list(range(100, 200)) + [0] + list(range(28, 77))
    lam, weight = learned(s, 150, False, True)
    got = gqa.decode_paged_diff_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), lam, norm_weight=weight)
    check_diff(got, q, s, owner, pos, lam, unit=CHUNK_UNIT, weight=weight)


@pytest.mark.parametrize("what", MODS)
@pytest.mark.parametrize("code,page_len,norm", [("int8", 16, True), ("e4m3", 64, False)])
def test_decode_masks_cap_and_bias(what, code, page_len, norm):
    lens = ODD_LENS + [513, 700, 90, 31]
    s = Setup(lens, seed=len(what), page_len=page_len, code=code)
    owner = list(range(len(lens)))
    rng = np.random.RandomState(3)
    pos = [int(rng.randint(0, max(1, n))) for n in lens]
    q = s.queries(len(lens))
    call, chk = modifiers(s, what, owner, pos)
    starts, ends = chk.get("starts", [0] * len(lens)), chk.get("ends", [0] * len(lens))
    s.poison(lambda b, p: not starts[b] <= p < max(pos[b] + 1, ends[b]))
    lam, weight = learned(s, len(lens), norm, norm)
    got = gqa.decode_paged_diff(q, s.cache, ints(s.table), ints(lens), lam, norm_weight=weight, query_positions=ints(pos),
                                **call)
    check_diff(got, q, s, owner, pos, lam, unit=DECODE_UNIT, weight=weight, **chk)


@pytest.mark.parametrize("counts,lens", [
    ([1], [1]), ([5], [5]), ([3], [300]), ([128], [8192]), ([1, 1, 1], [1, 90, 17]), ([6, 5, 1, 0, 7], [6, 900, 1, 30, 64]),
    ([33, 0, 1, 64, 65], [33, 10, 400, 64, 700]), ([257], [257]), ([5] * 40, [5 + 97 * i for i in range(40)]),
    ([31, 32, 33, 127, 129], [1000, 32, 500, 127, 200])])
@pytest.mark.parametrize("code,page_len,layout,norm", [("int8", 16, "position_major", True), ("e4m3", 64, "head_major", False)])
def test_chunked_lengths(counts, lens, code, page_len, layout, norm):
    s = Setup(lens, seed=sum(lens), page_len=page_len, code=code, layout=layout)
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    rows = first[-1]
    q = s.queries(rows + 3)
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]
    s.poison(lambda b, p: False)
    lam, weight = learned(s, rows + 3, not norm, norm)
    out = torch.full((rows + 3, 16, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    args = (q, s.cache, ints(s.table), ints(lens), ints(first), lam)
    got = gqa.decode_paged_diff_chunked(*args, norm_weight=weight, out_scale=0.7, out=out)
    assert got is out and bool((out[rows:] == 7.0).all())
    pick = sorted(set(range(0, rows, max(1, rows // 40))) | {rows - 1})
    check_diff(got[pick], q[pick], s, [owner[i] for i in pick], [pos[i] for i in pick], lam if norm else lam[pick],
               unit=CHUNK_UNIT, weight=weight, out_scale=0.7)
    again = gqa.decode_paged_diff_chunked(*args, norm_weight=weight, out_scale=0.7)
    assert torch.equal(got[:rows].view(torch.int16), again[:rows].view(torch.int16))
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("what", MODS)
@pytest.mark.parametrize("code,page_len,counts,lens", [("e4m3", 16, [40, 130, 1, 7], [40, 301, 77, 7]),
                                                       ("int8", 64, [4, 6, 1, 2], [400, 6, 77, 130])])
def test_chunked_masks_cap_and_bias(what, code, page_len, counts, lens):
    s = Setup(lens, seed=7 * len(what), page_len=page_len, code=code)
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]
    q = s.queries(first[-1])
    call, chk = modifiers(s, what, owner, pos)
    starts, ends = chk.get("starts", [0] * len(pos)), chk.get("ends", [0] * len(pos))
    visible = [set() for _ in lens]
    for i, b in enumerate(owner):
        visible[b] |= set(range(max(0, starts[i]), min(lens[b], max(pos[i] + 1, ends[i]))))
    s.poison(lambda b, p: p not in visible[b])
    lam, weight = learned(s, first[-1], True, True)
    got = gqa.decode_paged_diff_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), lam, norm_weight=weight, **call)
    check_diff(got, q, s, owner, pos, lam, unit=CHUNK_UNIT, weight=weight, **chk)


@pytest.mark.parametrize("counts,lens", [([1] * 5, [700, 65, 1, 0, 20000]), ([300, 64, 1], [9000, 64, 20]), ([5, 4, 6], [3000, 64, 20])])
def test_lambda_zero_is_the_first_map(counts, lens):
    """Without the second map and a norm the rows are those of the plain calls' even heads, to the bit."""
    s = Setup(lens, seed=5, page_len=32, code="e4m3")
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    q, zero = s.queries(first[-1]), torch.zeros(16, device="cuda")
    args = (q, s.cache, ints(s.table), ints(lens))
    if set(counts) == {1}:
        got, want = gqa.decode_paged_diff(*args, zero), gqa.decode_paged(*args)
    else:
        got = gqa.decode_paged_diff_chunked(*args, ints(first), zero)
        want = gqa.decode_paged_chunked(*args, ints(first))
    assert torch.equal(got, want[:, 0::2])
    second = torch.full((16,), -1.0, device="cuda")  # the sum of the maps
    both = (gqa.decode_paged_diff(*args, second) if set(counts) == {1} else
            gqa.decode_paged_diff_chunked(*args, ints(first), second))
    total = want[:, 0::2].float() + want[:, 1::2].float()
    size = want[:, 0::2].float().abs() + want[:, 1::2].float().abs()
    assert bool(((both.float() - total).abs() <= 2.0 ** -8 * (total.abs() + size) + 1e-30).all())


def test_equal_maps_cancel():
    """Where both heads ask the same and lambda is 1, nothing is left: within FP32's rounding of what was taken away."""
    lens = [700, 1, 65]
    s = Setup(lens, seed=9, page_len=64, code="int8")
    q = s.queries(3)
    q[:, 1::2] = q[:, 0::2]
    one = torch.ones(16, device="cuda")
    args = (q, s.cache, ints(s.table), ints(lens))
    assert not gqa.decode_paged_diff(*args, one).any()
    assert not gqa.decode_paged_diff(*args, one, norm_weight=torch.ones(128, device="cuda")).any()


@pytest.mark.parametrize("size", [1e-18, 1.0, 1e18, 1e30])
def test_norm_of_tiny_and_huge_values(size):
    """Values of any size a V scale takes: a row's squares may pass FP32's range, where eps is nothing beside them."""
    lens, first = [60, 129, 40], [0, 7, 136, 137]
    for chunked in (False, True):
        s = Setup(lens, seed=4, page_len=64, code="e4m3")
        s.cache.v_scale.mul_(size)
        rows = first[-1] if chunked else 3
        q = s.queries(rows)
        lam, weight = learned(s, rows, False, True)
        args = (q, s.cache, ints(s.table), ints(lens))
        if chunked:
            lens_used = [60, 129, 40]
            owner = [0] * 7 + [1] * 129 + [2]
            pos = list(range(53, 60)) + list(range(129)) + [39]
            got = gqa.decode_paged_diff_chunked(*args, ints(first), lam, norm_weight=weight)
        else:
            owner, pos = [0, 1, 2], [n - 1 for n in lens]
            got = gqa.decode_paged_diff(*args, lam, norm_weight=weight)
        assert bool(torch.isfinite(got).all())
        pick = list(range(0, rows, 9 if chunked else 1))
        check_diff(got[pick], q[pick], s, [owner[i] for i in pick], [pos[i] for i in pick], lam,
                   unit=CHUNK_UNIT if chunked else DECODE_UNIT, weight=weight)


def test_strided_rows_lambdas_and_out():
    lens, first = [90, 33], [0, 70, 71]
    s = Setup(lens, seed=6, page_len=16, code="int8", layout="position_major")
    big = s.queries(71 * 2).view(71, 2, 32, 128)
    q = big[:, 1]
    lam = torch.rand(71, 40, generator=s.gen, device="cuda")[:, 3:19]
    out = torch.full((71, 3, 16, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    gqa.decode_paged_diff_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), lam, out=out[:, 1])
    want = gqa.decode_paged_diff_chunked(q.contiguous(), s.cache, ints(s.table), ints(lens), ints(first), lam.contiguous())
    assert torch.equal(out[:, 1], want) and bool((out[:, 0] == 5).all()) and bool((out[:, 2] == 5).all())
    got = gqa.decode_paged_diff(q[:2], s.cache, ints(s.table), ints(lens), lam[:2], out=out[:2, 0])
    assert torch.equal(got, gqa.decode_paged_diff(q[:2].contiguous(), s.cache, ints(s.table), ints(lens), lam[:2].contiguous()))
    expanded = lam[:1].expand(71, 16)  # one row's for all
    a = gqa.decode_paged_diff_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), expanded)
    b = gqa.decode_paged_diff_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), lam[0].contiguous())
    assert torch.equal(a, b)


def test_graph_follows_the_lengths_and_plain_calls_between():
    """A captured step on a stream of its own, whose lengths and lambdas change; plain calls of the same stream share its
    workspace and counters."""
    lens = [3000, 64, 500, 1]
    s = Setup(lens, seed=8, page_len=64, code="e4m3")
    q, table, ln = s.queries(4), ints(s.table), ints(lens)
    lam, weight = learned(s, 4, True, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gqa.decode_paged_diff(q, s.cache, table, ln, lam, norm_weight=weight)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = gqa.decode_paged_diff(q, s.cache, table, ln, lam, norm_weight=weight)
            plain = gqa.decode_paged(q, s.cache, table, ln)
        for now in (lens, [2999, 63, 2, 0], [1, 64, 128, 1]):
            ln.copy_(ints(now))
            lam.mul_(0.9)
            graph.replay()
            assert torch.equal(out, gqa.decode_paged_diff(q, s.cache, table, ln, lam, norm_weight=weight))
            assert torch.equal(plain, gqa.decode_paged(q, s.cache, table, ln))
    side.synchronize()


def test_refusals():
    lens = [20, 30]
    s = Setup(lens, seed=1, page_len=16)
    q, lam = s.queries(2), torch.rand(16, device="cuda")
    args = (q, s.cache, ints(s.table), ints(lens))
    weight = torch.ones(128, device="cuda")
    for bad in (lam.double(), lam[:15], lam.cpu(), torch.rand(3, 16, device="cuda"), torch.rand(2, 32, device="cuda")[:, ::2]):
        with pytest.raises(ValueError, match="lambdas"):
            gqa.decode_paged_diff(*args, bad)
        with pytest.raises(ValueError, match="lambdas"):
            gqa.decode_paged_diff_chunked(*args, ints([0, 1, 2]), bad)
    for more, match in [(dict(norm_weight=weight[:64]), "norm_weight"), (dict(norm_weight=weight.bfloat16()), "norm_weight"),
                        (dict(norm_weight=weight, norm_eps=0.0), "norm_eps"), (dict(out_scale=math.inf), "out_scale"),
                        (dict(norm_weight=weight, norm_eps=math.nan), "norm_eps"),
                        (dict(out=torch.empty(2, 32, 128, dtype=torch.bfloat16, device="cuda")), "out must be"),
                        (dict(score_cap=-1.0), "score_cap")]:
        with pytest.raises(ValueError, match=match):
            gqa.decode_paged_diff(*args, lam, **more)
    with pytest.raises(gqa.GqaError, match="aligned"):
        gqa.decode_paged_diff(*args, lam, norm_weight=torch.ones(129, device="cuda")[1:])
