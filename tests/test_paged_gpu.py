"""GPU tests of the paged 8-bit cache against its definitions in 64 bits (oracle/paged.py)."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import _lib
from oracle import paged as ref

pytestmark = pytest.mark.gpu

THETA = 500000.0
DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ---- page planning -----------------------------------------------------------------------------------------------
def run_plan(lens, new, table, free, capacity, page_len, max_tokens, in_place=False):
    """Plan on the GPU from Python lists; returns (plan, table, free) with the tensors."""
    stack = ints(free + [-7] * (capacity - len(free)))
    n_free, t, ln = ints([len(free)]), ints(table), ints(lens)
    more = {"lens_out": ln, "n_free_out": n_free} if in_place else {}
    plan = gqa.plan_pages(ln, ints(new), t, stack, n_free, page_len=page_len, max_tokens=max_tokens, **more)
    return plan, t, stack


@pytest.mark.parametrize("requests,page_len,longest,most", [
    (1, 16, 40, 1), (1, 128, 300, 300), (3, 32, 70, 40), (64, 16, 300, 1), (64, 64, 500, 129),
    (1025, 16, 90, 50), (2500, 64, 200, 3), (8192, 16, 40, 2)])
def test_plan_follows_a_run_of_steps(requests, page_len, longest, most):
    rng = random.Random(requests * 131 + page_len)
    width = -(-(longest + most * 4) // page_len) + 1
    capacity = requests * width
    table = [[-1] * width for _ in range(requests)]
    free = list(range(capacity))
    rng.shuffle(free)
    lens = [0] * requests
    for step in range(4):
        new = [rng.randint(0, longest if step == 0 else most) for _ in range(requests)]
        if step >= 2:
            new = [-1 if rng.random() < 0.3 else a for a in new]
        max_tokens = sum(max(0, a) for a in new) + rng.randint(0, 5)
        plan, t, stack = run_plan(lens, new, table, free, capacity, page_len, max_tokens, in_place=step % 2 == 1)
        ok, lens, first, slots, positions, taken, given = ref.plan_step(lens, new, table, free, page_len, max_tokens,
                                                                        capacity)
        assert ok
        assert plan.counts.tolist() == [first[-1], taken, given, 0]
        assert plan.lens.tolist() == lens and plan.n_free.tolist() == [len(free)]
        assert plan.first_token.tolist() == first
        assert plan.slots.tolist() == slots and plan.positions.tolist() == positions
        got = t.tolist()
        for r, n in enumerate(lens):
            assert got[r][:-(-n // page_len)] == table[r][:-(-n // page_len)]
        assert stack.tolist()[:len(free)] == free
        plan.check()


@pytest.mark.parametrize("why", ["pages", "width", "tokens", "negative", "capacity"])
@pytest.mark.parametrize("requests", [3, 1500])
def test_plan_refuses_and_changes_nothing(why, requests):
    lens, new, width, capacity, free = [20] * requests, [5] * requests, 3, requests * 3, list(range(requests, requests * 2))
    max_tokens = 5 * requests
    table = [[r, -1, -1] for r in range(requests)]
    for row in table:
        row[1] = row[0] + 2 * requests
    new[0] = -1
    if why == "pages":
        new[2], free = 28, []
        new[0], max_tokens = 0, 5 * requests + 28
    elif why == "width":
        new[1], max_tokens = 40, 5 * requests + 40
    elif why == "tokens":
        max_tokens = 5 * (requests - 1) - 1
    elif why == "negative":
        lens[1] = -1
    else:
        capacity = len(free) + 1
    plan, t, stack = run_plan(lens, new, table, free, capacity, 16, max_tokens)
    before = [list(r) for r in table]
    assert not ref.plan_step(lens, new, table, list(free), 16, max_tokens, capacity)[0]
    assert plan.counts.tolist() == [0, 0, 0, _lib.GQA_ERR_PAGES]
    assert plan.lens.tolist() == lens and plan.n_free.tolist() == [len(free)]
    assert set(plan.slots.tolist()) <= {-1} and set(plan.first_token.tolist()) == {0}
    assert t.tolist() == before and stack.tolist()[:len(free)] == free
    with pytest.raises(gqa.GqaError, match="page planning refused"):
        plan.check()


# ---- append and read-back ----------------------------------------------------------------------------------------
def random_cache(gen, pages, page_len, code, layout, heads=8, fill=True):
    cache = gqa.paged_cache(pages, page_len, dtype=DTYPES[code], kv_heads=heads, layout=layout)
    if fill:
        for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            c = torch.randint(0, 256, t.shape, generator=gen, device="cuda", dtype=torch.uint8)
            if code == "e4m3":
                c[(c & 0x7F) == 0x7F] = 0x11  # no NaN codes
            else:
                c[c == 128] = 7  # codes are in [-127, 127]
            t.view(torch.uint8).copy_(c)
            s.copy_(torch.exp(0.5 * torch.randn(s.shape, generator=gen, device="cuda")) *
                    (1 / 127 if code == "int8" else 1 / 448))
    return cache


def words(t):
    """Codes of a cache tensor as uint8 [pages, page_len, heads, 128] on the host."""
    return t.view(torch.uint8).cpu().numpy()


def rows_of(cache, t):
    w = words(t)
    return w if cache.layout == "position_major" else w.transpose(0, 2, 1, 3)


def expect_append(codes, scale, x, slots, page_len, code):
    """Codes [pages, page_len, heads, 128] and scales after an append of float32 rows, one run at a time, in float32
    where the definition is (a division and two products, each rounded)."""
    codes, scale = codes.copy(), scale.copy()
    top = np.float32(ref.CODE_MAX[code])

    def encode(y):
        y = torch.from_numpy(np.clip(y, -top, top).astype(np.float32))
        if code == "int8":
            return y.round().to(torch.int8).view(torch.uint8).numpy()
        return y.to(torch.float8_e4m3fn).view(torch.uint8).numpy()

    def values(c):
        return ref.code_values(c, code).astype(np.float32)

    t = 0
    while t < len(slots):
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % page_len:
            n += 1
        if slots[t] >= 0:
            page, r = slots[t] // page_len, slots[t] % page_len
            old = scale[page] if r else np.zeros_like(scale[page])
            mine = np.maximum(np.abs(x[t:t + n]).max((0, 2)) / top, np.float32(ref.MIN_SCALE))
            now = np.maximum(mine, old)
            inv = np.float32(1) / now
            grew = mine > old
            again = encode((values(codes[page, :r]) * old[:, None]) * inv[:, None])
            codes[page, :r] = np.where(grew[:, None], again, codes[page, :r])
            codes[page, r:r + n] = encode(x[t:t + n] * inv[:, None])
            scale[page] = now
        t += n
    return codes, scale


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("layout", ["head_major", "position_major"])
@pytest.mark.parametrize("page_len", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_append_without_rope_is_exact(code, layout, page_len, heads):
    gen = torch.Generator("cuda").manual_seed(page_len + heads)
    cache = random_cache(gen, 12, page_len, code, layout, heads)
    # runs: a page's end, a whole page, a single row, a skipped slot, a short start, one row in mid-page, zeros
    runs = [(3, page_len - 3, 3), (7, 0, page_len), (1, 5, 1), (-1, 0, 2), (0, 0, 7), (9, page_len // 2, 1), (11, 0, 2)]
    slots = [page * page_len + r + i if page >= 0 else -1 for page, r, n in runs for i in range(n)]
    n = len(slots)
    k = (torch.randn(n, heads, 128, generator=gen, device="cuda") * 3).to(torch.bfloat16)
    v = torch.randn(n, heads, 128, generator=gen, device="cuda").to(torch.bfloat16)
    v[1] *= 100
    k[-2:] = 0
    want = {name: expect_append(rows_of(cache, t), s.cpu().numpy(), x.float().cpu().numpy(), slots, page_len, code)
            for name, t, s, x in (("k", cache.k, cache.k_scale, k), ("v", cache.v, cache.v_scale, v))}
    wide = torch.zeros(n, heads + 2, 256, dtype=torch.bfloat16, device="cuda")  # rows inside larger ones
    wide[:, 1:1 + heads, 128:] = k
    gqa.append_paged(cache, wide[:, 1:1 + heads, 128:], v, ints(slots, torch.int64))
    for name, t, s in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
        codes, scale = want[name]
        assert np.array_equal(s.cpu().numpy(), scale), name
        assert np.array_equal(rows_of(cache, t), codes), name
    # read-back: code * scale, rounded to BF16, in any order, with zeros for what is not there
    ask = [s for s in slots if s >= 0][::-1] + [-1, 12 * page_len]
    got = gqa.read_paged(cache, ints(ask, torch.int64))
    for (codes, scale), g in zip((want["k"], want["v"]), got):
        x = np.zeros((len(ask), heads, 128), np.float32)
        for i, s in enumerate(ask[:-2]):
            x[i] = ref.code_values(codes[s // page_len, s % page_len], code).astype(np.float32) * \
                scale[s // page_len][:, None]
        assert torch.equal(g.cpu(), torch.from_numpy(x).to(torch.bfloat16))


@pytest.mark.parametrize("page_len,code", [(16, "e4m3"), (32, "int8"), (64, "e4m3"), (128, "int8")])
def test_append_of_many_tokens_is_exact(page_len, code):
    """Prompts: more tokens than a step has, runs that fill pages and cross them."""
    gen = torch.Generator("cuda").manual_seed(page_len)
    lens, starts = [700, 1, page_len * 3, 331, 90], [5, page_len - 1, 0, page_len // 2, 3]
    table, slots = list(range(200))[::-1], []
    for n, a in zip(lens, starts):
        pages = [table.pop() for _ in range(-(-(a + n) // page_len))]
        slots += [pages[(a + i) // page_len] * page_len + (a + i) % page_len for i in range(n)]
    cache = random_cache(gen, 200, page_len, code, "position_major", 3)
    n = len(slots)
    assert n > 1024
    k, v = (torch.randn(n, 3, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    k[::100] *= 30
    want = {name: expect_append(rows_of(cache, t), s.cpu().numpy(), x.float().cpu().numpy(), slots, page_len, code)
            for name, t, s, x in (("k", cache.k, cache.k_scale, k), ("v", cache.v, cache.v_scale, v))}
    gqa.append_paged(cache, k, v, ints(slots, torch.int64))
    for name, t, s in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
        assert np.array_equal(s.cpu().numpy(), want[name][1]), name
        assert np.array_equal(rows_of(cache, t), want[name][0]), name
    # the same rows with rotation by zero, which is none: the same codes
    again = random_cache(gen, 200, page_len, code, "position_major", 3)
    again.k.view(torch.uint8).copy_(cache.k.view(torch.uint8))
    again.k_scale.copy_(cache.k_scale)
    gqa.append_paged(again, k, v, ints(slots, torch.int64), positions=torch.zeros(n, dtype=torch.int32, device="cuda"))
    assert torch.equal(again.k_scale, cache.k_scale) and np.array_equal(words(again.k), words(cache.k))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_rotates_k(code):
    """Stored K is RoPE(k) to half a step of its scale; the rotation's own error (FP32, about 2^-22 of the pair's
    size) can move a value across a rounding boundary, which the allowance of 2^-20 of the block's largest covers."""
    gen = torch.Generator("cuda").manual_seed(5)
    n, page_len = 300, 64
    cache = gqa.paged_cache(6, page_len, dtype=DTYPES[code])
    k = torch.randn(n, 8, 128, generator=gen, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 1 << 20, (n,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.arange(3, n + 3, device="cuda")
    gqa.append_paged(cache, k, k, slots, positions=pos, rope_theta=THETA)
    want = ref.rope(k.float().cpu().numpy(), pos.cpu().numpy(), THETA)
    s = slots.cpu().numpy()
    scale = cache.k_scale.cpu().numpy().astype(np.float64)[s // page_len][..., None]
    got = ref.code_values(rows_of(cache, cache.k)[s // page_len, s % page_len], code) * scale
    half = scale / 2 if code == "int8" else np.maximum(np.abs(want) * 2.0 ** -4, scale * 2.0 ** -10)
    assert (np.abs(got - want) <= half * (1 + 2 ** -6) + scale * ref.CODE_MAX[code] * 2.0 ** -20).all()
    for page in range(6):
        mine = np.abs(want[s // page_len == page]).max((0, 2)) / ref.CODE_MAX[code] if (s // page_len == page).any() else 0
        assert np.allclose(cache.k_scale[page].cpu().numpy(), mine, rtol=2.0 ** -20)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_of_a_non_finite_row_marks_its_block(bad):
    gen = torch.Generator("cuda").manual_seed(6)
    cache = random_cache(gen, 4, 16, "e4m3", "head_major")
    before = words(cache.v).copy()
    k = torch.randn(20, 8, 128, generator=gen, device="cuda").to(torch.bfloat16)
    v = k.clone()
    v[17, 3, 5] = bad
    gqa.append_paged(cache, k, v, torch.arange(18, 38, device="cuda"))
    vs, ks = cache.v_scale.cpu(), cache.k_scale.cpu()
    assert torch.isnan(vs[2, 3]) and int(torch.isnan(vs).sum()) == 1 and not torch.isnan(ks).any()
    after = words(cache.v)
    assert (after[2, 3, :6] == 0).all()
    assert np.array_equal(after[0], before[0]) and np.array_equal(after[3], before[3])
    k2, v2 = gqa.read_paged(cache, ints([35, 20], torch.int64))
    assert torch.isnan(v2[0, 3]).all() and not torch.isnan(v2[0, :3]).any() and not torch.isnan(v2[1]).any()
    # a later append to the block keeps the mark, and starting the page again clears it
    gqa.append_paged(cache, k[:1], k[:1], ints([38], torch.int64))
    assert torch.isnan(cache.v_scale[2, 3])
    gqa.append_paged(cache, k[:1], k[:1], ints([32], torch.int64))
    assert not torch.isnan(cache.v_scale).any()


def test_append_in_many_steps_matches_rows_within_their_steps():
    """One row at a time: every stored value stays within half a step of each scale it was rounded to."""
    gen = torch.Generator("cuda").manual_seed(8)
    cache = gqa.paged_cache(2, 32, dtype=torch.int8)
    x = torch.randn(40, 8, 128, generator=gen, device="cuda").to(torch.bfloat16)
    x *= torch.linspace(0.2, 4, 40, device="cuda").to(torch.bfloat16)[:, None, None]
    for i in range(40):
        gqa.append_paged(cache, x[i:i + 1], x[i:i + 1], ints([i], torch.int64))
    k, v = gqa.read_paged(cache, torch.arange(40, device="cuda"))
    assert torch.equal(k, v)
    scale = cache.k_scale[torch.arange(40, device="cuda") // 32][..., None]
    # each of the (at most 32) growths of a block's scale adds half a step of that scale; the scales grow to the last
    grown = torch.cummax(x.abs().amax(-1).float(), 0).values / 127
    steps = torch.zeros(40, 8, device="cuda")
    for i in range(40):
        last = 32 if i < 32 else 40
        s = torch.unique_consecutive(grown[i:last], dim=0) if i < 32 else \
            torch.unique_consecutive(torch.cummax(x[32:].abs().amax(-1).float(), 0).values[i - 32:] / 127, dim=0)
        steps[i] = s.sum(0) / 2
    assert ((v.float() - x.float()).abs() <= steps[..., None] * 1.01 + x.float().abs() * 2 ** -8 + scale * 2 ** -10).all()


# ---- attention ---------------------------------------------------------------------------------------------------
class Setup:
    """Sequences in a shuffled cache, with values the tests can put anywhere."""

    def __init__(self, lens, *, seed, page_len=64, code="int8", layout="head_major", heads=8, width=None, spare=2):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.lens, self.page_len, self.code, self.heads = lens, page_len, code, heads
        need = [-(-n // page_len) for n in lens]
        pages = sum(need) + spare
        self.cache = random_cache(gen, pages, page_len, code, layout, heads)
        order = torch.randperm(pages, generator=gen, device="cuda").tolist()
        width = width or max(1, max(need))
        self.table = [[-1] * width for _ in lens]
        for b, n in enumerate(need):
            self.table[b][:n] = [order.pop() for _ in range(n)]
        self.unused = order
        self.gen = gen

    def queries(self, rows):
        return torch.randn(rows, 4 * self.heads, 128, generator=self.gen, device="cuda").to(torch.bfloat16)

    def poison(self, spoiled):
        """NaN codes and scales where no visible key is: the pages of no sequence, and of each sequence b the keys
        that ``spoiled(b, p)`` names (only whole pages of them get a NaN scale)."""
        n = self.page_len
        bad = 0x7F if self.code == "e4m3" else 0x80
        for c, s in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            rows = c.view(torch.uint8)
            rows = rows if self.cache.layout == "position_major" else rows.transpose(1, 2)
            for page in self.unused:
                rows[page] = bad
                s[page] = math.nan
            for b, length in enumerate(self.lens):
                for col in range(-(-length // n)):
                    gone = [r for r in range(n) if col * n + r >= length or spoiled(b, col * n + r)]
                    rows[self.table[b][col], gone] = bad
                    if len(gone) == n:
                        s[self.table[b][col]] = math.nan

    def values(self, b):
        n, page_len = self.lens[b], self.page_len
        p = np.arange(n)
        page = np.array(self.table[b])[p // page_len] if n else p
        out = []
        for c, s in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            x = ref.code_values(rows_of(self.cache, c)[page, p % page_len], self.code)
            out.append(x * s.cpu().numpy().astype(np.float64)[page][..., None])
        return out


#: Relative size of what each kernel rounds beside its output: the decode kernel keeps Q and the weights in two FP16
#: parts (22 bits) and the codes are exact; the chunked kernel keeps one FP16 part of Q, the weights, and the scaled
#: codes of K and V (2^-11 each).
DECODE_UNIT, CHUNK_UNIT = 2.0 ** -20, 2.0 ** -11


def check(got, q, setup, owner, positions, *, unit, q_rotated=False, cap=0.0, slopes=None, starts=None, ends=None,
          scale=1 / math.sqrt(128)):
    """Every output against 64 bits.  A score is off by at most 2 units of the sum of its terms' sizes (Q and K), plus
    FP32's 2^-20 of that (rotation, sums), of the cap and of the bias; a weight by e to twice that, plus a unit for its
    rounding and one for V's; the output by a BF16 rounding (8 significant bits: 2^-8 of it at most)."""
    got = got.float().cpu().numpy().astype(np.float64)
    x = q.float().cpu().numpy().astype(np.float64)
    if not q_rotated:
        x = ref.rope(x, np.array(positions), THETA)
    slopes = slopes.cpu().numpy().astype(np.float64) if slopes is not None else None
    kv = {b: setup.values(b) for b in set(owner)}
    for i, (b, m) in enumerate(zip(owner, positions)):
        p = np.arange(setup.lens[b])
        end = max(m + 1, ends[i] if ends is not None else 0)
        seen = (p >= (starts[i] if starts is not None else 0)) & (p < end)
        k, v = kv[b]
        out, size, most = ref.attend(x[i], k, v, m, seen, scale=scale, cap=cap, slopes=slopes)
        far = np.abs(m - p).max() * slopes.max() if slopes is not None and len(p) else 0.0
        z = (2 * unit + 2.0 ** -20) * most + 2.0 ** -20 * cap + 2.0 ** -22 * far
        tol = 2.0 ** -8 * np.abs(out) + (math.expm1(2 * z) + 3 * unit + 2.0 ** -20) * size * 1.01 + 1e-30
        bad = ~(np.abs(got[i] - out) <= tol)
        assert not bad.any(), (i, b, m, int(bad.sum()), float((np.abs(got[i] - out) / tol)[~np.isnan(got[i])].max()))


ODD_LENS = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 2, 1000]


@pytest.mark.parametrize("page_len", [16, 32, 64, 128])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("layout", ["head_major", "position_major"])
def test_decode_lengths(page_len, code, layout):
    s = Setup(ODD_LENS, seed=page_len, page_len=page_len, code=code, layout=layout)
    q = s.queries(len(ODD_LENS))
    s.poison(lambda b, p: False)
    got = gqa.decode_paged(q, s.cache, ints(s.table), ints(ODD_LENS))
    check(got, q, s, list(range(len(ODD_LENS))), [n - 1 for n in ODD_LENS], unit=DECODE_UNIT)
    again = gqa.decode_paged(q, s.cache, ints(s.table), ints(ODD_LENS))
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("lens", [[30], [1], [4096], [20000], [5000, 1, 700]])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_decode_few_sequences(lens, code):
    s = Setup(lens, seed=sum(lens), page_len=16 if lens == [30] else 64, code=code)
    q = s.queries(len(lens))
    got = gqa.decode_paged(q, s.cache, ints(s.table), ints(lens))
    check(got, q, s, list(range(len(lens))), [n - 1 for n in lens], unit=DECODE_UNIT)


@pytest.mark.parametrize("heads", [1, 2, 3, 5])
def test_head_shards(heads):
    lens = [200, 1, 77]
    s = Setup(lens, seed=heads, page_len=32, code="e4m3", heads=heads, layout="position_major")
    q = s.queries(3)
    check(gqa.decode_paged(q, s.cache, ints(s.table), ints(lens)), q, s, [0, 1, 2], [199, 0, 76], unit=DECODE_UNIT)
    first = [0, 100, 101, 150]
    q = s.queries(150)
    owner = [0] * 100 + [1] + [2] * 49
    pos = list(range(100, 200)) + [0] + list(range(28, 77))
    check(gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first)), q, s, owner, pos,
          unit=CHUNK_UNIT)


MODS = ["cap", "slopes", "docs", "prefix", "cap slopes", "cap slopes docs prefix"]


def modifiers(s, what, owner, positions):
    """Keyword arguments of a call and of ``check`` for the named score changes; some rows see nothing."""
    rng = np.random.RandomState(len(what))
    call, chk = {}, {}
    if "cap" in what:
        call["score_cap"] = chk["cap"] = 5.0
    if "slopes" in what:
        chk["slopes"] = call["distance_slopes"] = 2.0 ** (-8 * torch.arange(1, 4 * s.heads + 1, device="cuda") / (4 * s.heads))
        call["q_rotated"] = chk["q_rotated"] = True
    if "docs" in what:
        starts = [int(rng.randint(-3, max(1, m + 1))) for m in positions]
        for i in range(0, len(starts), 4):
            starts[i] = s.lens[owner[i]] + int(rng.randint(0, 3))  # nothing visible
        call["doc_starts"], chk["starts"] = ints(starts), starts
    if "prefix" in what:
        ends = [int(rng.randint(-2, s.lens[b] + 40)) for b in owner]
        call["prefix_ends"], chk["ends"] = ints(ends), ends
    return call, chk


@pytest.mark.parametrize("what", MODS)
@pytest.mark.parametrize("code,page_len", [("int8", 16), ("e4m3", 64)])
def test_decode_masks_cap_and_bias(what, code, page_len):
    lens = ODD_LENS + [513, 700, 90, 31]
    s = Setup(lens, seed=len(what), page_len=page_len, code=code)
    owner = list(range(len(lens)))
    rng = np.random.RandomState(3)
    pos = [int(rng.randint(0, max(1, n))) for n in lens]
    q = s.queries(len(lens))
    call, chk = modifiers(s, what, owner, pos)
    starts, ends = chk.get("starts", [0] * len(lens)), chk.get("ends", [0] * len(lens))
    s.poison(lambda b, p: not starts[b] <= p < max(pos[b] + 1, ends[b]))
    got = gqa.decode_paged(q, s.cache, ints(s.table), ints(lens), query_positions=ints(pos), **call)
    check(got, q, s, owner, pos, unit=DECODE_UNIT, **chk)


@pytest.mark.parametrize("counts,lens", [
    ([1], [1]), ([5], [5]), ([3], [300]), ([128], [8192]), ([1, 1, 1], [1, 90, 17]),
    ([33, 0, 1, 64, 65], [33, 10, 400, 64, 700]), ([257], [257]), ([31, 32, 33, 127, 129], [1000, 32, 500, 127, 200])])
@pytest.mark.parametrize("code,page_len,layout", [("int8", 16, "position_major"), ("e4m3", 64, "head_major"),
                                                  ("int8", 128, "head_major"), ("e4m3", 32, "position_major")])
def test_chunked_lengths(counts, lens, code, page_len, layout):
    s = Setup(lens, seed=sum(lens), page_len=page_len, code=code, layout=layout)
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    rows = first[-1]
    q = s.queries(rows + 3)
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]
    s.poison(lambda b, p: False)
    out = torch.full((rows + 3, 32, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), out=out)
    assert got is out and bool((out[rows:] == 7.0).all())
    pick = sorted(set(range(0, rows, max(1, rows // 40))) | {rows - 1})
    check(got[pick], q[pick], s, [owner[i] for i in pick], [pos[i] for i in pick], unit=CHUNK_UNIT)
    again = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first))
    assert torch.equal(got[:rows].view(torch.int16), again[:rows].view(torch.int16))
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("what", MODS)
@pytest.mark.parametrize("code,page_len", [("e4m3", 16), ("int8", 64)])
def test_chunked_masks_cap_and_bias(what, code, page_len):
    counts, lens = [40, 130, 1, 7], [40, 301, 77, 7]
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
    got = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), **call)
    check(got, q, s, owner, pos, unit=CHUNK_UNIT, **chk)


def test_chunked_and_decode_agree():
    """One query a sequence through both: the same rows within the chunked kernel's bound of the definition."""
    lens = [700, 65, 1]
    s = Setup(lens, seed=12, page_len=32, code="e4m3")
    q = s.queries(3)
    a = gqa.decode_paged(q, s.cache, ints(s.table), ints(lens))
    b = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints([0, 1, 2, 3]))
    for got, unit in ((a, DECODE_UNIT), (b, CHUNK_UNIT)):
        check(got, q, s, [0, 1, 2], [699, 64, 0], unit=unit)


def test_strided_rows_and_scale():
    lens = [90, 200]
    s = Setup(lens, seed=4, page_len=16)
    wide = torch.zeros(2, 40, 256, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 3:35, 64:192]
    q.copy_(s.queries(2))
    out = torch.zeros(2, 34, 136, dtype=torch.bfloat16, device="cuda")
    wide_table = torch.full((2, 50), 9999, dtype=torch.int32, device="cuda")
    wide_table[:, :len(s.table[0])] = ints(s.table)
    got = gqa.decode_paged(q, s.cache, wide_table[:, :len(s.table[0])], ints(lens), out=out[:, 1:33, :128], scale=0.3)
    check(got, q, s, [0, 1], [89, 199], unit=DECODE_UNIT, scale=0.3)
    assert bool((out[:, 0] == 0).all()) and bool((out[:, 33] == 0).all()) and bool((out[..., 128:] == 0).all())


def test_table_bounds_are_kept():
    """A length past what the table can name is cut to it, and page numbers outside the cache read as zeros."""
    s = Setup([64, 64], seed=14, page_len=32)
    q = s.queries(2)
    table = ints(s.table)
    want = gqa.decode_paged(q, s.cache, table, ints([64, 64]), query_positions=ints([63, 63]))
    got = gqa.decode_paged(q, s.cache, table, ints([1 << 30, 65]), query_positions=ints([63, 63]))
    assert torch.equal(want, got)
    for page in (-5, s.cache.pages, 1 << 30):
        table[1, 0] = page
        got = gqa.decode_paged(q, s.cache, table, ints([64, 64]))
        assert torch.equal(got[0], want[0])
        zero = Setup([64, 64], seed=14, page_len=32)
        rows = zero.cache.k.view(torch.uint8), zero.cache.v.view(torch.uint8)
        for r in rows:
            r[zero.table[1][0]] = 0
        check(got, q, zero, [0, 1], [63, 63], unit=DECODE_UNIT)
        rows = gqa.decode_paged_chunked(q, s.cache, table, ints([64, 64]), ints([0, 1, 2]))
        check(rows, q, zero, [0, 1], [63, 63], unit=CHUNK_UNIT)


def test_large_and_tiny_scales_and_queries():
    """Scales and queries of very different sizes in one sequence: no part overflows or vanishes."""
    lens = [200]
    for big, small in ((1e4, 1e-6), (1e18, 1e12), (1e-18, 1e-20)):
        s = Setup(lens, seed=21, page_len=16, code="e4m3")
        col = ints(s.table[0])[:13].long()
        s.cache.v_scale[col] = ints([big if i % 3 == 0 else small for i in range(13)], torch.float32)[:, None] / 448
        s.cache.k_scale[col] = 1e-3
        q = s.queries(1)
        q[:, ::2] *= 64
        check(gqa.decode_paged(q, s.cache, ints(s.table), ints(lens)), q, s, [0], [199], unit=DECODE_UNIT)
    s = Setup(lens, seed=22, page_len=16)
    s.cache.k_scale.mul_(1e-25)
    q = s.queries(1) * 1e25
    check(gqa.decode_paged(q, s.cache, ints(s.table), ints(lens)), q, s, [0], [199], unit=DECODE_UNIT)


def test_a_visible_nan_reaches_its_rows_only():
    lens = [100, 100]
    s = Setup(lens, seed=15, page_len=16, code="int8")
    s.cache.v_scale[s.table[0][3], 2] = math.nan
    s.cache.k_scale[s.table[1][6], 5] = math.nan
    q = s.queries(2)
    for got in (gqa.decode_paged(q, s.cache, ints(s.table), ints(lens)),
                gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints([0, 1, 2]))):
        nan = torch.isnan(got).any(-1)
        want = torch.zeros_like(nan)
        want[0, 8:12] = True
        want[1, 20:24] = True
        assert torch.equal(nan, want)


def test_offsets_past_32_bits():
    """Pages more than 4 GB into the cache."""
    pages = 36000
    k, v = (torch.empty(pages, 8, 128, 128, dtype=torch.uint8, device="cuda").view(torch.int8) for _ in range(2))
    ks, vs = (torch.empty(pages, 8, dtype=torch.float32, device="cuda") for _ in range(2))
    cache = gqa.PagedCache(k, v, ks, vs)
    lens = [300, 40]
    s = Setup(lens, seed=16, page_len=128, spare=0)
    far = [35999, 17, 35000, 34000]
    table, at = [[-1] * 3 for _ in lens], 0
    for b, n in enumerate((3, 1)):
        for col in range(n):
            src, dst = s.table[b][col], far[at]
            k[dst], v[dst], ks[dst], vs[dst] = s.cache.k[src], s.cache.v[src], s.cache.k_scale[src], s.cache.v_scale[src]
            table[b][col] = dst
            at += 1
    q = s.queries(2)
    check(gqa.decode_paged(q, cache, ints(table), ints(lens)), q, s, [0, 1], [299, 39], unit=DECODE_UNIT)
    check(gqa.decode_paged_chunked(q, cache, ints(table), ints(lens), ints([0, 1, 2])), q, s, [0, 1], [299, 39],
          unit=CHUNK_UNIT)
    x = torch.randn(2, 8, 128, device="cuda").to(torch.bfloat16)
    slots = ints([35000 * 128 + 44, 35000 * 128 + 45], torch.int64)
    gqa.append_paged(cache, x, x, slots)
    assert float((gqa.read_paged(cache, slots)[1].float() - x.float()).abs().max()) < 0.05


def test_side_streams_and_graphs():
    """The whole step on a side stream, then as a CUDA graph replayed with other lengths."""
    page_len, batch = 16, 5
    gen = torch.Generator("cuda").manual_seed(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache = gqa.paged_cache(64, page_len)
    lens, new = ints([0] * batch), ints([20, 1, 16, 33, 5])
    table, free, n_free = ints([[-1] * 8] * batch), torch.arange(64, device="cuda", dtype=torch.int32), ints([64])
    k, v = (torch.randn(batch * 33, 8, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(batch, 32, 128, generator=gen, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)

    def step():
        plan = gqa.plan_pages(lens, new, table, free, n_free, page_len=page_len, max_tokens=batch * 33, lens_out=lens,
                              n_free_out=n_free)
        gqa.append_paged(cache, k, v, plan.slots, positions=plan.positions)
        gqa.decode_paged(q, cache, table, lens, out=out)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    first = out.clone()
    assert lens.tolist() == [20, 1, 16, 33, 5] and bool(first.abs().sum() > 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for adds in ([1, 0, 1, 1, 1], [0, 30, 1, 0, -1], [2, 2, 2, 2, 2]):
        before = lens.tolist()
        new.copy_(ints(adds))
        graph.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [0 if a < 0 else n + a for n, a in zip(before, adds)]
        want = gqa.decode_paged(q, cache, table, lens)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_calls_of_different_sizes_share_a_workspace():
    """Calls in turn on one stream: what one leaves in the workspace does not reach the next."""
    calls = []
    for lens, page_len, heads in (([3000, 500] * 20, 64, 8), ([4000], 16, 1), ([900, 2000, 40] * 5, 32, 8),
                                  ([20000], 64, 8), ([129] * 300, 16, 2)):
        s = Setup(lens, seed=len(lens), page_len=page_len, heads=heads)
        calls.append((s, s.queries(len(lens)), ints(s.table), ints(lens)))
    first = [gqa.decode_paged(q, s.cache, t, n) for s, q, t, n in calls]
    for _ in range(3):
        again = [gqa.decode_paged(q, s.cache, t, n) for s, q, t, n in calls]
        for a, b in zip(first, again):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    for (s, q, _, _), got in zip(calls, again):
        pick = list(range(0, len(s.lens), max(1, len(s.lens) // 6)))
        check(got[pick], q[pick], s, pick, [s.lens[i] - 1 for i in pick], unit=DECODE_UNIT)


def test_nothing_visible_at_all():
    lens = [70, 0, 200]
    s = Setup(lens, seed=41, page_len=16, code="e4m3")
    q = s.queries(3)
    out = torch.full((3, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    gqa.decode_paged(q, s.cache, ints(s.table), ints(lens), doc_starts=ints([70, 0, 900]), out=out)
    assert not out.any()
    first = [0, 70, 70, 150]
    q = s.queries(150)
    out = torch.full((150, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), doc_starts=ints([300] * 150), out=out)
    assert not out.any()
    out = torch.full((150, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints([0, 0, 0, 0]), out=out)
    assert bool((out == 5.0).all())  # no sequence has a query


def test_first_query_is_kept_within_the_rows():
    """Numbers in first_query that name rows the call does not have are cut to those it has."""
    lens = [100, 100]
    s = Setup(lens, seed=42, page_len=32)
    q = s.queries(10)
    guard = torch.full((30, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    for first in ([0, 4, 1 << 30], [-7, 4, 10], [0, 12, 11], [10, 4, 2]):
        gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), out=guard[10:20])
        assert bool((guard[:10] == 5.0).all()) and bool((guard[20:] == 5.0).all())
    assert gqa.read_device_status() == 0


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    setups = [Setup(lens, seed=50 + i, page_len=64) for i, lens in enumerate(([5000, 300] * 8, [900, 2000, 40] * 6))]
    work, want = [], []
    for s in setups:
        n = len(s.lens)
        first = [0]
        for length in s.lens:
            first.append(first[-1] + min(length, 40))
        work.append((s, s.queries(n), s.queries(first[-1]), ints(s.table), ints(s.lens), ints(first)))
    run = lambda s, q, qc, t, n, f: (gqa.decode_paged(q, s.cache, t, n),  # noqa: E731
                                     gqa.decode_paged_chunked(qc, s.cache, t, n, f))
    want = [run(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[] for _ in work]
    for _ in range(10):
        for i, (w, st) in enumerate(zip(work, streams)):
            with torch.cuda.stream(st):
                got[i].append(run(*w))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for pair in g:
            for a, b in zip(pair, w):
                assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_the_largest_batch():
    lens = [(i * 53) % 40 for i in range(8192)]
    s = Setup(lens, seed=31, page_len=16, heads=1)
    q = s.queries(8192)
    got = gqa.decode_paged(q, s.cache, ints(s.table), ints(lens))
    pick = list(range(0, 8192, 409)) + [8191]
    check(got[pick], q[pick], s, pick, [lens[i] - 1 for i in pick], unit=DECODE_UNIT)
    rows = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(list(range(8193))))
    check(rows[pick], q[pick], s, pick, [lens[i] - 1 for i in pick], unit=CHUNK_UNIT)
    assert gqa.read_device_status() == 0


def test_many_sequences():
    lens = [(i * 37) % 150 for i in range(1500)]
    s = Setup(lens, seed=30, page_len=16, code="e4m3", heads=2)
    q = s.queries(1500)
    got = gqa.decode_paged(q, s.cache, ints(s.table), ints(lens))
    pick = list(range(0, 1500, 61)) + [1499]
    sub = [got[i] for i in pick]
    check(torch.stack(sub), q[pick], s, pick, [lens[i] - 1 for i in pick], unit=DECODE_UNIT)
    rows = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(list(range(1501))))
    check(rows[pick], q[pick], s, pick, [lens[i] - 1 for i in pick], unit=CHUNK_UNIT)


# ---- a few queries a sequence: a kernel of its own, which keeps one FP16 part of Q and of the weights (so CHUNK_UNIT's
# bound holds for it: it rounds a subset of what the chunked kernel does) --------------------------------------------
@pytest.mark.parametrize("counts,lens", [
    ([6], [6]), ([2], [31]), ([4], [33]), ([6], [20000]),             # one unit, cut by up to every CTA
    ([1, 2, 3, 4, 5, 6], [1, 2, 300, 64, 5, 3000]),                   # every number of queries
    ([7, 0, 5, 13, 1, 6, 0, 12], [7, 9, 1000, 13, 40, 700, 0, 65]),   # several units a sequence, and none
    ([5] * 60, [5 + 37 * i for i in range(60)])])                     # many units a share
@pytest.mark.parametrize("code,page_len,layout", [("int8", 16, "position_major"), ("e4m3", 64, "head_major"),
                                                  ("int8", 128, "head_major"), ("e4m3", 32, "position_major")])
def test_few_queries_a_sequence(counts, lens, code, page_len, layout):
    assert sum(counts) <= 6 * len(counts)
    s = Setup(lens, seed=sum(lens), page_len=page_len, code=code, layout=layout)
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    rows = first[-1]
    q = s.queries(rows + 2)
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]
    s.poison(lambda b, p: False)
    out = torch.full((rows + 2, 32, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), out=out)
    assert bool((out[rows:] == 7.0).all())
    pick = sorted(set(range(0, rows, max(1, rows // 40))) | {rows - 1})
    check(got[pick], q[pick], s, [owner[i] for i in pick], [pos[i] for i in pick], unit=CHUNK_UNIT)
    again = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first))
    assert torch.equal(got[:rows].view(torch.int16), again[:rows].view(torch.int16))
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("what", MODS)
@pytest.mark.parametrize("code,page_len", [("e4m3", 16), ("int8", 64)])
def test_few_queries_masks_cap_and_bias(what, code, page_len):
    counts, lens = [6, 5, 1, 11, 2, 0, 4], [6, 301, 77, 700, 1500, 8, 130]
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
    got = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first), **call)
    check(got, q, s, owner, pos, unit=CHUNK_UNIT, **chk)
    assert gqa.read_device_status() == 0


@pytest.mark.parametrize("counts,lens", [
    ([1] * 20 + [100], [40] * 20 + [3000]),        # the long one has the keys, too: cut as chunks
    ([100] + [1] * 20, [130] + [2000] * 20),       # it has few of them: cut as few queries
    ([0] * 20 + [120], [5] * 20 + [121]),
    ([2] * 7, [0] * 7)])                           # more rows than keys: most of them see nothing
def test_one_chunk_among_single_tokens(counts, lens):
    s = Setup(lens, seed=5, page_len=32, code="int8")
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]
    q = s.queries(first[-1])
    s.poison(lambda b, p: False)
    got = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first))
    check(got, q, s, owner, pos, unit=CHUNK_UNIT)
    assert gqa.read_device_status() == 0


def test_few_queries_reach_every_page_and_head_shard():
    """Table entries outside the cache are zeros, not reads; a shard's heads match the whole cache's."""
    lens, counts = [200, 64, 33], [5, 6, 2]
    s = Setup(lens, seed=9, page_len=16, code="e4m3", heads=3)
    first = np.concatenate([[0], np.cumsum(counts)]).tolist()
    owner = [b for b, n in enumerate(counts) for _ in range(n)]
    pos = [lens[b] - n + i for b, n in enumerate(counts) for i in range(n)]
    q = s.queries(first[-1])
    s.poison(lambda b, p: False)
    got = gqa.decode_paged_chunked(q, s.cache, ints(s.table), ints(lens), ints(first))
    check(got, q, s, owner, pos, unit=CHUNK_UNIT)
    table = [[-5 if c % 2 else 1 << 30 for c in range(len(row))] for row in s.table]
    out = gqa.decode_paged_chunked(q, s.cache, ints(table), ints(lens), ints(first))
    assert bool((out == 0).all())  # codes and scales of such pages count as 0
    assert gqa.read_device_status() == 0


def test_a_workspace_for_the_largest_call_holds_every_smaller_one():
    import ctypes

    from attention_accelerator_b200 import _lib
    cache = gqa.paged_cache(2, 16)
    first = ints([0, 1])

    def need(batch, rows):
        p = _lib.GqaPagedParams()
        p.batch, p.rows, p.first_query = batch, rows, first.data_ptr()
        return _lib.load().gqa_paged_workspace_bytes(ctypes.byref(cache.c), ctypes.byref(p))

    sizes = [[need(batch, rows) for rows in (1, 6, 12, 13, 64, 384, 385, 8192, 100000)] for batch in (1, 2, 63, 64, 1000, 8192)]
    assert all(x > 0 for row in sizes for x in row)
    assert all(row == sorted(row) for row in sizes)
    assert all(list(col) == sorted(col) for col in zip(*sizes))
