"""The paged 8-bit cache's refusals and its oracle, without a GPU."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import _lib
from oracle import paged as ref

CPU = torch.device("cpu")


def host_cache(pages=4, page_len=16, heads=8, layout="head_major", dtype=torch.int8):
    return gqa.paged_cache(pages, page_len, kv_heads=heads, layout=layout, dtype=dtype, device=CPU)


def test_e4m3_values_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.E4M3, want, equal_nan=True)


def test_cache_describes_its_tensors():
    for layout, row, head in (("head_major", 128, 16 * 128), ("position_major", 3 * 128, 128)):
        c = host_cache(heads=3, layout=layout)
        assert (c.pages, c.page_len, c.kv_heads) == (4, 16, 3)
        assert (c.c.row_stride, c.c.head_stride, c.c.page_stride) == (row, head, 3 * 16 * 128)
    one = host_cache(pages=1, heads=1)
    assert one.c.page_stride % 16 == 0 and one.c.head_stride >= 128


def test_cache_refuses_wrong_tensors():
    k = torch.zeros(4, 8, 16, 128, dtype=torch.int8)
    s = torch.zeros(4, 8)
    good = dict(k=k, v=k.clone(), k_scale=s, v_scale=s.clone())
    gqa.PagedCache(**good)
    for change, match in [
            (dict(v=k.view(torch.uint8).view(torch.float8_e4m3fn)), "both be int8"),
            (dict(k=k.float(), v=k.float()), "both be int8"), (dict(v=k[:3]), "k and v must be"),
            (dict(k=k[..., :64], v=k[..., :64]), "k and v must be"),
            (dict(v=torch.zeros(4, 8, 32, 128, dtype=torch.int8)[:, :, :16]), "same strides"),
            (dict(k=k[:, :, :12], v=k[:, :, :12]), "page_len"), (dict(layout="position_major"), "page_len"),
            (dict(layout="rows"), "layout"), (dict(k_scale=s[:3]), "k_scale"), (dict(v_scale=s.double()), "v_scale"),
            (dict(v_scale=torch.zeros(4, 16)[:, :8]), "same strides")]:
        with pytest.raises(ValueError, match=match):
            gqa.PagedCache(**{**good, **change})
    wide = torch.zeros(4, 9, 16, 128, dtype=torch.int8)
    with pytest.raises(ValueError, match="1 to 8"):
        gqa.PagedCache(wide, wide, torch.zeros(4, 9), torch.zeros(4, 9))


def test_cache_refuses_scales_whose_pages_overlap():
    """An expanded scale tensor has fewer floats than pages times heads."""
    for heads in (1, 8):
        k = torch.zeros(4, heads, 16, 128, dtype=torch.int8)
        whole, one = torch.zeros(4, heads), torch.zeros(1, heads).expand(4, heads)
        for scales in (dict(k_scale=one, v_scale=one), dict(k_scale=one, v_scale=whole), dict(k_scale=whole, v_scale=one)):
            with pytest.raises(ValueError, match="overlap|same strides"):
                gqa.PagedCache(k, k.clone(), **scales)
        skewed = torch.zeros(64).as_strided((4, heads), (max(1, heads - 1), 1))
        if heads > 1:
            with pytest.raises(ValueError, match="overlap"):
                gqa.PagedCache(k, k.clone(), skewed, skewed)
        one_page = torch.zeros(1, heads).expand(1, heads)
        gqa.PagedCache(k[:1], k[:1].clone(), one_page, one_page.clone())


def test_calls_refuse_host_tensors():
    c = host_cache()
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    rows = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    q = torch.zeros(2, 32, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.plan_pages(i32, i32, table, i32, i32[:1], page_len=16, max_tokens=4)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.append_paged(c, rows, rows, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        gqa.read_paged(c, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        gqa.decode_paged(q, c, table, i32)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.decode_paged_chunked(q, c, table, i32, torch.zeros(3, dtype=torch.int32))


def c_cache(**change):
    base = dict(k=4096, v=8192, k_scale=4096, v_scale=4096, code=0, kv_heads=8, page_len=16, pages=4,
                page_stride=16384, row_stride=128, head_stride=2048, scale_page_stride=8)
    return _lib.GqaPagedCache(**{**base, **change})


def c_params(**change):
    base = dict(batch=2, rows=2, block_table=4096, table_stride=3, table_width=3, flags=0, seq_lens=4096,
                first_query=4096, scale=0.1, score_cap=0.0, rope_theta=5e5, q_row_stride=4096, q_head_stride=128,
                out_row_stride=4096, out_head_stride=128)
    return _lib.GqaPagedParams(**{**base, **change})


def status(name, cache, params=None):
    """Status of a call with made-up addresses: everything here is refused before a pointer is looked at."""
    lib = _lib.load()
    c = ctypes.byref(cache)
    if name == "append":
        return lib.gqa_append_paged(4096, 4096, 2, 1024, 128, 1024, 128, 4096, None, 5e5, c, None)
    if name == "read":
        return lib.gqa_read_paged(c, 4096, 2, 4096, 4096, None)
    fn = lib.gqa_decode_paged if name == "decode" else lib.gqa_decode_paged_chunked
    return fn(4096, 4096, c, ctypes.byref(params or c_params()), None, 0, None)


@pytest.mark.parametrize("change,want", [
    (dict(k=None), "NULL_POINTER"), (dict(v_scale=None), "NULL_POINTER"), (dict(kv_heads=0), "KV_HEADS"),
    (dict(kv_heads=9), "KV_HEADS"), (dict(code=2), "FLAGS"), (dict(page_len=8), "KV_BLOCK_LEN"),
    (dict(page_len=48), "KV_BLOCK_LEN"), (dict(page_len=256), "KV_BLOCK_LEN"), (dict(pages=0), "KV_RANGE"),
    (dict(k=4104), "ALIGNMENT"), (dict(v_scale=4098), "ALIGNMENT"), (dict(row_stride=120), "ALIGNMENT"),
    (dict(page_stride=16392), "ALIGNMENT"), (dict(head_stride=-2048), "ALIGNMENT"),
    (dict(page_stride=1 << 40), "ALIGNMENT"), (dict(scale_page_stride=7), "ALIGNMENT")])
@pytest.mark.parametrize("name", ["append", "read", "decode", "chunked"])
def test_c_refuses_bad_caches(name, change, want):
    assert status(name, c_cache(**change)) == getattr(_lib, "GQA_ERR_" + want)


@pytest.mark.parametrize("change,want", [
    (dict(block_table=None), "NULL_POINTER"), (dict(seq_lens=None), "NULL_POINTER"), (dict(batch=0), "BATCH"),
    (dict(batch=8193, rows=8193), "BATCH"), (dict(rows=-1), "BATCH"), (dict(table_width=0), "BATCH"),
    (dict(table_stride=2), "BATCH"), (dict(table_width=(1 << 26) + 1, table_stride=1 << 27), "BATCH"), (dict(reserved=1), "BATCH"), (dict(flags=1), "FLAGS"), (dict(flags=2), "FLAGS"),
    (dict(scale=0.0), "SCALE"), (dict(scale=math.nan), "SCALE"), (dict(score_cap=-1.0), "SCALE"),
    (dict(score_cap=math.inf), "SCALE"), (dict(rope_theta=0.0), "ROPE_THETA"), (dict(q_row_stride=4), "ALIGNMENT"),
    (dict(out_head_stride=-128), "ALIGNMENT")])
@pytest.mark.parametrize("name", ["decode", "chunked"])
def test_c_refuses_bad_calls(name, change, want):
    assert status(name, c_cache(), c_params(**change)) == getattr(_lib, "GQA_ERR_" + want)


def test_c_refuses_what_only_one_call_takes():
    assert status("decode", c_cache(), c_params(rows=3)) == _lib.GQA_ERR_BATCH
    assert status("chunked", c_cache(), c_params(first_query=None)) == _lib.GQA_ERR_NULL_POINTER
    lib = _lib.load()
    ok = [4096, 4096, 2, 4096, 3, 3, 4096, 10, 4096, 16, 4, 4096, 4096, 4096, 4096, 4096, 4096, None, 0, None]
    for at, value, want in [(0, None, "NULL_POINTER"), (2, 0, "BATCH"), (2, 8193, "BATCH"), (4, 2, "BATCH"),
                            (5, 0, "BATCH"), (7, -1, "BATCH"), (9, 24, "KV_BLOCK_LEN"), (10, -1, "BATCH"),
                            (16, None, "NULL_POINTER"), (17, None, "WORKSPACE")]:
        args = list(ok)
        args[at] = value
        assert lib.gqa_plan_pages(*args) == getattr(_lib, "GQA_ERR_" + want), (at, value)


def test_capture_mode_refuses_what_is_no_mode():
    lib, before = _lib.load(), ctypes.c_int(-1)
    for mode in (-1, 3):
        assert lib.gqa_capture_mode(mode, ctypes.byref(before)) == _lib.GQA_ERR_FLAGS and before.value == -1
    assert lib.gqa_capture_mode(_lib.GQA_CAPTURE_RELAXED, None) == _lib.GQA_ERR_NULL_POINTER


def test_oracle_plan_allocates_every_page_once():
    table, free = [[-1] * 4 for _ in range(3)], list(range(8))
    ok, lens, first, slots, positions, taken, given = ref.plan_step([0, 0, 0], [17, 0, 16], table, free, 16, 40, 8)
    assert ok and lens == [17, 0, 16] and first == [0, 17, 17, 33] and (taken, given) == (3, 0)
    assert table[0][:2] == [7, 6] and table[2][0] == 5 and free == [0, 1, 2, 3, 4]
    assert slots[:17] == [7 * 16 + i for i in range(16)] + [96] and positions[17:33] == list(range(16))
    ok, lens, first, slots, positions, taken, given = ref.plan_step(lens, [-1, 2, 1], table, free, 16, 3, 8)
    assert ok and lens == [0, 2, 17] and (taken, given) == (2, 2) and free == [0, 1, 2, 3, 4]
    assert table[1][0] == 6 and table[2][1] == 7 and slots == [96, 97, 112]


def test_oracle_attention_by_differences():
    """The 64-bit attention against itself: the output is a weighted mean, an empty row is 0, the cap and the bias
    act as their formulas say."""
    rng = np.random.RandomState(0)
    q, k, v = rng.randn(4, 128), rng.randn(9, 1, 128), rng.randn(9, 1, 128)
    seen = np.ones(9, bool)
    out, size, most = ref.attend(q, k, v, 8, seen, scale=0.1)
    assert (np.abs(out) <= size + 1e-12).all() and most > 0
    assert not ref.attend(q, k, v, 8, ~seen, scale=0.1)[0].any()
    flat = ref.attend(q, k, v, 8, seen, scale=0.1, cap=1e-9)[0]
    assert np.allclose(flat, v[:, 0].mean(0), atol=1e-8)
    near = ref.attend(q, k, v, 8, seen, scale=0.1, slopes=np.full(4, 1e3))[0]
    assert np.allclose(near, v[8, 0])
