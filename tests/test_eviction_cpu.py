"""Differential attention and eviction over the paged cache: refusals and their oracle, without a GPU."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import attention_accelerator_b200 as gqa
from attention_accelerator_b200 import _lib
from oracle import paged as ref
from test_paged_cpu import CPU, c_cache, c_params, host_cache


def host_weights(requests=2, capacity=48, heads=8):
    return gqa.key_weights(requests, capacity, kv_heads=heads, device=CPU)


def test_calls_refuse_host_tensors():
    c, w = host_cache(), host_weights()
    i32, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    q, first = torch.zeros(2, 32, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    lam = torch.zeros(16)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.decode_paged_diff(q, c, table, i32, lam)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.decode_paged_diff_chunked(q, c, table, i32, first, lam)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.decode_paged_weights(q, c, table, i32, w)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.add_key_weights(q, c, table, i32, first, w)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.plan_eviction(w, i32, i32, table, i32, i32[:1], page_len=16, max_keep=8)
    plan = gqa.EvictionPlan(torch.zeros(2, 8, 8, dtype=torch.int32), i32, i32, i32[:1], i32)
    with pytest.raises(ValueError, match="CUDA"):
        gqa.evict_paged(c, table, w, plan)


def test_key_weights_refuse_wrong_tensors():
    w = torch.zeros(2, 8, 48)
    p, e = torch.zeros(2, 8, 48, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = gqa.KeyWeights(w, p, e)
    assert (good.requests, good.kv_heads, good.capacity) == (2, 8, 48)
    assert good[1:].requests == 1 and good[1:].c.weight == w[1:].data_ptr()
    for args, match in [((w.double(), p, e), "weight"), ((w[..., :40], p, e), "weight"), ((torch.zeros(2, 9, 48), p, e), "weight"),
                        ((w[0], p, e), "weight"), ((w, p.long(), e), "position"), ((w, p[:, :4], e), "position"),
                        ((w, p, e[:1]), "evicted"), ((w, p, e.float()), "evicted")]:
        with pytest.raises(ValueError, match=match):
            gqa.KeyWeights(*args)


def diff(**change):
    base = dict(lambdas=4096, lambda_row_stride=16, norm_weight=4096, norm_eps=1e-5, out_scale=1.0)
    return _lib.GqaPagedDiff(**{**base, **change})


@pytest.mark.parametrize("name", ["gqa_decode_paged_diff", "gqa_decode_paged_chunked_diff"])
def test_c_refuses_bad_differences(name):
    """Refused before any pointer is looked at but by the memory check, which made-up addresses do not pass."""
    fn = getattr(_lib.load(), name)

    def status(d, params=None):
        return fn(4096, 4096, ctypes.byref(c_cache()), ctypes.byref(params or c_params()), d, None, 0, None)

    # The call's own checks come first.
    assert status(ctypes.byref(diff()), c_params(scale=0.0)) == _lib.GQA_ERR_SCALE
    assert status(None, c_params(seq_lens=None)) == _lib.GQA_ERR_NULL_POINTER
    assert status(ctypes.byref(diff()), c_params(flags=1)) == _lib.GQA_ERR_FLAGS


def weights(**change):
    return _lib.GqaKeyWeights(**{**dict(weight=4096, position=4096, evicted=4096, capacity=48), **change})


def test_c_refuses_bad_planning_with_weights():
    lib = _lib.load()
    ok = [4096, 4096, 2, 4096, 3, 3, 4096, 10, 4096, 16, 4, 4096, 4096, 4096, 4096, 4096, 4096, 4096, None, 0, None]
    for at, value, want in [(0, None, "NULL_POINTER"), (16, None, "NULL_POINTER"), (16, 4098, "ALIGNMENT"),
                            (17, None, "NULL_POINTER"), (2, 0, "BATCH"), (9, 24, "KV_BLOCK_LEN"), (18, None, "WORKSPACE")]:
        args = list(ok)
        args[at] = value
        assert lib.gqa_plan_pages_evicted(*args) == getattr(_lib, "GQA_ERR_" + want), (at, value)


def test_c_refuses_bad_evictions():
    lib = _lib.load()
    w = weights()
    ok = [ctypes.byref(w), 8, 4096, 4096, 2, 4096, 3, 3, 4096, 10, 4096, 16, 8, 4, 32, 4096, 4096, 4096, 4096, 4096, None, 0, None]
    for at, value, want in [(0, None, "NULL_POINTER"), (0, weights(weight=None), "NULL_POINTER"),
                            (0, weights(evicted=None), "NULL_POINTER"), (0, weights(position=4098), "ALIGNMENT"),
                            (0, weights(capacity=0), "KV_RANGE"), (0, weights(capacity=(1 << 30) + 1), "KV_RANGE"),
                            (2, None, "NULL_POINTER"), (3, None, "NULL_POINTER"), (15, None, "NULL_POINTER"),
                            (17, None, "NULL_POINTER"), (19, None, "NULL_POINTER")]:
        args = list(ok)
        args[at] = ctypes.byref(value) if isinstance(value, ctypes.Structure) else value
        assert lib.gqa_plan_eviction(*args) == getattr(_lib, "GQA_ERR_" + want), (at, want)
    for requests, heads, keep in ((0, 8, 8), (8193, 8, 8), (2, 0, 8), (2, 9, 8), (2, 8, 0), (2, 8, (1 << 30) + 1)):
        assert lib.gqa_plan_eviction_workspace_bytes(requests, heads, keep) == 0
    assert lib.gqa_plan_eviction_workspace_bytes(2, 8, 100) == 256 + 2 * 8 * 2 * 100 * 4
    c = c_cache()
    ok = [ctypes.byref(c), 4096, 3, 3, ctypes.byref(w), 4096, 4096, 2, 8, None]
    for at, value, want in [(0, None, "NULL_POINTER"), (1, None, "NULL_POINTER"), (5, None, "NULL_POINTER"),
                            (6, None, "NULL_POINTER"), (0, c_cache(page_len=8), "KV_BLOCK_LEN"),
                            (0, c_cache(kv_heads=9), "KV_HEADS"), (4, None, "NULL_POINTER"),
                            (4, weights(capacity=-1), "KV_RANGE")]:
        args = list(ok)
        args[at] = ctypes.byref(value) if isinstance(value, ctypes.Structure) else value
        assert lib.gqa_evict_paged(*args) == getattr(_lib, "GQA_ERR_" + want), (at, want)


@pytest.mark.parametrize("change,want", [
    (dict(seq_lens=None), "NULL_POINTER"), (dict(batch=0), "BATCH"), (dict(scale=math.nan), "SCALE"), (dict(flags=1), "FLAGS"),
    (dict(rope_theta=0.0), "ROPE_THETA"), (dict(q_row_stride=4), "ALIGNMENT"), (dict(table_stride=2), "BATCH")])
def test_c_refuses_bad_weight_calls(change, want):
    lib, w = _lib.load(), weights()
    c, p = c_cache(), c_params(**change)
    assert lib.gqa_decode_paged_weights(4096, 4096, ctypes.byref(c), ctypes.byref(p), ctypes.byref(w), None, 0, None) == \
        getattr(_lib, "GQA_ERR_" + want)
    assert lib.gqa_add_key_weights(4096, ctypes.byref(c), ctypes.byref(p), ctypes.byref(w), None, None, 0, None) == \
        getattr(_lib, "GQA_ERR_" + want)


def test_weights_workspace_is_0_for_what_is_no_call():
    lib, c = _lib.load(), c_cache()
    for change in (dict(batch=0), dict(rows=-1), dict(table_width=0), dict(batch=8193), dict(table_width=1 << 27)):
        assert lib.gqa_key_weights_workspace_bytes(ctypes.byref(c), ctypes.byref(c_params(**change))) == 0
    assert lib.gqa_key_weights_workspace_bytes(None, ctypes.byref(c_params())) == 0


def test_oracle_rounds_to_the_nearest_code():
    rng = np.random.RandomState(0)
    x = np.concatenate([rng.randn(5000) * np.exp(3 * rng.randn(5000)), np.linspace(-460, 460, 4001)])
    want = torch.from_numpy(x).float().clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.round_code(torch.from_numpy(x).float().double().numpy(), "e4m3"), want)
    assert np.array_equal(ref.round_code(np.array([0.5, 1.5, -2.5, 200.0]), "int8"), [0, 2, -2, 127])


def test_oracle_difference_and_norm():
    rng = np.random.RandomState(1)
    q, k, v = rng.randn(4, 128), rng.randn(9, 1, 128), rng.randn(9, 1, 128)
    seen = np.ones(9, bool)
    maps = ref.attend(q, k, v, 8, seen, scale=0.1)[0]
    out = ref.attend_diff(q, k, v, 8, seen, [0.5, 2.0], scale=0.1, out_scale=0.3)[0]
    assert np.allclose(out, 0.3 * np.stack([maps[0] - 0.5 * maps[1], maps[2] - 2 * maps[3]]))
    out, size, _ = ref.attend_diff(q, k, v, 8, seen, [0.5, 2.0], scale=0.1, norm_weight=np.ones(128), eps=1e-12)
    assert np.allclose((out ** 2).mean(-1), 1)
    # The bound of what an error of the maps becomes, against differences.
    for _ in range(20):
        d = 1e-6 * rng.randn(*v.shape) * np.abs(v)
        moved = ref.attend_diff(q, k, v + d, 8, seen, [0.5, 2.0], scale=0.1, norm_weight=np.ones(128), eps=1e-12)[0]
        assert np.all(np.abs(moved - out) <= 1e-6 * 5 * size)


def test_oracle_plan_keeps_the_heaviest():
    weight = np.zeros((1, 1, 16))
    weight[0, 0, :10] = [5, 1, 9, 1, 7, 1, 8, 2, 6, 0]
    position = np.arange(16).reshape(1, 1, 16)
    free = [40]
    ok, take, lens, evicted, cuts, rows, given = ref.plan_eviction(weight, position, [10], [0], [4], [[3]], free, 16, 8,
                                                                  max_keep=8, sinks=1, recent=1)
    assert ok and lens == [4] and evicted == [6] and (cuts, rows, given) == (1, 6, 0) and free == [40]
    assert take[0, 0].tolist() == [-1, 6, -1, 9, -1, -1, -1, -1]  # rows 0 (a sink), 2, 6 and 9 (the last) stay
