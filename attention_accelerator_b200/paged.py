"""Paged 8-bit KV cache: page planning, append, read-back and attention.

The cache is a pool of pages of ``page_len`` tokens; every (page, KV head) block of K and of V holds int8 or FP8
(e4m3) codes and one FP32 scale.  A serving step is

    plan = plan_pages(lens, new_lens, block_table, free_pages, n_free, page_len=P, max_tokens=T)
    append_paged(cache, k, v, plan.slots, positions=plan.positions)
    out = decode_paged(q, cache, block_table, plan.lens)                              # one token a sequence, or
    out = decode_paged_chunked(q, cache, block_table, plan.lens, plan.first_token)    # any number

with every length in device memory: no call waits for the GPU, and a captured CUDA graph of the step follows the
lengths.  A graph keeps the workspace of the stream that it was captured on: graphs captured on one stream, and that
stream's own calls, are not to run at the same time.  K is rotated when it is appended (as :func:`rope_k_cache` does for a BF16 cache), Q when it is used.

The geometry is the library's: 4 Q heads to each KV head and 128 dims; 1 to 8 KV heads (a head shard's cache holds
only its own).  Everything runs in ``lib/libgqa_b200.so``; the C side is ``include/gqa_b200.h``.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field

import torch

from . import _lib, api
from ._lib import GqaPagedCache, GqaPagedParams
from .api import GROUP_SIZE, HEAD_DIM, N_KV_HEADS, ROPE_THETA, GqaError, _check, _check_cuda, _check_out, _stream_ptr

PAGE_LENS = (16, 32, 64, 128)
_CODES = {torch.int8: _lib.GQA_CODE_INT8, torch.float8_e4m3fn: _lib.GQA_CODE_E4M3}


@dataclass(frozen=True)
class PagedCache:
    """The pages of a cache and their scales.

    ``k``/``v``: int8 or float8_e4m3fn, ``[pages, page_len, heads, 128]`` (``layout="position_major"``) or
    ``[pages, heads, page_len, 128]`` (``"head_major"``), with the same strides (views of one buffer may be given).
    ``k_scale``/``v_scale``: float32 ``[pages, heads]``.  :func:`paged_cache` allocates one.
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    layout: str = "head_major"
    c: GqaPagedCache = field(init=False, repr=False, compare=False)

    def __post_init__(self):
        k, v = self.k, self.v
        if self.layout not in api.LAYOUTS:
            raise ValueError(f"layout must be one of {api.LAYOUTS}")
        if k.dtype not in _CODES or v.dtype != k.dtype:
            raise ValueError("k and v must both be int8 or both float8_e4m3fn")
        if k.dim() != 4 or k.shape[-1] != HEAD_DIM or v.shape != k.shape or k.stride(-1) != 1:
            raise ValueError(f"k and v must be [pages, page_len, heads, {HEAD_DIM}] or [pages, heads, page_len, "
                             f"{HEAD_DIM}] with a contiguous last dim")
        if v.stride() != k.stride():
            raise ValueError("k and v must have the same strides")
        row, head = (1, 2) if self.layout == "position_major" else (2, 1)
        pages, page_len, heads = k.shape[0], k.shape[row], k.shape[head]
        if page_len not in PAGE_LENS:
            raise ValueError(f"page_len must be one of {PAGE_LENS}, got {page_len}")
        if not 1 <= heads <= N_KV_HEADS:
            raise ValueError(f"a cache holds 1 to {N_KV_HEADS} KV heads, got {heads}")
        if pages < 1:
            raise ValueError("a cache holds at least one page")
        for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale)):
            if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) or t.stride(-1) != 1 and heads > 1:
                raise ValueError(f"{name} must be float32 [{pages}, {heads}] with a contiguous last dim")
            if pages > 1 and t.stride(0) < heads:  # (an expanded tensor: an append writes each page's own scale)
                raise ValueError(f"{name}'s pages must not overlap (row stride {t.stride(0)} for {heads} heads)")
        if self.v_scale.stride(0) != self.k_scale.stride(0) and pages > 1:
            raise ValueError("k_scale and v_scale must have the same strides")
        for name, t in (("v", v), ("k_scale", self.k_scale), ("v_scale", self.v_scale)):
            if t.device != k.device:
                raise ValueError(f"{name} is on {t.device}, k on {k.device}")
        # The stride of a dimension of one element says nothing: the smallest valid one stands for it.
        stride = [s if n > 1 else max(HEAD_DIM, -(-s // 16) * 16) for s, n in zip(k.stride(), k.shape)]
        object.__setattr__(self, "c", GqaPagedCache(
            k=k.data_ptr(), v=v.data_ptr(), k_scale=self.k_scale.data_ptr(), v_scale=self.v_scale.data_ptr(),
            code=_CODES[k.dtype], kv_heads=heads, page_len=page_len, pages=pages, page_stride=stride[0],
            row_stride=stride[row], head_stride=stride[head],
            scale_page_stride=max(heads, self.k_scale.stride(0))))

    @property
    def pages(self) -> int:
        return self.c.pages

    @property
    def page_len(self) -> int:
        return self.c.page_len

    @property
    def kv_heads(self) -> int:
        return self.c.kv_heads

    @property
    def device(self) -> torch.device:
        return self.k.device


def paged_cache(pages: int, page_len: int, *, dtype: torch.dtype = torch.float8_e4m3fn, kv_heads: int = N_KV_HEADS,
                layout: str = "head_major", device: torch.device | None = None) -> PagedCache:
    """Allocate an empty cache.  ``head_major`` keeps a (page, head) block in one piece."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    shape = (pages, page_len, kv_heads, HEAD_DIM) if layout == "position_major" else (pages, kv_heads, page_len, HEAD_DIM)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2))
    return PagedCache(k, v, ks, vs, layout=layout)


def _paged_workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """Zeroed once and kept for the paged calls of a stream: they leave counters past the header at zero, where the
    other calls' workspace holds partial rows."""
    return api._workspace(device, ("paged", stream), nbytes)


def _need(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> int:
    """Pointer of a contiguous tensor of a call, or of None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on {device}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")
    return t.data_ptr()


def _table(block_table: torch.Tensor, rows: int, device: torch.device) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != rows \
            or block_table.shape[1] < 1 or block_table.stride(1) != 1 or block_table.device != device:
        raise ValueError(f"block_table must be int32 [{rows}, width] on {device} with a contiguous last dim")


@dataclass(frozen=True)
class PagePlan:
    """What :func:`plan_pages` laid out, all in device memory."""
    lens: torch.Tensor         # int32 [requests]: tokens held after the step
    n_free: torch.Tensor       # int32 [1]: height of the free stack after the step
    first_token: torch.Tensor  # int32 [requests + 1]: running sum of the new tokens
    slots: torch.Tensor        # int64 [max_tokens]: page * page_len + row, -1 past the last new token
    positions: torch.Tensor    # int32 [max_tokens]
    counts: torch.Tensor       # int32 [4]: new tokens, pages taken, pages given back, status

    def check(self) -> None:
        """Wait for the plan; raise :class:`GqaError` if it was refused (nothing was changed then)."""
        _check(int(self.counts[3]), "plan_pages")


def plan_pages(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               n_free: torch.Tensor, *, page_len: int, max_tokens: int, lens_out: torch.Tensor | None = None,
               n_free_out: torch.Tensor | None = None) -> PagePlan:
    """Pages, slots and positions of a step's new tokens, from lengths in device memory.

    ``lens``/``new_lens``: int32 ``[requests]``; ``new_lens[r] < 0`` ends request r: its pages go back to the free
    stack and its length becomes 0.  ``block_table``: int32 ``[requests, width]`` and ``free_pages``: int32
    ``[capacity]``, entries below ``n_free`` (int32 ``[1]``) valid, are updated in place.  ``lens_out`` and
    ``n_free_out`` may be ``lens`` and ``n_free``.  A step that cannot be met (too few free pages, a row of the table
    too short, more than ``max_tokens`` new tokens) changes nothing and says so in ``counts[3]``
    (:meth:`PagePlan.check`).
    """
    lib = _lib.load()
    device = lens.device
    if device.type != "cuda":
        raise ValueError("plan_pages takes CUDA tensors")
    if page_len not in PAGE_LENS:
        raise ValueError(f"page_len must be one of {PAGE_LENS}, got {page_len}")
    n = lens.shape[0] if lens.dim() == 1 else 0
    if not 1 <= n <= _lib.PAGED_MAX_BATCH:
        raise ValueError(f"lens must be [requests] with 1 to {_lib.PAGED_MAX_BATCH} requests")
    _table(block_table, n, device)
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be one-dimensional")
    if not 0 <= max_tokens <= 0x7FFFFFFF:
        raise ValueError(f"max_tokens must be in [0, 2^31), got {max_tokens}")
    i32 = torch.int32
    slots = lens.new_empty(max_tokens, dtype=torch.int64)
    room = [n if lens_out is None else 0, 1 if n_free_out is None else 0, n + 1, max_tokens, 4]  # in one allocation
    new_lens_out, new_n_free, first, positions, counts = lens.new_empty(sum(room), dtype=i32).split(room)
    lens_out = new_lens_out if lens_out is None else lens_out
    n_free_out = new_n_free if n_free_out is None else n_free_out
    stream = _stream_ptr(device)
    ws = _paged_workspace(device, stream, _lib.CHUNKED_WORKSPACE_BYTES)
    _check(lib.gqa_plan_pages(
        _need("lens", lens, i32, (n,), device), _need("new_lens", new_lens, i32, (n,), device), n,
        block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        _need("free_pages", free_pages, i32, tuple(free_pages.shape), device), free_pages.shape[0],
        _need("n_free", n_free, i32, (1,), device), page_len, max_tokens,
        _need("lens_out", lens_out, i32, (n,), device), _need("n_free_out", n_free_out, i32, (1,), device),
        first.data_ptr(), slots.data_ptr(), positions.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.numel(),
        stream), "plan_pages")
    return PagePlan(lens_out, n_free_out, first, slots, positions, counts)


def _rows(name: str, t: torch.Tensor, heads: int, device: torch.device) -> None:
    if t.dtype is not torch.bfloat16 or t.dim() != 3 or t.shape[1:] != (heads, HEAD_DIM) or t.stride(2) != 1 \
            or t.device != device:
        raise ValueError(f"{name} must be bfloat16 [rows, {heads}, {HEAD_DIM}] on {device} with a contiguous last dim")


def append_paged(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
                 positions: torch.Tensor | None = None, rope_theta: float = ROPE_THETA) -> None:
    """Store new K and V rows (BF16 ``[tokens, heads, 128]``, any token and head strides) at ``slots`` (int64).

    With ``positions`` (int32) K is rotated first; without, it is stored as it is.  The rows of one page must be
    consecutive with consecutive slots, as :func:`plan_pages` lays them out; slot -1 is skipped.  A block's scale is
    the largest magnitude it holds over 127 (int8) or 448 (e4m3): where new rows raise it, the block's earlier codes
    are rounded again.  A NaN or infinity makes its block's scale NaN.
    """
    lib = _lib.load()
    device = cache.device
    if device.type != "cuda":
        raise ValueError("append_paged takes CUDA tensors")
    _rows("k", k, cache.kv_heads, device)
    _rows("v", v, cache.kv_heads, device)
    n = k.shape[0]
    if v.shape[0] != n:
        raise ValueError(f"{n} rows of K, {v.shape[0]} of V")
    _check(lib.gqa_append_paged(
        k.data_ptr(), v.data_ptr(), n, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        _need("slots", slots, torch.int64, (n,), device), _need("positions", positions, torch.int32, (n,), device),
        rope_theta, ctypes.byref(cache.c), _stream_ptr(device)), "append_paged") if n else None


def read_paged(cache: PagedCache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows of ``slots`` (int64 ``[n]``) as BF16 ``[n, heads, 128]``: code * scale; zeros for slot -1.
    (K as it was stored: rotated if it was appended with positions.)"""
    lib = _lib.load()
    device = cache.device
    if device.type != "cuda":
        raise ValueError("read_paged takes CUDA tensors")
    n = slots.shape[0] if slots.dim() == 1 else -1
    ptr = _need("slots", slots, torch.int64, (n,), device)
    shape = (n, cache.kv_heads, HEAD_DIM)
    k, v = slots.new_empty(shape, dtype=torch.bfloat16), slots.new_empty(shape, dtype=torch.bfloat16)
    if n:
        _check(lib.gqa_read_paged(ctypes.byref(cache.c), ptr, n, k.data_ptr(), v.data_ptr(), _stream_ptr(device)),
               "read_paged")
    return k, v


def _attend(name: str, q, cache, block_table, seq_lens, first_query, query_positions, scale, rope_theta, q_rotated,
            score_cap, distance_slopes, doc_starts, prefix_ends, out):
    lib = _lib.load()
    device = q.device
    if device.type != "cuda":
        raise ValueError(f"{name} takes CUDA tensors")
    heads = cache.kv_heads * GROUP_SIZE
    _rows("q", q, heads, device)
    rows = q.shape[0]
    batch = seq_lens.shape[0] if seq_lens.dim() == 1 else 0
    if not 1 <= batch <= _lib.PAGED_MAX_BATCH:
        raise ValueError(f"seq_lens must be [batch] with 1 to {_lib.PAGED_MAX_BATCH} sequences")
    if first_query is None and rows != batch:
        raise ValueError(f"{rows} query rows for {batch} sequences")
    _check_cuda(device, cache=cache.k)
    _table(block_table, batch, device)
    if score_cap is not None and not (score_cap > 0.0 and math.isfinite(score_cap)):
        raise ValueError("score_cap must be positive and finite, or None")
    if out is None:
        out = q.new_empty((rows, heads, HEAD_DIM))
    else:
        _check_out(out, (rows, heads, HEAD_DIM), torch.bfloat16, device)
    i32 = torch.int32
    p = GqaPagedParams(
        batch=batch, rows=rows, block_table=block_table.data_ptr(), table_stride=block_table.stride(0),
        table_width=block_table.shape[1], flags=_lib.GQA_FLAG_Q_ROTATED if q_rotated else 0,
        seq_lens=_need("seq_lens", seq_lens, i32, (batch,), device),
        query_positions=_need("query_positions", query_positions, i32, (batch,), device),
        first_query=_need("first_query", first_query, i32, (batch + 1,), device),
        doc_starts=_need("doc_starts", doc_starts, i32, (rows,), device),
        prefix_ends=_need("prefix_ends", prefix_ends, i32, (rows,), device),
        slopes=_need("distance_slopes", distance_slopes, torch.float32, (heads,), device),
        scale=1.0 / math.sqrt(HEAD_DIM) if scale is None else scale, score_cap=score_cap or 0.0,
        rope_theta=rope_theta, reserved=0, q_row_stride=q.stride(0), q_head_stride=q.stride(1),
        out_row_stride=out.stride(0), out_head_stride=out.stride(1))
    if rows == 0:
        return out
    stream = _stream_ptr(device)
    fn = lib.gqa_decode_paged if first_query is None else lib.gqa_decode_paged_chunked
    c = ctypes.byref(cache.c)
    ws = _paged_workspace(device, stream, _lib.CHUNKED_WORKSPACE_BYTES)
    status = fn(q.data_ptr(), out.data_ptr(), c, ctypes.byref(p), ws.data_ptr(), ws.numel(), stream)
    if status == _lib.GQA_ERR_WORKSPACE:  # nothing was launched: the stream's first call, or a larger one
        nbytes = lib.gqa_paged_workspace_bytes(c, ctypes.byref(p))
        if nbytes == 0:
            raise GqaError(_lib.GQA_ERR_CUDA, f"{name}: workspace sizing failed (no supported GPU?)")
        ws = _paged_workspace(device, stream, nbytes)
        status = fn(q.data_ptr(), out.data_ptr(), c, ctypes.byref(p), ws.data_ptr(), ws.numel(), stream)
    _check(status, name)
    return out


def decode_paged(q: torch.Tensor, cache: PagedCache, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                 query_positions: torch.Tensor | None = None, scale: float | None = None,
                 rope_theta: float = ROPE_THETA, q_rotated: bool = False, score_cap: float | None = None,
                 distance_slopes: torch.Tensor | None = None, doc_starts: torch.Tensor | None = None,
                 prefix_ends: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token a sequence over the paged cache; returns BF16 ``[batch, 4 * heads, 128]``.

    ``q``: BF16 ``[batch, 4 * heads, 128]``; ``block_table``: int32 ``[batch, width]``; ``seq_lens``: int32
    ``[batch]`` (0: nothing visible).  ``query_positions`` (int32, default ``seq_lens - 1``) are where the queries
    stand and, unless ``q_rotated``, the angle they are turned by.

    Scores are ``z = scale * q.k``, then ``score_cap * tanh(z / score_cap)``, then minus ``distance_slopes[head] *
    |query position - key position|`` (float32 ``[4 * heads]``).  Query row i sees the keys p with
    ``doc_starts[i] <= p < min(seq_len, max(position + 1, prefix_ends[i]))`` (int32 per row: its document's first
    key, and the end of a prefix that is visible from everywhere).  A row that sees no key is 0.
    """
    return _attend("decode_paged", q, cache, block_table, seq_lens, None, query_positions, scale, rope_theta,
                   q_rotated, score_cap, distance_slopes, doc_starts, prefix_ends, out)


def decode_paged_chunked(q: torch.Tensor, cache: PagedCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         first_query: torch.Tensor, *, scale: float | None = None, rope_theta: float = ROPE_THETA,
                         q_rotated: bool = False, score_cap: float | None = None,
                         distance_slopes: torch.Tensor | None = None, doc_starts: torch.Tensor | None = None,
                         prefix_ends: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Any number of queries a sequence, packed: ``q`` BF16 ``[rows, 4 * heads, 128]``, sequence b's queries in rows
    ``first_query[b]`` to ``first_query[b + 1]`` (int32 ``[batch + 1]``); they are its last tokens, so query i of n
    stands at ``seq_lens[b] - n + i``.  Whole prompts, chunks of one, and drafted tokens to verify; otherwise as
    :func:`decode_paged`.  Rows at or past ``first_query[batch]`` are not written."""
    return _attend("decode_paged_chunked", q, cache, block_table, seq_lens, first_query, None, scale, rope_theta,
                   q_rotated, score_cap, distance_slopes, doc_starts, prefix_ends, out)
