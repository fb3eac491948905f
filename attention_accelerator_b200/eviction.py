"""Eviction from the paged 8-bit KV cache by accumulated attention weight.

Beside the cache a program keeps, for every row (held key) of every request and KV head, the attention weight that its
queries have given it so far (:class:`KeyWeights`).  Requests that hold more rows than their budget lose those of the
least weight:

    out = decode_paged_weights(q, cache, block_table, lens, weights)               # decode_paged, and its weights
    add_key_weights(q, cache, block_table, lens, first_query, weights)             # those of a prompt, or of its end
    plan = plan_eviction(weights, lens, keep, block_table, free_pages, n_free, page_len=P, max_keep=M,
                         lens_out=lens, n_free_out=n_free)
    evict_paged(cache, block_table, weights, plan)

K was rotated at its token's position when it was appended, so that a row may move: the rows that stay but lie past the
new length fill the holes below it, each head its own.  Afterwards a row's number is no longer its position.  A request's
next token has row ``lens[r]`` and position ``lens[r] + weights.evicted[r]``: append it with that position
(``append_paged(..., positions=...)``) behind ``plan_pages(..., weights=weights)``, which sets ``evicted`` of a request that
ends, or holds no rows yet, to 0 (a program that ends requests in another way does so before the first append of the next
one in that row); ``decode_paged_weights`` and ``add_key_weights`` place their queries so by
themselves, ``decode_paged`` takes ``query_positions``, and ``decode_paged_chunked`` queries that were rotated before
(``q_rotated``).  Distance bias, document and prefix masks go by rows and no longer apply.  The pages of a request that is
cut must be its own.  As with the other paged calls every length is in device memory, no call waits for the GPU, and a
captured graph keeps the workspace of the stream that it was captured on.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import NamedTuple

import torch

from . import _lib, api
from ._lib import GqaKeyWeights
from .api import N_KV_HEADS, ROPE_THETA, _check, _stream_ptr
from .paged import PAGE_LENS, PagedCache, _attend, _need, _table


@dataclass(frozen=True)
class KeyWeights:
    """What the rows of ``requests`` requests have been given, ``capacity`` rows each: at least what a row of the block
    table can name.  ``weight``: float32 ``[requests, heads, capacity]``; ``position``: int32, the same shape, of each
    row's token; ``evicted``: int32 ``[requests]``, tokens evicted so far.  :func:`key_weights` allocates one.
    (``weights[a:b]`` of the first dimension may be given for some of the requests.)"""
    weight: torch.Tensor
    position: torch.Tensor
    evicted: torch.Tensor
    c: GqaKeyWeights = field(init=False, repr=False, compare=False)

    def __post_init__(self):
        w = self.weight
        if w.dtype != torch.float32 or w.dim() != 3 or not w.is_contiguous() or w.shape[0] < 1 or w.shape[2] < 1 \
                or not 1 <= w.shape[1] <= N_KV_HEADS:
            raise ValueError(f"weight must be contiguous float32 [requests, 1 to {N_KV_HEADS} heads, capacity]")
        _need("position", self.position, torch.int32, tuple(w.shape), w.device)
        _need("evicted", self.evicted, torch.int32, (w.shape[0],), w.device)
        object.__setattr__(self, "c", GqaKeyWeights(weight=w.data_ptr(), position=self.position.data_ptr(),
                                                    evicted=self.evicted.data_ptr(), capacity=w.shape[2]))

    @property
    def requests(self) -> int:
        return self.weight.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.weight.shape[1]

    @property
    def capacity(self) -> int:
        return self.weight.shape[2]

    @property
    def device(self) -> torch.device:
        return self.weight.device

    def __getitem__(self, rows: slice) -> "KeyWeights":
        return KeyWeights(self.weight[rows], self.position[rows], self.evicted[rows])


def key_weights(requests: int, capacity: int, *, kv_heads: int = N_KV_HEADS,
                device: torch.device | None = None) -> KeyWeights:
    """Allocate the weights of ``requests`` requests of up to ``capacity`` rows."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    shape = (requests, kv_heads, capacity)
    return KeyWeights(torch.zeros(shape, dtype=torch.float32, device=device),
                      torch.zeros(shape, dtype=torch.int32, device=device),
                      torch.zeros(requests, dtype=torch.int32, device=device))


def _check_weights(weights: KeyWeights, cache: PagedCache, block_table: torch.Tensor, requests: int) -> None:
    rows, heads, capacity = weights.weight.shape
    if weights.weight.device != cache.k.device:
        raise ValueError(f"weights are on {weights.device}; every tensor of this call must be on {cache.device}")
    if rows != requests or heads != cache.c.kv_heads:
        raise ValueError(f"weights are of {rows} requests and {heads} heads, the call of {requests} and {cache.kv_heads}")
    if block_table.dim() == 2 and capacity < block_table.shape[1] * cache.c.page_len:
        raise ValueError(f"weights hold {capacity} rows a request, a row of block_table names "
                         f"{block_table.shape[1] * cache.page_len}")


def decode_paged_weights(q: torch.Tensor, cache: PagedCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         weights: KeyWeights, *, scale: float | None = None, rope_theta: float = ROPE_THETA,
                         q_rotated: bool = False, score_cap: float | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`decode_paged`, adding to ``weights`` the softmax weights that the 4 Q heads of a KV head give each of its
    rows.  The last row is the query's own token: its weight starts at 0, its position, and the query's, is
    ``seq_lens - 1 + evicted``.  (A sequence of one row is a new one: its ``evicted`` becomes 0.)"""
    _check_weights(weights, cache, block_table, seq_lens.shape[0] if seq_lens.dim() else 0)
    lib = _lib.load()
    return _attend("decode_paged_weights", q, cache, block_table, seq_lens, None, None, scale, rope_theta, q_rotated,
                   score_cap, None, None, None, out, extra=(ctypes.byref(weights.c),),
                   entry=lib.gqa_decode_paged_weights, sizes=lib.gqa_key_weights_workspace_bytes)


def add_key_weights(q: torch.Tensor, cache: PagedCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    first_query: torch.Tensor, weights: KeyWeights, *, known: torch.Tensor | None = None,
                    scale: float | None = None, rope_theta: float = ROPE_THETA, q_rotated: bool = False,
                    score_cap: float | None = None) -> None:
    """Add the softmax weights of any number of queries a sequence, packed as for :func:`decode_paged_chunked`: of a
    prompt's tokens, or of its last ones.  Query i of n stands at row ``seq_lens - n + i`` and sees the rows up to it.

    Rows from ``known`` on (int32 ``[batch]``; default: from the first query's row on) are new: their weight starts at 0,
    their position is ``row + evicted``.  Where ``known`` is 0 the sequence is a new one, and its ``evicted`` becomes 0:
    give zeros for prompts of which only the last tokens are looked at.  Sequences without queries stay as they are."""
    _check_weights(weights, cache, block_table, seq_lens.shape[0] if seq_lens.dim() else 0)
    lib = _lib.load()
    k = _need("known", known, torch.int32, (weights.requests,), cache.device)
    if first_query is None:
        raise ValueError("first_query must be given")
    _need("first_query", first_query, torch.int32, (weights.requests + 1,), cache.device)
    _attend("add_key_weights", q, cache, block_table, seq_lens, first_query, None, scale, rope_theta, q_rotated, score_cap,
            None, None, None, None, out_heads=0, extra=(ctypes.byref(weights.c), k), entry=lib.gqa_add_key_weights,
            sizes=lib.gqa_key_weights_workspace_bytes)


class EvictionPlan(NamedTuple):
    """What :func:`plan_eviction` chose, all in device memory."""
    take: torch.Tensor     # int32 [requests, heads, max_keep]: the row that moves to row i, -1 where none does
    lens: torch.Tensor     # int32 [requests]: rows held after the step
    evicted: torch.Tensor  # int32 [requests]: tokens evicted after the step
    n_free: torch.Tensor   # int32 [1]: height of the free stack after the step
    counts: torch.Tensor   # int32 [4]: requests cut, rows evicted a head (2^31 - 1 at most), pages given back, status

    def check(self) -> None:
        """Wait for the plan; raise ``GqaError`` if it was refused (nothing was changed then)."""
        _check(int(self.counts[3]), "plan_eviction")


def plan_eviction(weights: KeyWeights, lens: torch.Tensor, keep: torch.Tensor, block_table: torch.Tensor,
                  free_pages: torch.Tensor, n_free: torch.Tensor, *, page_len: int, max_keep: int, sinks: int = 4,
                  recent: int = 32, lens_out: torch.Tensor | None = None, evicted_out: torch.Tensor | None = None,
                  n_free_out: torch.Tensor | None = None) -> EvictionPlan:
    """Choose what stays of the requests that hold more rows than ``keep`` (int32 ``[requests]``; 0 leaves a request as it
    is; at most ``max_keep`` counts): for each head the rows of the highest weight, first of those at a position below
    ``sinks`` or among the ``recent`` last tokens, then of the others; of equal weights the lower rows.

    Pages past the new lengths are pushed on ``free_pages`` (int32 ``[capacity]``, entries below ``n_free``, int32
    ``[1]``, valid).  ``lens_out``, ``evicted_out`` and ``n_free_out`` may be ``lens``, ``weights.evicted`` and
    ``n_free``; where ``evicted_out`` is not given it is ``weights.evicted`` if ``lens_out`` is ``lens`` (the same memory),
    else new.  A step that cannot be met (a length past the table's row, no room on the stack) changes nothing and says so
    in ``counts[3]`` (:meth:`EvictionPlan.check`).  Follow it with :func:`evict_paged` before anything takes pages or
    changes the lengths.
    """
    lib = _lib.load()
    device = lens.device
    if device.type != "cuda":
        raise ValueError("plan_eviction takes CUDA tensors")
    if page_len not in PAGE_LENS:
        raise ValueError(f"page_len must be one of {PAGE_LENS}, got {page_len}")
    n = lens.shape[0] if lens.dim() == 1 else 0
    if not 1 <= n <= _lib.PAGED_MAX_BATCH:
        raise ValueError(f"lens must be [requests] with 1 to {_lib.PAGED_MAX_BATCH} requests")
    requests, heads, _ = weights.weight.shape
    if requests != n or weights.weight.device != device:
        raise ValueError(f"weights are of {weights.requests} requests on {weights.device}, lens of {n} on {device}")
    _table(block_table, n, device)
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be one-dimensional")
    if not 1 <= max_keep <= 1 << 30:
        raise ValueError(f"max_keep must be in [1, 2^30], got {max_keep}")
    if not (0 <= sinks <= 0x7FFFFFFF and 0 <= recent <= 0x7FFFFFFF):
        raise ValueError("sinks and recent must not be negative")
    i32 = torch.int32
    if evicted_out is None and lens_out is not None and lens_out.data_ptr() == lens.data_ptr():
        evicted_out = weights.evicted
    lens_ptr = _need("lens", lens, i32, (n,), device)
    given = [_need("lens_out", lens_out, i32, (n,), device), _need("evicted_out", evicted_out, i32, (n,), device),
             _need("n_free_out", n_free_out, i32, (1,), device)]
    take = lens.new_empty((n, heads, max_keep))
    room = [n if lens_out is None else 0, n if evicted_out is None else 0, 1 if n_free_out is None else 0, 4]
    new_lens, new_evicted, new_n_free, counts = lens.new_empty(sum(room)).split_with_sizes(room)
    lens_out = new_lens if lens_out is None else lens_out
    evicted_out = new_evicted if evicted_out is None else evicted_out
    n_free_out = new_n_free if n_free_out is None else n_free_out
    stream = _stream_ptr(device)
    nbytes = lib.gqa_plan_eviction_workspace_bytes(n, heads, max_keep)
    ws = api._workspace(device, ("eviction", stream), nbytes)
    _check(lib.gqa_plan_eviction(
        ctypes.byref(weights.c), heads, lens_ptr, _need("keep", keep, i32, (n,), device), n, block_table.data_ptr(),
        block_table.stride(0), block_table.shape[1],
        _need("free_pages", free_pages, i32, free_pages.shape, device), free_pages.shape[0],
        _need("n_free", n_free, i32, (1,), device), page_len, max_keep, sinks, recent, take.data_ptr(),
        given[0] or lens_out.data_ptr(), given[1] or evicted_out.data_ptr(), given[2] or n_free_out.data_ptr(),
        counts.data_ptr(), ws.data_ptr(), ws.numel(), stream),
        "plan_eviction")
    return EvictionPlan(take, lens_out, evicted_out, n_free_out, counts)


def evict_paged(cache: PagedCache, block_table: torch.Tensor, weights: KeyWeights, plan: EvictionPlan) -> None:
    """Move the rows of ``plan``: K and V codes in ``cache``, and their weights and positions.  A block's scale grows
    where a row needs it, and the block's other codes are rounded again (as in :func:`append_paged`)."""
    lib = _lib.load()
    device = cache.device
    if device.type != "cuda":
        raise ValueError("evict_paged takes CUDA tensors")
    n = plan.lens.shape[0] if plan.lens.dim() == 1 else 0
    _check_weights(weights, cache, block_table, n)
    _table(block_table, n, device)
    max_keep = plan.take.shape[2] if plan.take.dim() == 3 else 0
    i32 = torch.int32
    take = _need("plan.take", plan.take, i32, (n, cache.kv_heads, max_keep), device)
    _check(lib.gqa_evict_paged(ctypes.byref(cache.c), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                               ctypes.byref(weights.c), _need("plan.lens", plan.lens, i32, (n,), device), take, n,
                               max_keep, _stream_ptr(device)), "evict_paged")
