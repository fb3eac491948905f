"""A serving loop over the paged 8-bit KV cache with a budget of keys a request.

Prompts are stored whole; what their last tokens look at decides which of their keys stay.  Every decode step then adds
the weights of its own attention, and a request that has grown past its budget by ``--slack`` keys loses those of the
least weight, whose pages go back to the pool.  Lengths, weights, pages and the choice live on the GPU throughout.  One
attention layer with random projections stands in for the model.

    python examples/paged_budget.py [--requests 16] [--steps 40] [--budget 256] [--slack 16] [--differential]

``--differential`` answers each step with differential attention as well (two softmax maps a head, their difference
normalised) over the keys that stayed.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import attention_accelerator_b200 as gqa  # noqa: E402

HEADS, KV_HEADS, DIM = gqa.N_Q_HEADS, gqa.N_KV_HEADS, gqa.HEAD_DIM


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--prompt", type=int, default=1500, help="longest prompt")
    ap.add_argument("--budget", type=int, default=256)
    ap.add_argument("--slack", type=int, default=16)
    ap.add_argument("--window", type=int, default=32, help="last tokens of a prompt whose weights count")
    ap.add_argument("--page-len", type=int, default=32, choices=(16, 32, 64, 128))
    ap.add_argument("--dtype", default="int8", choices=("int8", "e4m3"))
    ap.add_argument("--differential", action="store_true")
    args = ap.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(dev).manual_seed(0)
    n, page_len = args.requests, args.page_len
    width = -(-max(args.prompt, args.budget + args.slack + 1) // page_len)
    i32 = dict(dtype=torch.int32, device=dev)
    cache = gqa.paged_cache(n * width, page_len, dtype=torch.int8 if args.dtype == "int8" else torch.float8_e4m3fn)
    weights = gqa.key_weights(n, width * page_len)
    table = torch.full((n, width), -1, **i32)
    free, n_free = torch.arange(n * width, **i32), torch.full((1,), n * width, **i32)
    lens = torch.zeros(n, **i32)

    def rows(count: int, heads: int) -> torch.Tensor:
        return torch.randn(count, heads, DIM, generator=gen, device=dev).to(torch.bfloat16)

    def append(new: list[int]):
        """``new[r]`` tokens join request r, at the positions behind all it has had; returns the plan and their queries."""
        total = sum(new)
        plan = gqa.plan_pages(lens, torch.tensor(new, **i32), table, free, n_free, page_len=page_len, max_tokens=total,
                              lens_out=lens, n_free_out=n_free, weights=weights)
        owner = torch.searchsorted(plan.first_token[1:], torch.arange(total, **i32), right=True)
        gqa.append_paged(cache, rows(total, KV_HEADS), rows(total, KV_HEADS), plan.slots,
                         positions=plan.positions + weights.evicted[owner])
        return plan, rows(total, HEADS)

    def cut(keep: torch.Tensor) -> gqa.EvictionPlan:
        plan = gqa.plan_eviction(weights, lens, keep, table, free, n_free, page_len=page_len, max_keep=args.budget,
                                 recent=args.window, lens_out=lens, n_free_out=n_free)
        gqa.evict_paged(cache, table, weights, plan)
        return plan

    prompts = [1 + (r * 7919) % args.prompt for r in range(n)]
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    plan, q = append(prompts)
    out = gqa.decode_paged_chunked(q, cache, table, lens, plan.first_token)
    seen = [min(p, args.window) for p in prompts]
    ends = [sum(prompts[:r + 1]) for r in range(n)]
    first = torch.tensor([0] + [sum(seen[:r + 1]) for r in range(n)], **i32)
    last = torch.cat([q[e - s:e] for e, s in zip(ends, seen)])
    gqa.add_key_weights(last, cache, table, lens, first, weights, known=torch.zeros(n, **i32))
    budget = torch.full((n,), args.budget, **i32)
    cut(budget)
    lambdas = torch.full((2 * KV_HEADS,), 0.5, device=dev)
    gain = torch.ones(DIM, device=dev)
    for _ in range(args.steps):
        _, q = append([1] * n)
        out = gqa.decode_paged_weights(q, cache, table, lens, weights)
        if args.differential:
            out = gqa.decode_paged_diff(q, cache, table, lens, lambdas, norm_weight=gain, out_scale=0.5,
                                        query_positions=lens - 1 + weights.evicted)
        plan = cut(torch.where(lens >= budget + args.slack, budget, 0).to(torch.int32))
    stop.record()
    torch.cuda.synchronize()
    plan.check()
    held = lens.tolist()
    tokens = [p + args.steps for p in prompts]
    return {"tokens": sum(tokens), "held": sum(held), "longest": max(held),
            "accounted": [h + e for h, e in zip(held, weights.evicted.tolist())] == tokens,
            "pages_used": n * width - int(n_free), "pages_needed": sum(-(-h // page_len) for h in held),
            "ms": start.elapsed_time(stop), "finite": bool(torch.isfinite(out).all()),
            "device_status": gqa.read_device_status()}


if __name__ == "__main__":
    for name, value in main().items():
        print(f"{name}: {value}")
