"""A serving loop over the paged 8-bit KV cache: prompts, decode steps, drafted tokens, and pages that come back.

Requests with ragged prompts are admitted together, decode one token a step, verify a few drafted tokens now and
then, and finish at different times; finished requests' pages go to new requests.  Lengths, pages and slots live on
the GPU throughout: the loop's only host decisions are who joins and who leaves.  One attention layer with random
projections stands in for the model.

    python examples/paged_serving.py [--requests 32] [--steps 40] [--page-len 64] [--dtype int8] [--check]

``--check`` keeps a BF16 copy of every request's K and V beside the cache and compares the last step's outputs with
``decode_batch`` over it: what remains is the 8 bits.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import attention_accelerator_b200 as gqa  # noqa: E402

HEADS, KV_HEADS, DIM = gqa.N_Q_HEADS, gqa.N_KV_HEADS, gqa.HEAD_DIM


class Server:
    """Slots for ``requests`` running requests over a pool of pages."""

    def __init__(self, requests: int, pages: int, page_len: int, longest: int, dtype: torch.dtype, seed: int = 0):
        dev = torch.device("cuda", torch.cuda.current_device())
        i32 = dict(dtype=torch.int32, device=dev)
        self.gen = torch.Generator(dev).manual_seed(seed)
        self.requests, self.page_len = requests, page_len
        self.cache = gqa.paged_cache(pages, page_len, dtype=dtype)
        self.table = torch.full((requests, -(-longest // page_len)), -1, **i32)
        self.free = torch.arange(pages, **i32)
        self.n_free = torch.full((1,), pages, **i32)
        self.lens = torch.zeros(requests, **i32)
        self.copy = None  # per request: lists of BF16 K (rotated) and V rows

    def rows(self, n: int, heads: int) -> torch.Tensor:
        return torch.randn(n, heads, DIM, generator=self.gen, device=self.lens.device).to(torch.bfloat16)

    def step(self, new: list[int]) -> torch.Tensor:
        """``new[r]`` tokens join request r (-1: it ends); returns the attention rows of the new tokens."""
        new_lens = torch.tensor(new, dtype=torch.int32).pin_memory().to(self.lens.device, non_blocking=True)
        tokens = sum(n for n in new if n > 0)
        plan = gqa.plan_pages(self.lens, new_lens, self.table, self.free, self.n_free, page_len=self.page_len,
                              max_tokens=tokens, lens_out=self.lens, n_free_out=self.n_free)
        q, k, v = self.rows(tokens, HEADS), self.rows(tokens, KV_HEADS), self.rows(tokens, KV_HEADS)
        gqa.append_paged(self.cache, k, v, plan.slots, positions=plan.positions)
        if self.copy is not None:
            self.keep(new, plan, k, v)
        if all(n == 1 for n in new):
            return gqa.decode_paged(q, self.cache, self.table, self.lens)
        return gqa.decode_paged_chunked(q, self.cache, self.table, self.lens, plan.first_token)

    def keep(self, new, plan, k, v):
        k = gqa.rope_k_cache(k, plan.positions)
        at = 0
        for r, n in enumerate(new):
            if n < 0:
                self.copy[r] = []
            elif n:
                self.copy[r].append((k[at:at + n], v[at:at + n]))
                at += n

    def difference(self) -> float:
        """Largest difference of a decode over the pages from one over the BF16 copy, over the latter's RMS."""
        held = [r for r in range(self.requests) if self.copy[r]]
        k, v = (torch.cat([x[i] for r in held for x in self.copy[r]]) for i in (0, 1))
        lens = [sum(x[0].shape[0] for x in self.copy[r]) for r in held]
        q = self.rows(len(held), HEADS)
        index = torch.tensor(held, device=self.lens.device)
        want = gqa.decode_batch(q, k, v, gqa.plan_batch(lens), k_rotated=True).float()
        got = gqa.decode_paged(q, self.cache, self.table[index].contiguous(), self.lens[index]).float()
        return float((got - want).abs().max() / want.square().mean().sqrt())


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--prompt", type=int, default=700, help="longest prompt")
    ap.add_argument("--page-len", type=int, default=64, choices=(16, 32, 64, 128))
    ap.add_argument("--dtype", default="e4m3", choices=("int8", "e4m3"))
    ap.add_argument("--check", action="store_true")
    args = ap.parse_args(argv)
    longest = args.prompt + 6 * args.steps
    pages = args.requests * -(-longest // args.page_len)
    server = Server(args.requests, pages, args.page_len, longest,
                    torch.int8 if args.dtype == "int8" else torch.float8_e4m3fn)
    if args.check:
        server.copy = [[] for _ in range(args.requests)]
    prompts = [1 + (r * 7919) % args.prompt for r in range(args.requests)]
    tokens, start, stop = 0, torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for step in range(args.steps):
        if step == 0:
            new = prompts
        elif step % 10 == 9:  # a tenth of the requests end; new ones take their places in the next step
            new = [-1 if (r + step) % 10 == 0 else 1 for r in range(args.requests)]
        elif step % 10 == 0:
            new = [prompts[r] if (r + step - 1) % 10 == 0 else 1 for r in range(args.requests)]
        elif step % 4 == 3:   # drafted tokens to verify
            new = [1 + r % 5 for r in range(args.requests)]
        else:
            new = [1] * args.requests
        out = server.step(new)
        tokens += sum(n for n in new if n > 0)
    stop.record()
    torch.cuda.synchronize()
    used = int(sum(-(-n // args.page_len) for n in server.lens.tolist()))
    result = {"tokens": tokens, "tokens_per_s": tokens / start.elapsed_time(stop) * 1e3,
              "pages_used": used, "pages_free": int(server.n_free), "pages": pages,
              "finite": bool(torch.isfinite(out).all()), "device_status": gqa.read_device_status()}
    if args.check:
        result["difference"] = server.difference()
    return result


if __name__ == "__main__":
    for name, value in main().items():
        print(f"{name}: {value}")
