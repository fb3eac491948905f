"""The paged 8-bit KV cache's operators as measured cases: page planning, append and read-back, and attention over the
cache for one token a sequence and for many, with capped scores, distance bias, document and prefix masks.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes a program's
inputs, ``run(state)`` is one pass -- in elementary torch operations, or through ``attention_accelerator_b200`` where
``own`` is true -- ``work(case)`` counts what a pass cannot do without and ``exact(case, seed)`` is the same answer in
64 bits.
"""
import math

import numpy as np
import torch

own = False

HEADS, GROUP, DIM = 8, 4, 128        # KV heads, Q heads of each, head_dim
THETA = 500000.0
SCALE = 1.0 / math.sqrt(DIM)
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
CODE_TYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MIN_SCALE = 2.0 ** -100


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # A decode step of 64 running requests: one new token each, some requests just finished.
        {"name": "pages-step-64", "op": "pages", "requests": 64, "page": 16, "longest": 8192, "new": 1, "budget": 64},
        # A wave of prompts: 1024 requests share a budget of 131072 new tokens.
        {"name": "pages-prompts-1024", "op": "pages", "requests": 1024, "page": 64, "longest": 8192, "new": 256,
         "budget": 131072},
        # The K/V rows of that decode step go into half-filled pages.
        {"name": "append-step-64", "op": "append", "requests": 64, "new": 1, "cached": 8192, "page": 64,
         "code": "e4m3", "layout": "head_major"},
        # Eight ragged prompts are stored whole.
        {"name": "append-prompts-8", "op": "append", "requests": 8, "new": 4095, "cached": 100, "page": 32,
         "code": "int8", "layout": "position_major"},
        # The shortest call: one sequence of 30 keys, where latency is everything.
        {"name": "decode-1x30", "op": "decode", "batch": 1, "low": 30, "high": 30, "page": 16, "code": "int8",
         "layout": "head_major", "cap": 0.0, "slopes": False, "docs": False, "rope": True},
        # The serving batch: 64 ragged sequences of 512 to 8192 keys.
        {"name": "decode-64-ragged", "op": "decode", "batch": 64, "low": 512, "high": 8192, "page": 64, "code": "e4m3",
         "layout": "head_major", "cap": 0.0, "slopes": False, "docs": False, "rope": True},
        # One long context.
        {"name": "decode-1x131072", "op": "decode", "batch": 1, "low": 131072, "high": 131072, "page": 128,
         "code": "int8", "layout": "position_major", "cap": 0.0, "slopes": False, "docs": False, "rope": True},
        # Capped scores with a distance bias, each token in a document of its own sequence; some rows see nothing.
        {"name": "decode-33-cap-bias-docs", "op": "decode", "batch": 33, "low": 0, "high": 4099, "page": 32,
         "code": "e4m3", "layout": "position_major", "cap": 30.0, "slopes": True, "docs": True, "rope": False},
        # Chunks of 128 queries at the end of 8192 keys, 16 sequences.
        {"name": "chunk-16x128-8192", "op": "chunk", "batch": 16, "low": 8192, "high": 8192, "queries": 128, "page": 64,
         "code": "e4m3", "layout": "head_major", "cap": 0.0, "slopes": False, "masks": "", "rope": True},
        # Whole ragged prompts, the first part of each visible to all its tokens, capped scores.
        {"name": "chunk-prompts-prefix-cap", "op": "chunk", "batch": 8, "low": 1, "high": 2051, "queries": 2051,
         "page": 16, "code": "int8", "layout": "position_major", "cap": 50.0, "slopes": False, "masks": "prefix",
         "rope": True},
        # One packed sequence of documents with a distance bias.
        {"name": "chunk-docs-bias-8192", "op": "chunk", "batch": 1, "low": 8192, "high": 8192, "queries": 8192,
         "page": 128, "code": "e4m3", "layout": "head_major", "cap": 0.0, "slopes": True, "masks": "docs",
         "rope": False},
        # Five drafted tokens of each of 48 ragged sequences are verified in one call.
        {"name": "chunk-verify-48x5", "op": "chunk", "batch": 48, "low": 5, "high": 8191, "queries": 5, "page": 64,
         "code": "int8", "layout": "head_major", "cap": 0.0, "slopes": False, "masks": "", "rope": True},
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 1))) - 0.5))))

    op = rng.choice(["pages", "append", "decode", "decode", "chunk", "chunk"])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.choice(["head_major", "position_major"])
    code = rng.choice(["int8", "e4m3"])
    if op == "pages":
        n = log(1, 1024)
        new = rng.choice([1, log(1, 256)])
        return {"op": op, "requests": n, "page": page, "longest": log(64, 8192), "new": new,
                "budget": min(131072, n * new)}
    if op == "append":
        n = log(1, 256)
        return {"op": op, "requests": n, "new": rng.choice([1, log(1, max(1, 16384 // n))]), "cached": log(1, 8192),
                "page": page, "code": code, "layout": layout}
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    slopes = rng.random() < 0.3
    if op == "decode":
        n = log(1, 128)
        high = log(1, min(131072, 262144 // n))
        return {"op": op, "batch": n, "low": rng.choice([0, high // 8, high]), "high": high, "page": page, "code": code,
                "layout": layout, "cap": cap, "slopes": slopes, "docs": rng.random() < 0.3, "rope": not slopes}
    n = log(1, 48)
    queries = log(2, max(2, 4096 // n))
    high = max(queries, log(2, min(32768, 131072 // n)))
    high = max(queries, min(high, 16777216 // (n * queries)))
    return {"op": op, "batch": n, "low": rng.choice([1, high]), "high": high, "queries": queries, "page": page,
            "code": code, "layout": layout, "cap": cap, "slopes": slopes,
            "masks": rng.choice(["", "", "docs", "prefix", "docs prefix"]), "rope": not slopes}


def lengths(case):
    """The sequences' lengths, spread over [low, high] in no order."""
    low, high = case["low"], case["high"]
    return [low + int((high - low) * ((i * 0.6180339887 + 0.999) % 1.0) + 0.5) for i in range(case["batch"])]


def query_counts(case):
    """New tokens of each sequence: at most what it holds, and ragged where the case asks for whole prompts."""
    return [min(s, case["queries"]) for s in lengths(case)]


def append_lengths(case):
    """(cached, new) tokens of each request of an append."""
    n, new = case["requests"], case["new"]
    cached = [int(case["cached"] * ((i * 0.7548776662 + 0.37) % 1.0)) for i in range(n)]
    fresh = [1 if new == 1 else 1 + int((new - 1) * ((i * 0.5698402910 + 0.93) % 1.0)) for i in range(n)]
    return cached, fresh


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def quantise(x, code):
    """Codes and one scale per leading block of ``x`` [blocks, heads, rows, DIM]."""
    s = (x.abs().amax((-1, -2)) * (1.0 / CODE_MAX[code])).clamp(min=MIN_SCALE)
    y = x * (1.0 / s)[..., None, None]
    return (y.round().clamp(-127, 127) if code == "int8" else y.clamp(-448, 448)).to(CODE_TYPE[code]), s


def make_cache(gen, pages, page, code, layout):
    """A filled cache: keys with strong channels, as real ones have, and values whose size differs from page to page."""
    channel = torch.exp(0.5 * torch.randn(HEADS, 1, DIM, device="cuda", generator=gen))
    parts = {"k": [], "v": [], "k_scale": [], "v_scale": []}
    for at in range(0, pages, 4096):
        n = min(4096, pages - at)
        shape = (n, HEADS, page, DIM)
        k = torch.randn(shape, device="cuda", generator=gen) * channel
        v = torch.randn(shape, device="cuda", generator=gen)
        v *= torch.exp(0.5 * torch.randn(n, HEADS, 1, 1, device="cuda", generator=gen))
        for name, x in (("k", k), ("v", v)):
            c, s = quantise(x, code)
            parts[name].append(c if layout == "head_major" else c.view(torch.uint8).transpose(1, 2).contiguous().view(c.dtype))
            parts[name + "_scale"].append(s)
    return {name: torch.cat([x.view(torch.uint8) for x in p]).view(p[0].dtype) if name in ("k", "v") else torch.cat(p)
            for name, p in parts.items()}


def make_table(gen, lens, page, width=None):
    """A block table over pages in no order, and how many pages there are."""
    need = [-(-s // page) for s in lens]
    pages = max(1, sum(need))
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    width = width or max(1, max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    host, at = order.cpu(), 0
    for b, n in enumerate(need):
        table[b, :n] = host[at:at + n]
        at += n
    return table.cuda(), pages


def cuda_ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case), "op": case["op"]}
    s.update({"pages": prepare_pages, "append": prepare_append, "decode": prepare_attention,
              "chunk": prepare_attention}[case["op"]](case, seed, gen))
    if own and case["op"] != "pages":
        import attention_accelerator_b200 as gqa
        c = s["cache"]
        s["handle"] = gqa.PagedCache(c["k"], c["v"], c["k_scale"], c["v_scale"], layout=case["layout"])
    return s


def prepare_pages(case, seed, gen):
    r = np.random.RandomState(seed % (1 << 31))
    n, page = case["requests"], case["page"]
    lens = r.randint(0, case["longest"] + 1, n)
    new = np.minimum(r.randint(1, case["new"] + 1, n), max(1, case["budget"] // n))
    done = r.rand(n) < 0.1
    new = np.where(done, -1, new)
    need = -(-lens // page)
    width = int(-(-(case["longest"] + case["new"]) // page))
    table, held = make_table(gen, [int(x) for x in lens], page, width)
    spare = int((-(-(lens + np.maximum(new, 0)) // page) - need).sum()) + 64
    free = np.full(n * width + 64, -1, np.int32)
    free[:spare] = held + r.permutation(spare)
    return {"lens": cuda_ints(lens.tolist()), "new": cuda_ints(new.tolist()), "table": table,
            "free": torch.from_numpy(free).cuda(), "n_free": cuda_ints([spare])}


def prepare_append(case, seed, gen):
    page = case["page"]
    cached, fresh = append_lengths(case)
    table, pages = make_table(gen, [a + b for a, b in zip(cached, fresh)], page)
    host = table.cpu()
    slots, positions, read = [], [], []
    for b, (a, n) in enumerate(zip(cached, fresh)):
        first = a - a % page  # the pages that change, from their first row on
        pos = torch.arange(first, a + n)
        at = host[b, pos // page].to(torch.int64) * page + pos % page
        read.append(at)
        slots.append(at[a - first:])
        positions.append(pos[a - first:].to(torch.int32))
    slots, positions, read = (torch.cat(x).cuda() for x in (slots, positions, read))
    rows = (slots.numel(), HEADS, DIM)
    size = torch.exp(0.5 * torch.randn(rows[0], 1, 1, device="cuda", generator=gen))
    k = (torch.randn(rows, device="cuda", generator=gen) * size).to(torch.bfloat16)
    v = (torch.randn(rows, device="cuda", generator=gen) * size).to(torch.bfloat16)
    return {"cache": make_cache(gen, pages, page, case["code"], case["layout"]), "k": k, "v": v, "slots": slots,
            "positions": positions, "read": read}


def prepare_attention(case, seed, gen):
    lens = lengths(case)
    counts = [1] * len(lens) if case["op"] == "decode" else query_counts(case)
    table, pages = make_table(gen, lens, case["page"])
    s = {"cache": make_cache(gen, pages, case["page"], case["code"], case["layout"]), "table": table,
         "lens": cuda_ints(lens), "longest": max(lens), "most": max(counts)}
    rows = sum(counts)
    s["q"] = torch.randn(rows, HEADS * GROUP, DIM, device="cuda", generator=gen).to(torch.bfloat16)
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    s["first"] = cuda_ints(first)
    s["slopes"] = (torch.pow(2.0, -8.0 * torch.arange(1, HEADS * GROUP + 1, device="cuda") / (HEADS * GROUP))
                   if case["slopes"] else None)
    starts, ends = mask_rows(case, lens, counts)
    s["doc_starts"] = cuda_ints(starts) if starts is not None else None
    s["prefix_ends"] = cuda_ints(ends) if ends is not None else None
    return s


def mask_rows(case, lens, counts):
    """Each query's first visible key (documents) and the end of the keys that all see (prefixes), or None."""
    docs = case["docs"] if case["op"] == "decode" else "docs" in case["masks"]
    prefix = case["op"] == "chunk" and "prefix" in case["masks"]
    starts, ends = [], []
    for b, (length, n) in enumerate(zip(lens, counts)):
        edges = [0]  # documents of 200 to 1000 tokens
        while edges[-1] < length:
            edges.append(edges[-1] + 200 + (len(edges) * 389 + b * 151) % 801)
        at = 0
        for i in range(n):
            m = length - n + i
            while at + 1 < len(edges) and edges[at + 1] <= m:
                at += 1
            empty = case["op"] == "decode" and b % 11 == 5
            starts.append(length if empty else edges[at])
            ends.append(min(length, (edges[at] if docs else 0) + (length // 3 if not docs else 100)))
    return starts if docs else None, ends if prefix else None


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
def run(state):
    return (run_own if own else run_plain)(state)


def run_own(s):
    import attention_accelerator_b200 as gqa
    case = s["case"]
    if s["op"] == "pages":
        p = gqa.plan_pages(s["lens"], s["new"], s["table"], s["free"], s["n_free"], page_len=case["page"],
                           max_tokens=case["budget"])
        return {"table": s["table"], "free": s["free"], "lens": p.lens, "n_free": p.n_free,
                "first": p.first_token, "slots": p.slots, "positions": p.positions, "counts": p.counts}
    if s["op"] == "append":
        gqa.append_paged(s["handle"], s["k"], s["v"], s["slots"], positions=s["positions"], rope_theta=THETA)
        k, v = gqa.read_paged(s["handle"], s["read"])
        return {"k": k, "v": v, "k_scale": s["cache"]["k_scale"], "v_scale": s["cache"]["v_scale"]}
    more = {"score_cap": case["cap"] or None, "distance_slopes": s["slopes"], "doc_starts": s["doc_starts"],
            "prefix_ends": s["prefix_ends"], "q_rotated": not case["rope"], "rope_theta": THETA}
    if s["op"] == "decode":
        return gqa.decode_paged(s["q"], s["handle"], s["table"], s["lens"], **more)
    return gqa.decode_paged_chunked(s["q"], s["handle"], s["table"], s["lens"], s["first"], **more)


def run_plain(s):
    return {"pages": plain_pages, "append": plain_append, "decode": plain_attention, "chunk": plain_attention}[s["op"]](s)


def plain_pages(s):
    lens, new, table, page, budget = s["lens"], s["new"], s["table"], s["case"]["page"], s["case"]["budget"]
    n, width = table.shape
    done = new < 0
    add = new.clamp(min=0)
    held = (lens + page - 1) // page
    after = torch.where(done, 0, lens + add)
    need = torch.where(done, 0, (lens + add + page - 1) // page - held)
    give = torch.where(done, held, 0)
    first = torch.cumsum(add, 0) - add
    column = torch.arange(width, device="cuda")[None]
    # Released pages go on top of the free stack, in the order of requests and columns.
    gone = done[:, None] & (column < held[:, None])
    place = s["n_free"] + (torch.cumsum(give, 0) - give)[:, None] + column
    stack = torch.cat([s["free"], s["free"][:1]])
    stack.scatter_(0, torch.where(gone, place, s["free"].numel()).reshape(-1), table.reshape(-1))
    stack = stack[:-1]
    top = s["n_free"] + give.sum()
    # New pages come off its top.
    taken = (torch.cumsum(need, 0) - need)[:, None] + column - held[:, None]
    fresh = (column >= held[:, None]) & (column < (held + need)[:, None])
    pages = torch.where(fresh, stack[(top - 1 - taken).clamp(0, stack.numel() - 1)], table)
    token = torch.arange(budget, device="cuda")
    request = torch.searchsorted(torch.cumsum(add, 0), token, right=True).clamp(max=n - 1)
    position = lens[request] + token - first[request]
    slot = pages[request, (position // page).clamp(max=width - 1)].to(torch.int64) * page + position % page
    real = token < add.sum()
    ok = (need.sum() <= top) & ((after + page - 1) // page <= width).all() & (add.sum() <= budget)
    total = torch.cat([add.sum()[None], need.sum()[None], give.sum()[None], torch.zeros_like(give[:1])])
    ends = torch.cat([torch.zeros_like(add[:1]), torch.cumsum(add, 0)])
    whole = torch.int32
    return {"table": torch.where(ok, pages, table), "free": torch.where(ok, stack, s["free"]),
            "lens": torch.where(ok, after, lens).to(whole),
            "n_free": torch.where(ok, top - need.sum(), s["n_free"]).to(whole),
            "first": torch.where(ok, ends, 0).to(whole), "slots": torch.where(ok & real, slot, -1),
            "positions": torch.where(ok & real, position, -1).to(whole),
            "counts": torch.where(ok, total, (~ok).reshape(1)).to(whole)}


def rotate(x, positions):
    """RoPE of rows [n, heads, DIM] at their positions, in 32 bits."""
    turn = torch.pow(THETA, -torch.arange(DIM // 2, device="cuda", dtype=torch.float32) / (DIM // 2))
    angle = positions.float()[:, None, None] * turn
    a, b = x.float().split(DIM // 2, -1)
    c, d = angle.cos(), angle.sin()
    return torch.cat([a * c - b * d, a * d + b * c], -1)


def plain_append(s):
    case, cache = s["case"], s["cache"]
    page, slots, top = case["page"], s["slots"], CODE_MAX[case["code"]]
    block, row = slots // page, slots % page
    out = {}
    for name, x in (("k", rotate(s["k"], s["positions"])), ("v", s["v"].float())):
        codes, old = cache[name], cache[name + "_scale"]
        by_row = codes if case["layout"] == "position_major" else codes.transpose(1, 2)
        pages = old.shape[0]
        index = block[:, None].expand(-1, HEADS)
        most = torch.zeros_like(old).scatter_reduce_(0, index, x.abs().amax(-1), "amax")
        start = torch.full((pages,), page, device="cuda").scatter_reduce_(0, block, row, "amin")
        before = torch.where((start == 0)[:, None], 0.0, old)
        scale = torch.where((start < page)[:, None], torch.maximum(before, (most / top).clamp(min=MIN_SCALE)), old)
        # What the changed pages held before the new rows is rounded again where their scale grew.
        earlier = s["read"][(s["read"] % page) < start[s["read"] // page]]
        b, r = earlier // page, earlier % page
        held = by_row[b, r].float()
        again = (held * old[b][..., None]) * (1.0 / scale[b])[..., None]
        held = torch.where((scale[b] > old[b])[..., None], again, held)
        fresh = x * (1.0 / scale[block])[..., None]
        where = torch.cat([b, block]), torch.cat([r, row])
        y = torch.cat([held, fresh])
        y = y.round().clamp(-127, 127) if case["code"] == "int8" else y.clamp(-448, 448)
        by_row.view(torch.uint8)[where] = y.to(codes.dtype).view(torch.uint8)
        old.copy_(scale)
        b, r = s["read"] // page, s["read"] % page
        out[name] = (by_row.view(torch.uint8)[b, r].view(codes.dtype).float() * scale[b][..., None]).to(torch.bfloat16)
        out[name + "_scale"] = old
    return out


def plain_attention(s):
    case = s["case"]
    q, lens, first, page, most = s["q"], s["lens"], s["first"], case["page"], s["most"]
    batch, width = s["table"].shape
    keys = width * page
    # The sequences' queries side by side: [batch, most], rows past a sequence's own are not used.
    i = torch.arange(most, device="cuda")[None]
    count = (first[1:] - first[:-1])[:, None]
    if case["op"] == "decode":
        position = lens[:, None] - 1
    else:
        position = lens[:, None] - count + i
    row = (first[:-1, None] + i).clamp(max=q.shape[0] - 1)
    q = (rotate(q, torch.where(i < count, position, 0)[i < count]) if case["rope"] else q.float())[row]
    q = q.reshape(batch, most, HEADS, GROUP, DIM).permute(0, 2, 3, 1, 4).reshape(batch, HEADS, GROUP * most, DIM)

    def dense(name):
        table = s["table"].clamp(min=0).long()
        x = s["cache"][name].view(torch.uint8)[table].view(s["cache"][name].dtype).float()
        if case["layout"] == "head_major":
            x = x.transpose(2, 3)
        x = x * s["cache"][name + "_scale"][table][:, :, None, :, None]
        return x.reshape(batch, keys, HEADS, DIM).transpose(1, 2)

    z = (q @ dense("k").transpose(-1, -2) * SCALE).reshape(batch, HEADS, GROUP, most, keys)
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    key = torch.arange(keys, device="cuda")
    if s["slopes"] is not None:
        far = (position[..., None] - key).abs().float()
        z = z - s["slopes"].reshape(HEADS, GROUP, 1, 1) * far[:, None, None]
    end = position + 1
    if s["prefix_ends"] is not None:
        end = torch.maximum(end, s["prefix_ends"][row])
    end = torch.minimum(end, lens[:, None])
    start = s["doc_starts"][row] if s["doc_starts"] is not None else torch.zeros_like(end)
    seen = ((key >= start[..., None]) & (key < end[..., None]))[:, None, None]
    z = torch.where(seen, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    w = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    v = torch.where((key < lens[:, None])[:, None, :, None], dense("v"), 0.0)
    o = w.reshape(batch, HEADS, GROUP * most, keys) @ v
    o = o.reshape(batch, HEADS, GROUP, most, DIM) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, most, HEADS * GROUP, DIM)
    return o[i < count].to(torch.bfloat16)


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    row = HEADS * DIM
    if case["op"] == "pages":
        n = case["requests"]
        tokens = min(case["budget"], n * (case["new"] + 1) / 2)
        return {"bytes": n * 24 + tokens * 12 + 8 * tokens / case["page"], "flops": 4 * tokens}
    if case["op"] == "append":
        cached, fresh = append_lengths(case)
        tokens = sum(fresh)
        read = sum(a % case["page"] + n for a, n in zip(cached, fresh))
        # BF16 in and codes out for the new rows, then codes in and BF16 out for the rows read back.
        return {"bytes": 2 * row * (3 * tokens + 3 * read) + 8 * HEADS * 2 * (read // case["page"] + len(fresh)),
                "flops": 2 * row * (6 * tokens + read)}
    lens = lengths(case)
    counts = [1] * len(lens) if case["op"] == "decode" else query_counts(case)
    starts, ends = mask_rows(case, lens, counts)
    pairs = keys = at = 0
    for length, n in zip(lens, counts):
        low, high = length, 0
        for i in range(n):
            lo = starts[at] if starts is not None else 0
            hi = min(length, max(length - n + i + 1, ends[at] if ends is not None else 0))
            at += 1
            pairs += max(0, hi - lo)
            if hi > lo:
                low, high = min(low, lo), max(high, hi)
        keys += max(0, high - low)
    scales = 2 * 4 * HEADS * (keys // case["page"] + len(lens))
    return {"bytes": 2 * keys * row + scales + 2 * 2 * sum(counts) * row * GROUP, "flops": 4 * DIM * HEADS * GROUP * pairs}


# ----------------------------------------------------------------------------------------------------------------------
# the same in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers
    s = prepare(case, seed)
    return exact_append(s) if case["op"] == "append" else exact_attention(s)


def turned(x, position):
    """Rows [n, heads, DIM] as complex pairs turned by their positions, in 64 bits."""
    x = x.double()
    z = torch.complex(x[..., :DIM // 2], x[..., DIM // 2:])
    angle = torch.tensor([THETA ** (-2.0 * j / DIM) for j in range(DIM // 2)], dtype=torch.float64, device="cuda")
    z = z * torch.exp(1j * position.double()[:, None, None] * angle)
    return torch.cat([z.real, z.imag], -1)


def code_value(y, code):
    if code == "int8":
        return torch.round(y).clamp(-127, 127)
    return y.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()


def exact_append(s):
    case, cache = s["case"], s["cache"]
    page, code = case["page"], case["code"]
    cached, fresh = append_lengths(case)
    new = {"k": turned(s["k"], s["positions"]), "v": s["v"].double()}
    out = {}
    for name in ("k", "v"):
        codes = cache[name].float().double()
        codes = codes if case["layout"] == "position_major" else codes.transpose(1, 2).contiguous()  # [pages, rows, heads, DIM]
        scale = cache[name + "_scale"].double()
        at = 0
        for a, n in zip(cached, fresh):
            done = 0
            while done < n:
                r = (a + done) % page
                m = min(page - r, n - done)
                b = int(s["slots"][at]) // page
                x = new[name][at:at + m]
                old = scale[b] if r else torch.zeros_like(scale[b])
                least = torch.full_like(old, MIN_SCALE)
                now = torch.maximum(torch.maximum(old, x.abs().amax((0, 2)) / CODE_MAX[code]), least).float().double()
                grew = (now > old)[None, :, None]
                codes[b, :r] = torch.where(grew, code_value(codes[b, :r] * (old / now)[None, :, None], code), codes[b, :r])
                codes[b, r:r + m] = code_value(x / now[None, :, None], code)
                scale[b] = now
                at += m
                done += m
        b, r = s["read"] // page, s["read"] % page
        out[name] = codes[b, r] * scale[b][..., None]
        out[name + "_scale"] = scale
    return out


def exact_attention(s):
    case = s["case"]
    page, cache, lens = case["page"], s["cache"], s["lens"].tolist()
    first, rows = s["first"].tolist(), s["q"].shape[0]
    out = torch.zeros(rows, HEADS * GROUP, DIM, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        n = first[b + 1] - first[b]
        m = torch.arange(length - n, length, device="cuda")
        if case["op"] == "decode":
            m = torch.tensor([length - 1], device="cuda")
        q = s["q"][first[b]:first[b + 1]]
        q = turned(q, m) if case["rope"] else q.double()
        if length == 0:
            continue
        p = torch.arange(length, device="cuda")
        block = s["table"][b].long()[p // page]
        end = m + 1
        if s["prefix_ends"] is not None:
            end = torch.maximum(end, s["prefix_ends"][first[b]:first[b + 1]].long())
        start = s["doc_starts"][first[b]:first[b + 1]].long() if s["doc_starts"] is not None else torch.zeros_like(m)
        hidden = (p[None] < start[:, None]) | (p[None] >= end[:, None])
        for h in range(HEADS):
            part = {}
            for name in ("k", "v"):
                c = cache[name] if case["layout"] == "position_major" else cache[name].transpose(1, 2)
                c = c.view(torch.uint8)[block, p % page, h].view(cache[name].dtype).float().double()
                part[name] = c * cache[name + "_scale"][block, h].double()[:, None]
            for g in range(GROUP):
                head = h * GROUP + g
                z = q[:, head] @ part["k"].T / math.sqrt(DIM)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if s["slopes"] is not None:
                    z = z - float(s["slopes"][head]) * (m[:, None] - p[None]).abs()
                z.masked_fill_(hidden, -math.inf)
                w = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)).nan_to_num_(nan=0.0)
                out[first[b]:first[b + 1], head] = w @ part["v"]
    return out
