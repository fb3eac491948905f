"""More operators of the paged 8-bit KV cache as measured cases: differential attention for one token a sequence and for
many, and eviction by accumulated attention weight -- the weights of a decode step's keys and of a prompt's, the choice of
what stays, and the move.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes a program's
inputs, ``run(state)`` is one pass -- in elementary torch operations, or through ``attention_accelerator_b200`` where
``own`` is true -- ``work(case)`` counts what a pass cannot do without and ``exact(case, seed)`` is the same answer in
64 bits.
"""
import math

import torch

own = False

HEADS, GROUP, DIM = 8, 4, 128        # KV heads, Q heads of each, head_dim
PAIRS = HEADS * GROUP // 2           # differential heads: Q heads 2 j and 2 j + 1
THETA = 500000.0
SCALE = 1.0 / math.sqrt(DIM)
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
CODE_TYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MIN_SCALE = 2.0 ** -100
LAMBDA_INIT = 0.8 - 0.6 * math.exp(-0.3 * 8)   # of a ninth layer
NORM_EPS = 1e-5
SINKS = 4


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # The shortest call: one sequence of 30 keys, where latency is everything.
        {"name": "diff-1x30", "op": "diff", "batch": 1, "low": 30, "high": 30, "page": 16, "code": "int8",
         "layout": "head_major", "cap": 0.0, "slopes": False, "docs": False, "norm": True, "by_row": False},
        # The serving batch: a token each of 64 ragged sequences, lambdas projected from the tokens.
        {"name": "diff-64-ragged", "op": "diff", "batch": 64, "low": 512, "high": 8192, "page": 64, "code": "e4m3",
         "layout": "head_major", "cap": 0.0, "slopes": False, "docs": False, "norm": True, "by_row": True},
        # Five drafted tokens of each of 48 ragged sequences are verified in one call.
        {"name": "diff-verify-48x5", "op": "diffchunk", "batch": 48, "low": 5, "high": 8191, "queries": 5, "page": 64,
         "code": "int8", "layout": "head_major", "cap": 0.0, "slopes": False, "docs": False, "norm": True,
         "by_row": False},
        # Whole ragged prompts of packed documents with capped scores; the head norm left to the program.
        {"name": "diff-prompts-docs-cap", "op": "diffchunk", "batch": 8, "low": 1, "high": 2051, "queries": 2051,
         "page": 16, "code": "e4m3", "layout": "position_major", "cap": 50.0, "slopes": False, "docs": True,
         "norm": False, "by_row": True},
        # A decode step of 33 sequences, some empty, capped scores.
        {"name": "weights-33-cap", "op": "weights", "batch": 33, "low": 0, "high": 4099, "page": 32, "code": "e4m3",
         "layout": "position_major", "cap": 30.0},
        # A decode step of the serving batch, in sequences that were evicted from before.
        {"name": "weights-64-ragged", "op": "weights", "batch": 64, "low": 512, "high": 8192, "page": 64,
         "code": "int8", "layout": "head_major", "cap": 0.0},
        # What the last 64 tokens of 8 prompts look at: the prompts are cut to a budget after it.
        {"name": "observe-8x64-16384", "op": "observe", "batch": 8, "low": 9001, "high": 16384, "queries": 64,
         "page": 64, "code": "e4m3", "layout": "head_major", "cap": 0.0, "all_new": True},
        # Every token of ragged prompts counts, capped scores.
        {"name": "observe-prompts-cap", "op": "observe", "batch": 6, "low": 1, "high": 2051, "queries": 2051,
         "page": 16, "code": "int8", "layout": "position_major", "cap": 50.0, "all_new": False},
        # A decode step of 64 requests with a budget of 1024 keys (some of half as many): one row too many each.
        {"name": "plan-step-64", "op": "plan", "requests": 64, "low": 1025, "high": 1025, "keep": 1024, "recent": 32,
         "page": 16, "room": 1040},
        # Eight long prompts are cut to 4096 keys.
        {"name": "plan-prompts-8", "op": "plan", "requests": 8, "low": 20000, "high": 32768, "keep": 4096,
         "recent": 64, "page": 64, "room": 32768},
        # A few rows a request, as after some steps or some drafted tokens.
        {"name": "evict-step-64", "op": "evict", "requests": 64, "low": 258, "high": 272, "keep": 257, "page": 64,
         "code": "int8", "layout": "position_major"},
        # The rows of eight prompts of up to 16384 that are cut to 2000.
        {"name": "evict-prompts-8", "op": "evict", "requests": 8, "low": 9001, "high": 16384, "keep": 2000, "page": 32,
         "code": "e4m3", "layout": "head_major"},
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 1))) - 0.5))))

    op = rng.choice(["diff", "diffchunk", "weights", "observe", "plan", "evict"])
    case = {"op": op, "page": rng.choice([16, 32, 64, 128])}
    if op in ("plan", "evict"):
        n = log(1, 64)
        high = log(16, min(32768, (131072 if op == "evict" else 262144) // n))
        keep = log(1, int(0.9 * high))
        case.update({"requests": n, "low": rng.choice([1, high // 2, high]), "high": high, "keep": keep})
        if op == "plan":
            return {**case, "recent": rng.choice([0, log(1, keep)]),
                    "room": -(-high // case["page"]) * case["page"]}
    case.update({"code": rng.choice(["int8", "e4m3"]), "layout": rng.choice(["head_major", "position_major"])})
    if op == "evict":
        return case
    case["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    if op in ("diff", "weights"):
        n = log(1, 128)
        high = log(1, min(131072, 262144 // n))
        case.update({"batch": n, "low": rng.choice([0, high // 8, high]), "high": high})
        if op == "weights":
            return case
    else:
        n = log(1, 48)
        queries = log(2, max(2, 4096 // n))
        high = max(queries, log(2, min(32768, 131072 // n)))
        high = max(queries, min(high, 8388608 // (n * queries)))
        case.update({"batch": n, "low": rng.choice([1, high]), "high": high, "queries": queries})
        if op == "observe":
            return {**case, "all_new": rng.random() < 0.5}
    return {**case, "slopes": rng.random() < 0.3, "docs": rng.random() < 0.3, "norm": rng.random() < 0.6,
            "by_row": rng.random() < 0.5}


def lengths(case):
    """The sequences' lengths, spread over [low, high] in no order."""
    low, high = case["low"], case["high"]
    n = case["batch"] if "batch" in case else case["requests"]
    return [low + int((high - low) * ((i * 0.6180339887 + 0.999) % 1.0) + 0.5) for i in range(n)]


def query_counts(case):
    """Queries of each sequence: one, or at most what it holds."""
    return [min(s, case["queries"]) if "queries" in case else 1 for s in lengths(case)]


def known_rows(case):
    """The rows of each sequence that had weights before the pass."""
    if case.get("all_new"):
        return [0] * case["batch"]
    return [max(0, s - n) for s, n in zip(lengths(case), query_counts(case))]


def document_rows(case):
    """Each query's first visible key, in documents of 200 to 1000 tokens; some rows of a decode step see nothing."""
    starts = []
    for b, (length, n) in enumerate(zip(lengths(case), query_counts(case))):
        edges = [0]
        while edges[-1] < length:
            edges.append(edges[-1] + 200 + (len(edges) * 389 + b * 151) % 801)
        at = 0
        for i in range(n):
            m = length - n + i
            while at + 1 < len(edges) and edges[at + 1] <= m:
                at += 1
            starts.append(length if case["op"] == "diff" and b % 11 == 5 else edges[at])
    return starts


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
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
            s = (x.abs().amax((-1, -2)) * (1.0 / CODE_MAX[code])).clamp(min=MIN_SCALE)
            c = to_codes(x * (1.0 / s)[..., None, None], code)
            parts[name].append(c if layout == "head_major" else
                               c.view(torch.uint8).transpose(1, 2).contiguous().view(c.dtype))
            parts[name + "_scale"].append(s)
    return {name: torch.cat([x.view(torch.uint8) for x in p]).view(p[0].dtype) if name in ("k", "v") else torch.cat(p)
            for name, p in parts.items()}


def to_codes(y, code):
    return (y.round().clamp(-127, 127) if code == "int8" else y.clamp(-448, 448)).to(CODE_TYPE[code])


def make_table(gen, lens, page, width=None):
    """A block table over pages in no order, and how many pages there are."""
    need = [-(-s // page) for s in lens]
    pages = max(1, sum(need))
    host = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).cpu()
    table = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = host[at:at + n]
        at += n
    return table.cuda(), pages


def cuda_ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case), "op": case["op"]}
    s.update({"slopes": None, "doc_starts": None})
    s.update({"plan": prepare_plan, "evict": prepare_evict}.get(case["op"], prepare_attention)(case, gen))
    if own:
        import attention_accelerator_b200 as gqa
        if "cache" in s:
            c = s["cache"]
            s["handle"] = gqa.PagedCache(c["k"], c["v"], c["k_scale"], c["v_scale"], layout=case["layout"])
        if "weight" in s:
            s["keys"] = gqa.KeyWeights(s["weight"], s["position"], s["evicted"])
        if case["op"] == "evict":
            s["plan"] = gqa.EvictionPlan(take=s["take"], lens=s["lens"], evicted=s["evicted"], n_free=None,
                                         counts=None)
    return s


def earlier_rows(gen, lens, room):
    """What a program has of the rows that it holds: weights, positions with gaps where rows went before, and how many did."""
    n = len(lens)
    evicted = torch.randint(0, 300, (n,), device="cuda", generator=gen).to(torch.int32)
    evicted[::3] = 0
    # Long-tailed weights, a quarter of them equal to another's, as those of keys that are hardly looked at.
    weight = 0.01 * torch.exp(2.5 * torch.randn(n, HEADS, room, device="cuda", generator=gen))
    weight = torch.where(weight < 0.002, (weight * 4000).round() / 4000, weight)
    gap = torch.randint(0, 300, (n, HEADS, 1), device="cuda", generator=gen)
    row = torch.arange(room, device="cuda")
    position = row + torch.where(row >= gap, evicted[:, None, None], 0)
    return weight, position.to(torch.int32), evicted


def prepare_attention(case, gen):
    lens, counts = lengths(case), query_counts(case)
    table, pages = make_table(gen, lens, case["page"])
    s = {"cache": make_cache(gen, pages, case["page"], case["code"], case["layout"]), "table": table,
         "lens": cuda_ints(lens), "most": max(counts)}
    rows = sum(counts)
    s["q"] = (1.5 * torch.randn(rows, HEADS * GROUP, DIM, device="cuda", generator=gen)).to(torch.bfloat16)
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    s["first"] = cuda_ints(first)
    s["slopes"] = (torch.pow(2.0, -8.0 * torch.arange(1, HEADS * GROUP + 1, device="cuda") / (HEADS * GROUP))
                   if case.get("slopes") else None)
    s["doc_starts"] = cuda_ints(document_rows(case)) if case.get("docs") else None
    if case["op"] in ("diff", "diffchunk"):
        if case["by_row"]:  # from a projection of each token
            s["lambdas"] = torch.sigmoid(torch.randn(rows, PAIRS, device="cuda", generator=gen))
        else:               # exp(a . b) - exp(c . d) + lambda_init of four learned vectors a head
            x = 0.1 * torch.randn(4, PAIRS, DIM, device="cuda", generator=gen)
            s["lambdas"] = torch.exp((x[0] * x[1]).sum(-1)) - torch.exp((x[2] * x[3]).sum(-1)) + LAMBDA_INIT
        s["norm_weight"] = 1.0 + 0.1 * torch.randn(DIM, device="cuda", generator=gen) if case["norm"] else None
    else:
        s["weight"], s["position"], s["evicted"] = earlier_rows(gen, lens, table.shape[1] * case["page"])
        s["known"] = cuda_ints(known_rows(case))
    return s


def prepare_plan(case, gen):
    lens, page, room = lengths(case), case["page"], case["room"]
    width = -(-room // page)
    table, pages = make_table(gen, lens, page, width)
    weight, position, evicted = earlier_rows(gen, lens, width * page)
    keep = torch.full((len(lens),), case["keep"], dtype=torch.int32, device="cuda")
    keep[2::5] = max(1, case["keep"] // 2)  # requests of a smaller budget
    if len(lens) > 3:
        keep[3] = 0                         # and one without any
    free = torch.full((pages + 64,), -1, dtype=torch.int32, device="cuda")
    free[:50] = pages + torch.randperm(50, device="cuda", generator=gen).to(torch.int32)
    return {"weight": weight, "position": position, "evicted": evicted, "lens": cuda_ints(lens), "keep": keep,
            "table": table, "free": free, "n_free": cuda_ints([50])}


def prepare_evict(case, gen):
    """A plan: of rows chosen at random, those at or past the budget fill the holes below it in order."""
    lens, page = lengths(case), case["page"]
    table, pages = make_table(gen, lens, page)
    room = table.shape[1] * page
    weight, position, evicted = earlier_rows(gen, lens, room)
    held = cuda_ints(lens)
    after = held.clamp(max=case["keep"])
    mark = torch.rand(len(lens), HEADS, room, device="cuda", generator=gen)
    row = torch.arange(room, device="cuda")
    take = chosen(torch.where(row < held[:, None, None], mark, -1.0), after)[..., :case["keep"]].to(torch.int32)
    take = torch.where((after < held)[:, None, None], take, -1).contiguous()
    # The rows to look at afterwards: all that stay.
    b, i = torch.nonzero(torch.arange(room)[None] < after.cpu()[:, None], as_tuple=True)
    read = table.cpu()[b, i // page].to(torch.int64) * page + i % page
    return {"cache": make_cache(gen, pages, page, case["code"], case["layout"]), "table": table, "take": take,
            "lens": after, "weight": weight, "position": position, "evicted": evicted, "read": read.cuda()}


def chosen(mark, keep):
    """take[..., i]: the row that fills row i, or -1: of each row of `mark` the `keep` highest stay (ties: the lowest),
    those at or past `keep` move into the holes below it, in order."""
    order = torch.sort(mark, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, torch.arange(mark.shape[-1], device="cuda").expand_as(order))
    k = keep[:, None, None]
    row = torch.arange(mark.shape[-1], device="cuda")
    stays, low = rank < k, row < k
    hole, mover = low & ~stays, ~low & stays
    # Row numbers of the movers, by their count; holes look up theirs.
    place = torch.where(mover, torch.cumsum(mover, -1) - 1, mark.shape[-1])
    source = torch.full((*mark.shape[:-1], mark.shape[-1] + 1), -1, device="cuda", dtype=torch.int64)
    source.scatter_(-1, place, row.expand_as(place).contiguous())
    return torch.where(hole, source.gather(-1, (torch.cumsum(hole, -1) - 1).clamp(min=0)), -1)


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
def run(state):
    return (run_own if own else run_plain)(state)


def run_own(s):
    import attention_accelerator_b200 as gqa
    case, op = s["case"], s["op"]
    if op in ("diff", "diffchunk"):
        more = {"norm_weight": s["norm_weight"], "norm_eps": NORM_EPS, "out_scale": 1.0 - LAMBDA_INIT,
                "score_cap": case["cap"] or None, "distance_slopes": s["slopes"], "doc_starts": s["doc_starts"],
                "rope_theta": THETA}
        if op == "diff":
            return gqa.decode_paged_diff(s["q"], s["handle"], s["table"], s["lens"], s["lambdas"], **more)
        return gqa.decode_paged_diff_chunked(s["q"], s["handle"], s["table"], s["lens"], s["first"], s["lambdas"], **more)
    if op == "weights":
        out = gqa.decode_paged_weights(s["q"], s["handle"], s["table"], s["lens"], s["keys"],
                                       score_cap=case["cap"] or None, rope_theta=THETA)
        return {"out": out, "weight": s["weight"], "position": s["position"], "evicted": s["evicted"]}
    if op == "observe":
        gqa.add_key_weights(s["q"], s["handle"], s["table"], s["lens"], s["first"], s["keys"],
                            known=s["known"] if case["all_new"] else None, score_cap=case["cap"] or None,
                            rope_theta=THETA)
        return {"weight": s["weight"], "position": s["position"], "evicted": s["evicted"]}
    if op == "plan":
        p = gqa.plan_eviction(s["keys"], s["lens"], s["keep"], s["table"], s["free"], s["n_free"],
                              page_len=case["page"], max_keep=case["keep"], sinks=SINKS, recent=case["recent"])
        return {"take": p.take, "lens": p.lens, "evicted": p.evicted, "free": s["free"], "n_free": p.n_free,
                "counts": p.counts}
    gqa.evict_paged(s["handle"], s["table"], s["keys"], s["plan"])
    k, v = gqa.read_paged(s["handle"], s["read"])
    return {"k": k, "v": v, "k_scale": s["cache"]["k_scale"], "v_scale": s["cache"]["v_scale"], "weight": s["weight"],
            "position": s["position"]}


def run_plain(s):
    return {"diff": plain_diff, "diffchunk": plain_diff, "weights": plain_weights, "observe": plain_weights,
            "plan": plain_plan, "evict": plain_evict}[s["op"]](s)


def rotate(x, positions):
    """RoPE of rows [n, heads, DIM] at their positions: the angles in 64 bits, the rest in 32."""
    turn = torch.pow(THETA, -torch.arange(DIM // 2, device="cuda", dtype=torch.float64) / (DIM // 2))
    angle = positions.double()[:, None, None] * turn
    a, b = x.float().split(DIM // 2, -1)
    c, d = angle.cos().float(), angle.sin().float()
    return torch.cat([a * c - b * d, a * d + b * c], -1)


def dense(s, name):
    """K or V of every sequence side by side, [batch, heads, keys, DIM]."""
    table = s["table"].clamp(min=0).long()
    x = s["cache"][name].view(torch.uint8)[table].view(s["cache"][name].dtype).float()
    if s["case"]["layout"] == "head_major":
        x = x.transpose(2, 3)
    x = x * s["cache"][name + "_scale"][table][:, :, None, :, None]
    return x.reshape(table.shape[0], -1, HEADS, DIM).transpose(1, 2)


def plain_map(s, shift=None):
    """The softmax maps [batch, HEADS, GROUP, most, keys], the sequences' queries side by side, and which query rows these
    are; `shift`: what the queries' positions are ahead of their rows."""
    case, lens, first = s["case"], s["lens"], s["first"]
    batch, keys = s["table"].shape[0], s["table"].shape[1] * case["page"]
    i = torch.arange(s["most"], device="cuda")[None]
    count = (first[1:] - first[:-1])[:, None]
    real = i < count
    at = lens[:, None] - count + i                          # the row that each query's token has
    row = (first[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = rotate(s["q"], (at if shift is None else at + shift[:, None])[real])[row]
    q = q.reshape(batch, s["most"], HEADS, GROUP, DIM).permute(0, 2, 3, 1, 4).reshape(batch, HEADS, -1, DIM)
    z = (q @ dense(s, "k").transpose(-1, -2) * SCALE).reshape(batch, HEADS, GROUP, s["most"], keys)
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    key = torch.arange(keys, device="cuda")
    if s["slopes"] is not None:
        z = z - s["slopes"].reshape(HEADS, GROUP, 1, 1) * (at[..., None] - key).abs().float()[:, None, None]
    start = s["doc_starts"][row] if s["doc_starts"] is not None else torch.zeros_like(at)
    seen = (key >= start[..., None]) & (key < torch.minimum(at + 1, lens[:, None])[..., None])
    z = torch.where((seen & real[..., None])[:, None, None], z, -math.inf)
    top = z.amax(-1, keepdim=True)
    w = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    return w / torch.where(total > 0, total, 1.0), real, row


def values(s, w):
    """The maps [batch, HEADS, each, most, keys] times V: [batch, most, HEADS * each, DIM]."""
    batch, _, each, most, keys = w.shape
    key = torch.arange(keys, device="cuda")
    v = torch.where((key < s["lens"][:, None])[:, None, :, None], dense(s, "v"), 0.0)
    o = (w.reshape(batch, HEADS, -1, keys) @ v).reshape(batch, HEADS, each, most, DIM)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most, HEADS * each, DIM)


def plain_diff(s):
    w, real, row = plain_map(s)
    lam = s["lambdas"][row] if s["case"]["by_row"] else s["lambdas"].expand(*row.shape, PAIRS)
    w = w.unflatten(2, (GROUP // 2, 2))
    by_head = lam.unflatten(-1, (HEADS, GROUP // 2)).permute(0, 2, 3, 1)[..., None]
    o = values(s, w[:, :, :, 0] - by_head * w[:, :, :, 1])
    if s["norm_weight"] is not None:
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + NORM_EPS) * s["norm_weight"]
    return (o * (1.0 - LAMBDA_INIT))[real].to(torch.bfloat16)


def plain_weights(s):
    lens, known = s["lens"], s["known"]
    # A sequence that had no rows before is a new one: nothing was evicted from it.
    s["evicted"].copy_(torch.where((known == 0) & (lens > 0), 0, s["evicted"]))
    w, real, _ = plain_map(s, s["evicted"])
    key = torch.arange(w.shape[-1], device="cuda")
    held = (key < lens[:, None])[:, None]
    fresh = held & (key >= known[:, None])[:, None]
    seen = torch.where(fresh, 0.0, s["weight"]) + w.sum((2, 3))
    s["weight"].copy_(torch.where(held, seen, s["weight"]))
    s["position"].copy_(torch.where(fresh, key + s["evicted"][:, None, None], s["position"]))
    state = {"weight": s["weight"], "position": s["position"], "evicted": s["evicted"]}
    if s["op"] == "observe":
        return state
    return {"out": values(s, w)[real].to(torch.bfloat16), **state}


def plain_plan(s):
    case, lens, table, page = s["case"], s["lens"], s["table"], s["case"]["page"]
    keep = s["keep"].clamp(max=case["keep"])
    cut = (keep > 0) & (keep < lens)
    after = torch.where(cut, keep, lens)
    row = torch.arange(s["weight"].shape[-1], device="cuda")
    tokens = (lens + s["evicted"])[:, None, None]
    safe = (s["position"] < SINKS) | (s["position"] >= tokens - case["recent"])
    # Weights are not negative: their bits order as whole numbers, rows to be spared above all others.
    mark = s["weight"].view(torch.int32).long() + (safe.long() << 32)
    mark = torch.where(row < lens[:, None, None], mark, -1)
    take = torch.where(cut[:, None, None], chosen(mark, after), -1)
    if take.shape[-1] < case["keep"]:
        take = torch.nn.functional.pad(take, (0, case["keep"] - take.shape[-1]), value=-1)
    # Pages past the new length go on top of the free stack, in the order of requests and columns.
    held, stay = (lens + page - 1) // page, (after + page - 1) // page
    give = held - stay
    column = torch.arange(table.shape[1], device="cuda")[None]
    gone = (column >= stay[:, None]) & (column < held[:, None])
    place = s["n_free"] + (torch.cumsum(give, 0) - give)[:, None] + column - stay[:, None]
    stack = torch.cat([s["free"], s["free"][:1]])
    stack.scatter_(0, torch.where(gone, place, s["free"].numel()).reshape(-1), table.reshape(-1))
    s["free"].copy_(stack[:-1])
    whole = torch.int32
    counts = torch.stack([cut.sum(), (lens - after).sum(), give.sum(), torch.zeros_like(give[0])])
    return {"take": take[..., :case["keep"]].to(whole), "lens": after.to(whole),
            "evicted": (s["evicted"] + lens - after).to(whole), "free": s["free"],
            "n_free": (s["n_free"] + give.sum()).to(whole), "counts": counts.to(whole)}


def plain_evict(s):
    case, cache, take, table = s["case"], s["cache"], s["take"], s["table"].long()
    page, top = case["page"], CODE_MAX[case["code"]]
    b, h, to = torch.nonzero(take >= 0, as_tuple=True)
    source = take[b, h, to].long()
    page_to, row_to = table[b, to // page], to % page
    page_from, row_from = table[b, source // page], source % page
    out = {}
    for name in ("k", "v"):
        codes, old = cache[name], cache[name + "_scale"]
        # By (page, head, row), a view.
        at = codes.view(torch.uint8)
        at = at if case["layout"] == "head_major" else at.transpose(1, 2)
        x = at[page_from, h, row_from].view(codes.dtype).float() * old[page_from, h][:, None]
        most = torch.zeros_like(old).view(-1).scatter_reduce_(0, page_to * HEADS + h, x.abs().amax(-1), "amax")
        moved = torch.zeros_like(old, dtype=torch.bool)
        moved[page_to, h] = True
        scale = torch.where(moved, torch.maximum(old, (most.view_as(old) / top).clamp(min=MIN_SCALE)), old)
        # The other rows of a block whose scale grew are rounded again.
        p, g = torch.nonzero(scale > old, as_tuple=True)
        again = at[p, g].view(codes.dtype).float() * old[p, g][:, None, None] * (1.0 / scale[p, g])[:, None, None]
        at[p, g] = to_codes(again, case["code"]).view(torch.uint8)
        at[page_to, h, row_to] = to_codes(x * (1.0 / scale[page_to, h])[:, None], case["code"]).view(torch.uint8)
        old.copy_(scale)
        p, r = s["read"] // page, s["read"] % page
        rows = at.transpose(1, 2)[p, r].view(codes.dtype).float()
        out[name] = (rows * scale[p][..., None]).to(torch.bfloat16)
        out[name + "_scale"] = old
    for name in ("weight", "position"):
        s[name][b, h, to] = s[name][b, h, source]
        out[name] = s[name]
    return out


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    row, op = HEADS * DIM, case["op"]
    if op == "plan":
        held = sum(lengths(case))
        # A row's weight and position, and where each row that stays comes from.
        return {"bytes": HEADS * (8 * held + 4 * case["keep"] * case["requests"]) + 16 * case["requests"],
                "flops": HEADS * held}
    if op == "evict":
        # What moves, where the choice is spread evenly: codes out and in, weights and positions, and the plan.  Then the
        # codes of all that stay in, and BF16 out.
        stay = [(n, min(n, case["keep"])) for n in lengths(case)]
        moved = sum(c * (n - c) / n for n, c in stay)
        return {"bytes": HEADS * (moved * (4 * DIM + 16) + 4 * case["keep"] * case["requests"])
                + 6 * row * sum(c for _, c in stay), "flops": 4 * row * moved + 2 * row * sum(c for _, c in stay)}
    lens, counts = lengths(case), query_counts(case)
    starts = document_rows(case) if case.get("docs") else None
    pairs = keys = at = 0
    for length, n in zip(lens, counts):
        low = length
        for i in range(n):
            lo, hi = (starts[at] if starts else 0), max(0, min(length, length - n + i + 1))
            at += 1
            pairs += max(0, hi - lo)
            low = min(low, lo)
        keys += length - low
    scales = 2 * 4 * HEADS * (keys // case["page"] + len(lens))
    queries = 2 * sum(counts) * row * GROUP
    product = 2 * DIM * HEADS * GROUP * pairs
    if op == "observe":
        known = sum(known_rows(case))
        return {"bytes": keys * row + scales // 2 + queries + 4 * HEADS * (2 * keys + (keys - known)), "flops": product}
    if op == "weights":
        return {"bytes": 2 * keys * row + scales + 2 * queries + 8 * HEADS * keys, "flops": 2 * product}
    lambdas = 4 * PAIRS * (sum(counts) if case["by_row"] else 1)
    return {"bytes": 2 * keys * row + scales + queries + queries // 2 + lambdas, "flops": 2 * product}


# ----------------------------------------------------------------------------------------------------------------------
# the same in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "evict":
        return exact_evict(s)
    if sum(n * m for n, m in zip(lengths(case), query_counts(case))) > 1 << 25:
        return None
    return exact_diff(s) if case["op"] in ("diff", "diffchunk") else exact_weights(s)


def turned(x, position):
    """Rows [n, heads, DIM] as complex pairs turned by their positions, in 64 bits."""
    x = x.double()
    z = torch.complex(x[..., :DIM // 2], x[..., DIM // 2:])
    angle = torch.tensor([THETA ** (-2.0 * j / DIM) for j in range(DIM // 2)], dtype=torch.float64, device="cuda")
    z = z * torch.exp(1j * position.double()[:, None, None] * angle)
    return torch.cat([z.real, z.imag], -1)


def exact_maps(s, b, shift):
    """(head, its softmax map [n, length], V) of each Q head of sequence b."""
    case, cache, page = s["case"], s["cache"], s["case"]["page"]
    first, length = s["first"].tolist(), int(s["lens"][b])
    n = first[b + 1] - first[b]
    m = torch.arange(length - n, length, device="cuda")
    q = turned(s["q"][first[b]:first[b + 1]], m + shift)
    p = torch.arange(length, device="cuda")
    block = s["table"][b].long()[p // page]
    hidden = p[None] > m[:, None]
    if s["doc_starts"] is not None:
        hidden = hidden | (p[None] < s["doc_starts"][first[b]:first[b + 1]].long()[:, None])
    for h in range(HEADS):
        part = {}
        for name in ("k", "v"):
            c = cache[name] if case["layout"] == "position_major" else cache[name].transpose(1, 2)
            c = c.view(torch.uint8)[block, p % page, h].view(cache[name].dtype).float().double()
            part[name] = c * cache[name + "_scale"][block, h].double()[:, None]
        for g in range(GROUP):
            z = q[:, h * GROUP + g] @ part["k"].T / math.sqrt(DIM)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if s["slopes"] is not None:
                z = z - float(s["slopes"][h * GROUP + g]) * (m[:, None] - p[None]).abs()
            z.masked_fill_(hidden, -math.inf)
            yield h * GROUP + g, torch.exp(z - torch.logsumexp(z, -1, keepdim=True)).nan_to_num_(nan=0.0), part["v"]


def exact_diff(s):
    first, rows = s["first"].tolist(), s["q"].shape[0]
    out = torch.zeros(rows, PAIRS, DIM, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        here = slice(first[b], first[b + 1])
        for head, w, v in exact_maps(s, b, 0):
            if head % 2 == 0:
                out[here, head // 2] = w @ v
                continue
            lam = s["lambdas"][here, head // 2] if s["case"]["by_row"] else s["lambdas"][head // 2].expand(w.shape[0])
            out[here, head // 2] -= lam.double()[:, None] * (w @ v)
    if s["norm_weight"] is not None:
        out = out / torch.sqrt((out * out).mean(-1, keepdim=True) + NORM_EPS) * s["norm_weight"].double()
    return out * (1.0 - LAMBDA_INIT)


def exact_weights(s):
    first, rows = s["first"].tolist(), s["q"].shape[0]
    out = torch.zeros(rows, HEADS * GROUP, DIM, dtype=torch.float64, device="cuda")
    weight = s["weight"].double()
    for b, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        known = int(s["known"][b])
        weight[b, :, known:length] = 0.0
        for head, w, v in exact_maps(s, b, int(s["evicted"][b]) if known > 0 else 0):
            weight[b, head // GROUP, :length] += w.sum(0)
            out[first[b]:first[b + 1], head] = w @ v
    state = {"weight": weight, "position": None, "evicted": None}
    return state if s["op"] == "observe" else {"out": out, **state}


def code_value(y, code):
    if code == "int8":
        return torch.round(y).clamp(-127, 127)
    return y.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()


def exact_evict(s):
    case, cache, take, table = s["case"], s["cache"], s["take"], s["table"]
    page, code = case["page"], case["code"]
    out = {}
    where = torch.nonzero((take >= 0).any(1).cpu()).tolist()
    blocks = sorted({(b, i // page) for b, i in where})
    for name in ("k", "v"):
        codes = cache[name].float().double()
        codes = codes.transpose(1, 2) if case["layout"] == "position_major" else codes  # [pages, heads, rows, DIM]
        before, codes = codes, codes.clone()
        scale = cache[name + "_scale"].double()
        held = scale.clone()
        for b, column in blocks:
            to = int(table[b, column])
            source = take[b, :, column * page:(column + 1) * page].long()  # [heads, rows of this page]
            n = source.shape[1]
            moves = source >= 0
            from_page = table[b].long()[source.clamp(min=0) // page]
            head = torch.arange(HEADS, device="cuda")[:, None].expand(-1, n)
            x = before[from_page, head, source.clamp(min=0) % page] * held[from_page, head][..., None]
            most = torch.where(moves[..., None], x.abs(), 0.0).amax((1, 2)) / CODE_MAX[code]
            now = torch.maximum(held[to], most.clamp(min=MIN_SCALE)).float().double()
            now = torch.where(moves.any(1), now, held[to])
            grew = (now > held[to])[:, None, None]
            codes[to] = torch.where(grew, code_value(codes[to] * (held[to] / now)[:, None, None], code), codes[to])
            codes[to, :, :n] = torch.where(moves[..., None], code_value(x / now[:, None, None], code), codes[to, :, :n])
            scale[to] = now
        p, r = s["read"] // page, s["read"] % page
        out[name] = codes.transpose(1, 2)[p, r] * scale[p][..., None]
        out[name + "_scale"] = scale
    b, h, to = torch.nonzero(take >= 0, as_tuple=True)
    weight = s["weight"].double()
    weight[b, h, to] = s["weight"][b, h, take[b, h, to].long()].double()
    return {**out, "weight": weight, "position": None}
