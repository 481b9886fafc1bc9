"""What a serving loop does around a model's matrices, as cases that can be timed: bookkeeping of cache pages, query and key
heads on their way into the cache, attention over the cache, and the choice of the next token.

`listed()` names the cases, `draw(rng)` gives another one of the same ranges, `prepare(case, seed)` makes what a program holds
before the call, `run(state)` is one pass through an operator, `work(case)` says what a pass cannot do without, and
`exact(case, seed)` is the operator's definition in 64 bits.  `run` computes the plain form (elementary torch operations in 32
bits, in 64 where a border decides) unless `own` is set; then it makes the calls a user of this library makes.

Operators:

* plan    `paged.PagePool.plan`: block tables and slot maps from request lengths.  Pages come from a stack of free ones.
* heads   `paged.enter` / `paged.rotate`: norm of every query and key head, rotation, and the write into the paged cache.
* attend  `paged.attend`: causal attention of ragged queries over a paged cache of 16 or 4 bits, with a sliding window and
          first tokens that stay visible.
* sample  `sampling.sample`: temperature, top-k, top-p and min-p, from given uniform numbers.

A cache of 4 bits holds groups of 64 values of a head as codes 0 .. 15 with a scale and a lowest value in bf16
(value = low + scale * code).  The eight codes of 8 consecutive values share a 32-bit word, the first in the lowest bits; a
row of `dim` codes is stored as [8][dim / 64] words, word (i, g) holding values 64 g + 8 i .. 64 g + 8 i + 7.
"""

import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
GROUP = 64

# heads of the models this library runs: query heads, KV heads, head dim, rotated dims
HEADS = {"0.8b": (8, 2, 256, 64), "27b": (24, 4, 256, 64), "35b": (16, 2, 256, 64), "26b": (16, 8, 256, 256)}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the step of a full batch of the large engines: eight requests, one token each
        {"name": "plan, 8 requests", "op": "plan", "requests": 8, "page": 64, "max_pages": 64, "room": 8, "prompts": 0.0, "ended": 0.0},
        # a serving step of many users: most decode, some bring prompts, some have ended or were cut back
        {"name": "plan, 1000 requests, prompts among them", "op": "plan", "requests": 1000, "page": 32, "max_pages": 512, "room": 16384, "prompts": 0.1, "ended": 0.1},
        # decoding: the heads of eight tokens of the 27B model enter a 4-bit cache, straight from the projection's fp32 row
        {"name": "heads, 8 tokens, 27b, 4 bits", "op": "heads", "heads": "27b", "tokens": 8, "source": "fp32", "cache": "int4", "type": "bf16", "gated": True, "page": 64},
        # a prompt's heads of the 26B model (plain norm weights, all dims rotated) enter a bf16 cache
        {"name": "heads, 4000 tokens, 26b, bf16 cache", "op": "heads", "heads": "26b", "tokens": 4000, "source": "bf16", "cache": "bf16", "type": "bf16", "gated": False, "page": 64},
        # a prompt's heads of the 35B model enter a 4-bit cache
        {"name": "heads, 2048 tokens, 35b, 4 bits", "op": "heads", "heads": "35b", "tokens": 2048, "source": "bf16", "cache": "int4", "type": "bf16", "gated": True, "page": 64},
        # one user of the small model in the middle of a reply: latency
        {"name": "attend, 1 x 700, 0.8b, bf16 cache", "op": "attend", "heads": "0.8b", "cache": "bf16", "type": "bf16", "requests": 1, "context": 700, "new": 1, "window": 0, "sinks": 0, "page": 64, "ragged": False},
        # a full batch of the 27B model at long contexts, which a 4-bit cache is for
        {"name": "attend, 8 x 32000, 27b, 4 bits", "op": "attend", "heads": "27b", "cache": "int4", "type": "bf16", "requests": 8, "context": 32000, "new": 1, "window": 0, "sinks": 0, "page": 64, "ragged": True},
        # many users of a sliding-window layer of the 26B model, the first tokens kept visible
        {"name": "attend, 48 x 6000, 26b, window 1024 + 4", "op": "attend", "heads": "26b", "cache": "bf16", "type": "bf16", "requests": 48, "context": 6000, "new": 1, "window": 1024, "sinks": 4, "page": 32, "ragged": True},
        # two prompts continue behind contexts held in 4 bits
        {"name": "attend, 2 x 1500 of 4000, 27b, 4 bits", "op": "attend", "heads": "27b", "cache": "int4", "type": "bf16", "requests": 2, "context": 4000, "new": 1500, "window": 0, "sinks": 0, "page": 64, "ragged": True},
        # a long prompt through a sliding-window layer
        {"name": "attend, prompt of 8192, 26b, window 1024 + 4", "op": "attend", "heads": "26b", "cache": "bf16", "type": "bf16", "requests": 1, "context": 8192, "new": 8192, "window": 1024, "sinks": 4, "page": 64, "ragged": False},
        # one user's next token of the small model
        {"name": "sample, 1 x 151936", "op": "sample", "rows": 1, "vocab": 151936, "type": "fp32", "mixed": False, "top_k": 20, "top_p": 0.95, "min_p": 0.0, "temperature": 0.6},
        # the next tokens of many users, each with settings of their own
        {"name": "sample, 64 x 248320, mixed", "op": "sample", "rows": 64, "vocab": 248320, "type": "fp32", "mixed": True, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["plan", "heads", "attend", "attend", "sample"])
    if op == "plan":
        requests = _log(rng, 1, 2000)
        return {"op": op, "requests": requests, "page": rng.choice([16, 32, 64, 128]), "max_pages": _log(rng, 8, 512), "room": _log(rng, requests, 16384),
                "prompts": rng.choice([0.0, 0.02, 0.1]), "ended": rng.choice([0.0, 0.05, 0.2])}
    heads = rng.choice(sorted(HEADS))
    if op == "heads":
        return {"op": op, "heads": heads, "tokens": _log(rng, 1, 4000), "source": rng.choice(["fp32", "bf16", "fp16"]), "cache": rng.choice(["int4", "int4", "bf16", "fp16", "none"]),
                "type": "bf16", "gated": heads != "26b", "page": rng.choice([16, 32, 64, 128])}
    if op == "attend":
        kind = rng.choice(["bf16", "fp16", "int4", "int4"])
        c = {"op": op, "heads": heads, "cache": kind, "type": kind if kind != "int4" else rng.choice(["bf16", "fp16"]), "page": rng.choice([16, 32, 64, 128])}
        window = rng.choice([0, 0, _log(rng, 64, 4096)])
        c.update(window=window, sinks=rng.choice([0, 1, 4, 16, 100]) if window else 0, ragged=rng.random() < 0.7)
        if rng.random() < 0.6:
            requests = _log(rng, 1, 64)
            c.update(requests=requests, context=_log(rng, 16, min(32000, 256000 // requests)), new=rng.choice([1, 1, 1, 2, 4]))
        else:
            requests = _log(rng, 1, 4)
            context = _log(rng, 100, 4000 // (1 if requests == 1 else 2))
            c.update(requests=requests, context=context, new=_log(rng, 9, context))
        return c
    return {"op": op, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 262144), "type": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "mixed": rng.random() < 0.5,
            "top_k": rng.choice([0, 1, 20, 50, 1000]), "top_p": rng.choice([1.0, 0.99, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
            "temperature": rng.choice([0.0, 0.3, 0.6, 0.7, 1.0, 1.0, 1.5])}


# ---------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _uniform(g, n):
    return torch.rand(n, generator=g, device=DEVICE)


def _whole(g, n, lo, hi):
    """n whole numbers of lo .. hi."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32)


def prepare(case, seed):
    return {"plan": _plan_state, "heads": _heads_state, "attend": _attend_state, "sample": _sample_state}[case["op"]](case, _gen(seed))


def _plan_state(c, g):
    """Requests in flight with the pages of their tokens; some bring a prompt, some have ended (length 0, nothing new), some were
    cut back behind rejected drafts.  The pool is large enough for nearly all of them."""
    R, page, P, room = c["requests"], c["page"], c["max_pages"], c["room"]
    longest = page * P
    had = (torch.exp(_uniform(g, R) * math.log(max(2, longest - 8))).int()).clamp(1, longest - 8 if longest > 16 else 1)
    held = (had + page - 1) // page
    kind = _uniform(g, R)
    prompt = torch.minimum(_whole(g, R, 2, max(2, 4 * room // max(1, R))), (longest - had).clamp(min=0))
    length = torch.where(kind < c["ended"], torch.zeros_like(had), had)
    new = torch.where(kind < c["ended"], torch.zeros_like(had), torch.where(kind > 1 - c["prompts"], prompt, torch.ones_like(had)))
    length = torch.where((kind > 0.5) & (kind < 0.55), (length - 3).clamp(min=0), length)
    total = int(held.sum())
    pages = 1 + R * P                                          # page 0 is the null page; most of the others serve elsewhere
    spare = min(pages - 1 - total, R + room // page + 8)
    order = (torch.randperm(pages - 1, generator=g, device=DEVICE) + 1).int()
    col = torch.arange(P, device=DEVICE)
    first = torch.cumsum(held, 0) - held
    at = first[:, None] + col[None]
    live = col[None] < held[:, None]
    table = torch.where(live, order[at.clamp(max=pages - 2).long()], torch.zeros((), dtype=torch.int32, device=DEVICE)).int()
    free = torch.zeros(pages - 1, dtype=torch.int32, device=DEVICE)
    free[:spare] = order[total: total + spare]
    return {"op": "plan", "page": page, "room": room, "pages": pages, "lengths": length.int(), "new": new.int(), "table": table, "held": held.int(), "free": free,
            "n_free": torch.tensor([spare], dtype=torch.int32, device=DEVICE)}


def _angles(g, longest, pairs):
    inv = 1e6 ** (-torch.arange(pairs, dtype=torch.float64, device=DEVICE) / pairs)
    a = torch.arange(longest, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _heads_state(c, g):
    """One row per token as a projection leaves it: query heads (each with its gate where the model has one), keys, values."""
    nq, nkv, dim, rot = HEADS[c["heads"]]
    T, page = c["tokens"], c["page"]
    qs = 2 * dim if c["gated"] else dim
    width = nq * qs + 2 * nkv * dim
    y = torch.randn(T, width, generator=g, device=DEVICE) * (0.5 + 2 * _uniform(g, T)[:, None])
    y = y.to(TYPES[c["source"]])
    longest = 8192
    cos, sin = _angles(g, longest, rot // 2)
    pages = 1 + -(-T // page) + 4
    start = int(_whole(g, 1, 0, longest - T))
    at = torch.arange(T, device=DEVICE)
    order = (torch.randperm(pages - 1, generator=g, device=DEVICE) + 1)
    slots = (order[at // page] * page + at % page).int()
    if T > 4:
        slots[T - 1] = -1                                      # a padding row
    s = {"op": "heads", "heads": (nq, nkv, dim, rot), "page": page, "cache": c["cache"], "type": TYPES[c["type"]],
         "q": y[:, : nq * qs].view(T, nq, qs)[..., :dim], "k": y[:, nq * qs: nq * qs + nkv * dim].view(T, nkv, dim), "v": y[:, nq * qs + nkv * dim:].view(T, nkv, dim),
         "positions": (start + at).int(), "slots": slots, "cos": cos, "sin": sin, "offset": 1.0 if c["gated"] else 0.0,
         "q_norm": torch.randn(dim, generator=g, device=DEVICE) * 0.1 + (0.0 if c["gated"] else 1.0),
         "k_norm": torch.randn(dim, generator=g, device=DEVICE) * 0.1 + (0.0 if c["gated"] else 1.0)}
    if c["cache"] == "int4":
        for n in "kv":
            s[n + "_codes"] = torch.zeros(pages, nkv, page, dim // 2, dtype=torch.uint8, device=DEVICE)
            s[n + "_scales"] = torch.zeros(pages, nkv, page, dim // GROUP, 2, dtype=torch.bfloat16, device=DEVICE)
    elif c["cache"] != "none":
        for n in "kv":
            s[n + "_cache"] = torch.zeros(pages, nkv, page, dim, dtype=TYPES[c["cache"]], device=DEVICE)
        s["type"] = TYPES[c["cache"]]
    return s


def _attend_state(c, g):
    nq, nkv, dim, _ = HEADS[c["heads"]]
    R, page, dtype = c["requests"], c["page"], TYPES[c["type"]]
    full, new = c["context"], c["new"]
    lo = max(new if new <= 4 else 2, full // 3)
    lengths = _gen(R + full)                                   # a case's lengths, the same for every seed
    context = _whole(lengths, R, min(lo, full), full) if c["ragged"] else torch.full((R,), full, dtype=torch.int32, device=DEVICE)
    context[0] = full
    fresh = torch.full((R,), new, dtype=torch.int32, device=DEVICE)
    if new > 4 and c["ragged"]:
        fresh[1:] = torch.minimum(_whole(lengths, R, 1, new), context)[1:]
    fresh = torch.minimum(fresh, context)
    P = -(-full // page)
    pages = 1 + int(((context + page - 1) // page).sum())
    order = (torch.randperm(pages - 1, generator=g, device=DEVICE) + 1).int()
    held = (context + page - 1) // page
    col = torch.arange(P, device=DEVICE)
    at = (torch.cumsum(held, 0) - held)[:, None] + col[None]
    table = torch.where(col[None] < held[:, None], order[at.clamp(max=pages - 2).long()], torch.zeros((), dtype=torch.int32, device=DEVICE)).int()
    counts = fresh.tolist()
    starts = torch.zeros(R + 1, dtype=torch.int32, device=DEVICE)
    starts[1:] = torch.cumsum(fresh, 0)
    T = sum(counts)
    s = {"op": "attend", "heads": (nq, nkv, dim), "page": page, "cache": c["cache"], "type": dtype, "window": c["window"], "sinks": c["sinks"], "new": max(counts),
         "q": (torch.randn(T, nq, dim, generator=g, device=DEVICE) * 1.5).to(dtype), "table": table, "context": context.int(), "starts": starts, "scale": dim ** -0.5}
    if c["cache"] == "int4":
        for n in "kv":
            s[n + "_codes"] = torch.randint(0, 256, (pages, nkv, page, dim // 2), generator=g, device=DEVICE, dtype=torch.uint8)
            spread = 2.5 + torch.rand(pages, nkv, page, dim // GROUP, generator=g, device=DEVICE)
            s[n + "_scales"] = torch.stack([spread * (2 / 15), -spread + 0.2 * torch.randn(spread.shape, generator=g, device=DEVICE)], -1).to(torch.bfloat16)
    else:
        for n in "kv":
            s[n + "_cache"] = torch.randn(pages, nkv, page, dim, generator=g, device=DEVICE).to(dtype)
    return s


def _sample_state(c, g):
    """Logits as a language model gives them: a broad floor, and a few hundred candidates above it."""
    B, V = c["rows"], c["vocab"]
    x = torch.randn(B, V, generator=g, device=DEVICE) * 1.7
    raised = torch.rand(B, V, generator=g, device=DEVICE) * V < 300
    x = torch.where(raised, 3 + 9 * torch.rand(B, V, generator=g, device=DEVICE) ** 2, x)
    pick = lambda *v: torch.tensor(v, device=DEVICE)[torch.randint(0, len(v), (B,), generator=g, device=DEVICE)]      # noqa: E731
    if c["mixed"]:
        t, k, p, m = pick(0.0, 0.6, 0.7, 1.0, 1.0, 1.3), pick(0, 0, 1, 20, 50, 1000), pick(1.0, 1.0, 0.95, 0.9, 0.8), pick(0.0, 0.0, 0.05)
    else:
        t, k, p, m = (torch.full((B,), v, device=DEVICE) for v in (c["temperature"], c["top_k"], c["top_p"], c["min_p"]))
    return {"op": "sample", "logits": x.to(TYPES[c["type"]]), "u": _uniform(g, B), "temperature": t.float(), "top_k": k.int(), "top_p": p.float(), "min_p": m.float()}


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"plan": _plan_own, "heads": _heads_own, "attend": _attend_own, "sample": _sample_own}[state["op"]](state)
    return {"plan": _plan, "heads": _heads, "attend": _attend, "sample": _sample}[state["op"]](state)


def _plan_own(s):
    from megakernels_b200 import paged
    if "pool" not in s:                                        # the pool a program keeps, in the state that the requests left it in
        pool = s["pool"] = paged.PagePool(requests=s["table"].shape[0], pages=s["pages"], max_pages=s["table"].shape[1], page=s["page"], max_tokens=s["room"], device=DEVICE)
        pool.table.copy_(s["table"]), pool.held.copy_(s["held"]), pool.free.copy_(s["free"]), pool.n_free.copy_(s["n_free"])
    pool = s["pool"]
    p = pool.plan(s["lengths"], s["new"])
    return {"table": p.table, "slots": p.slots, "positions": p.positions, "rows": p.rows, "starts": p.starts, "context": p.context, "granted": p.granted,
            "held": pool.held, "free": pool.free, "n_free": pool.n_free}


def _plan(s):
    """In request order: what a request holds beyond its first `lengths` tokens goes back on the stack of free pages, then
    pages for its new tokens come from the top.  The first request that does not fit, and all behind it, wait."""
    page, room, table, held, free = s["page"], s["room"], s["table"], s["held"], s["free"]
    R, P = table.shape
    length, new = s["lengths"], s["new"]
    need = (length + new + page - 1) // page
    valid = need <= P
    base = torch.minimum(held, (length + page - 1) // page)
    back = held - base
    take = torch.where(valid, need - base, 0)
    tokens = torch.where(valid, new, 0)
    col = torch.arange(P, device=DEVICE)
    # returned pages, the first request's on top
    n, returned = s["n_free"], back.sum()
    above = torch.cumsum(back, 0) - back
    gone = (col[None] >= base[:, None]) & (col[None] < held[:, None])
    to = torch.where(gone, n + returned - 1 - (above[:, None] + col[None] - base[:, None]), free.numel())
    wide = torch.cat([free, free.new_zeros(1)])
    wide.scatter_(0, to.flatten().long(), table.flatten())
    free.copy_(wide[:-1])
    # pages taken
    have = n + returned
    taken = torch.cumsum(take, 0)
    fits = (taken <= have) & (torch.cumsum(tokens, 0) <= room)
    granted = valid & (fits | ((take == 0) & (tokens == 0)))
    take, tokens = torch.where(granted, take, 0), torch.where(granted, tokens, 0)
    holds = torch.where(granted, need, base)
    j = col[None] - base[:, None]
    from_top = (have - 1 - ((taken - take)[:, None] + j)).clamp(0, free.numel() - 1)
    table.copy_(torch.where(col[None] < base[:, None], table, torch.where(col[None] < holds[:, None], free[from_top.long()], 0)))
    held.copy_(holds)
    n.copy_(have - take.sum())
    # the new tokens, one after the other
    starts = torch.zeros(R + 1, dtype=torch.int32, device=DEVICE)
    starts[1:] = torch.cumsum(tokens, 0)
    at = torch.arange(room, device=DEVICE)
    live = at < starts[R]
    row = torch.where(live, torch.searchsorted(starts[1:].contiguous(), at, right=True), 0).clamp(max=R - 1)
    position = torch.where(live, length[row] + at - starts[row], 0)
    slot = torch.where(live, table[row, (position // page).long()] * page + position % page, -1)
    return {"table": table, "slots": slot.int(), "positions": position.int(), "rows": torch.where(live, row, -1).int(), "starts": starts,
            "context": torch.where(granted, length + new, torch.where(valid, length, 0)).int(), "granted": granted.int(), "held": held, "free": free, "n_free": n}


def _cache(s):
    """The cache object a program keeps."""
    from megakernels_b200 import paged
    if "handle" not in s:
        if s["cache"] == "int4":
            s["handle"] = paged.Cache.of_codes(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
        else:
            s["handle"] = paged.Cache.of(s["k_cache"], s["v_cache"])
    return s["handle"]


def _heads_own(s):
    from megakernels_b200 import paged
    kw = dict(rope=(s["cos"], s["sin"]), rot=s["heads"][3], q_norm=s["q_norm"], k_norm=s["k_norm"], norm_offset=s["offset"], eps=1e-6, dtype=s["type"])
    if s["cache"] == "none":
        return paged.rotate(s["q"], s["k"], s["positions"], **kw)
    cache = _cache(s)
    q = paged.enter(s["q"], s["k"], s["v"], s["positions"], s["slots"], cache, **kw)
    if s["cache"] == "int4":
        return (q, *cache.rows(s["slots"]))
    return q, cache.k, cache.v


def _turn(x, weight, s):
    """Norm and rotation of heads [T, n, dim], in 32 bits."""
    x = x.float()
    half = s["heads"][3] // 2
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (s["offset"] + weight)
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    a, b = x[..., :half], x[..., half: 2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _bf16_down(x):
    """The largest bf16 value that is not above x."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    cut = torch.where((bits < 0) & (cut != bits), cut + 65536, cut)
    return cut.view(torch.float32)


def _codes(x):
    """fp32 [..., dim] -> (packed codes [..., dim / 2], (scale, low) bf16 [..., dim / 64, 2])."""
    lead, dim = x.shape[:-1], x.shape[-1]
    x = x.reshape(*lead, dim // GROUP, GROUP)
    low = _bf16_down(x.amin(-1))
    scale = -_bf16_down(-((x.amax(-1) - low) / 15))
    c = torch.where(scale[..., None] > 0, torch.round((x - low[..., None]) / scale[..., None]), 0.0).clamp(0, 15).to(torch.uint8)
    c = c.reshape(*lead, dim // GROUP, 8, 4, 2).transpose(-4, -3).reshape(*lead, dim // 2, 2)
    return c[..., 0] | (c[..., 1] << 4), torch.stack([scale, low], -1).to(torch.bfloat16)


def _values(codes, scales):
    """The inverse: fp32 [..., dim]."""
    lead, dim = codes.shape[:-1], codes.shape[-1] * 2
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*lead, 8, dim // GROUP, 8).transpose(-3, -2).reshape(*lead, dim // GROUP, GROUP)
    f = scales.float()
    return (c.float() * f[..., :1] + f[..., 1:]).reshape(*lead, dim)


def _heads(s):
    """A row whose slot is -1 is padding: its queries are zeros and nothing is written."""
    q, k, v = _turn(s["q"], s["q_norm"], s), _turn(s["k"], s["k_norm"], s), s["v"].float()
    if s["cache"] == "none":
        return q.to(s["type"]), k.to(s["type"])
    live = s["slots"] >= 0
    slot = s["slots"].long().clamp(min=0)                      # padding rows write the null page, which nothing reads
    at, off = slot // s["page"], slot % s["page"]
    q = torch.where(live[:, None, None], q, 0.0).to(s["type"])
    if s["cache"] != "int4":
        for name, x in (("k_cache", k), ("v_cache", v)):
            s[name][at, :, off] = torch.where(live[:, None, None], x, 0.0).to(s[name].dtype)
        return q, s["k_cache"], s["v_cache"]
    back = []
    for name, x in (("k", k), ("v", v)):
        codes, scales = _codes(x)
        s[name + "_codes"][at, :, off] = codes
        s[name + "_scales"][at, :, off] = scales
        back.append(torch.where(live[:, None, None], _values(s[name + "_codes"][at, :, off], s[name + "_scales"][at, :, off]), 0.0))
    return q, back[0], back[1]


def _attend_own(s):
    from megakernels_b200 import paged
    return paged.attend(s["q"], _cache(s), s["table"], s["context"], starts=s["starts"], max_new=s["new"], scale=s["scale"], window=s["window"], sinks=s["sinks"])


def _attend(s):
    """All requests side by side, padded to the longest; in 32 bits."""
    nq, nkv, dim = s["heads"]
    context, starts, table = s["context"].long(), s["starts"].long(), s["table"].long()
    R, P = table.shape
    if s["cache"] == "int4":
        k, v = (_values(s[n + "_codes"][table], s[n + "_scales"][table]) for n in "kv")
    else:
        k, v = (s[n + "_cache"][table].float() for n in "kv")
    k, v = (x.transpose(1, 2).reshape(R, nkv, -1, dim) for x in (k, v))                   # [R, nkv, L, dim]
    L, N = k.shape[2], s["new"]
    i, j = torch.arange(N, device=DEVICE), torch.arange(L, device=DEVICE)
    count = starts[1:] - starts[:-1]
    live = i[None] < count[:, None]
    rows = torch.where(live, starts[:-1, None] + i[None], 0)
    q = s["q"].float()[rows].reshape(R, N, nkv, nq // nkv, dim).permute(0, 2, 3, 1, 4).reshape(R, nkv, -1, dim)
    position = (context - count)[:, None] + i[None]                                       # [R, N]
    d = position[:, :, None] - j
    seen = d >= 0
    if s["window"]:
        seen &= (d < s["window"]) | (j < s["sinks"])
    score = (q @ k.transpose(2, 3)).view(R, nkv, nq // nkv, N, L).mul_(s["scale"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = score.sum(-1, keepdim=True)
    score = score / torch.where(total > 0, total, 1.0)
    o = (score.view(R, nkv, -1, L) @ v).view(R, nkv, nq // nkv, N, dim).permute(0, 3, 1, 2, 4).reshape(R, N, nq, dim)
    return o[live].to(s["type"])


def _sample_own(s):
    from megakernels_b200 import sampling
    r = sampling.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"ids": r.ids, "logprobs": r.logprobs, "kept": r.kept}


def _sample(s):
    """Candidates in the order (value falling, index rising): the first top_k, of these the fewest that hold top_p of their
    weight, of these the ones with at least min_p of the largest weight.  The token is the first, by index, at which the
    running weight of the kept ones passes u times their sum.  Temperature 0 takes the largest.  In 64 bits: a border decides."""
    x = s["logits"].double()
    V = x.shape[1]
    t = s["temperature"].double()[:, None]
    k = torch.where(s["top_k"] > 0, s["top_k"], V).clamp(max=V)[:, None]
    k = torch.where(t > 0, k, 1)
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((value - value[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(V, device=DEVICE)[None]
    w = torch.where(rank < k, w, 0.0)
    run_sum = torch.cumsum(w, 1)
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((run_sum - w < p * run_sum[:, -1:]) | (p >= 1)) & (w >= s["min_p"].double()[:, None])
    kept = keep.sum(1)
    weight = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))            # by index again
    run_sum = torch.cumsum(weight, 1)
    total = run_sum[:, -1]
    ids = (run_sum <= s["u"].double()[:, None] * total[:, None]).sum(1)
    chosen = weight.gather(1, ids[:, None])[:, 0]
    return {"ids": ids.int(), "logprobs": torch.log(chosen / total).float(), "kept": kept.int()}


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def _visible(position, window, sinks):
    """Keys that a query at `position` sees."""
    if not window or position < window:
        return position + 1
    return window + min(sinks, position - window + 1)


def work(c):
    if c["op"] == "plan":
        R = c["requests"]
        tokens = min(c["room"], max(1, round(R * (1 - c["ended"]))))
        return {"bytes": 4 * (8 * R + 3 * c["room"] + 2 * tokens), "flops": 0}
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * (4 if c["type"] == "fp32" else 2) + 32), "flops": 0}
    nq, nkv, dim, _ = HEADS[c["heads"]]
    row = {"int4": 2 * (dim // 2 + dim // GROUP * 4), "none": 0}.get(c["cache"], 4 * dim)  # a token's K and V of one KV head
    if c["op"] == "heads":
        T, size = c["tokens"], 4 if c["source"] == "fp32" else 2
        read = T * size * dim * (nq + (1 if c["cache"] == "none" else 2) * nkv)
        wrote = T * (2 * dim * nq + (nkv * row if c["cache"] != "none" else 2 * dim * nkv))
        again = T * nkv * (row + 8 * dim) if c["cache"] == "int4" else 0                  # the rows as values
        return {"bytes": read + wrote + again, "flops": 0}
    mean = (c["context"] + max(c["new"], c["context"] // 3)) / 2 if c["ragged"] else c["context"]
    new = c["new"] if c["new"] <= 4 or not c["ragged"] or c["requests"] == 1 else (c["new"] + 1) / 2
    lengths = [c["context"]] + [mean] * (c["requests"] - 1)
    news = [min(c["new"], c["context"])] + [min(new, mean)] * (c["requests"] - 1)
    keys = pairs = 0.0
    for length, n in zip(lengths, news):
        first, last = length - n, length - 1
        keys += length if not c["window"] else min(length, n + c["window"] - 1 + c["sinks"])
        pairs += n * (_visible(first, c["window"], c["sinks"]) + _visible(last, c["window"], c["sinks"])) / 2
    return {"bytes": round(keys * nkv * row + sum(news) * nq * dim * 4), "flops": round(4 * dim * nq * pairs)}


# ---------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _plan_exact, "heads": _heads_exact, "attend": _attend_exact, "sample": _sample_exact}[case["op"]](s)


def _plan_exact(s):
    """Request by request, on lists."""
    page, room = s["page"], s["room"]
    length, new, held = s["lengths"].tolist(), s["new"].tolist(), s["held"].tolist()
    table, stack, n = s["table"].tolist(), s["free"].tolist(), int(s["n_free"])
    R, P = s["table"].shape
    returned = []
    for r in range(R):
        base = min(held[r], -(-length[r] // page))
        returned += table[r][base: held[r]]
        table[r][base: held[r]] = [0] * (held[r] - base)
        held[r] = base
    stack[n: n + len(returned)] = returned[::-1]
    n += len(returned)
    waiting, wanted, starts, granted, context = False, 0, [0], [0] * R, list(length)
    slots, positions, rows = [-1] * room, [0] * room, [-1] * room
    for r in range(R):
        need = -(-(length[r] + new[r]) // page)
        if need > P:
            context[r] = 0
        elif not waiting and need - held[r] <= n and wanted + new[r] <= room:
            granted[r], context[r] = 1, length[r] + new[r]
            while held[r] < need:
                n -= 1
                table[r][held[r]] = stack[n]
                held[r] += 1
            for i in range(new[r]):
                p = length[r] + i
                slots[wanted], positions[wanted], rows[wanted] = table[r][p // page] * page + p % page, p, r
                wanted += 1
        elif need == held[r] and new[r] == 0:
            granted[r] = 1
        else:
            waiting = True
        starts.append(wanted)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)                        # noqa: E731
    return {"table": t(table), "slots": t(slots), "positions": t(positions), "rows": t(rows), "starts": t(starts), "context": t(context), "granted": t(granted),
            "held": t(held), "free": t(stack), "n_free": t([n])}


def _heads_exact(s):
    nq, nkv, dim, rot = s["heads"]
    T, half, position = s["q"].shape[0], rot // 2, s["positions"].long()

    def turned(x, weight):
        x = x.double()
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / dim + 1e-6) * (weight.double() + s["offset"])
        out = x.clone()
        for d in range(half):
            c, n = s["cos"][position, d].double()[:, None], s["sin"][position, d].double()[:, None]
            out[..., d] = x[..., d] * c - x[..., d + half] * n
            out[..., d + half] = x[..., d + half] * c + x[..., d] * n
        return out

    q, k = turned(s["q"], s["q_norm"]), turned(s["k"], s["k_norm"])
    if s["cache"] == "none":
        return q, k
    live = torch.nonzero(s["slots"] >= 0)[:, 0]
    q[s["slots"] < 0] = 0
    if s["cache"] == "int4":
        return q, None, None                                   # codes next to a border have no 64-bit value of their own
    out = [q]
    for name, x in (("k_cache", k), ("v_cache", s["v"].double())):
        c = s[name].double()
        slot = s["slots"][live].long()
        c[slot // s["page"], :, slot % s["page"]] = x[live]
        out.append(c)
    return tuple(out)


def _attend_exact(s):
    nq, nkv, dim = s["heads"]
    table, context, starts, page = s["table"].long(), s["context"].tolist(), s["starts"].tolist(), s["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)

    def row_values(name, pages, head, length):
        if s["cache"] != "int4":
            return s[name + "_cache"][pages, head].double().reshape(-1, dim)[:length]
        words = s[name + "_codes"][pages, head].reshape(-1, 8, dim // GROUP, 4)[:length]
        sc = s[name + "_scales"][pages, head].double().reshape(-1, dim // GROUP, 2)[:length]
        v = torch.empty(length, dim // GROUP, 8, 8, dtype=torch.float64, device=DEVICE)
        for b in range(4):
            byte = words[..., b].transpose(1, 2)
            v[..., 2 * b], v[..., 2 * b + 1] = (byte % 16).double(), (byte // 16).double()
        return (sc[:, :, 1, None] + sc[:, :, 0, None] * v.reshape(length, dim // GROUP, GROUP)).reshape(length, dim)

    per = nq // nkv
    for r, length in enumerate(context):
        a, b = starts[r], starts[r + 1]
        pages = table[r, : -(-length // page)]
        key = torch.arange(length, device=DEVICE)
        for h in range(nkv):
            k, v = row_values("k", pages, h, length), row_values("v", pages, h, length)
            for lo in range(a, b, 1024):
                hi = min(b, lo + 1024)
                at = length - (b - a) + torch.arange(lo - a, hi - a, device=DEVICE)
                hidden = key[None] > at[:, None]
                if s["window"]:
                    hidden |= (key[None] <= at[:, None] - s["window"]) & (key[None] >= s["sinks"])
                for g in range(h * per, (h + 1) * per):
                    score = (s["q"][lo:hi, g].double() @ k.T) * s["scale"]
                    score[hidden] = -math.inf
                    out[lo:hi, g] = torch.softmax(score, -1) @ v
    return out


def _sample_exact(s):
    """Row by row, from a sorted list of candidates."""
    ids, logprobs, kept = [], [], []
    for b in range(s["logits"].shape[0]):
        x = s["logits"][b].double().cpu().numpy()
        t, k, p, m, u = (float(s[n][b]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        order = (-x).argsort(kind="stable")
        if t <= 0:
            t, k = 1.0, 1
        if k >= 1:
            order = order[: int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            total = w.sum()
            n = int((w.cumsum() < p * total).sum()) + 1
            order, w = order[:n], w[:n]
        stay = w >= m
        order, w = order[stay], w[stay]
        by_index = order.argsort(kind="stable")
        w_sorted = w[by_index]
        at = int((w_sorted.cumsum() <= u * w.sum()).sum())
        at = min(at, len(w_sorted) - 1)
        ids.append(int(order[by_index[at]]))
        logprobs.append(math.log(w_sorted[at] / w.sum()))
        kept.append(len(order))
    t = lambda v, dt: torch.tensor(v, dtype=dt, device=DEVICE)                             # noqa: E731
    return {"ids": t(ids, torch.int32), "logprobs": t(logprobs, torch.float64), "kept": t(kept, torch.int32)}

