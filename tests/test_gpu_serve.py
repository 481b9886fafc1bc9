"""Cache pages, heads, paged attention and sampling against 64 bits.

Tolerances, in half steps h of the output's type (bf16 2^-9, fp16 2^-12 of a value's power of two, so at most 2^-8 and 2^-11 of the value).
Heads: 32-bit arithmetic, so one rounding (h of the value) and 2^-20 of the head's largest value for the sums in between.  Attention: with E
the largest |out| bound sum p |v| <= max |v|: one rounding h |out|, plus the probabilities' rounding.  16-bit caches: bf16 probabilities are two pieces (2^-16) for
few queries per request and one (2^-8 of each, so at most 2^-8 sum p |v|) for many, whose product takes both operands of one type; fp16 ones one half (2^-11); scores are exact products in 32-bit sums whose error enters the exponent: 2^-20 max |score|.  4 bits: codes and queries are exact, probabilities and their
product with a scale are rounded to halves, lows too: 3 * 2^-11.  All of them times sum p |v| (for 4 bits sum p (|low| + 15 scale), at most 2 max |v| plus the low)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import serve_reference as R
from megakernels_b200 import paged, sampling

DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- pages -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("requests,page,max_pages,pages,room,seed", [
    (1, 16, 4, 6, 1, 0), (3, 16, 8, 12, 40, 1), (8, 64, 16, 40, 8, 2), (65, 32, 20, 400, 300, 3), (65, 1, 64, 900, 1500, 4), (1500, 16, 12, 6000, 5000, 5), (4096, 64, 5, 9000, 4096, 6)])
def test_plans_follow_the_lists(requests, page, max_pages, pages, room, seed):
    g = torch.Generator().manual_seed(seed)
    pool = paged.PagePool(requests, pages, max_pages, page=page, max_tokens=room, device=DEV)
    rnd = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))             # noqa: E731
    table, held, free, n = pool.table.tolist(), pool.held.tolist(), pool.free.tolist(), int(pool.n_free)
    length = [0] * requests
    for step in range(12):
        new = []
        for r in range(requests):
            what = rnd(0, 19)
            if what == 0:
                length[r] = 0                                  # ended, or replaced by a new prompt
            elif what == 1:
                length[r] = max(0, length[r] - rnd(1, page + 3))
            new.append(0 if what in (2, 3) else (rnd(1, 2 * page) if what < 6 else 1))
            if what == 19 and step % 3 == 0:
                new[r] = rnd(1, page * (max_pages + 1))        # may ask for more pages than a request can hold
        if step % 4 == 3:
            new[rnd(0, requests - 1)] = -1
        want = R.plan(length, new, table, held, free, n, page, room)
        got = pool.plan(ints(length), ints(new))
        table, held, free, n = want[:4]
        assert pool.table.tolist() == table and pool.held.tolist() == held, step
        assert int(pool.n_free) == n and pool.free[:n].tolist() == free[:n], step
        for name, w in zip(("slots", "positions", "rows", "starts", "context", "granted"), want[4:]):
            assert getattr(got, name).tolist() == w, (step, name)
        # no page twice, none lost
        mine = [p for r in range(requests) for p in table[r][: held[r]]]
        assert sorted(mine + free[:n]) == list(range(1, pages))
        length = [c if c or not length[r] else length[r] for r, c in enumerate(want[8])]
    torch.cuda.synchronize()


def test_a_plan_repeats_itself_and_replays_from_a_graph():
    pool = paged.PagePool(6, 60, 8, page=16, max_tokens=64, device=DEV)
    length, new = ints([0] * 6), ints([30, 1, 0, 17, 16, 0])
    first = [t.clone() for t in pool.plan(length, new)]
    again = pool.plan(length, new)                             # the same lengths: pages go back and come again
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = pool.plan(length, new)
    length.copy_(ints([30, 1, 0, 17, 16, 0])), new.fill_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert out.context.tolist() == [31, 2, 1, 18, 17, 1] and out.starts.tolist() == list(range(7))
    assert out.slots[6:].tolist() == [-1] * 58


# ---- heads -------------------------------------------------------------------------------------------------------
def tables(n, pairs):
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * 1e4 ** (-torch.arange(pairs, dtype=torch.float64, device=DEV) / pairs)
    return a.cos().float(), a.sin().float()


def near(got, want, half, extra):
    """|got - want| <= half |want| + extra."""
    d = (got.double() - want).abs()
    bad = d > half * want.abs() + extra
    assert not bool(bad.any()), (int(bad.sum()), float((d - half * want.abs()).max()), float(torch.as_tensor(extra).max()))


HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("source,dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("rot,pairs,interleaved,norm", [("all", None, False, True), ("part", None, False, True), ("part", "few", True, False), (None, None, False, True)])
def test_rotate(dim, source, dtype, rot, pairs, interleaved, norm):
    T, nq, nkv = 5, 3, 1
    g = gen(dim)
    width = nq * 2 * dim + nkv * dim + 8
    y = (torch.randn(T, width, generator=g, device=DEV) * torch.tensor([0.01, 1.0, 30.0, 1.0, 1.0], device=DEV)[:, None]).to(source)
    q, k = y[:, : nq * 2 * dim].view(T, nq, 2 * dim)[..., :dim], y[:, nq * 2 * dim: nq * 2 * dim + nkv * dim].view(T, nkv, dim)
    positions = ints([0, 1, 99, 40, 7])
    rope, r = None, None
    if rot:
        r = dim if rot == "all" else dim // 4
        rope = tables(100, r // 2 if pairs is None else max(1, r // 4))
    qn, kn = (torch.randn(dim, generator=g, device=DEV) * 0.2 for _ in "qk") if norm else (None, None)
    got = paged.rotate(q, k, positions, rope=rope, rot=r, q_norm=qn, k_norm=kn, norm_offset=1.0, eps=1e-6, interleaved=interleaved, dtype=dtype)
    for x, w, o in ((q, qn, got[0]), (k, kn, got[1])):
        want = R.heads(x, w, 1.0, 1e-6, rope, positions, r, interleaved)
        near(o, want, HALF[dtype], 2.0 ** -20 * want.abs().amax(-1, keepdim=True))
    assert got[0].dtype == dtype and got[0].is_contiguous()


def make_cache(kind, pages, nkv, dim, page, layout="pages"):
    return paged.Cache(pages, nkv, dim, page=page, dtype={"bf16": torch.bfloat16, "fp16": torch.float16, "int4": "int4"}[kind], device=DEV, layout=layout)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind,layout", [("bf16", "pages"), ("bf16", "serving"), ("fp16", "pages"), ("int4", "pages")])
def test_enter(dim, kind, layout):
    T, nq, nkv, page = 7, 4, 2, 16
    g = gen(dim + len(kind))
    q, k, v = (torch.randn(T, n, dim, generator=g, device=DEV, dtype=torch.float32) for n in (nq, nkv, nkv))
    v[3] = 2.5                                                  # a group of equal values
    v[4] = torch.linspace(-1e-6, 3e4, nkv * dim, device=DEV).view(nkv, dim)
    cache = make_cache(kind, 5, nkv, dim, page, layout)
    for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        if t is not None:
            t.fill_(3)
    slots, positions = ints([16, 17, 79, -1, 33, 80, 40]), ints([5, 6, 7, 8, 9, 10, 200])     # -1, 80: outside the cache; 200: outside the tables
    qn, kn = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV) for _ in "qk")
    rope = tables(100, dim // 2)
    before = [t.clone() for t in (cache.k, cache.v)]
    out = paged.enter(q, k, v, positions, slots, cache, rope=rope, q_norm=qn, k_norm=kn, v_norm=False, eps=1e-5)
    dead = [3, 5, 6]
    at = positions.clone()
    at[6] = 0
    want = R.heads(q, qn, 0.0, 1e-5, rope, at, dim, False)
    want[dead] = 0
    near(out, want, HALF[out.dtype], 2.0 ** -20 * want.abs().amax(-1, keepdim=True))
    wk = R.heads(k, kn, 0.0, 1e-5, rope, at, dim, False)
    live = [i for i in range(T) if i not in dead]
    slot = slots[live].long()
    pg, off = slot // page, slot % page
    if kind != "int4":
        near(cache.k[pg, :, off], wk[live], HALF[cache.dtype], 2.0 ** -20 * wk[live].abs().amax(-1, keepdim=True))
        if kind == "bf16":
            assert torch.equal(cache.v[pg, :, off], v[live].to(cache.dtype))
    else:
        # values as they are: the same codes; normed keys: within half a step and its rounding of what went in
        c, s, low = R.encode(v[live])
        assert torch.equal(cache.v_scales[pg, :, off, :, 0].float(), s) and torch.equal(cache.v_scales[pg, :, off, :, 1].float(), low)
        assert torch.equal(cache.v[pg, :, off], R.pack(c))
        step = cache.k_scales[pg, :, off, :, 0].double().repeat_interleave(64, -1)
        d = (R.decode(cache.k[pg, :, off], cache.k_scales[pg, :, off]) - wk[live]).abs()
        assert bool((d <= step * 0.5001 + 2.0 ** -20 * wk[live].abs().amax(-1, keepdim=True)).all())
        assert bool((step <= (wk[live].view(len(live), nkv, -1, 64).amax(-1) - wk[live].view(len(live), nkv, -1, 64).amin(-1) + 2.0 ** -7 * wk[live].view(len(live), nkv, -1, 64).amin(-1).abs()).repeat_interleave(64, -1) / 15 * 1.008 + 1e-30).all())
    # everything else is as it was
    for t, b in zip((cache.k, cache.v), before):
        same = torch.ones(t.shape[0], t.shape[2], dtype=torch.bool, device=DEV)
        same[pg, off] = False
        assert torch.equal(t.transpose(1, 2)[same], b.transpose(1, 2)[same])
    # and comes back as values
    rk, rv = cache.rows(slots)
    ref = [R.decode(c, s) if kind == "int4" else c.double() for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]
    for got, r in zip((rk, rv), ref):
        want = torch.zeros(T, nkv, dim, dtype=torch.float64, device=DEV)
        inside = [i for i in range(T) if 0 <= int(slots[i]) < 80]
        sl = slots[inside].long()
        want[inside] = r[sl // page, :, sl % page]
        # two roundings to 32 bits of a 4-bit value's product and sum
        near(got, want, 2.0 ** -23, 2.0 ** -23 * want.abs().amax(-1, keepdim=True))


def test_enter_normed_values_and_groups_that_are_not_finite():
    cache = make_cache("int4", 2, 1, 64, 16)
    v = torch.randn(4, 1, 64, generator=gen(0), device=DEV)
    v[1, 0, 5], v[2, 0, 6], v[3, 0, 7] = math.inf, -math.inf, math.nan
    q = torch.zeros(4, 1, 64, device=DEV)
    paged.enter(q, q, v, ints([0] * 4), ints([16, 17, 18, 19]), cache, v_norm=False)
    got = cache.rows(ints([16, 17, 18, 19]))[1]
    assert bool(got[0].isfinite().all()) and bool(got[1:].isnan().all())
    c16 = make_cache("bf16", 2, 1, 64, 16)
    x = torch.randn(3, 1, 64, generator=gen(1), device=DEV)
    paged.enter(q[:3], x, x, ints([0] * 3), ints([0, 1, 2]), c16, v_norm=True, eps=1e-6)
    want = R.heads(x, True, 0, 1e-6, None, None, 0, False)
    near(c16.v[0, :, :3].transpose(0, 1), want, HALF[torch.bfloat16], 2.0 ** -20 * want.abs().amax())
    assert torch.equal(c16.k[0, :, :3].transpose(0, 1), x.to(torch.bfloat16))


# ---- attention ---------------------------------------------------------------------------------------------------
def fill(cache, seed, spread=1.0):
    g = gen(seed)
    shape = (cache.pages, cache.kv_heads, cache.page, cache.head_dim)
    if cache.int4:
        for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
            c.copy_(torch.randint(0, 256, c.shape, generator=g, device=DEV, dtype=torch.uint8))
            size = spread * (0.5 + torch.rand(s.shape[:-1], generator=g, device=DEV))
            s.copy_(torch.stack([size / 7.5, -size * (0.8 + 0.4 * torch.rand(s.shape[:-1], generator=g, device=DEV))], -1))
        return R.decode(cache.k, cache.k_scales), R.decode(cache.v, cache.v_scales)
    for c in (cache.k, cache.v):
        c.copy_(torch.randn(shape, generator=g, device=DEV) * spread)
    return cache.k.double(), cache.v.double()


def case(kind, dtype, nq, nkv, dim, page, contexts, counts, window, sinks, seed=0, spread=1.0, layout="pages"):
    P = max(1, max(-(-c // page) for c in contexts)) + 1
    need = sum(-(-c // page) for c in contexts)
    cache = make_cache(kind, need + 2, nkv, dim, page, layout)
    k, v = fill(cache, seed, spread)
    g = torch.Generator().manual_seed(seed)
    order = (torch.randperm(need + 1, generator=g) + 1).tolist()
    table = torch.zeros(len(contexts), P, dtype=torch.int32)
    for r, c in enumerate(contexts):
        for j in range(-(-c // page)):
            table[r, j] = order.pop()
    T = sum(counts)
    q = (torch.randn(T, nq, dim, generator=gen(seed + 1), device=DEV) * 2).to(dtype)
    starts = ints([0] + torch.tensor(counts).cumsum(0).tolist()) if len(counts) else None
    return cache, k, v, table.to(DEV), ints(contexts), starts, q


def compare(got, want, cache, v, dtype, many=False):
    big = float((v.abs().amax() if not cache.int4 else (cache.v_scales[..., 1].abs() + 15 * cache.v_scales[..., 0]).amax()))
    slack = 2.0 ** -8 if many and cache.dtype == torch.bfloat16 else {"int4": 3 * 2.0 ** -11, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -11}[cache.dtype] + 2.0 ** -14
    near(got, want, HALF[dtype], slack * big)


SHAPES = [(8, 2, 256), (6, 1, 128), (24, 4, 256), (3, 3, 64), (16, 1, 128), (5, 1, 64)]


@pytest.mark.parametrize("kind,dtype", [("bf16", torch.bfloat16), ("fp16", torch.float16), ("int4", torch.bfloat16), ("int4", torch.float16)])
@pytest.mark.parametrize("nq,nkv,dim", SHAPES)
def test_attend_one_query_each(kind, dtype, nq, nkv, dim):
    contexts = [1, 2, 15, 16, 17, 64, 65, 700, 333]
    for page, window, sinks in ((16, 0, 0), (64, 50, 3), (32, 16, 40), (128, 1, 0)):
        cache, k, v, table, context, _, q = case(kind, dtype, nq, nkv, dim, page, contexts, [1] * len(contexts), window, sinks, seed=page)
        got = paged.attend(q, cache, table, context, window=window, sinks=sinks)
        compare(got, R.attend(q, k, v, table, context, None, dim ** -0.5, window, sinks), cache, v, dtype)
        again = paged.attend(q, cache, table, context, window=window, sinks=sinks)
        assert torch.equal(got, again)
    paged.check()


@pytest.mark.parametrize("kind,dtype", [("bf16", torch.bfloat16), ("fp16", torch.float16), ("int4", torch.bfloat16)])
@pytest.mark.parametrize("nq,nkv,dim", SHAPES[:4])
def test_attend_ragged_queries(kind, dtype, nq, nkv, dim):
    contexts, counts = [70, 1, 0, 300, 40, 129, 500], [3, 1, 0, 2, 40, 7, 200]
    for window, sinks in ((0, 0), (33, 2), (100, 0)):
        cache, k, v, table, context, starts, q = case(kind, dtype, nq, nkv, dim, 32, contexts, counts, window, sinks, seed=window)
        got = paged.attend(q, cache, table, context, starts=starts, window=window, sinks=sinks, scale=0.11)
        compare(got, R.attend(q, k, v, table, context, starts, 0.11, window, sinks), cache, v, dtype, many=True)
    paged.check()


@pytest.mark.parametrize("kind,dtype,dim", [("bf16", torch.bfloat16, 256), ("int4", torch.bfloat16, 256), ("fp16", torch.float16, 128), ("int4", torch.float16, 64)])
def test_attend_long_contexts_are_split(kind, dtype, dim):
    contexts = [9000, 5, 4097, 2500]
    for window in (0, 3000):
        cache, k, v, table, context, _, q = case(kind, dtype, 8, 2, dim, 64, contexts, [1] * 4, window, 4, seed=dim)
        got = paged.attend(q, cache, table, context, window=window, sinks=4)
        compare(got, R.attend(q, k, v, table, context, None, dim ** -0.5, window, 4), cache, v, dtype)
    paged.check()


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_attend_what_nobody_sees_is_not_looked_at(kind):
    """NaN behind a context, before a window, in the null page and in pages that no table names; rows without a key; bad pages."""
    contexts, counts = [100, 37, 0, 3, 64], [1, 2, 1, 5, 1]
    cache, k, v, table, context, starts, q = case(kind, torch.bfloat16, 4, 2, 128, 16, contexts, counts, 20, 2, seed=9)
    seen = torch.zeros(cache.pages, cache.page, dtype=torch.bool, device=DEV)
    for r, (c, n) in enumerate(zip(contexts, counts)):
        for j in range(c):
            if j < 2 or j > c - n - 20:
                seen[int(table[r, j // 16]), j % 16] = True
    table[0, 5], table[3, 0] = 10 ** 6, -7                      # keys 80 .. 95 of request 0 and all of request 3 are gone
    for t in (cache.k_scales, cache.v_scales) if kind == "int4" else (cache.k, cache.v):
        t.copy_(torch.where(seen[:, None, :].reshape(cache.pages, 1, cache.page, *([1] * (t.dim() - 3))), t, math.nan))
    got = paged.attend(q, cache, table, context, starts=starts, window=20, sinks=2)
    want = R.attend(q, torch.nan_to_num(k), torch.nan_to_num(v), table, context, starts, 128 ** -0.5, 20, 2)
    compare(got, want, cache, torch.nan_to_num(v) if kind == "bf16" else v, torch.bfloat16) if kind == "bf16" else near(got, want, HALF[torch.bfloat16], (3 * 2.0 ** -11 + 2.0 ** -14) * 1.5 * 2.2)
    assert bool((got[3] == 0).all()) and bool((got[4:9] == 0).all())


@pytest.mark.parametrize("kind,dtype,layout", [("bf16", torch.bfloat16, "pages"), ("fp16", torch.float16, "serving"), ("int4", torch.bfloat16, "pages")])
@pytest.mark.parametrize("nq,nkv,dim,page", [(24, 4, 256, 64), (8, 8, 128, 16), (32, 4, 64, 256)])
def test_attend_more_blocks_than_the_gpu_takes_at_once(kind, dtype, layout, nq, nkv, dim, page):
    """Every block of rows goes on where another one has been: requests of no, one and many queries, some of them with fewer positions than queries or none at all."""
    rng = torch.Generator().manual_seed(dim)
    counts = [int(x) for x in torch.randint(0, 130, (90,), generator=rng)] + [300, 0, 1, 2, 700]
    contexts = [c + int(x) for c, x in zip(counts, torch.randint(0, 500, (95,), generator=rng))]
    for r in (3, 4, 5, 6, 7, 40):
        contexts[r] = 0
    contexts[20], contexts[21] = counts[20] // 2, max(counts[21] - 1, 0)
    for window, sinks in ((0, 0), (100, 5)):
        cache, k, v, table, context, starts, q = case(kind, dtype, nq, nkv, dim, page, contexts, counts, window, sinks, seed=window, layout=layout)
        got = paged.attend(q, cache, table, context, starts=starts, window=window, sinks=sinks)
        paged.check()
        compare(got, R.attend(q, k, v, table, context, starts, dim ** -0.5, window, sinks), cache, v, dtype, many=True)
        assert torch.equal(got, paged.attend(q, cache, table, context, starts=starts, window=window, sinks=sinks))


def test_attend_leaves_other_rows_alone_and_takes_strides():
    cache, k, v, table, context, starts, q = case("bf16", torch.bfloat16, 4, 2, 64, 16, [50, 20], [2, 3], 0, 0, seed=3, layout="serving")
    wide = torch.full((8, 4, 192), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[1:6, :, 64:128] = q
    out = torch.full((8, 8, 64), 5.0, dtype=torch.bfloat16, device=DEV)
    big = torch.zeros(2, 40, dtype=torch.int32, device=DEV)
    big[:, : table.shape[1]] = table
    got = paged.attend(wide[:, :, 64:128], cache, big[:, : table.shape[1]], context, starts=starts + 1, out=out[:, ::2])
    want = R.attend(q, k, v, table, context, starts, 0.125)
    compare(got[1:6], want, cache, v, torch.bfloat16)
    assert bool((out[:, 1::2] == 5).all()) and bool((out[0] == 5).all()) and bool((out[6:] == 5).all())


@pytest.mark.parametrize("kind,layout", [("bf16", "pages"), ("fp16", "serving"), ("int4", "pages")])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 128), (256, 64)])
def test_attend_many_queries_of_views(kind, layout, dim, page):
    """Queries and outputs [heads, tokens, dim] and inside wider rows; a table inside a wider one; rows of out in front of and behind the queries."""
    dtype = torch.float16 if kind == "fp16" else torch.bfloat16
    cache, k, v, table, context, starts, q = case(kind, dtype, 6, 2, dim, page, [400, 130, 90], [150, 1, 90], 0, 0, seed=dim, layout=layout)
    T = q.shape[0]
    wide = torch.full((6, T + 9, dim + 8), 9.0, dtype=dtype, device=DEV)
    wide[:, 5:T + 5, :dim] = q.transpose(0, 1)
    out = torch.full((6, T + 9, dim + 64), 5.0, dtype=dtype, device=DEV)
    big = torch.full((3, 70), -3, dtype=torch.int32, device=DEV)
    big[:, 1: 1 + table.shape[1]] = table
    for window, sinks in ((0, 0), (60, 9)):
        got = paged.attend(wide[..., :dim].transpose(0, 1), cache, big[:, 1: 1 + table.shape[1]], context, starts=starts + 5, window=window, sinks=sinks, out=out[..., 64:].transpose(0, 1))
        compare(got[5:T + 5], R.attend(q, k, v, table, context, starts, dim ** -0.5, window, sinks), cache, v, dtype, many=True)
        assert bool((out[..., :64] == 5).all()) and bool((out[:, :5] == 5).all()) and bool((out[:, T + 5:] == 5).all())


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("dim", [64, 256])
def test_attend_many_queries_do_not_look_at_what_none_of_them_sees(kind, dim):
    contexts, counts, window, sinks = [600, 257, 0, 40], [190, 100, 70, 40], 20, 2
    cache, k, v, table, context, starts, q = case(kind, torch.bfloat16, 4, 2, dim, 16, contexts, counts, window, sinks, seed=19)
    table[0, 30], table[3, 0] = 10 ** 6, -7                     # keys 480 .. 495 of request 0, 0 .. 15 of request 3
    seen = torch.zeros(cache.pages, cache.page, dtype=torch.bool, device=DEV)
    for r, (c, n) in enumerate(zip(contexts, counts)):
        for j in range(c):
            page = int(table[r, j // 16])
            if (j < sinks or j > c - n - window) and 0 <= page < cache.pages:
                seen[page, j % 16] = True
    for t in (cache.k_scales, cache.v_scales) if kind == "int4" else (cache.k, cache.v):
        t.copy_(torch.where(seen[:, None, :].reshape(cache.pages, 1, cache.page, *([1] * (t.dim() - 3))), t, math.nan))
    got = paged.attend(q, cache, table, context, starts=starts, window=window, sinks=sinks)
    want = R.attend(q, torch.nan_to_num(k), torch.nan_to_num(v), table, context, starts, dim ** -0.5, window, sinks)
    near(got, want, HALF[torch.bfloat16], (2.0 ** -8 if kind == "bf16" else 3 * 2.0 ** -11 + 2.0 ** -14) * float(torch.nan_to_num(v).abs().max()) * (1 if kind == "bf16" else 2.2))
    assert bool((got[290:360] == 0).all())                      # the request without positions
    paged.check()


def test_attend_many_queries_in_graphs_and_on_streams_at_once():
    cache, k, v, table, context, starts, q = case("bf16", torch.bfloat16, 8, 2, 256, 64, [900, 600], [500, 400], 0, 0, seed=8)
    want = paged.attend(q, cache, table, context, starts=starts)
    outs, graphs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.attend(q, cache, table, context, starts=starts))
        graphs.append(graph)
    q.mul_(0.5)
    half = paged.attend(q, cache, table, context, starts=starts)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s, graph in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    few = paged.attend(q[:2], cache, table, context, stream=streams[2])
    also = paged.attend(q, cache, table, context, starts=starts, stream=streams[2])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], half) and torch.equal(outs[1], half) and torch.equal(also, half) and not torch.equal(want, half)
    assert torch.equal(few, paged.attend(q[:2], cache, table, context))
    paged.check("cuda")


@pytest.mark.parametrize("kind,dim", [("bf16", 64), ("bf16", 256), ("int4", 128)])
def test_attend_sharp_scores_of_many_queries(kind, dim):
    """Scores that rise far above what came before, tile after tile: what was added is scaled away each time."""
    cache, k, v, table, context, starts, q = case(kind, torch.bfloat16, 4, 2, dim, 64, [1500, 700], [900, 650], 0, 0, seed=16)
    q.mul_(20)
    got = paged.attend(q, cache, table, context, starts=starts)
    want = R.attend(q, k, v, table, context, starts, dim ** -0.5)
    # scores reach 20 * 2 * |k|'s 4 sigma over dim ** -0.5 sums: below 20 * 2 * 4 * 16; their 32-bit error, 2^-20 of that, is the exponent's, on either side of a quotient
    near(got, want, HALF[torch.bfloat16], (2.0 ** -8 + 3 * 2.0 ** -11 + 2 * 2.0 ** -20 * 2560) * 2 * float(v.abs().max()))
    paged.check()


@pytest.mark.parametrize("spread", [1e-6, 1.0, 3e4])
def test_attend_many_queries_on_values_of_any_size(spread):
    """4-bit values far below and above what a half can hold."""
    cache, k, v, table, context, starts, q = case("int4", torch.bfloat16, 4, 1, 128, 16, [900, 440], [700, 440], 0, 0, seed=15, spread=spread)
    cache.k_scales.copy_(cache.k_scales * (1 / spread))
    k = R.decode(cache.k, cache.k_scales)
    got = paged.attend(q, cache, table, context, starts=starts)
    compare(got, R.attend(q, k, v, table, context, starts, 128 ** -0.5), cache, v, torch.bfloat16, many=True)


def test_attend_takes_more_queries_than_it_was_told_of():
    """max_new chooses a kernel and bounds nothing."""
    cache, k, v, table, context, starts, q = case("bf16", torch.bfloat16, 4, 2, 64, 16, [90, 70], [33, 12], 0, 0, seed=4)
    got = paged.attend(q, cache, table, context, starts=starts, max_new=1)
    compare(got, R.attend(q, k, v, table, context, starts, 0.125), cache, v, torch.bfloat16, many=True)


@pytest.mark.parametrize("kind,dim,new", [("bf16", 256, 1), ("int4", 64, 9)])
def test_attend_of_the_most_requests(kind, dim, new):
    R_, T = 4096, 4096 * new
    cache = make_cache(kind, 65, 4, dim, 16)
    k, v = fill(cache, 2)
    table = (torch.arange(R_, dtype=torch.int32, device=DEV) % 64 + 1).view(R_, 1)
    context = torch.full((R_,), 16, dtype=torch.int32, device=DEV)
    starts = torch.arange(R_ + 1, dtype=torch.int32, device=DEV) * new
    q = torch.randn(64 * new, 16, dim, generator=gen(3), device=DEV).to(torch.bfloat16)
    got = paged.attend(q.repeat(64, 1, 1), cache, table, context, starts=starts, max_new=new)
    want = R.attend(q, k, v, table[:64], context[:64], starts[:65], dim ** -0.5)
    assert got.shape[0] == T and torch.equal(got.view(64, -1), got[: 64 * new].reshape(1, -1).expand(64, -1))
    compare(got[: 64 * new], want, cache, v, torch.bfloat16, many=True)


@pytest.mark.parametrize("kind,layout", [("bf16", "serving"), ("fp16", "pages")])
@pytest.mark.parametrize("source", [torch.float32, torch.bfloat16, torch.float16])
def test_put_writes_rows_as_they_are(kind, layout, source):
    cache = make_cache(kind, 4, 2, 64, 16, layout)
    k, v = (torch.randn(5, 2, 64, generator=gen(i), device=DEV).to(source) for i in range(2))
    slots = ints([17, -1, 63, 16, 64])
    cache.put(k, v, slots)
    got_k, got_v = cache.rows(slots)
    for got, x in ((got_k, k), (got_v, v)):
        assert torch.equal(got[[0, 2, 3]], x[[0, 2, 3]].to(cache.dtype)) and bool((got[[1, 4]] == 0).all())
    assert int((cache.k != 0).any(-1).sum()) == 6               # three rows of two heads


@pytest.mark.parametrize("spread", [1e-6, 1.0, 3e4])
@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_attend_values_of_any_size(spread, dtype):
    """4-bit values far below and above what a half can hold."""
    cache, k, v, table, context, starts, q = case("int4", dtype, 4, 1, 128, 16, [300, 40, 77], [1, 1, 50], 0, 0, seed=5, spread=spread)
    cache.k_scales.copy_(cache.k_scales * (1 / spread))
    k = R.decode(cache.k, cache.k_scales)
    got = paged.attend(q, cache, table, context, starts=starts)
    compare(got, R.attend(q, k, v, table, context, starts, 128 ** -0.5), cache, v, dtype)


def test_attend_sharp_scores():
    """One key far above the others, late in the context: what was added before is scaled away."""
    cache, k, v, table, context, starts, q = case("bf16", torch.bfloat16, 2, 1, 128, 16, [600, 333], [1, 90], 0, 0, seed=6)
    q.mul_(30)
    got = paged.attend(q, cache, table, context, starts=starts)
    want = R.attend(q, k, v, table, context, starts, 128 ** -0.5)
    # scores reach 30 * 2 * 40: their 32-bit error, 2^-20 of that, is the exponent's
    near(got, want, HALF[torch.bfloat16], (2.0 ** -8 + 2.0 ** -20 * 3000) * float(v.abs().max()))


def test_attend_in_graphs_and_on_another_stream():
    cache, k, v, table, context, starts, q = case("int4", torch.bfloat16, 8, 2, 128, 32, [900, 200], [1, 1], 0, 0, seed=7)
    plain = paged.attend(q, cache, table, context)
    outs, graphs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.attend(q, cache, table, context))
        graphs.append(graph)
    context.copy_(ints([500, 64]))
    want = paged.attend(q, cache, table, context)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for i, graph in enumerate(graphs):
        with torch.cuda.stream(s):
            graph.replay()
    other = paged.attend(q, cache, table, context, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(other, want) and not torch.equal(plain, want)


# ---- the next token ----------------------------------------------------------------------------------------------
def check_sample(x, u, t, k, p, m):
    got = sampling.sample(x, u, t, k, p, m)
    # (settings are fp32: 0.8 of fifty equals is 40.0000006 of them, so 41)
    at = lambda s, i: float(s[i]) if torch.is_tensor(s) else float(torch.tensor(s, dtype=torch.float32))   # noqa: E731
    for i in range(x.shape[0]):
        want = R.sample(x[i].double().cpu(), float(u[i]), at(t, i), int(at(k, i)), at(p, i), at(m, i))
        have = int(got.ids[i]), float(got.logprobs[i]), int(got.kept[i])
        assert have[0] == want[0] and have[2] == want[2], (i, have, want)
        assert have[1] == want[1] or abs(have[1] - want[1]) <= 2.0 ** -23 * max(1.0, abs(want[1])), (i, have, want)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.6, 20, 0.95, 0.0), (1.3, 0, 1.0, 0.05), (1.0, 50, 0.8, 0.02), (0.0, 0, 0.5, 0.0), (1.0, 1, 1.0, 0.0),
            (0.3, 1000, 0.999, 0.0), (5.0, 7, 0.3, 1.0), (2.0, 0, 0.01, 0.0)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 2049, 5000, 151936])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample(vocab, dtype):
    g = gen(vocab)
    rows = 3
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(dtype)
    u = torch.rand(rows, generator=g, device=DEV)
    u[0] = 0.0
    for s in SETTINGS if vocab < 100000 else SETTINGS[1::3]:
        check_sample(x, u, *s)


def test_sample_ties_masks_and_infinities():
    x = torch.full((8, 3000), -math.inf, device=DEV)
    x[0, 1000:2000] = 1.5                                      # equals only
    x[1, ::7] = torch.tensor(0.0)
    x[1, ::14] = -0.0                                          # equal to 0
    x[3, 17] = 5.0                                             # one candidate (row 2: none)
    x[4] = torch.finfo(torch.float32).min
    x[4, 2999] = torch.finfo(torch.float32).min
    x[5] = torch.randn(3000, generator=gen(1), device=DEV).round()
    x[5, 5:400] = math.nan
    x[6, 100:300] = 1.0
    x[6, 200], x[6, 250] = math.inf, math.inf
    x[7] = torch.randn(3000, generator=gen(2), device=DEV)
    x[7, 1500:] = torch.finfo(torch.float32).min
    for u in (0.0, 0.31, 0.99999994):
        for s in SETTINGS:
            check_sample(x, torch.full((8,), u, device=DEV), *s)
    h = x.clamp(min=torch.finfo(torch.float16).min).to(torch.float16)
    check_sample(h, torch.full((8,), 0.5, device=DEV), 1.0, 2000, 0.9, 0.0)


def test_sample_rows_with_settings_of_their_own_and_strides():
    g = gen(11)
    rows, vocab = 40, 20000
    wide = (torch.randn(rows, vocab + 24, generator=g, device=DEV) * 2.5)
    x = wide[:, 8: 8 + vocab]
    pick = lambda v, dt: torch.tensor(v, dtype=dt, device=DEV)[torch.randint(0, len(v), (rows,), generator=g, device=DEV)]   # noqa: E731
    t, k = pick([0.0, 0.5, 1.0, 2.0], torch.float32), pick([0, 1, 5, 300, 19999, 20000, 50000], torch.int32)
    p, m = pick([1.0, 0.99, 0.7, 0.1], torch.float32), pick([0.0, 0.01, 0.3, 1.0], torch.float32)
    check_sample(x, torch.rand(rows, generator=g, device=DEV), t, k, p, m)


def test_sample_follows_the_distribution():
    """Over evenly spread uniforms a token comes as often as its share of the kept weight says, to one draw."""
    x = torch.randn(1, 500, generator=gen(4), device=DEV)
    n = 4096
    u = (torch.arange(n, device=DEV) + 0.5) / n
    ids = sampling.sample(x.expand(n, 500), u, top_k=40).ids
    w = torch.softmax(x.double()[0], -1)
    keep = w.topk(40).indices
    share = torch.zeros_like(w)
    share[keep] = w[keep] / w[keep].sum()
    count = torch.bincount(ids.long(), minlength=500)
    assert bool(((count - n * share).abs() <= 1.001).all())


# ---- a step as a serving loop makes it -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_pages_heads_attention_and_choice_together(kind):
    nq, nkv, dim, page, requests, vocab = 4, 2, 64, 16, 3, 500
    g = gen(21)
    pool = paged.PagePool(requests, 30, 8, page=page, max_tokens=64, device=DEV)
    cache = make_cache(kind, 30, nkv, dim, page)
    w = torch.randn(nq * dim, vocab, generator=g, device=DEV, dtype=torch.float64) * 0.05
    rope = tables(128, dim // 2)
    norm = 1 + 0.1 * torch.randn(dim, generator=g, device=DEV)
    length, keys, values = [0] * requests, [[] for _ in range(requests)], [[] for _ in range(requests)]
    for step, new in enumerate(([20, 5, 0], [1, 1, 30], [1, 1, 1], [4, 0, 1], [1, 1, 1])):
        if step == 3:
            length[0] -= 1                                     # a rejected draft
        if step == 4:
            length[1] = 0                                      # another user takes the row
        plan = pool.plan(ints(length), ints(new))
        T = sum(new)
        q, k, v = (torch.randn(64, n, dim, generator=g, device=DEV).to(torch.bfloat16) for n in (nq, nkv, nkv))
        qr = paged.enter(q, k, v, plan.positions, plan.slots, cache, rope=rope, q_norm=norm, k_norm=norm)
        out = paged.attend(qr, cache, plan.table, plan.context, starts=plan.starts, window=24, sinks=2, out=torch.zeros_like(qr))
        ends = plan.starts[1:].long() - 1
        logits = (out[ends].double().reshape(requests, -1) @ w).float()
        pickd = sampling.sample(logits, torch.rand(requests, generator=g, device=DEV), 0.8, 30, 0.9, 0.0)
        assert int(pickd.ids.min()) >= 0 and int(pickd.ids.max()) < vocab and int(pickd.kept.max()) <= 30
        # the same, request by request
        kr = R.heads(k, norm, 0.0, 1e-6, rope, plan.positions, dim, False)
        i = 0
        for r in range(requests):
            keys[r], values[r] = keys[r][: length[r]], values[r][: length[r]]
            for _ in range(new[r]):
                for store, x in ((keys[r], kr[i]), (values[r], v[i].double())):
                    if kind == "int4":
                        c, s, low = R.encode(x)
                        x = (low.double()[..., None] + s.double()[..., None] * c.double()).reshape(nkv, dim)
                    else:
                        x = x.to(torch.bfloat16).double()
                    store.append(x)
                i += 1
            length[r] += new[r]
            if not new[r]:
                continue
            kk, vv = torch.stack(keys[r]), torch.stack(values[r])
            tail = qr[i - new[r]: i]
            one = R.attend(tail, kk.transpose(0, 1)[None], vv.transpose(0, 1)[None], torch.zeros(1, 1, dtype=torch.int32, device=DEV), ints([length[r]]),
                           ints([0, new[r]]), dim ** -0.5, 24, 2) if len(kk) else None
            # a key's code, or its last bf16 bit, may fall the other way; 2^-4 of the values' size covers a step of one key among those seen
            assert float((out[i - new[r]: i].double() - one).abs().max()) <= 2.0 ** -4 * float(vv.abs().max())
        assert T == int(plan.starts[-1]) and bool((out[T:] == 0).all())
