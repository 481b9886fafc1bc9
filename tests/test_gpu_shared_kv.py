"""Engines on pages that their sequences share, on a 4-bit cache, and with sampled tokens.

Shared pages change where keys lie and nothing else, so everything equals the engine with pages of its own, bit for bit.  A 4-bit cache holds
what the bf16 cache's engine would have stored, cut to 4 bits (the codes of the same values, as the first attention layer sees the same
inputs), and the layer's output is that of the definition over it: bf16 queries (2^-8 of the largest score in the exponent: scores here stay
below 8, so 2^-5 of the values) and the kernel's own roundings below that."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import serve_reference as R
from megakernels_b200 import gemma26b, paged, qwen27b, qwen35moe, sampling
from megakernels_b200.qwen27b.dims import FULL as FULL27
from megakernels_b200.qwen27b.runner import rope_tables

SMALL = FULL27.with_(hidden=1024, ffn=2048, vocab=4096, layers=8, nkh=4, nvh=12, nq=8, nkv=2)
PROMPTS = 3


@pytest.fixture(scope="module")
def packed():
    W = qwen27b.SynthWeights(SMALL, layers=8, init="realistic", device="cuda", fmt="mxfp4")
    return qwen27b.Packed(W, "cuda")


def prompts(vocab, n, M=PROMPTS):
    return [qwen27b.make_prompt(vocab, n, seed=j) for j in range(M)]


def feed(eng, ps, n):
    for t in range(n):
        eng.step(torch.tensor([p[t] for p in ps]).cuda())


def test_shared_pages_change_nothing_but_where_keys_lie(packed):
    ps = prompts(SMALL.vocab, 80)
    own, shared = qwen27b.Engine(packed, 3, maxlen=256), qwen27b.Engine(packed, 3, maxlen=256, kv_pages=3 * 3 + 1)
    for eng in (own, shared):
        eng.prefill([p[:70] for p in ps])
        eng.got = [eng.logits.clone()]
        for t in range(70, 75):
            eng.got.append(eng.step(torch.tensor([p[t] for p in ps]).cuda()).clone())
        eng.got.append(eng.generate(torch.tensor([5, 6, 7]).cuda(), 20))
        eng.got += [k for ai in range(2) for m in range(3) for k in eng.kv_rows(ai, m, 95)]
        eng.check()
    assert all(torch.equal(a, b) for a, b in zip(own.got, shared.got))
    assert int(shared.pages.pool.n_free) == 9 - 3 * 2


def test_a_sequence_without_pages_waits_and_goes_on_later(packed):
    eng, ref = qwen27b.Engine(packed, 2, maxlen=256, kv_pages=4), qwen27b.Engine(packed, 2, maxlen=256)       # three pages for two sequences
    ps = prompts(SMALL.vocab, 70, M=2)
    feed(ref, ps, 70)
    for t in range(64):
        eng.step(torch.tensor([p[t] for p in ps]).cuda())
    for t in range(64, 70):                                    # only sequence 0 gets a second page
        got = eng.step(torch.tensor([p[t] for p in ps]).cuda()).clone()
    assert eng.pos[:2].tolist() == [70, 64] and torch.equal(eng.ssm[:, 0], ref.ssm[:, 0])
    assert torch.equal(got[0], ref.logits[0])
    eng.release(0)
    for t in range(64, 70):
        got = eng.step(torch.tensor([ps[0][t - 64], ps[1][t]]).cuda()).clone()
    assert eng.pos[:2].tolist() == [6, 70] and torch.equal(got[1], ref.logits[1]) and torch.equal(eng.ssm[:, 1], ref.ssm[:, 1])
    fresh = qwen27b.Engine(packed, 2, maxlen=256)
    feed(fresh, ps, 6)
    assert torch.equal(got[0], fresh.logits[0]) and torch.equal(eng.ssm[:, 0], fresh.ssm[:, 0])
    eng.check()


def test_prompts_that_do_not_fit_are_refused(packed):
    eng = qwen27b.Engine(packed, 3, maxlen=256, kv_pages=5)
    with pytest.raises(RuntimeError, match="pages"):
        eng.prefill([p for p in prompts(SMALL.vocab, 100)])


def test_shared_pages_of_the_other_engines():
    W = gemma26b.SynthWeights(layers=6, init="realistic", device="cuda", draw_device="cuda")
    PK = gemma26b.Packed(W, "cuda")
    got = []
    for kw in ({}, dict(kv_pages=6)):
        eng = gemma26b.Engine(PK, 2, maxlen=192, **kw)
        ps = prompts(PK.shape.vocab, 20, M=2)
        eng.prefill(ps)
        got.append([eng.logits.clone(), eng.generate(torch.tensor([5, 6]).cuda(), 6)])
        eng.check()
    assert all(torch.equal(a, b) for a, b in zip(*got))


def check_layer(eng, ai, cos, sin, q_norm, before):
    """The gated output of attention layer `ai` (the last one: y and y2 still hold its rows) against the definition over the engine's cache."""
    s, M = eng.shape, eng.M
    hd, nq, nkv = 256, eng.shape.nq, eng.shape.nkv
    q = eng.y[:, : nq * 2 * hd].view(M, nq, 2 * hd)
    turned = R.heads(q[..., :hd], q_norm, 1.0, s.eps, (cos, sin), before, 64, False)
    c = eng.kv4.caches[ai]
    k, v = R.decode(c.k, c.k_scales), R.decode(c.v, c.v_scales)
    want = R.attend(turned, k, v, eng.bt, before + 1, None, hd ** -0.5) * torch.sigmoid(q[..., hd:].double())
    got = eng.y2[:, : nq * hd].view(M, nq, hd).double()
    assert float((got - want).abs().max()) <= 2.0 ** -5 * float(v.abs().max())


@pytest.mark.parametrize("how", ["steps", "prompt"])
def test_a_4_bit_cache_holds_what_the_bf16_engine_stores(packed, how):
    M, n = 3, 90
    ps = prompts(SMALL.vocab, n)
    eng, ref = qwen27b.Engine(packed, M, maxlen=256, kv_dtype="int4"), qwen27b.Engine(packed, M, maxlen=256)
    for e in (eng, ref):
        if how == "prompt":
            e.prefill([p[: n - 1] for p in ps])
            e.step(torch.tensor([p[n - 1] for p in ps]).cuda())
        else:
            feed(e, ps, n)
    before = torch.full((M,), n - 1, dtype=torch.int32, device="cuda")
    assert eng.pos[:M].tolist() == [n] * M
    # the first attention layer sees the same inputs in both; in a prompt, all layers do
    for ai in range(2 if how == "prompt" else 1):
        for m in range(M):
            for got, x in zip(eng.kv_rows(ai, m, n), ref.kv_rows(ai, m, n)):
                if how == "prompt":                            # cut from the bf16 rows: the same codes, up to the last token's, which was stepped
                    c, s, low = R.encode(x[:, : n - 1])
                    back = (low.double()[..., None] + s.double()[..., None] * c.double()).reshape(x[:, : n - 1].shape)
                    assert torch.equal(got[:, : n - 1].double(), back.float().double())
                    continue
                # cut from 32-bit values, the other side rounded to bf16: half a step (and the 2^-7 by which bf16 scales are wide) and half a bf16 step
                step = (x.reshape(*x.shape[:-1], -1, 64).amax(-1) - x.reshape(*x.shape[:-1], -1, 64).amin(-1)) / 15 * (1 + 2.0 ** -6) + x.abs().amax() * 2.0 ** -10
                d = (got - x).abs().reshape(*x.shape[:-1], -1, 64).amax(-1)
                assert bool((d <= 0.5 * step + x.abs().amax() * 2.0 ** -8).all())
    cos, sin = rope_tables(SMALL.theta, 256, "cuda")
    check_layer(eng, 1, cos, sin, packed.small[(7, "self_attn.q_norm.weight")], before)
    ids = eng.generate(torch.tensor([1, 2, 3]).cuda(), 5)
    assert ids.shape == (5, M) and eng.pos[:M].tolist() == [n + 5] * M and int(ids.min()) >= 0
    again = qwen27b.Engine(packed, M, maxlen=256, kv_dtype="int4")
    if how == "steps":
        feed(again, ps, n)
        assert torch.equal(again.generate(torch.tensor([1, 2, 3]).cuda(), 5), ids)
    eng.check(), paged.check()


def test_a_4_bit_cache_with_padding_rows_and_35b_experts():
    W = qwen35moe.SynthWeights(layers=4, init="realistic", device="cuda", draw_device="cuda")
    PK = qwen35moe.Packed(W, "cuda")
    eng = qwen35moe.Engine(PK, 2, maxlen=128, kv_dtype="int4", kv_pages=5)
    ps = prompts(PK.shape.vocab, 30, M=2)
    for t in range(30):
        eng.step(torch.tensor([p[t] for p in ps]).cuda(), valid=[True, t % 3 != 1])
    assert eng.pos[:2].tolist() == [30, 20]
    alone = qwen35moe.Engine(PK, 2, maxlen=128, kv_dtype="int4")
    kept = [p for t, p in enumerate(ps[1]) if t % 3 != 1]
    for t in range(20):
        alone.step(torch.tensor([ps[0][t], kept[t]]).cuda())
    for a, b in zip(eng.kv_rows(0, 1, 20), alone.kv_rows(0, 1, 20)):
        assert float((a - b).abs().max()) <= 2.0 ** -3 * float(b.abs().max())      # (the other column's expert order may round a code the other way)
    eng.check()


def test_engines_with_one_query_rounding_refuse_what_they_do_not_have(packed):
    for kw in (dict(kv_dtype="int4", kv_layout="serving"), dict(kv_dtype="fp8")):
        with pytest.raises(ValueError):
            qwen27b.Engine(packed, 1, **kw)


# ---- sampled tokens ------------------------------------------------------------------------------------------------
def test_sampled_generation_of_a_large_engine(packed):
    eng = qwen27b.Engine(packed, 2, maxlen=128)
    ps = prompts(SMALL.vocab, 10, M=2)
    feed(eng, ps, 9)
    ids = eng.generate(torch.tensor([p[9] for p in ps]).cuda(), 12, temperature=0.8, top_k=20, top_p=0.9, seed=5)
    ref = qwen27b.Engine(packed, 2, maxlen=128)
    feed(ref, ps, 9)
    u = torch.rand(12, 2, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    tok = torch.tensor([p[9] for p in ps]).cuda()
    for t in range(12):
        tok = sampling.sample(ref.step(tok), u[t], 0.8, 20, 0.9).ids
        assert tok.tolist() == ids[t].tolist()
    eng.reset(), ref.reset()
    feed(eng, ps, 9), feed(ref, ps, 9)
    first = torch.tensor([p[9] for p in ps]).cuda()
    assert torch.equal(eng.generate(first, 6, temperature=0.7, top_k=1), ref.generate(first, 6))       # one candidate: the greedy choice


def test_sampled_generation_of_the_small_engine():
    from megakernels_b200.config import qwen35_08b
    from megakernels_b200.engine import Megakernel
    from megakernels_b200.synth import make_prompt, make_weights
    cfg = qwen35_08b(n_layers=4, vocab=4096)
    w = make_weights(cfg, 0, init="realistic")
    prompt = make_prompt(cfg, 8)
    mk = Megakernel((cfg, w), max_seq=128, quant="int8", pack_device="cpu")
    kw = dict(max_new_tokens=10, temperature=0.9, top_k=30, top_p=0.95, min_p=0.01, seed=11)
    ids = list(mk.generate(prompt, **kw))
    assert len(ids) == 10 and mk.pos == 8 + 9 and mk.pending == ids[-1]
    mk.reset()
    u = torch.rand(10, generator=torch.Generator(device="cuda").manual_seed(11), device="cuda")
    pending = mk.prefill(prompt)
    for i in range(10):
        _, logits = mk.run([pending], n_generate=1, return_logits=True)
        pending, _, kept = R.sample(logits[-1].double().cpu(), float(u[i]), *(float(torch.tensor(v, dtype=torch.float32)) for v in (0.9,)), 30, float(torch.tensor(0.95)), float(torch.tensor(0.01)))
        assert pending == ids[i] and kept <= 30
    mk.reset()
    stop = ids[3]
    cut = list(mk.generate(prompt, stop_ids=[stop], **kw))
    assert cut == ids[: ids.index(stop) + 1]
    mk.reset()
    greedy = list(mk.generate(prompt, max_new_tokens=6))
    mk.reset()
    assert list(mk.generate(prompt, max_new_tokens=6, temperature=1.0, top_k=1)) == greedy
    mk.reset()
    with pytest.raises(ValueError):
        next(mk.generate(prompt, top_p=1.2))
