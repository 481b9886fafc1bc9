"""KV caches that the sequences of an engine share, and 4-bit ones.

`SharedPages`: the engine's block table is that of a `paged.PagePool`; every launch first asks the pool for the pages of the tokens about
to enter, on the GPU, so a cache needs pages for the tokens there are, not for M times the longest context.  A sequence for which there are
no pages waits: it is a padding row of that launch (`mk_stage_args.row_valid`), its state, caches and position are left alone.

`FourBitLayers`: the attention records of a program run outside the stage kernel, on a 4-bit cache: a step is the records up to an
attention layer in one launch, the layer's heads into the cache and attention over it (`paged.enter`, `paged.attend`), the records up
to the next one, and so on.  Prompts that begin a sequence go through the token-parallel path with a bf16 cache of their own, whose
rows are then cut to 4 bits.

The reference keeps one bf16 cache per engine (`qwen3.8-27b-gfx942/mk/runner.py:27-34,103-112`)."""

import ctypes

import torch

from .. import _lib, paged
from . import desc as D
from .runtime import MIN_ROWS_PATH, MAX_ROWS

ROOM = 1024                     # tokens per sequence that one call of the pool places


class SharedPages:
    def __init__(self, M, pages, max_pages, page, device):
        self.M = M
        self.pool = paged.PagePool(M, pages, max_pages, page=page, max_tokens=M * ROOM, device=device)
        self.new = torch.zeros(M, dtype=torch.int32, device=self.pool.device)
        self.live = torch.zeros(M, dtype=torch.int32, device=self.pool.device)

    def reset(self):
        self.pool.reset()

    def ask(self, lengths, n, valid=None):
        """Pages for `n` tokens behind `lengths` (int32 [M]) of every sequence, or of those with valid[m].  Returns (the pool's plan, i32 [M]: which
        sequences go ahead)."""
        if valid is None:
            self.new.fill_(n)
        else:
            torch.mul(valid[: self.M], n, out=self.new)
        plan = self.pool.plan(lengths, self.new)
        if valid is None:
            return plan, plan.granted
        torch.mul(plan.granted, valid[: self.M], out=self.live)
        return plan, self.live

    def ask_all(self, lengths, n):
        """Pages for `n` tokens of every sequence, any number; waits for the device and raises if there are not enough.  Returns the slots, int32 [M, n]."""
        slots = []
        for lo in range(0, n, ROOM):
            part = min(ROOM, n - lo)
            plan, _ = self.ask(lengths + lo, part)
            if int(plan.granted.min()) == 0:
                raise RuntimeError(f"the {self.pool.pages} pages of the cache do not hold {n} more tokens of every sequence")
            slots.append(plan.slots[: self.M * part].view(self.M, part).clone())
        return torch.cat(slots, 1)


class FourBitLayers:
    """`layers`: one dict per attention record of the engine's program, in order: `index` (of the record), `q_norm`, `k_norm` (fp32 [dim]).
    The engine has y, y2, pos, rt, M, device; its rotation tables are `rope`."""

    def __init__(self, eng, layers, rope, pages, page, max_pages):
        self.eng, self.layers, self.rope = eng, layers, rope
        rt, M, dev = eng.rt, eng.M, eng.device
        stages = eng.prog.stages
        self.records = [stages[l["index"]] for l in layers]
        f = lambda d, n: d.i[D.K["MKS_I_" + n]]                                        # noqa: E731
        d = self.records[0]
        self.nq, self.nkv, self.hd, self.rot = f(d, "NQ"), f(d, "NKV"), f(d, "HD"), f(d, "ROT")
        self.caches = [paged.Cache(pages, self.nkv, self.hd, page=page, dtype="int4", device=dev) for _ in layers]
        cuts = [-1] + [l["index"] for l in layers] + [len(stages)]
        self.parts = []
        for i in range(len(cuts) - 1):
            records = [D.StageDesc.from_buffer_copy(s) for s in stages[cuts[i] + 1: cuts[i + 1]]]
            last = i == len(cuts) - 2
            if i == 0:
                records[0].i[D.K["MKS_I_KEYS_VALID"]] = 0                              # the token is chosen behind the LM head
            if last:
                first = D.StageDesc.from_buffer_copy(stages[0])                        # an embedding of width 0: the choice at the end of the launch
                first.i[D.K["MKS_I_HIDDEN"]] = 0
                records = [first] + records
            self.parts.append(rt.upload(records))
        self.positions = torch.zeros(len(self.parts), D.MAX_BATCH, dtype=torch.int32, device=dev)      # every part but the last advances a copy
        self.max_pages, self.page = max_pages, page
        self._staged = None

    def _heads(self, y, d):
        """Views of a projection's rows: queries, their gates, keys, values."""
        f = lambda n: d.i[D.K["MKS_I_" + n]]                                           # noqa: E731
        M, hd = y.shape[0], self.hd
        qs = y[:, f("A_Q_OFF"): f("A_Q_OFF") + self.nq * f("A_Q_HSTRIDE")].view(M, self.nq, f("A_Q_HSTRIDE"))
        k, v = (y[:, o: o + self.nkv * hd].view(M, self.nkv, hd) for o in (f("A_K_OFF"), f("A_V_OFF")))
        return qs[..., :hd], qs[..., f("A_GATE_OFF"): f("A_GATE_OFF") + hd], k, v

    def step(self, plan, live, tokens_out=None, stream=None):
        """One decode step of the sequences that `live` marks (the token ids are in rt.tok)."""
        eng, rt, M = self.eng, self.eng.rt, self.eng.M
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(eng.device)):
            self.positions.copy_(rt.pos.expand_as(self.positions))
            at = self.positions[-1, :M]
            first = plan.starts[:M].long().clamp(max=plan.slots.shape[0] - 1)
            slots = torch.where(live > 0, plan.slots[first], -1)
            for i, part in enumerate(self.parts):
                last = i == len(self.parts) - 1
                rt.launch(1, program=part, pos=rt.pos if last else self.positions[i], row_valid=live, tokens_out=tokens_out if last else None)
                if last:
                    break
                d, layer = self.records[i], self.layers[i]
                q, gate, k, v = self._heads(eng.y, d)
                q = paged.enter(q, k, v, at, slots, self.caches[i], rope=self.rope, rot=self.rot, q_norm=layer["q_norm"], k_norm=layer["k_norm"], norm_offset=1.0,
                                eps=d.f[D.K["MKS_F_EPS"]], dtype=torch.bfloat16)
                out = paged.attend(q, self.caches[i], plan.table, plan.context, scale=d.f[D.K["MKS_F_SCALE"]])
                torch.mul(out, torch.sigmoid(gate), out=eng.y2[:, : self.nq * self.hd].view(M, self.nq, self.hd))

    def prefill(self, tokens):
        """Prompts [L, M] at the start of all sequences, all positions at once; False if that path does not take them (they step then)."""
        eng, rt, M = self.eng, self.eng.rt, self.eng.M
        L = tokens.shape[0]
        if L < MIN_ROWS_PATH or rt.tp != 1:
            return False
        nb = -(-L // self.page)
        shape = (len(self.layers), M * nb, self.page, self.nkv, self.hd)
        try:
            k, v = (torch.empty(shape, dtype=torch.bfloat16, device=eng.device) for _ in "kv")
        except torch.cuda.OutOfMemoryError:
            return False
        table = torch.arange(M * nb, dtype=torch.int32, device=eng.device).view(M, nb)
        host = (D.StageDesc * rt.n_stages)(*[D.StageDesc.from_buffer_copy(s) for s in rt.host])
        row = self.nkv * self.hd
        for i, layer in enumerate(self.layers):
            d = host[layer["index"]]
            d.i[D.K["MKS_I_MAX_PAGES"]], d.i[D.K["MKS_I_KV_BLOCK"]] = nb, self.page
            d.i[D.K["MKS_I_KV_S_PAGE"]], d.i[D.K["MKS_I_KV_S_HEAD"]], d.i[D.K["MKS_I_KV_S_POS"]] = self.page * row, self.hd, row
            d.p[D.K["MKS_P_K_CACHE"]], d.p[D.K["MKS_P_V_CACHE"]], d.p[D.K["MKS_P_BLOCK_TABLE"]] = k[i].data_ptr(), v[i].data_ptr(), table.data_ptr()
        each = -(-L // -(-L * M // MAX_ROWS))
        need = int(rt.lib.mk_stage_prefill_bytes(host, rt.n_stages, M, each, eng.device.index))
        if need == _lib.MK_ERR_UNSUPPORTED:
            return False
        if need < 0:
            _lib.check(need)
        if not rt.workspace_room(need):
            return False
        slots = eng.pages.ask_all(rt.pos[:M], L)
        whole, rt.host = rt.host, host
        try:
            rt.prefill(tokens)
        finally:
            rt.host = whole
        flat = slots.reshape(-1)
        for i, cache in enumerate(self.caches):
            rows = [x[i].view(M, nb * self.page, self.nkv, self.hd)[:, :L].reshape(M * L, self.nkv, self.hd) for x in (k, v)]
            cache.put(*rows, flat)
        return True


class SequenceCalls:
    """How an engine (with M, rt, pos, device, lm_head, logits) advances its sequences: over pages of its own, shared ones (`pages`) or a 4-bit cache (`kv4`), with
    the greedy choice of the kernel or a sampled one."""

    pages = kv4 = None

    def _advance(self, valid, stream=None, tokens_out=None):
        """One step of the tokens in rt.tok; `valid` as `_rows` returns it."""
        if self.pages is None:
            return self.rt.launch(1, stream=stream, row_valid=valid, tokens_out=tokens_out)
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(self.device)):
            plan, live = self.pages.ask(self.pos[: self.M], 1, valid)
            if self.kv4 is not None:
                self.kv4.step(plan, live, tokens_out)
            else:
                self.rt.launch(1, row_valid=live, tokens_out=tokens_out)

    def _advance_greedy(self, n_steps, out):
        """`n_steps` steps from the tokens in rt.tok, each fed the greedy choice of the one before; the choices to out [n_steps, M]."""
        if self.pages is None:
            return self.rt.launch(n_steps, tokens_out=out)
        if self.kv4 is not None:
            for t in range(n_steps):
                self._advance(None, tokens_out=out[t: t + 1])
            return
        for lo in range(0, n_steps, ROOM):
            part = out[lo: lo + ROOM]
            _, live = self.pages.ask(self.pos[: self.M], part.shape[0])
            self.rt.launch(part.shape[0], tokens_out=part, row_valid=live)

    def _sampled(self, temperature, top_k, top_p, min_p):
        """Whether the tokens are sampled; refuses settings that mean nothing."""
        from .. import sampling
        sampling.check_settings(temperature, top_k, top_p, min_p)
        return temperature > 0

    def _advance_sampled(self, tok, n_steps, temperature, top_k, top_p, min_p, seed):
        from .. import sampling
        return sampling.continue_from(lambda t: self.step(t), tok.to(self.device), n_steps, temperature, top_k, top_p, min_p, seed)

    def _take_in(self, tokens):
        """Prompts int32 [L, M] on the device enter; the logits are those after the last position."""
        if self.pages is None:
            return self.rt.prefill(tokens)
        if self.kv4 is None:
            self.pages.ask_all(self.pos[: self.M], tokens.shape[0])
            return self.rt.prefill(tokens)
        if int(self.pos[: self.M].max()) == 0 and self.kv4.prefill(tokens):
            return
        for t in range(tokens.shape[0]):
            self.rt.tok[: self.M].copy_(tokens[t])
            self._advance(None)

    def release(self, m):
        """Sequence m starts over: position 0 and an empty recurrent state.  Pages it shared are free again with the next step."""
        if not 0 <= m < self.M:
            raise ValueError(f"sequence {m} of {self.M}")
        self.pos[m] = 0
        for state in (getattr(self, "conv", None), getattr(self, "ssm", None)):
            if state is not None:
                state[:, m].zero_()
