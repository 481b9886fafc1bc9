"""The next token from logits: temperature, top-k, top-p and min-p, from given uniform numbers, in one launch (`mk_sample`).

The engines choose the arg-max or a Gumbel-max at a temperature inside their kernels (`qwen3.5-0.8b/qwen_mk/engine.py:198-250`
in the reference); what else a request asks for is chosen here, from the logits they return."""

from collections import namedtuple

import torch

from . import _lib, serve

Sample = namedtuple("Sample", "ids logprobs kept")


def check_settings(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Refuses settings (numbers) that mean nothing."""
    if not 0.0 <= temperature < float("inf"):
        raise ValueError(f"temperature {temperature} (0 or more; 0 takes the largest logit)")
    if not (0 <= top_k < 2 ** 31 and int(top_k) == top_k):
        raise ValueError(f"top_k {top_k} (a whole number; 0 keeps all)")
    if not 0.0 < top_p <= 1.0:
        raise ValueError(f"top_p {top_p} (above 0, at most 1)")
    if not 0.0 <= min_p <= 1.0:
        raise ValueError(f"min_p {min_p} (0 to 1)")


_NEUTRAL = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}


def _per_row(name, value, rows, device, stream):
    dtype = torch.int32 if name == "top_k" else torch.float32
    if torch.is_tensor(value):
        if value.dtype != dtype or value.shape != (rows,) or not value.is_contiguous():
            raise ValueError(f"{name}: a number or contiguous {dtype} [{rows}], got {value.dtype} {list(value.shape)}")
        return value
    check_settings(**{**_NEUTRAL, name: value})
    return serve.empty((rows,), dtype, device, stream)             # filled below: the refusals come first


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, stream=None):
    """logits [rows, vocab] (fp32, bf16 or fp16; rows may be apart), u fp32 [rows] in [0, 1) -> Sample(ids int32 [rows], logprobs fp32
    [rows], kept int32 [rows]).

    Per row, with weights w = exp((x - max) / temperature): candidates in the order (x falling, index rising); the first `top_k`
    (0: all); of these the fewest that hold `top_p` of their weight; of these those with w >= `min_p`.  The token is the first, by
    index, at which the running weight of the kept ones exceeds u times their sum; `logprobs` is the logarithm of its share, `kept` how
    many were left.  Temperature 0 takes the largest, the lowest index among equals.  Masked logits (-inf, NaN) are never kept; a row of
    nothing else gives id -1.  The settings are numbers, or one per row (fp32, `top_k` int32; their values are not looked at, which
    would wait for the device: top_p of 0 or less keeps one, 1 or more all, min_p above 1 counts as 1).  Asynchronous."""
    if logits.dim() != 2 or logits.dtype not in serve.TYPES or not 1 <= logits.shape[1] <= serve.MAX_VOCAB or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"logits: fp32, bf16 or fp16 [rows, vocab of at most {serve.MAX_VOCAB}] with neighbouring columns, got {logits.dtype} {list(logits.shape)}")
    rows, vocab = logits.shape
    if u.dtype != torch.float32 or u.shape != (rows,) or not u.is_contiguous():
        raise ValueError(f"u: contiguous fp32 [{rows}]")
    settings = (temperature, top_k, top_p, min_p)
    device = serve.on_gpu(logits, u, *[v for v in settings if torch.is_tensor(v)])
    lib = serve.lib()
    t, k, p, m = (_per_row(n, v, rows, device, stream) for n, v in zip(_NEUTRAL, settings))
    for have, asked in zip((t, k, p, m), settings):
        if have is not asked:
            if stream is None:
                have.fill_(asked)
            else:
                with torch.cuda.stream(stream):
                    have.fill_(asked)
    out = serve.empty((3, rows), torch.int32, device, stream)
    ids, logprobs, kept = out.unbind(0)
    logprobs = logprobs.view(torch.float32)
    if rows:
        a = serve.pack_sample(logits.data_ptr(), u.data_ptr(), t.data_ptr(), p.data_ptr(), m.data_ptr(), k.data_ptr(), ids.data_ptr(), logprobs.data_ptr(), kept.data_ptr(),
                              logits.stride(0), rows, vocab, serve.TYPES[logits.dtype], device)
        code = lib.mk_sample(a, serve.raw_stream(device, stream))
        if code:
            _lib.check(code)
    return Sample(ids, logprobs, kept)


def continue_from(step, tok, n_steps, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed=0):
    """`n_steps` sampled tokens of every sequence: `step(tok [rows]) -> logits [rows, vocab]` takes one token of each in.  The uniform numbers
    are those of a generator seeded with `seed`.  Returns int32 [n_steps, rows] on the device; nothing waits for it."""
    check_settings(temperature, top_k, top_p, min_p)
    rows, device = tok.shape[0], tok.device
    u = torch.rand(n_steps, rows, generator=torch.Generator(device=device).manual_seed(seed), device=device)
    settings = [torch.full((rows,), v, dtype=torch.int32 if n == "top_k" else torch.float32, device=device) for n, v in zip(_NEUTRAL, (temperature, top_k, top_p, min_p))]
    out = torch.empty(n_steps, rows, dtype=torch.int32, device=device)
    for t in range(n_steps):
        out[t] = sample(step(tok), u[t], *settings).ids
        tok = out[t].clamp(min=0)                                  # (a padding row's logits are nothing in particular)
    return out
