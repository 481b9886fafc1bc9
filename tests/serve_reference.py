"""The serving operators in 64 bits, one request, row or token at a time; what their tests compare with."""

import math

import torch

GROUP = 64


def plan(lengths, new, table, held, free, n, page, room):
    """Lists in, lists out: (table, held, free, n, slots, positions, rows, starts, context, granted)."""
    P = len(table[0])
    table, held, free = [list(t) for t in table], list(held), list(free)
    back = []
    for r, length in enumerate(lengths):
        base = min(held[r], -(-max(length, 0) // page))
        back += table[r][base: held[r]]
        table[r][base: held[r]] = [0] * (held[r] - base)
        held[r] = base
    for i, p in enumerate(reversed(back)):
        free[n + i] = p
    n += len(back)
    slots, positions, rows, starts, granted, context = [], [], [], [0], [], []
    open_, asked_pages, asked_tokens, height = True, 0, 0, n
    for r, (length, k) in enumerate(zip(lengths, new)):
        need = -(-(length + k) // page)
        ok = length >= 0 and k >= 0 and need <= P
        if not ok:
            granted.append(0), context.append(0), starts.append(len(slots))
            continue
        take = max(need - held[r], 0)
        asked_pages, asked_tokens = asked_pages + take, asked_tokens + k
        open_ = open_ and asked_pages <= height and asked_tokens <= room
        if open_ or (take == 0 and k == 0):
            for _ in range(take):
                n -= 1
                table[r][held[r]] = free[n]
                held[r] += 1
            for p in range(length, length + k):
                slots.append(table[r][p // page] * page + p % page), positions.append(p), rows.append(r)
            granted.append(1), context.append(length + k)
        else:
            granted.append(0), context.append(length)
        starts.append(len(slots))
    pad = room - len(slots)
    return table, held, free, n, slots + [-1] * pad, positions + [0] * pad, rows + [-1] * pad, starts, context, granted


def heads(x, weight, offset, eps, rope, positions, rot, interleaved):
    """Norm (weight None: none; True: without a weight) and rotation of [tokens, heads, dim], in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        if weight is not True:
            x = x * (offset + weight.double())
    if rope is None:
        return x
    cos, sin = (t.double()[positions.long()][:, None] for t in rope)
    out = x.clone()
    for d in range(cos.shape[-1]):
        i, j = (2 * d, 2 * d + 1) if interleaved else (d, d + rot // 2)
        a, b, c, s = x[..., i], x[..., j], cos[..., d], sin[..., d]
        out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    return out


def bf16_down(x):
    """Largest bf16 at or below the fp32 x."""
    y = x.to(torch.bfloat16).float()
    below = torch.nextafter(y.to(torch.bfloat16), torch.tensor(-math.inf, dtype=torch.bfloat16, device=x.device)).float()
    return torch.where(y > x, below, y)


def encode(x):
    """fp32 [..., dim] -> codes [..., dim / 64, 64] (whole numbers), scale, low [..., dim / 64]."""
    x = x.float().reshape(*x.shape[:-1], -1, GROUP)
    low = bf16_down(x.amin(-1))
    scale = -bf16_down(-((x.amax(-1) - low) * torch.full((), 1 / 15, device=x.device)))
    c = torch.where(scale[..., None] > 0, ((x - low[..., None]) / scale[..., None]).round(), 0.0).clamp(0, 15)
    return c, scale, low


def pack(c):
    """codes [..., groups, 64] -> uint8 [..., groups * 32] in the cache's order."""
    lead, g = c.shape[:-2], c.shape[-2]
    w = c.to(torch.int64).reshape(*lead, g, 8, 8).transpose(-3, -2)                     # [..., 8, groups, 8 codes]
    b = w[..., 0::2] | (w[..., 1::2] << 4)
    return b.reshape(*lead, g * 32).to(torch.uint8)


def decode(codes, scales):
    """The cache's tensors -> fp64 values [..., dim]."""
    lead, g = codes.shape[:-1], codes.shape[-1] // 32
    b = codes.reshape(*lead, 8, g, 4).transpose(-3, -2).to(torch.int64)
    c = torch.stack([b & 15, b >> 4], -1).reshape(*lead, g, GROUP).double()
    s = scales.double()
    return (s[..., 1:] + s[..., :1] * c).reshape(*lead, g * GROUP)


def attend(q, k, v, table, context, starts, scale, window=0, sinks=0, out=None):
    """q [tokens, heads, dim]; k, v fp64 [pages, kv heads, page, dim]."""
    T, nq, dim = q.shape
    pages, nkv, page = k.shape[:3]
    out = torch.zeros(T, nq, dim, dtype=torch.float64, device=q.device) if out is None else out.double().clone()
    starts = starts.tolist() if starts is not None else list(range(len(context) + 1))
    for r, length in enumerate(context.tolist()):
        a, b = starts[r], starts[r + 1]
        length = min(max(length, 0), table.shape[1] * page)
        ids = table[r, : -(-length // page)].long()
        good = (ids >= 0) & (ids < pages)
        ids = torch.where(good, ids, 0)
        kk = k[ids].transpose(1, 2).reshape(-1, nkv, dim)[:length] if length else k.new_zeros(0, nkv, dim)
        vv = v[ids].transpose(1, 2).reshape(-1, nkv, dim)[:length] if length else k.new_zeros(0, nkv, dim)
        key = torch.arange(length, device=q.device)
        there = good.repeat_interleave(page)[:length]
        for t in range(a, b):
            p = length - (b - t)
            seen = (key <= p) & there
            if window:
                seen &= (key > p - window) | (key < sinks)
            if not bool(seen.any()):
                out[t] = 0
                continue
            x = torch.einsum("gjd,ngd->gjn", q[t].double().view(nkv, nq // nkv, dim), kk[seen]) * scale
            out[t] = torch.einsum("gjn,ngd->gjd", torch.softmax(x, -1), vv[seen]).reshape(nq, dim)
    return out


def sample(x, u, t, k, p, m):
    """One row (numbers); x fp64 [vocab] on the host -> (id, logprob, kept)."""
    x = [v if v == v else -math.inf for v in x.tolist()]
    live = [i for i, v in enumerate(x) if v > -math.inf]
    if not live:
        return -1, -math.inf, 0
    order = sorted(live, key=lambda i: (-x[i], i))
    if not t > 0:
        t, k = 1.0, 1
    top = x[order[0]]
    w = lambda i: 1.0 if x[i] == top else math.exp((x[i] - top) / t)                   # noqa: E731
    if k > 0:
        order = order[:k]
    if p < 1:
        total, run, n = math.fsum(w(i) for i in order), 0.0, 0
        while n < len(order) and (n == 0 or run < p * total):
            run += w(order[n])
            n += 1
        order = order[:n]
    order = sorted(i for i in order if w(i) >= m)
    total, run = math.fsum(w(i) for i in order), 0.0
    for i in order:
        run += w(i)
        if run > u * total:
            break
    return i, math.log(w(i) / total) if w(i) > 0 else -math.inf, len(order)
