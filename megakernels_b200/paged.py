"""A paged KV cache as a serving loop uses it: which pages a request holds, how heads enter the cache, and attention over it.

`PagePool.plan` builds block tables and slot maps on the GPU from request lengths; `enter` norms and rotates query and key heads
and writes keys and values to their slots (`rotate`: without a cache); `attend` is attention of any number of queries per request
over the cache, with a sliding window and first tokens that stay visible.  A `Cache` holds 16-bit elements, in the layouts of the
engines' own caches (the reference's serving layout is described at `qwen3.8-27b-gfx942/mk/kernel.py:15-27`), or 4-bit codes.

Every call is asynchronous on the current stream (or `stream`), allocates what it returns and its workspace from PyTorch's allocator, and
can be captured into a CUDA graph.  PyTorch allocates device memory; the work goes through the C ABI of `include/mk_serve.h`."""

import ctypes
from collections import namedtuple

import torch

from . import _lib, serve

Plan = namedtuple("Plan", "table slots positions rows starts context granted")


class PagePool:
    """Pages of `page` tokens for up to `requests` requests of at most `max_pages` pages each.  Page 0 is the null page: never handed
    out, and what a table holds behind a request's pages."""

    def __init__(self, requests, pages, max_pages, page=64, max_tokens=None, device="cuda"):
        """`pages`: all pages of the cache, page 0 among them; `max_tokens`: new tokens of one call (the size of the slot maps)."""
        max_tokens = requests if max_tokens is None else max_tokens
        if not 1 <= requests <= serve.MAX_REQUESTS:
            raise ValueError(f"{requests} requests (1 to {serve.MAX_REQUESTS})")
        if page < 1 or page & (page - 1):
            raise ValueError(f"{page} tokens per page (a power of two)")
        if pages < 2 or max_pages < 1 or max_tokens < 1:
            raise ValueError(f"{pages} pages, at most {max_pages} per request, {max_tokens} tokens a call")
        if max(pages, max_pages) * page >= 2 ** 31:
            raise ValueError(f"{pages} pages, at most {max_pages} per request, of {page} tokens exceed 32-bit slots")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"a page pool on {dev}: the serving operators have no CPU path")
        if not torch.cuda.is_available():
            raise RuntimeError("the page pool needs a CUDA device; there is no CPU path")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.requests, self.pages, self.max_pages, self.page, self.max_tokens, self.device = requests, pages, max_pages, page, max_tokens, dev
        z = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)          # noqa: E731
        self.table, self.held, self.free, self.n_free = z(requests, max_pages), z(requests), z(pages - 1), z(1)
        self.slots, self.positions, self.rows = z(max_tokens), z(max_tokens), z(max_tokens)
        self.starts, self.context, self.granted = z(requests + 1), z(requests), z(requests)
        self.scratch = z(8 * requests + 8)
        self.lib = serve.lib()
        self._args = (*(t.data_ptr() for t in (self.table, self.held, self.free, self.n_free, self.scratch, self.slots, self.positions, self.rows, self.starts, self.context, self.granted)),
                      requests, max_pages, page, pages, max_tokens, dev.index)
        self._plan = Plan(self.table, self.slots, self.positions, self.rows, self.starts, self.context, self.granted)
        self.reset()

    def reset(self):
        """All pages free again; the lowest is handed out first."""
        self.table.zero_(), self.held.zero_()
        self.free.copy_(torch.arange(self.pages - 1, 0, -1, dtype=torch.int32, device=self.device))
        self.n_free.fill_(self.pages - 1)

    def plan(self, lengths, new, stream=None):
        """`lengths` int32 [requests]: tokens in the cache; `new` int32 [requests]: tokens about to enter (0: none).  Returns the pool's
        own buffers, overwritten by the next call:

        table [requests, max_pages], slots / positions / rows [max_tokens] (cache slot, position and request of every new token,
        requests one after the other; -1, 0, -1 behind the last), starts [requests + 1], context [requests] (tokens in the cache
        once the granted ones have entered), granted [requests].

        A request holds the pages of its first `lengths` tokens: what it holds beyond them (it has ended: length 0; drafts were
        rejected) is free again before pages for new tokens are taken, in request order.  The first request that does not fit, for
        want of pages or of `max_tokens`, and every later one that asks for anything, waits: granted 0, no slots.  A negative number, or more than `max_pages`
        pages, is not granted and holds up nobody.  The pool is one state: its calls belong on one stream, in order."""
        serve.whole("lengths", lengths, self.requests)
        serve.whole("new", new, self.requests)
        serve.on_gpu(self.table, lengths, new)
        code = self.lib.mk_page_plan(serve.pack_plan(lengths.data_ptr(), new.data_ptr(), *self._args), serve.raw_stream(self.device.index, stream))
        if code:
            _lib.check(code)
        return self._plan


class Cache:
    """Keys and values of one layer in pages.  16 bits: `k`, `v` [pages, kv heads, page, head dim] (views of any strides with
    neighbouring dims).  4 bits: `k`, `v` uint8 [pages, kv heads, page, head dim / 2] and `k_scales`, `v_scales` bf16 [pages, kv
    heads, page, head dim / 64, 2]: every 64 values of a head share (scale, low), value = low + scale * code, codes 0 .. 15.  The
    codes of 8 consecutive values share a 32-bit word, the first in the lowest bits; a row's words are stored [8][head dim / 64],
    word (i, g) holding values 64 g + 8 i .. 64 g + 8 i + 7."""

    def __init__(self, pages, kv_heads, head_dim, page=64, dtype=torch.bfloat16, device="cuda", layout="pages"):
        """`dtype`: torch.bfloat16, torch.float16 or "int4"; `layout` (16 bits): "pages", or "serving": memory ordered [page][position][kv head][dim]."""
        if layout not in ("pages", "serving") or (layout == "serving" and dtype == "int4"):
            raise ValueError("layout: 'pages', or 'serving' for 16-bit elements")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head dim {head_dim} (64, 128 or 256)")
        if dtype == "int4":
            k, v = (torch.zeros(pages, kv_heads, page, head_dim // 2, dtype=torch.uint8, device=device) for _ in "kv")
            ks, vs = (torch.zeros(pages, kv_heads, page, head_dim // serve.GROUP, 2, dtype=torch.bfloat16, device=device) for _ in "kv")
            self._take(k, v, ks, vs)
        else:
            shape = (pages, kv_heads, page, head_dim) if layout == "pages" else (pages, page, kv_heads, head_dim)
            k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in "kv")
            if layout == "serving":
                k, v = k.transpose(1, 2), v.transpose(1, 2)
            self._take(k, v, None, None)

    @classmethod
    def of(cls, k, v):
        """A cache over 16-bit tensors that exist already, [pages, kv heads, page, head dim] (an engine's; a serving layout as a transposed view)."""
        c = cls.__new__(cls)
        c._take(k, v, None, None)
        return c

    @classmethod
    def of_codes(cls, k, k_scales, v, v_scales):
        """A cache over 4-bit tensors that exist already, contiguous."""
        c = cls.__new__(cls)
        c._take(k, v, k_scales, v_scales)
        return c

    def _take(self, k, v, ks, vs):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v: [pages, kv heads, page, head dim] of one type and layout")
        self.pages, self.kv_heads, self.page = k.shape[:3]
        self.int4 = ks is not None
        self.head_dim = k.shape[3] * (2 if self.int4 else 1)
        self.k, self.v, self.k_scales, self.v_scales = k, v, ks, vs
        if self.head_dim not in (64, 128, 256):
            raise ValueError(f"head dim {self.head_dim} (64, 128 or 256)")
        if self.page < 16 or self.page & (self.page - 1):
            raise ValueError(f"{self.page} tokens per page (a power of two, 16 or more)")
        if not 1 <= self.pages * self.page < 2 ** 31 or self.kv_heads < 1:
            raise ValueError(f"{self.pages} pages of {self.page} tokens, {self.kv_heads} heads (slots have 32 bits)")
        self.device = torch.device("cuda", serve.on_gpu(k, v, ks, vs))
        if self.int4:
            shape = (self.pages, self.kv_heads, self.page, self.head_dim // serve.GROUP, 2)
            if k.dtype != torch.uint8 or not (k.is_contiguous() and v.is_contiguous()):
                raise ValueError("4-bit codes: contiguous uint8")
            if any(s.dtype != torch.bfloat16 or s.shape != shape or not s.is_contiguous() for s in (ks, vs)):
                raise ValueError(f"scales: contiguous bf16 {list(shape)}")
            self.dtype, strides = "int4", (0, 0, 0)
        else:
            if k.dtype not in (torch.bfloat16, torch.float16):
                raise ValueError(f"elements of {k.dtype} (bf16, fp16, or 4-bit codes)")
            if k.stride(3) != 1 or any(s % 8 for s in k.stride()[:3]):
                raise ValueError("strides: neighbouring dims, the others multiples of 8 elements")
            self.dtype, strides = k.dtype, k.stride()[:3]
        if any(t is not None and t.data_ptr() % 16 for t in (k, v, ks, vs)):
            raise ValueError("a cache tensor does not start on a 16-byte boundary")
        at = lambda t: t.data_ptr() if t is not None else 0                            # noqa: E731
        self._args = (at(k), at(v), at(ks), at(vs), *strides, serve.INT4 if self.int4 else serve.TYPES[k.dtype], self.pages, self.kv_heads, self.head_dim, self.page, 0)
        self.desc = serve.CacheDesc(*self._args)
        _status_of(self.device.index)

    def put(self, k, v, slots, stream=None):
        """Keys and values [tokens, kv heads, head dim] (fp32, bf16 or fp16) as they are to `slots` (int32 [tokens]); -1 is padding."""
        _heads(k[:, :0], k, v, slots, slots, self, None, None, None, None, 0.0, 0.0, False, False, self.dtype if not self.int4 else torch.bfloat16, None, stream)

    def rows(self, slots, stream=None):
        """Keys and values in `slots` (int32 [tokens]) as [tokens, kv heads, head dim]: fp32 from a 4-bit cache, else the cache's type; zeros
        for a slot outside it (-1)."""
        n = slots.numel()
        serve.whole("slots", slots, n)
        serve.on_gpu(self.k, slots)
        out = serve.empty((2, n, self.kv_heads, self.head_dim), torch.float32 if self.int4 else self.dtype, self.device.index, stream)
        k, v = out[0], out[1]
        if n:
            code = serve.lib().mk_cache_rows(ctypes.byref(self.desc), slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), self.device.index, serve.raw_stream(self.device.index, stream))
            if code:
                _lib.check(code)
        return k, v


def _heads(q, k, v, positions, slots, cache, rope, rot, q_norm, k_norm, norm_offset, eps, interleaved, v_norm, dtype, out, stream):
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q [tokens, query heads, dim] and k [tokens, KV heads, dim], got {list(q.shape)} and {list(k.shape)}")
    (T, nq, dim), (Tk, nkv, dim_k), source = q.shape, k.shape, q.dtype
    if T != Tk or dim != dim_k or nkv < 1:
        raise ValueError(f"q [tokens, query heads, dim] and k [tokens, KV heads, dim], got {list(q.shape)} and {list(k.shape)}")
    if dim not in (64, 128, 256):
        raise ValueError(f"head dim {dim} (64, 128 or 256)")
    if source not in serve.TYPES or k.dtype != source or (v is not None and (v.dtype != source or v.shape != k.shape)):
        raise ValueError("q, k, v: one type (fp32, bf16 or fp16), v like k")
    (qt, qh, qd), (kt, kh, kd), (vt, vh, vd) = q.stride(), k.stride(), v.stride() if v is not None else (0, 0, 1)
    if qd != 1 or kd != 1 or vd != 1:
        raise ValueError("q, k, v: neighbouring dims")
    serve.whole("positions", positions, T)
    if cache is not None:
        serve.whole("slots", slots, T)
        if cache.kv_heads != nkv or cache.head_dim != dim:
            raise ValueError(f"a cache of {cache.kv_heads} heads of {cache.head_dim}, keys of {nkv} of {dim}")
    if dtype is None:
        dtype = source if source != torch.float32 else (cache.dtype if cache is not None and not cache.int4 else torch.bfloat16)
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError(f"dtype {dtype} (bf16 or fp16)")
    for w in (q_norm, k_norm):
        if w is not None and (w.dtype != torch.float32 or w.shape != (dim,) or not w.is_contiguous()):
            raise ValueError(f"q_norm, k_norm: contiguous fp32 [{dim}]")
    cos = sin = None
    angles = longest = 0
    if rope is not None:
        cos, sin = rope
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape or not (cos.is_contiguous() and sin.is_contiguous()) or not cos.numel():
            raise ValueError("rope: (cos, sin), contiguous fp32 [positions, angles]")
        longest, angles = cos.shape
        rot = 2 * angles if rot is None else rot
        if not 2 <= rot <= dim or rot % (dim // 16) or angles > rot // 2:
            raise ValueError(f"{rot} rotated dims of {dim} with {angles} angles (rot a multiple of {dim // 16})")
    device = serve.on_gpu(q, k, v, positions, slots, cache.k if cache is not None else None, q_norm, k_norm, cos, sin, out)
    if out is None:
        out = serve.empty((T, nq, dim), dtype, device, stream)
    elif out.shape != q.shape or out.dtype != dtype or not out.is_contiguous():
        raise ValueError(f"out: contiguous {dtype} {list(q.shape)}")
    k_out = serve.empty((T, nkv, dim), dtype, device, stream) if cache is None else None
    if T:
        a = serve.pack_heads(q.data_ptr(), k.data_ptr(), v.data_ptr() if v is not None else 0, out.data_ptr(), k_out.data_ptr() if k_out is not None else 0, positions.data_ptr(),
                             slots.data_ptr() if slots is not None else 0, q_norm.data_ptr() if q_norm is not None else 0, k_norm.data_ptr() if k_norm is not None else 0,
                             cos.data_ptr() if cos is not None else 0, sin.data_ptr() if sin is not None else 0, qt, qh, kt, kh, vt, vh, *(cache._args if cache is not None else serve.NO_CACHE),
                             eps, norm_offset, T, nq, nkv, dim, serve.TYPES[source], serve.TYPES[dtype], rot or 0, angles, longest, bool(interleaved), bool(v_norm), device)
        code = serve.lib().mk_heads(a, serve.raw_stream(device, stream))
        if code:
            _lib.check(code)
    return out, k_out


def rotate(q, k, positions, rope=None, rot=None, q_norm=None, k_norm=None, norm_offset=0.0, eps=1e-6, interleaved=False, dtype=None, stream=None):
    """Norm and rotation of query and key heads in one pass: q [tokens, query heads, dim], k [tokens, KV heads, dim] (fp32, bf16 or
    fp16, any strides with neighbouring dims) -> (q', k') of `dtype` (default: the inputs', bf16 for fp32).

    y = x * rsqrt(mean(x^2) + eps) * (norm_offset + weight) where a weight is given; then pairs (d, d + rot / 2), or (2 d, 2 d + 1) if
    `interleaved`, turned by angle d of the row `positions[t]` of `rope` = (cos, sin), fp32 [positions, angles <= rot / 2] (dims
    without an angle stay).  A token at a position outside the tables is padding: zeros."""
    return _heads(q, k, None, positions, None, None, rope, rot, q_norm, k_norm, norm_offset, eps, interleaved, False, dtype, None, stream)


def enter(q, k, v, positions, slots, cache, rope=None, rot=None, q_norm=None, k_norm=None, norm_offset=0.0, eps=1e-6, interleaved=False, v_norm=False, dtype=None, out=None,
          stream=None):
    """`rotate`, with the keys and the values `v` (`v_norm`: normed without a weight) written to `slots` (int32 [tokens]) of `cache`
    instead of being returned; returns q' [tokens, query heads, dim].  A token whose slot lies outside the cache (-1) is padding:
    its queries are zeros and nothing is written.  No two tokens of a call may have the same slot."""
    if not isinstance(cache, Cache) or v is None or slots is None:
        raise ValueError("enter needs values, slots and a paged.Cache")
    return _heads(q, k, v, positions, slots, cache, rope, rot, q_norm, k_norm, norm_offset, eps, interleaved, v_norm, dtype, out, stream)[0]


_status, _bytes = {}, {}


def _status_of(index):
    """Where the calls on a device leave word of a wait that ran out.  Its zeros are there before any stream's first call: not part of a graph, which would
    write them at every replay."""
    st = _status.get(index)
    if st is None:
        with torch.cuda.device(index):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first paged.Cache of a device cannot be made inside a graph capture")
            st = torch.zeros(4, dtype=torch.int32, device=index)
            torch.cuda.current_stream().synchronize()
        _status[index] = st
    return st


def check(device=None):
    """Synchronise and raise if a device-side wait ran out in any call so far on this device (default: the current one)."""
    index = torch.device("cuda" if device is None else device).index
    if index is None:
        index = torch.cuda.current_device()
    st = _status_of(index).tolist()
    if st[0] != 0:
        _status_of(index).zero_()
        raise _lib.MkError(_lib.MK_ERR_TIMEOUT, f"a device-side wait ran out (site {st[1]}, CTA {st[2]}, thread {st[3]})")


def attend(q, cache, table, context, starts=None, max_new=None, scale=None, window=0, sinks=0, out=None, stream=None):
    """Causal attention over a paged cache: q [tokens, query heads, dim] (the cache's type; bf16 or fp16 over 4 bits) -> out of the same
    shape and type.

    `table` int32 [requests, pages]: page of every page number (rows may be apart); `context` int32 [requests]: tokens in the cache, the queries'
    own among them; `starts` int32 [requests + 1]: first query of every request (without it: one query per request, in order), of which none has
    more than `max_new` (default: any number).  Query t of request r is at position context[r] - (starts[r + 1] - t) and sees the keys j up to its
    own position with j > position - window or j < sinks (window 0: all of them).  A query that sees nothing gives
    zeros; keys in a page that the table does not place inside the cache are not seen; rows of `out` outside the requests' queries are
    left alone.  Query head h uses KV head h // (query heads / KV heads).  `scale` (positive) defaults to dim ** -0.5.

    What no query of the call sees is not looked at and may hold anything.  Values that some query sees have to be finite: neighbouring queries
    multiply the same tile of them, those that do not see a key by 0."""
    if not isinstance(cache, Cache):
        raise ValueError("cache: a paged.Cache")
    if q.dim() != 3 or q.dtype not in (torch.bfloat16, torch.float16) or (not cache.int4 and q.dtype != cache.dtype):
        raise ValueError(f"q: [tokens, query heads, dim] of the cache's 16-bit type, got {q.dtype} {list(q.shape)}")
    T, nq, dim = q.shape
    nkv = cache.kv_heads
    if dim != cache.head_dim or nq % nkv or not 1 <= nq // nkv <= serve.MAX_GROUP_HEADS:
        raise ValueError(f"{nq} query heads of {dim} over {nkv} KV heads of {cache.head_dim}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.stride(1) != 1:
        raise ValueError(f"table: int32 [requests, pages] with neighbouring columns, got {table.dtype} {list(table.shape)}")
    R, pages = table.shape
    if not 1 <= R <= serve.MAX_REQUESTS or not 1 <= pages * cache.page <= 2 ** 30:
        raise ValueError(f"{R} requests (1 to {serve.MAX_REQUESTS}) of up to {pages} pages (at most 2^30 tokens)")
    if R > 1 and table.stride(0) < pages:
        raise ValueError("table: rows overlap")
    serve.whole("context", context, R)
    if starts is not None:
        serve.whole("starts", starts, R + 1)
    elif T != R:
        raise ValueError(f"{T} queries for {R} requests: give starts")
    if max_new is None:
        max_new = 1 if starts is None else max(T, 1)
    if max_new < 1 or window < 0 or sinks < 0:
        raise ValueError(f"max_new {max_new} (1 or more), window {window}, sinks {sinks} (0 or more)")
    device = serve.on_gpu(q, cache.k, table, context, starts, out)
    lib = serve.lib()
    if out is None:
        out = serve.empty(q.shape, q.dtype, device, stream)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError(f"out: {q.dtype} {list(q.shape)}")
    if T == 0:
        return out
    (qt, qh, qd), (ot, oh, od) = q.stride(), out.stride()
    if qd != 1 or od != 1:
        raise ValueError("q, out: neighbouring dims")
    if (T > 1 and ot < dim) or (nq > 1 and oh < dim):
        raise ValueError(f"out: rows of {dim} overlap at strides {ot}, {oh}")
    fixed = (qt, qh, ot, oh, table.stride(0), *cache._args, 0, dim ** -0.5 if scale is None else scale, serve.TYPES[q.dtype], R, T, nq, pages, min(max_new, T),
             min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1), device)
    front = (q.data_ptr(), out.data_ptr(), table.data_ptr(), context.data_ptr(), starts.data_ptr() if starts is not None else 0)
    need = _bytes.get((device, dim))                               # it depends on nothing else
    if need is None:
        need = lib.mk_attend_bytes(serve.pack_attend(*front, 0, 0, *fixed))
        if need < 0:
            _lib.check(int(need))
        _bytes[device, dim] = need
    work = serve.empty((need,), torch.uint8, device, stream)
    code = lib.mk_attend(serve.pack_attend(*front, work.data_ptr(), _status_of(device).data_ptr(), *fixed), serve.raw_stream(device, stream))
    if code:
        _lib.check(code)
    return out
