"""ctypes binding of the serving operators (`include/mk_serve.h`) and the checks they share; `paged.py` and `sampling.py` are what a
program calls.  There is no CPU path: without the library and a GPU the calls raise."""

import ctypes
import os
import struct

import torch

from . import _lib

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mk_serve.h")
SERVE_EXPORTS = ["mk_page_plan", "mk_heads", "mk_cache_rows", "mk_attend_bytes", "mk_attend", "mk_sample"]
BF16, F16, F32, INT4 = 0, 1, 2, 3
TYPES = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
MAX_REQUESTS, GROUP, MAX_VOCAB, MAX_GROUP_HEADS = 4096, 64, 524288, 128

_u64, _i64, _i32, _f32 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


def _fields(*groups):
    return [(name, kind) for kind, names in groups for name in names.split()]


class PlanArgs(ctypes.Structure):
    _fields_ = _fields((_u64, "lengths new_tokens table held free_pages n_free scratch slots positions rows starts context granted"),
                       (_i32, "requests max_pages page pages room device"))


class CacheDesc(ctypes.Structure):
    _fields_ = _fields((_u64, "k v k_scales v_scales"), (_i64, "s_page s_head s_pos"), (_i32, "type pages kv_heads head_dim page reserved"))


class HeadsArgs(ctypes.Structure):
    _fields_ = _fields((_u64, "q k v q_out k_out positions slots q_norm k_norm cos sin"), (_i64, "q_tok q_head k_tok k_head v_tok v_head"), (CacheDesc, "cache"),
                       (_f32, "eps norm_offset"), (_i32, "tokens q_heads kv_heads head_dim source type rot pairs max_position interleaved v_norm device"))


class AttendArgs(ctypes.Structure):
    _fields_ = _fields((_u64, "q out table context starts workspace status"), (_i64, "q_tok q_head out_tok out_head table_stride"), (CacheDesc, "cache"),
                       (_i64, "spin_limit_ns"), (_f32, "scale"), (_i32, "type requests tokens q_heads max_pages max_new window sinks device"))


class SampleArgs(ctypes.Structure):
    _fields_ = _fields((_u64, "logits u temperature top_p min_p top_k ids logprobs kept"), (_i64, "stride"), (_i32, "rows vocab type device"))


_bound = False


def lib():
    global _bound
    L = _lib.load()
    if not _bound:
        packed, stream = ctypes.c_char_p, ctypes.c_void_p                # (what `pack_...` returns)
        L.mk_page_plan.argtypes = [packed, stream]
        L.mk_heads.argtypes = [packed, stream]
        L.mk_cache_rows.argtypes = [ctypes.POINTER(CacheDesc), _u64, ctypes.c_int, _u64, _u64, ctypes.c_int, stream]
        L.mk_attend_bytes.argtypes = [packed]
        L.mk_attend_bytes.restype = _i64
        L.mk_attend.argtypes = [packed, stream]
        L.mk_sample.argtypes = [packed, stream]
        for name in ("mk_page_plan", "mk_heads", "mk_cache_rows", "mk_attend", "mk_sample"):
            getattr(L, name).restype = ctypes.c_int
        _bound = True
    return L


def packer(struct_class):
    """A function that lays values out as `struct_class` does, field after field (nested descriptors flattened): several times cheaper
    than filling the class, and the small calls here are bound by what the host does."""
    letter = {_u64: "Q", _i64: "q", _i32: "i", _f32: "f"}

    def flat(cls):
        for _, kind in cls._fields_:
            yield from (flat(kind) if kind not in letter else letter[kind])
    layout = struct.Struct("<" + "".join(flat(struct_class)))
    pad = ctypes.sizeof(struct_class) - layout.size                # behind the last field
    return (lambda *values: layout.pack(*values) + bytes(pad)) if pad else layout.pack


pack_plan, pack_heads, pack_attend, pack_sample = (packer(c) for c in (PlanArgs, HeadsArgs, AttendArgs, SampleArgs))
NO_CACHE = (0,) * 13


def on_gpu(*tensors):
    """Refuses tensors (None aside) that are not on one CUDA device; returns its index."""
    first = -1
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()
        if at != first or at < 0:
            if at < 0:
                raise ValueError(f"a tensor on {t.device}: the serving operators have no CPU path")
            if first >= 0:
                raise ValueError(f"tensors on cuda:{first} and {t.device}")
            first = at
    return first


def whole(name, t, *shape):
    """Refuses what is not a contiguous int32 tensor of this shape."""
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def raw_stream(index, stream):
    """The stream a call on the device of this index goes to, as the C ABI takes it."""
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)


def empty(shape, dtype, index, stream):
    """Memory of PyTorch's allocator that belongs to the stream of the call."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=index)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=index)
