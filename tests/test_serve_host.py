"""include/mk_serve.h against the built library and the ctypes mirrors, and the refusals of the serving operators (none of which needs a GPU:
arguments are refused before any CUDA call)."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import serve_reference as R
from megakernels_b200 import _lib, paged, sampling, serve

MIRRORS = {"mk_plan_args": serve.PlanArgs, "mk_cache": serve.CacheDesc, "mk_heads_args": serve.HeadsArgs, "mk_attend_args": serve.AttendArgs, "mk_sample_args": serve.SampleArgs}


def header_text():
    with open(serve.HEADER) as f:
        return re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)


def test_every_declared_function_is_exported(lib_built):
    lib = ctypes.CDLL(lib_built)
    declared = set(re.findall(r"\b(mk_[a-z0-9_]+)\s*\(", header_text()))
    assert declared == set(serve.SERVE_EXPORTS)
    for name in declared:
        assert hasattr(lib, name), name


def test_constants_follow_the_header():
    value = lambda n: int(re.search(rf"{n}\s*=\s*(\d+)", header_text()).group(1))        # noqa: E731
    assert [value("MKV_" + n) for n in ("BF16", "F16", "F32", "INT4")] == [serve.BF16, serve.F16, serve.F32, serve.INT4]
    assert [value("MKV_" + n) for n in ("MAX_REQUESTS", "GROUP", "MAX_VOCAB", "MAX_GROUP_HEADS")] == [serve.MAX_REQUESTS, serve.GROUP, serve.MAX_VOCAB, serve.MAX_GROUP_HEADS]


def test_struct_layouts_match_the_c_compiler(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    lines, want = [], []
    for name, mirror in MIRRORS.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        want.append(ctypes.sizeof(mirror))
        for field, _ in mirror._fields_:
            lines.append(f'printf("%zu ", offsetof({name}, {field}));')
            want.append(getattr(mirror, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mk_serve.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.dirname(serve.HEADER), str(src), "-o", str(exe)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


@pytest.mark.parametrize("mirror,pack", [(serve.PlanArgs, serve.pack_plan), (serve.HeadsArgs, serve.pack_heads), (serve.AttendArgs, serve.pack_attend), (serve.SampleArgs, serve.pack_sample)])
def test_packed_arguments_are_those_of_the_mirror(mirror, pack):
    values, at = [], iter(range(1, 200))

    def fill(cls, obj):
        for name, kind in cls._fields_:
            if hasattr(kind, "_fields_"):
                fill(kind, getattr(obj, name))
            else:
                values.append(next(at))
                setattr(obj, name, values[-1])
    a = mirror()
    fill(mirror, a)
    assert pack(*values) == bytes(a)


def cache(**kw):
    d = dict(k=4096, v=8192, k_scales=0, v_scales=0, s_page=2 * 64 * 128, s_head=64 * 128, s_pos=128, type=serve.BF16, pages=10, kv_heads=2, head_dim=128, page=64, reserved=0)
    d.update(kw)
    return serve.CacheDesc(**d)


BAD_CACHES = [dict(type=serve.F32), dict(type=7), dict(head_dim=96), dict(head_dim=512), dict(page=8), dict(page=48), dict(pages=0), dict(pages=2 ** 27), dict(kv_heads=0), dict(k=0), dict(k=4097),
              dict(v=8), dict(s_pos=4), dict(s_page=-8), dict(type=serve.INT4), dict(type=serve.INT4, k_scales=16, v_scales=24)]


def refused(lib, code, code_name=_lib.MK_ERR_BADARG):
    assert code == code_name, (code, lib.mk_last_error())
    assert lib.mk_last_error()


def test_refusals_of_the_plan(lib_built):
    lib = serve.lib()
    good = dict({n: 4096 for n, k in serve.PlanArgs._fields_ if k is ctypes.c_uint64}, requests=4, max_pages=8, page=64, pages=33, room=16, device=0)
    assert lib.mk_page_plan(None, None) == _lib.MK_ERR_BADARG
    for bad in (dict(requests=0), dict(requests=4097), dict(page=0), dict(page=24), dict(max_pages=0), dict(pages=1), dict(pages=2 ** 26), dict(max_pages=2 ** 26), dict(room=0),
                dict(table=0), dict(slots=2), dict(scratch=4100)):
        refused(lib, lib.mk_page_plan(bytes(serve.PlanArgs(**dict(good, **bad))), None))


def test_refusals_of_the_heads(lib_built):
    lib = serve.lib()
    good = dict(q=4096, k=4096, v=4096, q_out=4096, k_out=0, positions=4096, slots=4096, q_norm=4096, k_norm=4096, cos=4096, sin=4096, q_tok=512, q_head=128, k_tok=256, k_head=128, v_tok=256,
                v_head=128, cache=cache(), eps=1e-6, norm_offset=0, tokens=3, q_heads=4, kv_heads=2, head_dim=128, source=serve.F32, type=serve.BF16, rot=64, pairs=32, max_position=100,
                interleaved=0, v_norm=0, device=0)
    assert lib.mk_heads(None, None) == _lib.MK_ERR_BADARG
    for bad in (dict(tokens=-1), dict(kv_heads=0), dict(q_heads=-1), dict(source=3), dict(type=2), dict(q=0), dict(v=0), dict(slots=0), dict(q_out=8), dict(q=4100), dict(q_tok=-4), dict(k_head=130),
                dict(sin=0), dict(rot=0), dict(rot=256), dict(pairs=33), dict(pairs=0), dict(max_position=0), dict(q_norm=4), dict(kv_heads=3), dict(cache=cache(head_dim=64)),
                dict(cache=serve.CacheDesc())):                                          # no cache and nowhere to put the keys
        refused(lib, lib.mk_heads(bytes(serve.HeadsArgs(**dict(good, **bad))), None))
    for bad in (dict(head_dim=512), dict(rot=20, pairs=5)):
        refused(lib, lib.mk_heads(bytes(serve.HeadsArgs(**dict(good, **bad))), None), _lib.MK_ERR_UNSUPPORTED)
    for bad in BAD_CACHES[1:]:
        if bad != dict(k=0):
            refused(lib, lib.mk_heads(bytes(serve.HeadsArgs(**dict(good, cache=cache(**bad)))), None))
    for bad in BAD_CACHES:
        refused(lib, lib.mk_cache_rows(ctypes.byref(cache(**bad)), 4096, 2, 4096, 4096, 0, None))
    for args in ((None, 4096, 2, 4096, 4096), (ctypes.byref(cache()), 0, 2, 4096, 4096), (ctypes.byref(cache()), 4096, -1, 4096, 4096), (ctypes.byref(cache()), 4096, 2, 4096, 4104)):
        refused(lib, lib.mk_cache_rows(*args, 0, None))
    assert lib.mk_heads(bytes(serve.HeadsArgs(**dict(good, tokens=0))), None) == _lib.MK_OK          # nothing to do


def test_refusals_of_attention(lib_built):
    lib = serve.lib()
    good = dict(q=4096, out=4096, table=4096, context=4096, starts=0, workspace=4096, status=4096, q_tok=512, q_head=128, out_tok=512, out_head=128, table_stride=8, cache=cache(), spin_limit_ns=0,
                scale=0.1, type=serve.BF16, requests=3, tokens=3, q_heads=4, max_pages=8, max_new=1, window=0, sinks=0, device=0)
    assert lib.mk_attend(None, None) == _lib.MK_ERR_BADARG and lib.mk_attend_bytes(None) == _lib.MK_ERR_BADARG
    both = [dict(type=serve.F32), dict(type=serve.F16), dict(requests=0), dict(requests=4097), dict(tokens=-1), dict(tokens=2), dict(max_pages=0), dict(max_pages=2 ** 25), dict(q_heads=3), dict(q_heads=0),
            dict(q_heads=2 * 129), dict(window=-1), dict(sinks=-1), dict(max_new=0), dict(tokens=2 ** 29, starts=4096)] + [dict(cache=cache(**b)) for b in BAD_CACHES]
    for bad in both:
        a = bytes(serve.AttendArgs(**dict(good, **bad)))
        refused(lib, lib.mk_attend_bytes(a))
        refused(lib, lib.mk_attend(a, None))
    for bad in (dict(q=0), dict(out=8), dict(table=0), dict(workspace=0), dict(status=0), dict(workspace=8), dict(q_tok=516), dict(out_head=-8), dict(table_stride=7)):
        refused(lib, lib.mk_attend(bytes(serve.AttendArgs(**dict(good, **bad))), None))
    assert lib.mk_attend(bytes(serve.AttendArgs(**dict(good, tokens=0, starts=4096))), None) == _lib.MK_OK


def test_refusals_of_sampling(lib_built):
    lib = serve.lib()
    good = dict({n: 4096 for n, k in serve.SampleArgs._fields_ if k is ctypes.c_uint64}, stride=1000, rows=2, vocab=1000, type=serve.BF16, device=0)
    assert lib.mk_sample(None, None) == _lib.MK_ERR_BADARG
    for bad in (dict(rows=-1), dict(vocab=0), dict(vocab=serve.MAX_VOCAB + 1), dict(type=serve.INT4), dict(stride=-1), dict(ids=0), dict(u=2), dict(logits=4097), dict(type=serve.F32, logits=4098)):
        refused(lib, lib.mk_sample(bytes(serve.SampleArgs(**dict(good, **bad))), None))
    assert lib.mk_sample(bytes(serve.SampleArgs(**dict(good, rows=0))), None) == _lib.MK_OK


def test_settings_of_sampling():
    sampling.check_settings(0.0, 0, 1.0, 0.0)
    for bad in (dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=2.5), dict(top_k=2 ** 31), dict(top_p=0.0), dict(top_p=1.1),
                dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.5)):
        with pytest.raises(ValueError):
            sampling.check_settings(**bad)


def test_python_refusals_come_before_the_gpu():
    x, u = torch.zeros(2, 10), torch.zeros(2)
    for args, kw in (((x, u), {}), ((x.double(), u), {}), ((x[0], u), {}), ((x.t(), u), {}), ((x, u[:1]), {}), ((x, u.double()), {}), ((x, u), dict(top_k=torch.zeros(2))), ((x, u), dict(top_p=2.0))):
        with pytest.raises(ValueError):
            sampling.sample(*args, **kw)
    k = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    for a in ((k, k), (k.float(), k.float()), (k[..., :96], k[..., :96]), (k[:, :, :12], k[:, :, :12]), (k, k[:3])):
        with pytest.raises(ValueError):
            paged.Cache.of(*a)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            paged.PagePool(4, 10, 4)
    for kw in (dict(requests=0), dict(requests=5000), dict(page=3), dict(pages=1), dict(max_pages=0), dict(max_tokens=0), dict(pages=2 ** 26, page=64)):
        with pytest.raises(ValueError):
            paged.PagePool(**dict(dict(requests=4, pages=10, max_pages=4), **kw))
    q = torch.zeros(3, 4, 128)
    at = torch.zeros(3, dtype=torch.int32)
    for args, kw in (((q, q[:2], at), {}), ((q, q.bfloat16(), at), {}), ((q, q, at.long()), {}), ((q, q, at[:2]), {}), ((q[..., :96], q[..., :96], at), {}), ((q, q, at), dict(dtype=torch.float32)),
                     ((q, q, at), dict(q_norm=torch.zeros(64))), ((q, q, at), dict(rope=(torch.zeros(9, 8), torch.zeros(9, 9)))), ((q, q, at), dict(rope=(torch.zeros(9, 8), torch.zeros(9, 8)), rot=20)),
                     ((q[..., ::2].repeat(1, 1, 2)[..., ::2], q[..., ::2], at), {}), ((q, q, at), {})):
        with pytest.raises(ValueError):
            paged.rotate(*args, **kw)
    with pytest.raises(ValueError):
        paged.enter(q, q, q, at, at, None)
    with pytest.raises(ValueError):
        paged.attend(q.bfloat16(), None, at, at)


def test_refusals_of_scales_and_of_rows_that_overlap(lib_built):
    lib = serve.lib()
    good = dict(q=4096, out=4096, table=4096, context=4096, starts=0, workspace=4096, status=4096, q_tok=512, q_head=128, out_tok=512, out_head=128, table_stride=8, cache=cache(), spin_limit_ns=0,
                scale=0.1, type=serve.BF16, requests=3, tokens=3, q_heads=4, max_pages=8, max_new=1, window=0, sinks=0, device=0)
    for scale in (0.0, -0.5, float("nan"), float("inf"), 2e30):
        refused(lib, lib.mk_attend(bytes(serve.AttendArgs(**dict(good, scale=scale))), None))
        refused(lib, lib.mk_attend_bytes(bytes(serve.AttendArgs(**dict(good, scale=scale)))))
    for bad in (dict(out_tok=0), dict(out_tok=64), dict(out_head=0), dict(out_head=120)):
        refused(lib, lib.mk_attend(bytes(serve.AttendArgs(**dict(good, **bad))), None))


def test_a_pool_belongs_on_a_gpu():
    with pytest.raises(ValueError, match="no CPU path"):
        paged.PagePool(4, 10, 4, device="cpu")


def test_engines_refuse_settings_that_mean_nothing():
    from megakernels_b200.stage.kv import SequenceCalls
    eng = SequenceCalls()
    assert eng._sampled(0.5, 10, 0.9, 0.0) and not eng._sampled(0.0, 0, 1.0, 0.0)
    for bad in ((-0.5, 0, 1.0, 0.0), (float("nan"), 0, 1.0, 0.0), (0.0, -1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 2.0)):
        with pytest.raises(ValueError):
            eng._sampled(*bad)


# ---- what the other tests compare with ---------------------------------------------------------------------------
def test_the_reference_attention_is_a_softmax():
    g = torch.Generator().manual_seed(0)
    k, v, q = torch.randn(1, 1, 16, 64, generator=g).double(), torch.randn(1, 1, 16, 64, generator=g).double(), torch.randn(2, 1, 64, generator=g)
    out = R.attend(q, k, v, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([9]), torch.tensor([0, 2]), 0.3, window=4, sinks=1)
    for t, p in ((0, 7), (1, 8)):
        keys = [0] + list(range(p - 3, p + 1))
        w = torch.exp(torch.tensor([float(q[t, 0].double() @ k[0, 0, j]) * 0.3 for j in keys], dtype=torch.float64))
        want = sum(w[i] / w.sum() * v[0, 0, j] for i, j in enumerate(keys))
        assert float((out[t, 0] - want).abs().max()) < 1e-12


def test_the_reference_codes_come_back():
    x = torch.randn(5, 3, 128, generator=torch.Generator().manual_seed(1)) * 4
    c, s, low = R.encode(x)
    back = R.decode(R.pack(c), torch.stack([s, low], -1).to(torch.bfloat16))
    assert bool(((back - x.double()).abs() <= s.double().repeat_interleave(64, -1) * 0.5001).all())
    assert bool((low.repeat_interleave(64, -1) <= x).all())
    row = R.pack(c)[0, 0]                                       # word (i, g) of a row of [8][2]: values 64 g + 8 i ...
    assert int(row[4 * (2 * 3 + 1)]) == int(c[0, 0, 1, 24]) + 16 * int(c[0, 0, 1, 25])


def test_the_reference_plan_returns_and_takes():
    table, held, free, n, slots, positions, rows, starts, context, granted = R.plan([4, 0, 3], [1, 0, 30], [[7, 0, 0], [5, 6, 0], [8, 0, 0]], [1, 2, 1], [1, 2, 3, 4, 0, 0, 0], 4, 4, 64)
    assert table == [[7, 5, 0], [0, 0, 0], [8, 0, 0]] and held == [2, 0, 1] and free[:5] == [1, 2, 3, 4, 6] and n == 5
    assert granted == [1, 1, 0] and starts == [0, 1, 1, 1] and slots[:2] == [20, -1] and context == [5, 0, 0]
