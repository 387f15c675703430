"""CPU checks of the C ABI of the decoding operators: every declared function is exported, and
host-side refusals come back as status codes with a message before any launch."""

import ctypes
import os
import re

import pytest

from test_serving_abi import Batch, State, _batch, _s

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nanochat_decoding_amd.h")

i32, i64, vp, f32, f64 = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_double
size_t = ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    import torch

    from nanochat_amd import _native as N
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: only where no kernel can be launched")
    lib = ctypes.CDLL(N.LIB_PATH)
    lib.ltv_last_error.restype = ctypes.c_char_p
    for name in ("ltv_paged_attention_fp4_workspace_size", "ltv_paged_cache_reorder_workspace_size",
                 "ltv_beam_select_workspace_size"):
        getattr(lib, name).restype = size_t
    return lib


def test_declared_functions_are_exported(lib):
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"^\s*(?:int|size_t)\s+(ltv_[a-z0-9_]+)\s*\(", src, flags=re.M))
    assert len(names) == 10, sorted(names)
    assert not [n for n in names if not hasattr(lib, n)]
    assert lib.ltv_decoding_abi_version() == 1


def _batch4(**kw):
    return _batch(**(dict(page_size=16) | kw))


def _rotary(lib, dtype=1, batch=None, NH=4, NKVH=2, D=64, fmt=1, eps=0.0, positions=64, tab=1, q=16,
            cos=16, page=None, pages=16):
    s = _s(256, 64, 64)
    row = D // 2 + D // 32
    p = page or (_s(2 * 16 * row, 16 * row, row) if fmt == 1 else _s(2 * 16 * D, 16 * D, D))
    f = lib.ltv_paged_rotary_append
    f.argtypes = [i32, vp, vp, vp, vp, vp, vp, vp, i64, vp, i64, i32, i64, f64, vp, vp, vp, vp, vp, vp,
                  i32, vp, i32, i32, i32, vp]
    return f(dtype, q, s, 16, s, 16, s, cos, D // 2, cos, D // 2, tab, positions, eps, 16, s, pages, p,
             pages, p, fmt, ctypes.byref(batch or _batch4()), NH, NKVH, D, None)


def _refused(lib, rc, code, word):
    assert rc == code, (rc, lib.ltv_last_error())
    assert word in lib.ltv_last_error().decode(), lib.ltv_last_error()


def test_rotary_refusals(lib):
    for kw, code, word in [
            (dict(dtype=7), 1, "dtype"), (dict(fmt=2), 1, "format"), (dict(tab=9), 1, "tables"),
            (dict(positions=63), 1, "positions"), (dict(eps=float("inf")), 1, "norm_eps"),
            (dict(D=12), 2, "head_dim"), (dict(D=136), 2, "head_dim"), (dict(D=48), 2, "4-bit"),
            (dict(NH=-1), 1, "heads"), (dict(q=None), 1, "null"), (dict(cos=None), 1, "null"),
            (dict(pages=None), 1, "null"), (dict(pages=24), 2, "aligned"),
            (dict(page=_s(2 * 16 * 34, 16 * 34, 35)), 2, "dense"),
            (dict(page=_s(2 * 16 * 34 + 8, 16 * 34, 34)), 2, "dense"),
            (dict(batch=_batch4(page_size=24), positions=96), 2, "16 tokens"),
            (dict(batch=_batch4(B=70000, total=70000, num_slots=70000)), 2, "65,535"),
            (dict(batch=_batch4(T=1 << 26, total=1 << 27, B=2)), 2, "too many"),
            (dict(batch=_batch4(total=3)), 1, "B * T"), (dict(batch=_batch4(page_table=None)), 1, "null")]:
        _refused(lib, _rotary(lib, **kw), code, word)
    assert _rotary(lib, batch=_batch4(B=0, total=0)) == 0
    assert _rotary(lib, batch=_batch4(T=0, total=0)) == 0


def test_append_refusals(lib):
    s, p = _s(256, 64, 64), _s(2 * 16 * 34, 16 * 34, 34)
    f = lib.ltv_paged_cache_append_fp4
    f.argtypes = [i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, vp]

    def call(dtype=1, k=16, kp=16, p=p, D=64, NKVH=2, batch=None):
        return f(dtype, k, s, k, s, kp, p, kp, p, ctypes.byref(batch or _batch4()), NKVH, D, None)

    for kw, code, word in [(dict(dtype=3), 1, "dtype"), (dict(k=None), 1, "null"),
                           (dict(D=40), 2, "4-bit"), (dict(kp=8), 2, "aligned"),
                           (dict(p=_s(2 * 16 * 34, 16 * 34, 33)), 2, "dense"),
                           (dict(batch=_batch4(page_size=8)), 2, "16 tokens")]:
        _refused(lib, call(**kw), code, word)
    assert call(batch=_batch4(num_pages=0)) == 0


def test_read_refusals(lib):
    p = _s(2 * 16 * 34, 16 * 34, 34)
    f = lib.ltv_paged_cache_read
    f.argtypes = [i32, i32, vp, vp, vp, vp, vp, vp, vp, i32, i32, vp]

    def call(dtype=1, fmt=1, kp=16, p=p, out=16, D=64, NKVH=2, batch=None):
        return f(dtype, fmt, kp, p, kp, p, ctypes.byref(batch or _batch4()), out, out, NKVH, D, None)

    for kw, code, word in [(dict(dtype=3), 1, "dtype"), (dict(fmt=5), 1, "format"),
                           (dict(out=None), 1, "null"), (dict(out=8), 2, "16-byte"),
                           (dict(D=40), 2, "4-bit"), (dict(kp=None), 1, "null"),
                           (dict(batch=_batch4(B=65535, total=65535, num_slots=65535)), 2, "65,534")]:
        _refused(lib, call(**kw), code, word)
    assert call(batch=_batch4(T=0, total=0)) == 0


def test_attention_refusals(lib):
    s, p = _s(256, 64, 64), _s(2 * 16 * 34, 16 * 34, 34)
    f = lib.ltv_paged_attention_fp4
    f.argtypes = [i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, size_t, i32, i32, i32, i32, f32, vp]

    def call(dtype=1, q=16, kp=16, p=p, out=16, os=s, ws=16, nws=1 << 40, NH=4, NKVH=2, D=64, scale=0.1,
             batch=None):
        return f(dtype, q, s, kp, p, kp, p, ctypes.byref(batch or _batch4()), out, os, None, ws, nws, NH,
                 NKVH, D, 64, scale, None)

    far = _s(1 << 33, 16 * 34, 34)
    for kw, code, word in [
            (dict(dtype=3), 1, "dtype"), (dict(NH=3), 1, "heads"), (dict(D=72), 2, "4-bit"),
            (dict(scale=0.0), 1, "scale"), (dict(scale=float("inf")), 1, "scale"),
            (dict(q=None), 1, "null"), (dict(kp=None), 1, "null"), (dict(kp=24), 2, "aligned"),
            (dict(p=_s(2 * 16 * 34, 16 * 34, 64)), 2, "dense"), (dict(p=far), 2, "32 GiB"),
            (dict(p=_s(-1088, 16 * 34, 34)), 2, "negative"), (dict(ws=None), 4, "workspace"),
            (dict(nws=16), 4, "workspace"), (dict(ws=8), 4, "workspace"), (dict(out=8), 2, "aligned"),
            (dict(os=_s(252, 60, 60)), 2, "aligned"),
            (dict(batch=_batch4(page_size=24)), 2, "16 tokens"),
            (dict(batch=_batch4(T=1 << 28, total=1 << 29)), 2, "too many")]:
        _refused(lib, call(**kw), code, word)
    assert call(batch=_batch4(T=0, total=0)) == 0
    size = lib.ltv_paged_attention_fp4_workspace_size
    size.argtypes = [i32, vp, i32, i32, i32, i32]
    assert size(1, None, 4, 2, 64, 64) == 0 and size(1, ctypes.byref(_batch4()), 4, 2, 64, 64) > 0


def test_reorder_refusals(lib):
    f = lib.ltv_paged_cache_reorder
    f.argtypes = [vp, vp, vp, i32, vp, size_t, vp]
    lib.ltv_paged_cache_reorder_workspace_size.argtypes = [i32, i32]
    assert lib.ltv_paged_cache_reorder_workspace_size(3, 7) == 96
    assert lib.ltv_paged_cache_reorder_workspace_size(0, 7) == 0
    st = State(16, 16, 16, 4, 2, 4, 8, 16)

    def call(state=st, slots=16, n=2, ws=16, nws=40):
        return f(ctypes.byref(state), slots, slots, n, ws, nws, None)

    for kw, code, word in [(dict(n=-1), 1, "entries"), (dict(slots=None), 1, "null"),
                           (dict(n=65536, nws=1 << 30), 2, "65,535"), (dict(nws=39), 4, "workspace"),
                           (dict(ws=None), 4, "workspace"), (dict(ws=8), 4, "workspace"),
                           (dict(state=State(16, 16, None, 4, 2, 4, 8, 16)), 1, "null"),
                           (dict(state=State(16, 16, 16, 3, 2, 4, 8, 16)), 1, "bad state")]:
        _refused(lib, call(**kw), code, word)
    assert call(n=0) == 0 and call(state=State(None, None, None, 4, 0, 4, 0, 16)) == 0


def test_beam_refusals(lib):
    f = lib.ltv_beam_select
    f.argtypes = [i32, vp, i64, vp, vp, vp, vp, vp, vp, size_t, i64, i32, i32, i32, f32, vp]
    size = lib.ltv_beam_select_workspace_size
    size.argtypes = [i64, i32, i32, i32]

    def call(dtype=1, x=16, scores=16, out=16, ws=16, nws=1 << 40, groups=2, beams=4, V=100, k=8, cap=15.0):
        return f(dtype, x, V, scores, None, out, out, out, ws, nws, groups, beams, V, k, cap, None)

    for kw, code, word in [(dict(dtype=3), 1, "dtype"), (dict(k=0), 1, "shape"), (dict(k=401), 1, "shape"),
                           (dict(k=65), 2, "64"), (dict(beams=17, k=64), 2, "1024"),
                           (dict(beams=1025, V=1, k=1025), 2, "1024"), (dict(groups=-1), 1, "shape"),
                           (dict(groups=1 << 19), 2, "too many"), (dict(cap=-1.0), 1, "softcap"),
                           (dict(cap=float("inf")), 1, "softcap"), (dict(cap=float("nan")), 1, "softcap"),
                           (dict(x=None), 1, "null"), (dict(out=None), 1, "null"),
                           (dict(ws=None), 4, "workspace"), (dict(nws=8), 4, "workspace"),
                           (dict(beams=0), 1, "shape"), (dict(V=0), 1, "shape")]:
        _refused(lib, call(**kw), code, word)
    assert call(groups=0) == 0
    assert size(0, 4, 100, 8) == 0 and size(2, 4, 100, 8) == 8 * (8 * 8 + 12)
