"""CPU checks of the serving operators' C ABI: every declared function is exported, and
host-side refusals come back as status codes with a message before any launch."""

import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nanochat_serving_amd.h")

i32, i64, vp = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p


class Batch(ctypes.Structure):
    _fields_ = [("page_table", vp), ("seq_lens", vp), ("slots", vp), ("starts", vp),
                ("table_stride", i64), ("total", i64), ("B", i32), ("T", i32),
                ("num_slots", i32), ("num_pages", i32), ("table_width", i32),
                ("page_size", i32)]


class State(ctypes.Structure):
    _fields_ = [("page_table", vp), ("seq_lens", vp), ("ref_counts", vp), ("table_stride", i64),
                ("num_slots", i32), ("table_width", i32), ("num_pages", i32), ("page_size", i32)]


class Blocks(ctypes.Structure):
    _fields_ = [("k", vp), ("v", vp), ("k_page_bytes", i64), ("k_layer_bytes", i64),
                ("v_page_bytes", i64), ("v_layer_bytes", i64), ("block_bytes", i64),
                ("layers", i32), ("num_pages", i32)]


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
    for name in ("ltv_paged_attention_workspace_size", "ltv_paged_cache_reserve_workspace_size",
                 "ltv_paged_cache_compact_workspace_size"):
        getattr(lib, name).restype = ctypes.c_size_t
    return lib


def test_declared_functions_are_exported(lib):
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"^\s*(?:int|size_t)\s+(ltv_[a-z0-9_]+)\s*\(", src, flags=re.M))
    assert len(names) == 14, sorted(names)
    assert not [n for n in names if not hasattr(lib, n)]
    assert lib.ltv_serving_abi_version() == 1


def _s(*v):
    return (i64 * len(v))(*v)


def _batch(**kw):
    b = dict(page_table=16, seq_lens=16, slots=None, starts=None, table_stride=4, total=2, B=2,
             T=1, num_slots=2, num_pages=8, table_width=4, page_size=16)
    b.update(kw)
    return Batch(**b)


def _attention(lib, dtype=1, batch=None, NH=4, NKVH=2, D=64, scale=0.1, q=16):
    s = _s(64, 64, 64)
    lib.ltv_paged_attention.argtypes = [
        i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, ctypes.c_size_t, i32, i32, i32, i32,
        ctypes.c_float, vp]
    return lib.ltv_paged_attention(dtype, q, s, 16, s, 16, s,
                                   ctypes.byref(batch or _batch()), 16, s, None, None, 0, NH,
                                   NKVH, D, 64, scale, None)


def test_attention_refusals(lib):
    # (the pointers are never read: each call is refused on the host)
    for code, kw in ((1, dict(dtype=7)), (1, dict(NH=5)), (1, dict(NKVH=0)), (1, dict(D=0)),
                     (2, dict(D=60)), (2, dict(D=136)), (1, dict(scale=0.0)),
                     (1, dict(scale=float("nan"))), (1, dict(q=None)),
                     (1, dict(batch=_batch(page_size=0))), (1, dict(batch=_batch(B=-1))),
                     (1, dict(batch=_batch(total=3))), (1, dict(batch=_batch(table_stride=3))),
                     (1, dict(batch=_batch(B=3, total=3))),
                     (1, dict(batch=_batch(seq_lens=None))),
                     (2, dict(batch=_batch(page_size=1 << 20, table_width=1 << 12,
                                           table_stride=1 << 12)))):
        assert _attention(lib, **kw) == code, kw
        assert lib.ltv_last_error() != b""
    # nothing to do: no launch
    assert _attention(lib, batch=_batch(B=0, total=0)) == 0
    assert _attention(lib, NH=0) == 0


def _state(**kw):
    s = dict(page_table=16, seq_lens=16, ref_counts=16, table_stride=4, num_slots=2,
             table_width=4, num_pages=8, page_size=16)
    s.update(kw)
    return State(**s)


def _blocks(**kw):
    b = dict(k=16, v=16, k_page_bytes=64, k_layer_bytes=512, v_page_bytes=64, v_layer_bytes=512,
             block_bytes=64, layers=1, num_pages=8)
    b.update(kw)
    return Blocks(**b)


def test_cache_refusals(lib):
    def reserve(state=None, blocks=None, n=1, ws=16, bytes_=1 << 20, slots=16):
        return lib.ltv_paged_cache_reserve(ctypes.byref(state or _state()),
                                           ctypes.byref(blocks or _blocks()), vp(slots), vp(16),
                                           n, vp(16), vp(ws), ctypes.c_size_t(bytes_), None)

    for code, kw in ((1, dict(n=0)), (1, dict(slots=None)), (4, dict(bytes_=8)),
                     (1, dict(state=_state(page_size=0))), (1, dict(state=_state(num_pages=9))),
                     (1, dict(state=_state(ref_counts=None))),
                     (2, dict(blocks=_blocks(block_bytes=24))), (2, dict(blocks=_blocks(k=8))),
                     (2, dict(blocks=_blocks(v_page_bytes=40))), (1, dict(blocks=_blocks(v=None)))):
        assert reserve(**kw) == code, kw
    st, bl = _state(), _blocks()
    assert lib.ltv_paged_cache_fork(ctypes.byref(st), None, None, 0, None) == 0
    assert lib.ltv_paged_cache_fork(ctypes.byref(st), None, None, 1, None) == 1
    assert lib.ltv_paged_cache_free(ctypes.byref(st), vp(16), 70000, None) == 2
    assert lib.ltv_paged_cache_copy(ctypes.byref(bl), None, None, 2, None) == 1
    assert lib.ltv_paged_cache_compact(ctypes.byref(st), ctypes.byref(bl), vp(16), vp(16),
                                       ctypes.c_size_t(4), None) == 4
    b, s = _batch(), _s(64, 64, 64)
    assert lib.ltv_paged_cache_append(9, vp(16), s, vp(16), s, vp(16), s, vp(16), s,
                                      ctypes.byref(b), 2, 64, None) == 1
    assert lib.ltv_paged_cache_append(1, None, s, vp(16), s, vp(16), s, vp(16), s,
                                      ctypes.byref(b), 2, 64, None) == 1


def test_logprobs_refusals(lib):
    f = lib.ltv_token_logprobs_forward
    f.argtypes = [i32, vp, i64, vp, vp, vp, vp, vp, vp, vp, ctypes.c_size_t, i64, i32, i32,
                  ctypes.c_float, vp]

    def call(dtype=0, x=16, lp=16, top=16, N=2, V=100, k=0, cap=0.0, ws=None, nws=0):
        return f(dtype, x, V, 16, lp, None, None, top, top, ws, nws, N, V, k, cap, None)

    for code, kw in ((1, dict(dtype=5)), (1, dict(V=0)), (1, dict(k=101)), (2, dict(k=65)),
                     (1, dict(k=-1)), (1, dict(cap=-1.0)), (1, dict(cap=float("inf"))),
                     (1, dict(cap=float("nan"))), (1, dict(x=None)), (1, dict(lp=None)),
                     (1, dict(k=2, top=None)), (1, dict(N=-1)), (4, dict(V=65536)),
                     (4, dict(V=65536, nws=1 << 20)), (4, dict(V=65536, ws=8, nws=1 << 20))):
        assert call(**kw) == code, kw
    assert call(N=0) == 0
