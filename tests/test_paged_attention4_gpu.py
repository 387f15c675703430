"""Attention over a paged cache held in 4 bits against float64 over the values that it holds,
element by element, within the bound of its roundings."""

from __future__ import annotations

import math

import pytest
import torch

from fp4_test_utils import Cache4, parts4
from paged_test_utils import DEV, attention64, attention_bound, lse_bound

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _run(cache, q, new, packed, slots=None, scale=None, **hints):
    """Per-sequence (out, lse) of the operator; q: list of (n_i, NH, D)."""
    kw = dict(hints)
    if slots is not None:
        kw["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
    if packed:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        kw["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        x = torch.cat(q)
    else:
        x = torch.stack(q)
    out, lse = _ops().paged_attention(x, cache.k_pages, cache.v_pages, cache.table, cache.lens,
                                      scale=scale, return_lse=True, **kw)
    assert out.shape == x.shape and out.dtype == x.dtype and lse.shape == x.shape[:-1]
    if packed:
        return list(zip(out.split(list(new)), lse.split(list(new))))
    return list(zip(out, lse))


def _check(got, want, dtype, D, lens):
    """attention_bound's, and of bfloat16 the output's own rounding as torch.finfo has it (2^-8 of
    the value, where that bound counts 2^-9 of the sum of the terms' sizes)."""
    for i, ((out, lse), (o64, l64, mag, big)) in enumerate(zip(got, want)):
        bound = attention_bound(dtype, D, lens[i], mag, big)
        if dtype == BF:
            bound = bound + 2.0 ** -8 * o64.abs()
        err = (out.double() - o64).abs()
        nan = o64.isnan()
        assert torch.equal(out.isnan(), nan), i
        assert bool((err <= bound)[~nan].all()), (
            i, float((err / bound)[~nan].max()), float(err[~nan].max()))
        empty = l64 == -math.inf
        assert torch.equal(lse == -math.inf, empty), i
        assert bool((out[empty] == 0).all())
        e = (lse.double() - l64)[~empty]
        assert torch.equal(e.isnan(), l64[~empty].isnan())
        ok = (e.abs() <= lse_bound(D, lens[i], l64[~empty], big)) | e.isnan()
        assert bool(ok.all()), (i, float(e.abs().max()))


# Pages that a table has room for where tiles of 128 rows are to be taken: the calls that are small by
# their rows and by the longest sequence that there may be go in tiles of 16.
ROOM = 1 << 14


def _widen(cache, room):
    if room:
        cache.table = torch.nn.functional.pad(cache.table, (0, room), value=-1)


def _case(dtype, NH, NKVH, D, page, new, cached, packed, seed=0, slots=None, layout="dense",
          qscale=1.0, poison=None, room=0, **hints):
    lens = [a + b for a, b in zip(new, cached)]
    order = list(range(len(lens))) if slots is None else slots
    held = [0] * (max(order) + 1 if order else 0)
    for s, n in zip(order, lens):
        held[s] = n
    cache = Cache4(held, NKVH, D, page, seed, layout=layout)
    _widen(cache, room)
    if poison is not None:
        poison(cache)
        cache.decode()
    q = [(cache.rand(n, NH, D) * qscale).to(dtype) for n in new]
    got = _run(cache, q, new, packed, slots, **hints)
    want = attention64(q, cache, order, new, D ** -0.5)
    _check(got, want, dtype, D, lens)


HEADS = [(6, 6, 128, 64), (8, 4, 128, 16), (10, 5, 64, 48), (8, 1, 96, 32), (3, 1, 32, 16),
         (16, 2, 128, 128), (32, 1, 64, 16), (40, 2, 96, 304), (5, 5, 32, 48), (12, 12, 64, 32)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D,page", HEADS)
def test_decode(NH, NKVH, D, page, dtype):
    """One token per sequence; lengths around the tiles' and pages' ends."""
    cached = [0, 1, 2, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 127, 128, 255, 400, 511, 1000]
    _case(dtype, NH, NKVH, D, page, [1] * len(cached), cached, packed=False)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D,page", HEADS)
def test_chunks(NH, NKVH, D, page, dtype):
    """Ragged chunks in one call, a sequence without new tokens among them."""
    _case(dtype, NH, NKVH, D, page, [1, 5, 0, 33, 64, 2, 130], [0, 7, 20, 0, 65, 300, 131],
          packed=True, seed=1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("T,cached", [(1, 3000), (3, 2049), (17, 900), (40, 1500), (257, 100), (512, 0)])
def test_longer(T, cached, D, dtype):
    _case(dtype, 4, 2, D, 32, [T] * 2, [cached, cached // 3], packed=False, seed=2, qscale=3.0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D,page", HEADS)
def test_chunks_of_many_rows(NH, NKVH, D, page, dtype):
    """.. in tiles of 128 rows."""
    n = 8192 // NH
    _case(dtype, NH, NKVH, D, page, [1, 5, 0, 33, n, 2, 130], [0, 7, 20, 0, 65, 300, 131],
          packed=True, seed=1, room=ROOM)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("T,cached", [(257, 100), (512, 0), (300, 1700)])
def test_longer_of_many_rows(T, cached, D, dtype):
    _case(dtype, 20, 2, D, 32, [T] * 2, [cached, cached // 3], packed=False, seed=2, qscale=3.0,
          room=ROOM)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D", [(4, 1, 64), (6, 6, 128), (24, 1, 96)])
def test_long_context_split_over_many(NH, NKVH, D, dtype):
    """Few rows, a long and a short context: the keys are split and joined."""
    _case(dtype, NH, NKVH, D, 64, [1, 1, 2], [40000, 10, 9000], packed=True, seed=3, qscale=2.0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B", [257, 700])
def test_many_sequences(B, dtype):
    """More sequences than a workgroup has threads, most of them short, some in chunks."""
    new = [1 + (i % 97 == 5) * (i % 150) for i in range(B)]
    new[B // 2] = 0
    _case(dtype, 4, 2, 64, 16, new, [(i * 37) % 230 for i in range(B)], packed=True, seed=23)


@pytest.mark.parametrize("max_len", [None, 1, 64, 100000])
@pytest.mark.parametrize("max_new", [None, 1, 40])
def test_hints(max_new, max_len):
    """They choose launch shapes, not which keys are read."""
    _case(BF, 4, 2, 64, 16, [1, 40, 3], [700, 60, 0], packed=True, seed=4, max_new=max_new,
          max_len=max_len)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["dense", "apart"])
def test_slots_layouts_scale(layout, dtype):
    _case(dtype, 4, 2, 96, 16, [1, 3, 40], [90, 0, 33], packed=True, slots=[2, 0, 3], layout=layout,
          seed=5)


def _nan_scale(cache, which, slot, pos, block=0):
    pages = getattr(cache, which)
    s = parts4(pages)[1]
    s[int(cache.table[slot, pos // cache.page]), :, block, pos % cache.page] = 255


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("which", ["k_pages", "v_pages"])
@pytest.mark.parametrize("NH,new", [(2, 1), (2, 5), (16, 1), (4, 40), (2, 300), (32, 100)])
def test_nan_in_sight(NH, new, which, dtype):
    """32 channels that are NaN: of a key every row that sees it is NaN, of a value those channels."""

    def poison(cache):
        _nan_scale(cache, which, 0, 30, 1)
        _nan_scale(cache, which, 1, 100 + new // 2, 0)

    _case(dtype, NH, 2, 64, 16, [new] * 3, [80, 100, 50], packed=False, seed=6, poison=poison,
          room=ROOM if NH == 32 else 0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 3, 40, 300, 1100])
def test_nan_out_of_sight(new, dtype):
    """What no row sees -- past the end, in pages of no sequence, behind the causal mask -- does not
    reach one, whatever its bytes are."""

    def poison(cache):
        ps = cache.page
        for which in ("k_pages", "v_pages"):
            codes, s = parts4(getattr(cache, which))
            for slot, n in enumerate(cache.lens.tolist()):
                page = int(cache.table[slot, (n - 1) // ps])
                s[page, :, :, (n - 1) % ps + 1:] = 255
            used = set(cache.table.flatten().tolist())
            for p in range(cache.P):
                if p not in used:
                    s[p] = 255
            _nan_scale(cache, which, 1, int(cache.lens[1]) - 1)

    _case(dtype, 4, 2, 128, 16, [new] * 2, [83, 100], packed=False, seed=7, poison=poison,
          room=ROOM if new == 1100 else 0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 20, 200, 1100])
def test_missing_pages(new, dtype):
    """Ids outside the pages hold no keys; a sequence of none gives 0 and -inf."""

    def poison(cache):
        cache.table[0, 2] = -1
        cache.table[0, 4] = cache.P + 3
        cache.table[1, :] = -5

    _case(dtype, 4, 2, 64, 16, [new] * 2, [150, 30], packed=False, seed=8, poison=poison,
          room=ROOM if new == 1100 else 0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [5, 90, 1100])
def test_more_new_than_tokens(new, dtype):
    """Tokens at negative positions see nothing."""
    cache = Cache4([3, 40], 2, 64, 16, 9)
    _widen(cache, ROOM if new == 1100 else 0)
    q = [cache.rand(new, 4, 64, dtype=dtype) for _ in range(2)]
    got = _run(cache, q, [new] * 2, False)
    want = attention64(q, cache, [0, 1], [new] * 2, 64 ** -0.5)
    _check(got, want, dtype, 64, [3, 40])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 70, 1100])
def test_large_scores(new, dtype):
    """Scores of thousands: one key takes all, exponents far from 0."""
    _case(dtype, 4, 2, 64, 16, [new] * 2, [300, 20], packed=False, seed=10, qscale=3000.0,
          room=ROOM if new == 1100 else 0)


@pytest.mark.parametrize("new", [1, 60, 1100])
def test_extreme_scales(new):
    """Scales at both ends of their range."""

    def poison(cache):
        for which, low in (("k_pages", 60), ("v_pages", 2)):
            s = parts4(getattr(cache, which))[1]
            s.copy_(torch.randint(low, low + 3, s.shape, device=DEV))
            s[:, :, 0] = 120

    _case(F32, 4, 2, 64, 16, [new] * 2, [100, 20], packed=False, seed=11, poison=poison,
          room=ROOM if new == 1100 else 0)

    def large(cache):
        s = parts4(cache.v_pages)[1]
        s.fill_(249)

    _case(BF, 4, 2, 64, 16, [new] * 2, [100, 20], packed=False, seed=12, poison=large,
          room=ROOM if new == 1100 else 0)


def test_pages_past_32_bits():
    """Pages of 5 GiB: appended to, attended to and read as those of a small array are."""
    ops, D, ps, NKVH = _ops(), 128, 64, 8
    row = ops.fp4_row_bytes(D)
    P = 5 * 2 ** 30 // (NKVH * ps * row)
    small = Cache4([300, 90], NKVH, D, ps, 20)
    far = torch.cat([torch.arange(P - 4, P), torch.arange(4)]).flip(0).to(DEV, torch.int32)
    table = torch.full_like(small.table, -1)
    k, v = (torch.empty(P, NKVH, ps, row, dtype=torch.uint8, device=DEV) for _ in range(2))
    place = {}
    for i, page in enumerate(p for p in small.table.flatten().tolist() if 0 <= p < small.P):
        place[page] = int(far[i])
        k[far[i].long()] = small.k_pages[page]
        v[far[i].long()] = small.v_pages[page]
    for old, new in place.items():
        table[small.table == old] = new
    assert max(place.values()) * NKVH * ps * row > 2 ** 32
    new = [small.rand(2, 5, NKVH, D, dtype=BF) for _ in range(2)]
    for kp, vp, t in ((small.k_pages, small.v_pages, small.table), (k, v, table)):
        ops.paged_cache_append(*new, kp, vp, t, small.lens)
    for T, NH in ((1, 8), (30, 64), (2, 64)):
        q = small.rand(2, T, NH, D, dtype=BF)
        f = lambda *c: ops.paged_attention(q, *c, small.lens)  # noqa: E731
        assert torch.equal(f(small.k_pages, small.v_pages, small.table), f(k, v, table))
        wide = [torch.nn.functional.pad(t, (0, ROOM), value=-1) for t in (small.table, table)]
        assert torch.equal(f(small.k_pages, small.v_pages, wide[0]), f(k, v, wide[1]))
    for a, b in zip(ops.paged_cache_read(small.k_pages, small.v_pages, small.table, small.lens, 90),
                    ops.paged_cache_read(k, v, table, small.lens, 90)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("max_len", [None, 2048])
@pytest.mark.parametrize("new", [1, 256])
def test_probabilities_are_not_rounded_to_bfloat16(new, max_len):
    """All keys of a row but one have the same probability, so that its roundings would add up: outputs
    are within their own rounding (half a step of bfloat16), float32 sums, and the two bfloat16 parts of
    a probability, whose second is off by 2^-8 of at most 2^-8, whatever room for keys there is."""
    NH, NKVH, D, n = 8, 2, 64, 2000
    cache = Cache4([n, n // 3], NKVH, D, 16, 30)
    _widen(cache, ROOM)
    for which in ("k_pages", "v_pages"):
        codes, s = parts4(getattr(cache, which))
        s.fill_(127)
        if which == "k_pages":
            codes.zero_()
            for i in range(2):  # the first key: 1 in the first channel
                codes[int(cache.table[i, 0]), :, 0, 0] = 2
        else:
            codes.copy_((torch.arange(D // 2, device=DEV) % 7 + 1) * 17)
            for i in range(2):
                codes[int(cache.table[i, 0]), :, 0] = 0
    cache.decode()
    lens = [n, n // 3]
    q = [torch.zeros(new, NH, D, dtype=BF, device=DEV) for _ in lens]
    for x in q:
        x[..., 0] = (4.0 + 40.0 * torch.rand(new, NH, generator=cache.g, device=DEV)).to(BF)
    got = _run(cache, q, [new] * 2, False, max_len=max_len)
    for i, ((out, _), (o64, _, mag, big)) in enumerate(
            zip(got, attention64(q, cache, [0, 1], [new] * 2, D ** -0.5))):
        u = 2.0 ** -24
        off = mag * (2.0 ** -16 + u * (4 * (D + 8) * (1 + big) + 2 * lens[i] + 64))
        half = 2.0 ** ((o64.abs() + off).clamp(min=1e-30).log2().floor() - 8)
        err = (out.double() - o64).abs()
        assert bool((err <= half + off).all()), (i, float((err / (half + off)).max()))


def test_query_strides():
    cache = Cache4([90, 33], 2, 64, 16, 13)
    big = cache.rand(2, 4, 9, 70, dtype=BF)
    q = big[:, :, 1:8, 3:67].transpose(1, 2)
    f = lambda q: _ops().paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.lens)  # noqa: E731
    assert torch.equal(f(q), f(q.contiguous()))
    assert torch.equal(f(q), f(q.transpose(2, 3).contiguous().transpose(2, 3)))


@pytest.mark.parametrize("new", [1, 50, 1100])
def test_rows_of_no_sequence_and_again(new):
    """A call does not depend on the one before, nor write rows of no sequence."""
    cache = Cache4([400, 33], 2, 64, 16, 14)
    _widen(cache, ROOM if new == 1100 else 0)
    q = cache.rand(2, new, 4, 64, dtype=BF)
    a = _ops().paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.lens)
    other = Cache4([900] * 5, 2, 64, 16, 15)
    _ops().paged_attention(other.rand(5, 3, 4, 64, dtype=BF), other.k_pages, other.v_pages, other.table,
                           other.lens)
    b = _ops().paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.lens)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("new,cached", [([1, 1, 1], [5000, 3, 90]), ([40, 1, 200], [60, 3000, 700]),
                                        ([1100, 0, 3], [200, 5, 0])])
def test_rows_of_no_sequence_are_left(new, cached, room, dtype):
    """Rows before the first sequence and behind the last one, and what is between the heads' rows,
    stay as they were, in the output and in the log-sum-exps; cut tiles among them."""
    import ctypes

    from nanochat_amd import _native as N
    from test_serving_abi import Batch, _s

    _ops()
    N.torch_ext()
    lib = ctypes.CDLL(N.LIB_PATH)
    vp, i32 = ctypes.c_void_p, ctypes.c_int
    NH, NKVH, D, ps, before, behind = 8, 2, 64, 16, 3, 5
    lens = [a + b for a, b in zip(new, cached)]
    cache = Cache4(lens, NKVH, D, ps, 31)
    _widen(cache, room)
    starts = [before]
    for n in new:
        starts.append(starts[-1] + n)
    total = starts[-1] + behind
    q = cache.rand(total, NH, D, dtype=dtype)
    out = torch.full((total, NH, D + 16), 77.0, dtype=dtype, device=DEV)
    lse = torch.full((total, NH), 77.0, device=DEV)
    st = torch.tensor(starts, dtype=torch.int32, device=DEV)
    b = Batch(page_table=cache.table.data_ptr(), seq_lens=cache.lens.data_ptr(), slots=None,
              starts=st.data_ptr(), table_stride=cache.table.stride(0), total=total, B=len(new),
              T=max(new), num_slots=len(new), num_pages=cache.P, table_width=cache.table.shape[1],
              page_size=ps)
    max_len = cache.table.shape[1] * ps
    code = 0 if dtype == F32 else 1
    size = lib.ltv_paged_attention_fp4_workspace_size
    size.restype, size.argtypes = ctypes.c_size_t, [i32, vp, i32, i32, i32, i32]
    nws = size(code, ctypes.byref(b), NH, NKVH, D, max_len)
    ws = torch.empty(nws, dtype=torch.uint8, device=DEV)
    row = D // 2 + D // 32
    pages = _s(NKVH * ps * row, ps * row, row)
    f = lib.ltv_paged_attention_fp4
    f.argtypes = [i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, ctypes.c_size_t, i32, i32, i32, i32,
                  ctypes.c_float, vp]
    rc = f(code, q.data_ptr(), _s(0, NH * D, D), cache.k_pages.data_ptr(), pages,
           cache.v_pages.data_ptr(), pages, ctypes.byref(b), out.data_ptr(),
           _s(0, NH * (D + 16), D + 16), lse.data_ptr(), ws.data_ptr(), nws, NH, NKVH, D, max_len,
           D ** -0.5, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    rows = slice(starts[0], starts[-1])
    for x in (out[:before], out[starts[-1]:], out[..., D:], lse[:before], lse[starts[-1]:]):
        assert bool((x == 77.0).all())
    qs, outs, lses = (x[rows].split(new) for x in (q, out[..., :D], lse))
    _check(list(zip(outs, lses)), attention64(list(qs), cache, [0, 1, 2], new, D ** -0.5), dtype, D,
           lens)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40, 1100])
def test_captured(new, dtype):
    """Lengths, tables and pages change between replays; two graphs side by side."""
    cache = Cache4([2000, 600], 2, 64, 16, 16)
    _widen(cache, ROOM if new == 1100 else 0)
    q = cache.rand(2, new, 4, 64, dtype=dtype)
    f = lambda: _ops().paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.lens,  # noqa: E731
                                       return_lse=True)
    f()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for a, b in ((2000, 600), (64, 64), (1999, 100), (300, 1)):
        cache.lens.copy_(torch.tensor([a, b]))
        q.copy_(cache.rand(*q.shape))
        for g, out in zip(graphs, outs):
            g.replay()
        want = f()
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_other_stream():
    cache = Cache4([2000, 600], 2, 64, 16, 17)
    q = cache.rand(2, 3, 4, 64, dtype=BF)
    f = lambda: _ops().paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.lens)  # noqa: E731
    want = f()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = f()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_compiled():
    cache = Cache4([200, 60], 2, 64, 16, 18)
    q = cache.rand(2, 3, 4, 64, dtype=BF)
    f = lambda q: _ops().paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.lens)  # noqa: E731
    assert torch.equal(torch.compile(f, fullgraph=True, backend="eager")(q), f(q))


def test_pages_of_all_layers_move():
    """reserve, copy and compact of 4-bit pages: bytes as any others."""
    ops = _ops()
    ps, row = 16, ops.fp4_row_bytes(64)
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randint(0, 256, (3, 9, 2, ps, row), generator=g, device=DEV, dtype=torch.uint8)
            for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table, lens, refs = ints([[3, 4, -1], [3, 4, -1]]), ints([20, 20]), ints([0, 0, 0, 2, 2, 0, 0, 1, 0])
    was = k.clone(), v.clone()
    assert int(ops.paged_cache_reserve(table, lens, refs, ints([0, 1]), ints([1, 14]), k, v)) == 0
    assert table.tolist() == [[3, 0, -1], [3, 4, 1]] and lens.tolist() == [21, 34]
    for x, w in zip((k, v), was):
        assert torch.equal(x[:, 0], w[:, 4]) and torch.equal(x[:, 2:], w[:, 2:])
    assert int(ops.paged_cache_compact(table, refs, k, v)) == 5
    assert table.tolist() == [[3, 0, -1], [3, 4, 1]]
    for x, w in zip((k, v), was):
        assert torch.equal(x[:, 2], w[:, 7])


def test_refusals():
    cache = Cache4([40], 2, 64, 16, 1)
    q = cache.rand(1, 4, 4, 64, dtype=BF)

    def attn(q=q, kp=cache.k_pages, vp=cache.v_pages, **kw):
        return _ops().paged_attention(q, kp, vp, cache.table, cache.lens, **kw)

    attn()
    with pytest.raises(ValueError, match="head_dim"):
        attn(q=q[..., :32])
    with pytest.raises(ValueError):
        attn(q=q[..., :3, :])
    with pytest.raises(TypeError):
        attn(q=q.half())
    with pytest.raises(TypeError):
        attn(vp=torch.zeros(cache.v_pages.shape, dtype=torch.int8, device=DEV))
    with pytest.raises(ValueError):
        attn(vp=cache.v_pages[:-1])
    with pytest.raises(ValueError, match="scale"):
        attn(scale=0.0)
    with pytest.raises(RuntimeError):
        attn(q=q.float().requires_grad_())
    with pytest.raises(ValueError, match="multiple of 16"):
        bad = torch.zeros(4, 2, 24, 34, dtype=torch.uint8, device=DEV)
        attn(kp=bad, vp=bad)


def test_nothing():
    cache = Cache4([40, 7], 2, 64, 16, 1)
    q = cache.rand(2, 4, 4, 64, dtype=BF)
    f = _ops().paged_attention
    out, lse = f(q, cache.k_pages[:0], cache.v_pages[:0], cache.table, cache.lens, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    out, lse = f(q, cache.k_pages, cache.v_pages, cache.table[:, :0], cache.lens, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    assert f(q[:0], cache.k_pages, cache.v_pages, cache.table, cache.lens,
             slots=torch.zeros(0, dtype=torch.int32, device=DEV)).numel() == 0
    assert f(q[:, :0], cache.k_pages, cache.v_pages, cache.table, cache.lens).numel() == 0
