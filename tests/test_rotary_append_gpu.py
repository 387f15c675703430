"""Rotation on the way into the paged cache, 16, 32 and 4-bit pages, and what they hold read
back, against float64."""

from __future__ import annotations

import math

import pytest
import torch

from fp4_test_utils import Cache4, held4, rotated64, values4
from paged_test_utils import DEV, Cache

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _tables(n, D, dtype):
    f = 10000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * f
    return a.cos().to(dtype), a.sin().to(dtype)


def _half_step(dtype):
    """One rounding by way of float32: half a step of the type and a float32 rounding, relative
    (2 eps of float64 for the sums), and half the smallest subnormal."""
    e = torch.finfo(dtype).eps / 2
    return e * (1 + 2.0 ** -14), torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def _pages(cache):
    return (cache.k_pages, cache.v_pages) if isinstance(cache, Cache4) else (cache.k, cache.v)


def _call(cache, q, k, v, cos, sin, new, packed, slots=None, **kw):
    if slots is not None:
        kw["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
    if packed:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        kw["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    else:
        q, k, v = (x.unflatten(0, (len(new), -1)) for x in (q, k, v))
    y = _ops().paged_rotary_append(q, k, v, cos, sin, *_pages(cache), cache.table, cache.lens, **kw)
    assert y.shape == q.shape and y.dtype == q.dtype and y.is_contiguous()
    return y if packed else y.flatten(0, 1)


def _positions(cache, order, new):
    out = []
    for s, n in zip(order, new):
        length = int(cache.lens[s]) if 0 <= s < len(cache.lens) else 0
        out.append(torch.arange(length - n, length, device=DEV))
    return out


def _expect(cache, order, new, pos, k64, v64):
    """The pages' values (float64) after the call."""
    k, v = cache.k.double().clone(), cache.v.double().clone()
    at = 0
    for s, n, p in zip(order, new, pos):
        for t in range(n):
            i = int(p[t])
            if i < 0 or not 0 <= s < len(cache.lens):
                continue
            page = int(cache.table[s, i // cache.page])
            if 0 <= page < cache.P:
                k[page, :, i % cache.page] = k64[at + t]
                v[page, :, i % cache.page] = v64[at + t]
        at += n
    return k, v


def _near(got, want, dtype):
    rel, tiny = _half_step(dtype)
    err = (got.double() - want).abs()
    ok = (err <= rel * want.abs() + tiny) | (got.double() == want)
    ok |= got.isnan() & want.isnan()
    assert bool(ok.all()), float((err / want.abs().clamp(min=1e-30)).max())


def _case(dtype, tab, bits, NH, NKVH, D, page, new, cached, packed, eps, seed=0, slots=None,
          layout=None, scale=1.0):
    lens = [max(a + b, 0) for a, b in zip(new, cached)]
    order = list(range(len(lens))) if slots is None else slots
    held = [0] * (max([0, *order]) + 1)
    for s, n in zip(order, lens):
        if s >= 0:
            held[s] = n
    if bits == 4:
        cache = Cache4(held, NKVH, D, page, seed, layout=layout or "dense")
    else:
        cache = Cache(held, NKVH, D, page, dtype, seed, layout=layout or "head")
    N = sum(new)
    q, k, v = ((cache.rand(N, n, D) * scale).to(dtype) for n in (NH, NKVH, NKVH))
    cos, sin = _tables(cache.table.shape[1] * page, D, tab)
    pos = _positions(cache, order, new)
    allpos = torch.cat(pos) if pos else torch.zeros(0, device=DEV)
    k64, v64 = rotated64(k, cos, sin, allpos, eps), v.double()
    if bits == 4:
        k64, v64 = held4(k64)[0], held4(v64)[0]
    want_k, want_v = _expect(cache, order, new, pos, k64, v64)
    y = _call(cache, q, k, v, cos, sin, new, packed, slots, norm_eps=eps)
    _near(y, rotated64(q, cos, sin, allpos, eps), dtype)
    if bits == 4:
        assert torch.equal(values4(cache.k_pages), want_k)
        assert torch.equal(values4(cache.v_pages), want_v)
    else:
        _near(cache.k, want_k, dtype)
        assert torch.equal(cache.v.double(), want_v)
    return cache


# heads, page size; widths whose halves are no multiple of eight among them
HEADS = [(6, 6, 128, 64), (8, 4, 64, 16), (10, 5, 72, 48), (3, 1, 8, 1), (6, 2, 40, 5),
         (1, 1, 120, 300), (12, 3, 96, 32), (64, 8, 16, 7)]


@pytest.mark.parametrize("eps", [None, 2.0 ** -23])
@pytest.mark.parametrize("tab", [BF, F32])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D,page", HEADS)
def test_values(NH, NKVH, D, page, dtype, tab, eps):
    _case(dtype, tab, 16, NH, NKVH, D, page, [1, 5, 0, 33, 64, 2, 130], [0, 7, 20, 0, 65, 300, 131],
          True, eps)
    _case(dtype, tab, 16, NH, NKVH, D, page, [1] * 9, [0, 1, 2, 15, 16, 31, 64, 400, 511], False, eps)


HEADS4 = [(6, 6, 128, 64), (8, 4, 64, 16), (5, 5, 32, 48), (12, 3, 96, 32), (1, 1, 128, 304)]


@pytest.mark.parametrize("eps", [None, 2.0 ** -23])
@pytest.mark.parametrize("tab", [BF, F32])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D,page", HEADS4)
def test_four_bits(NH, NKVH, D, page, dtype, tab, eps):
    _case(dtype, tab, 4, NH, NKVH, D, page, [1, 5, 0, 33, 64, 2, 130], [0, 7, 20, 0, 65, 300, 131],
          True, eps)
    _case(dtype, tab, 4, NH, NKVH, D, page, [1] * 9, [0, 1, 2, 15, 16, 31, 64, 400, 511], False, eps,
          layout="apart")


@pytest.mark.parametrize("layout", ["token", "both"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts_of_pages(dtype, layout):
    _case(dtype, BF, 16, 4, 2, 64, 16, [1, 40, 3], [5, 60, 0], True, 1e-6, layout=layout)


@pytest.mark.parametrize("bits", [4, 16])
def test_slots_and_missing(bits):
    """Slots in another order, one out of range, a sequence shorter than its new tokens and
    pages that are missing: dropped, and their queries as everywhere, or 0 before position 0."""
    _case(BF, BF, bits, 4, 2, 64, 16, [3, 2, 5, 1], [20, 4, -3, 0], True, 1e-6, slots=[2, -1, 0, 1])
    cache = Cache4([40], 2, 64, 16, 3) if bits == 4 else Cache([40], 2, 64, 16, BF, 3)
    cache.table[0, 1] = cache.P + 5
    pages = [p.clone() for p in _pages(cache)]
    cos, sin = _tables(cache.table.shape[1] * 16, 64, BF)
    x = cache.rand(1, 24, 2, 64, dtype=BF)
    y = _ops().paged_rotary_append(x, x, x, cos, sin, *_pages(cache), cache.table, cache.lens)
    pos = torch.arange(16, 40, device=DEV)
    _near(y[0], rotated64(x[0], cos, sin, pos, None), BF)
    # page 1 of the table is missing: only the third is written
    for p, was in zip(_pages(cache), pages):
        third = int(cache.table[0, 2])
        others = [i for i in range(cache.P) if i != third]
        assert torch.equal(p[others], was[others]) and not torch.equal(p[third], was[third])


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides(dtype, bits):
    """Head-major inputs, slices that are not aligned, rows that are not contiguous."""
    cache = Cache4([40, 33], 3, 64, 16, 5) if bits == 4 else Cache([40, 33], 3, 64, 16, dtype, 5)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, F32)
    wide = torch.cat([cos, sin], 1)
    big = cache.rand(2, 6, 9, 70, dtype=dtype)
    outs = []
    for make in (lambda: (big[:, :, 1:8, 3:67].transpose(1, 2), big[:, :3, 2:9, 5:69].transpose(1, 2),
                          big[:, 3:, 2:9, 1:65].transpose(1, 2), wide[:, :32], wide[:, 32:]),
                 lambda: (*(x.contiguous() for x in (big[:, :, 1:8, 3:67].transpose(1, 2),
                                                     big[:, :3, 2:9, 5:69].transpose(1, 2),
                                                     big[:, 3:, 2:9, 1:65].transpose(1, 2))), cos, sin),
                 lambda: (*(x.transpose(2, 3).contiguous().transpose(2, 3) for x in (
                     big[:, :, 1:8, 3:67].transpose(1, 2), big[:, :3, 2:9, 5:69].transpose(1, 2),
                     big[:, 3:, 2:9, 1:65].transpose(1, 2))), cos.t().contiguous().t(), sin)):
        q, k, v, c, s = make()
        for p in _pages(cache):
            p.zero_()
        y = _ops().paged_rotary_append(q, k, v, c, s, *_pages(cache), cache.table, cache.lens,
                                       norm_eps=0.0)
        outs.append([y, *(p.clone() for p in _pages(cache))])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 16])
def test_sizes_of_values(dtype, bits):
    """Squares past float32, all zeros, infinities and NaN, values that are nearly 0."""
    cache = Cache4([8], 1, 64, 16, 1) if bits == 4 else Cache([8], 1, 64, 16, dtype, 1)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, F32)
    x = cache.rand(8, 1, 64)
    x[0] *= 1e30
    x[1] = 0.0
    x[2, 0, 5] = math.inf
    x[3, 0, 40] = math.nan
    x[4] *= 1e-30
    x = x.to(dtype)
    pos = torch.arange(8, device=DEV)
    for eps in (None, 0.0, 1e-5):
        want = rotated64(x, cos, sin, pos, eps)
        y = _ops().paged_rotary_append(x[None], x[None], x[None], cos, sin, *_pages(cache),
                                       cache.table, cache.lens, norm_eps=eps)[0]
        _near(y, want, dtype)
        page = int(cache.table[0, 0])
        if bits == 4:
            got = values4(cache.k_pages)[page, 0, :8], values4(cache.v_pages)[page, 0, :8]
            for g, w in zip(got, (held4(want)[0], held4(x)[0])):
                w = w[:, 0]
                assert torch.equal(torch.nan_to_num(g, 9e9), torch.nan_to_num(w, 9e9))
        else:
            _near(cache.k[page, 0, :8], want[:, 0], dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_results_below_float32(dtype):
    """Rotated keys that float32 does not hold are 0 in 4 bits, of both signs, beside others."""
    cache = Cache4([16], 1, 64, 16, 1)
    x = cache.rand(16, 1, 64)
    x[:, :, ::3] *= 2.0 ** -126
    x[::2] *= 2.0 ** -100
    x = x.to(dtype)
    c = torch.full((16, 32), 2.0 ** -40, device=DEV)
    s = torch.full((16, 32), 2.0 ** -60, device=DEV)
    _ops().paged_rotary_append(x[None], x[None], x[None], c, s, cache.k_pages, cache.v_pages,
                               cache.table, cache.lens)
    page = int(cache.table[0, 0])
    want = held4(rotated64(x, c, s, torch.arange(16, device=DEV), None))[0][:, 0]
    assert torch.equal(values4(cache.k_pages)[page, 0, :16], want)
    assert torch.equal(values4(cache.v_pages)[page, 0, :16], held4(x)[0][:, 0])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_results_near_borders(dtype):
    """Rotated keys a fraction of a float32 step, or some, from where a code or a scale ends."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], device=DEV)
    cache = Cache4([64], 1, 64, 16, 1)
    x = torch.cat([borders, -borders]).repeat(64, 4)
    x[32:, 7::8] = 6.0  # (the scale is theirs, or that of those beside 7)
    powers = torch.tensor([1.0, 2.0 ** -9, 2.0 ** 40], device=DEV).repeat(22)[:64]
    x = (x * powers[:, None])[:, None].to(dtype)
    near = torch.arange(64, device=DEV, dtype=torch.float64) % 32 - 15.5
    near = torch.where(near.abs() > 12, near * 16, near) * 2.0 ** -26
    c, s = torch.ones(64, 32, device=DEV), near.float()[:, None].expand(64, 32).contiguous()
    _ops().paged_rotary_append(x[None], x[None], x[None], c, s, cache.k_pages, cache.v_pages,
                               cache.table, cache.lens)
    pos = torch.arange(64, device=DEV)
    want = held4(rotated64(x, c, s, pos, None))[0][:, 0]
    got = values4(cache.k_pages)[cache.table[0, (pos // 16).long()].long(), 0, pos % 16]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_results_beyond_float32(dtype):
    """Rotated keys that are finite but past float32 are held as the largest there is."""
    cache = Cache4([16], 1, 64, 16, 1)
    x = (cache.rand(16, 1, 64).sign() * 3e38).to(dtype)
    x[4:, :, 32:] = 0.0
    x[8, 0, 3] = math.inf
    c = torch.full((16, 32), 0.75, device=DEV)
    s = torch.full((16, 32), 0.75, device=DEV)
    _ops().paged_rotary_append(x[None], x[None], x[None], c, s, cache.k_pages, cache.v_pages,
                               cache.table, cache.lens)
    page = int(cache.table[0, 0])
    want = held4(rotated64(x, c, s, torch.arange(16, device=DEV), None))[0][:, 0]
    got = values4(cache.k_pages)[page, 0, :16]
    assert torch.equal(got.isnan(), want.isnan()) and bool(got[8].isnan().all())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_borders_of_codes(dtype):
    """Every tie, the ends of the scales and what is beyond them, by ``paged_cache_append``."""
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0], device=DEV)
    eps = 2.0 ** -7 if dtype == BF else 2.0 ** -23
    rows = []
    for e in (-140, -130, -127, -126, -125, -124, -20, -1, 0, 1, 40, 120, 124, 125):
        for top in (4.0, 6.0, 7.0, 7.0 * (1 + eps), 7.9):
            v = torch.cat([base, base * (1 + eps), base * (1 - eps), torch.tensor([top, -top], device=DEV)])
            v = (v.double().clamp(max=top) * 2.0 ** e).float()
            v[1::2] *= -1
            rows.append(v)
    x = torch.stack(rows)  # (n, 32)
    n = len(x)
    x = x.to(dtype)[:, None]
    cache = Cache4([n], 1, 32, 16, 0)
    _ops().paged_cache_append(x[None], x[None].flip(-1), cache.k_pages, cache.v_pages, cache.table,
                              cache.lens)
    k, v = _ops().paged_cache_read(cache.k_pages, cache.v_pages, cache.table, cache.lens, n,
                                   dtype=F32)
    want = held4(x)[0]
    assert torch.equal(k[0].double(), want)
    assert torch.equal(v[0].double(), held4(x.flip(-1))[0])


@pytest.mark.parametrize("NH,NKVH,D,page", HEADS4)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_and_read(dtype, NH, NKVH, D, page):
    """``paged_cache_append`` into 4-bit pages, and back; rows of no sequence and of no page are 0."""
    new, cached = [1, 5, 0, 33, 64, 2, 130], [0, 7, 20, 0, 65, 300, 131]
    cache = Cache4([a + b for a, b in zip(new, cached)], NKVH, D, page, 2, layout="apart")
    N = sum(new)
    k, v = cache.rand(N + 3, NKVH, D, dtype=dtype), cache.rand(N + 3, NKVH, D, dtype=dtype) * 3
    starts = [1]
    for n in new:
        starts.append(starts[-1] + n)
    starts = torch.tensor(starts, dtype=torch.int32, device=DEV)
    before = cache.k.clone(), cache.v.clone()
    _ops().paged_cache_append(k, v, cache.k_pages, cache.v_pages, cache.table, cache.lens,
                              starts=starts)
    order = list(range(len(new)))
    pos = _positions(cache, order, new)
    want = _expect(cache, order, new, pos, held4(k[1:])[0], held4(v[1:])[0])
    cache.decode()
    assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])
    assert not torch.equal(cache.k, before[0]) and not torch.equal(cache.v, before[1])
    for out in (BF, F32):
        for hint in (None, 1, 130):
            a, b = _ops().paged_cache_read(cache.k_pages, cache.v_pages, cache.table, cache.lens, N + 3,
                                           starts=starts, dtype=out, max_new=hint)
            assert a.dtype == out and a.shape == (N + 3, NKVH, D)
            assert not a[0].any() and not a[N + 1:].any() and not b[N + 1:].any()
            assert torch.equal(a[1:N + 1].double(), held4(k[1:N + 1])[0])
            assert torch.equal(b[1:N + 1].double(), held4(v[1:N + 1])[0])
    a, b = _ops().paged_cache_read(cache.k_pages, cache.v_pages, cache.table, cache.lens, 7,
                                   slots=torch.tensor([5, 9, 0], device=DEV))
    assert a.shape == (3, 7, NKVH, D) and not a[1].any() and not a[2, :6].any()
    p = torch.arange(295, 302, device=DEV)
    pages = cache.table[5, (p // page).long()].long()
    assert torch.equal(a[0].double(), cache.k[pages, :, p % page])
    assert torch.equal(b[0].double(), cache.v[pages, :, p % page])


@pytest.mark.parametrize("layout", ["head", "token", "both"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,page", [(128, 64), (72, 7), (40, 5), (8, 1)])
def test_read_values(D, page, dtype, layout):
    cache = Cache([40, 0, 9, 131], 3, D, page, dtype, 4, layout=layout)
    cache.table[0, 0] = -1
    k, v = _ops().paged_cache_read(cache.k, cache.v, cache.table, cache.lens, 40)
    assert k.dtype == dtype and k.shape == (4, 40, 3, D)
    for b, n in enumerate([40, 0, 9, 131]):
        for t in range(40):
            i = n - 40 + t
            page_id = int(cache.table[b, i // page]) if i >= 0 else -1
            want = [x[page_id, :, i % page] if page_id >= 0 else torch.zeros(3, D, device=DEV)
                    for x in (cache.k, cache.v)]
            assert torch.equal(k[b, t], want[0].to(dtype)) and torch.equal(v[b, t], want[1].to(dtype))


def test_many_sequences():
    B = 700
    new = [1 + (i % 97 == 5) * (i % 150) for i in range(B)]
    cached = [(i * 37) % 230 for i in range(B)]
    N = sum(new)
    cache = Cache4([a + b for a, b in zip(new, cached)], 2, 64, 16, 6)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, BF)
    x = cache.rand(N, 2, 64, dtype=BF)
    y = _call(cache, x, x, x, cos, sin, new, True, norm_eps=1e-6)
    pos = torch.cat(_positions(cache, list(range(B)), new))
    want = rotated64(x, cos, sin, pos, 1e-6)
    _near(y, want, BF)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    k, v = _ops().paged_cache_read(cache.k_pages, cache.v_pages, cache.table, cache.lens, N,
                                   starts=torch.tensor(starts, device=DEV))
    assert torch.equal(k.double(), held4(want)[0]) and torch.equal(v.double(), held4(x)[0])


@pytest.mark.parametrize("bits", [4, 16])
def test_captured(bits):
    """Lengths change between replays."""
    cache = Cache4([64], 2, 64, 16, 7) if bits == 4 else Cache([64], 2, 64, 16, BF, 7)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, BF)
    x = cache.rand(1, 4, 2, 64, dtype=BF)
    lens = cache.lens
    call = lambda: (_ops().paged_rotary_append(x, x, x, cos, sin, *_pages(cache), cache.table, lens,  # noqa: E731
                                               norm_eps=1e-6),
                    *_ops().paged_cache_read(*_pages(cache), cache.table, lens, 4))
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for n in (4, 2, 17, 64, 33):
        lens.fill_(n)
        x.copy_(cache.rand(1, 4, 2, 64))
        for p in _pages(cache):
            p.zero_()
        graph.replay()
        torch.cuda.synchronize()
        saved = [t.clone() for t in (*got, *_pages(cache))]
        for p in _pages(cache):
            p.zero_()
        want = [*call(), *_pages(cache)]
        assert all(torch.equal(a, b) for a, b in zip(saved, want))


def test_other_stream():
    cache = Cache4([64], 2, 64, 16, 8)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, BF)
    x = cache.rand(1, 4, 2, 64, dtype=BF)
    want = _ops().paged_rotary_append(x, x, x, cos, sin, *_pages(cache), cache.table, cache.lens)
    read = _ops().paged_cache_read(*_pages(cache), cache.table, cache.lens, 4)
    cache.k_pages.zero_(), cache.v_pages.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _ops().paged_rotary_append(x, x, x, cos, sin, *_pages(cache), cache.table, cache.lens)
        again = _ops().paged_cache_read(*_pages(cache), cache.table, cache.lens, 4)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(again, read))


def test_compiled_and_traced():
    cache = Cache4([64], 2, 64, 16, 9)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, BF)
    x = cache.rand(1, 4, 2, 64, dtype=BF)

    def f(x):
        y = _ops().paged_rotary_append(x, x, x, cos, sin, *_pages(cache), cache.table, cache.lens,
                                       norm_eps=1e-6)
        k, v = _ops().paged_cache_read(*_pages(cache), cache.table, cache.lens, 4)
        return y, k, v

    want = f(x)
    got = torch.compile(f, fullgraph=True, backend="eager")(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    cache = Cache4([40], 2, 64, 16, 1)
    cos, sin = _tables(cache.table.shape[1] * 16, 64, BF)
    x = cache.rand(1, 4, 2, 64, dtype=BF)
    ops = _ops()

    def rot(q=x, k=x, v=x, cos=cos, sin=sin, kp=cache.k_pages, vp=cache.v_pages, **kw):
        return ops.paged_rotary_append(q, k, v, cos, sin, kp, vp, cache.table, cache.lens, **kw)

    rot()
    with pytest.raises(ValueError, match="positions"):
        rot(cos=cos[:-1], sin=sin[:-1])
    with pytest.raises(ValueError, match="cos and sin"):
        rot(cos=cos[:, :31], sin=sin[:, :31])
    with pytest.raises(ValueError, match="norm_eps"):
        rot(norm_eps=-1e-6)
    with pytest.raises(ValueError, match="norm_eps"):
        rot(norm_eps=math.inf)
    with pytest.raises(TypeError):
        rot(sin=sin.float())
    with pytest.raises(TypeError):
        rot(k=x.float(), v=x.float())
    with pytest.raises(TypeError):
        rot(q=x.half(), k=x.half(), v=x.half())
    with pytest.raises(ValueError):
        rot(k=x[:, :3], v=x[:, :3])
    with pytest.raises(ValueError):
        rot(k=x[..., :1, :], v=x[..., :1, :])
    with pytest.raises(ValueError):
        rot(q=x[..., :32])
    with pytest.raises(RuntimeError, match="q"):
        rot(q=x.float().requires_grad_(), k=x.float(), v=x.float())
    with pytest.raises(RuntimeError):
        rot(cos=cos.cpu())
    with pytest.raises(RuntimeError):
        rot(q=x.cpu(), k=x.cpu(), v=x.cpu())
    with pytest.raises(TypeError):
        rot(vp=cache.v_pages.to(torch.int8))
    with pytest.raises(ValueError, match="multiple of 16"):
        bad = torch.zeros(4, 2, 8, 34, dtype=torch.uint8, device=DEV)
        rot(kp=bad, vp=bad)
    with pytest.raises(ValueError, match="17 bytes"):
        bad = torch.zeros(4, 2, 16, 33, dtype=torch.uint8, device=DEV)
        rot(kp=bad, vp=bad)
    with pytest.raises(ValueError, match="dense"):
        bad = torch.zeros(4, 16, 2, 34, dtype=torch.uint8, device=DEV).transpose(1, 2)
        rot(kp=bad, vp=bad)
    with pytest.raises(ValueError, match="dense"):
        bad = torch.zeros(4 * 2 * 16 * 34 + 8, dtype=torch.uint8, device=DEV)[8:].view(4, 2, 16, 34)
        rot(kp=bad, vp=bad)
    with pytest.raises(ValueError):
        ops.paged_cache_append(x[..., :32], x[..., :32], cache.k_pages, cache.v_pages, cache.table,
                               cache.lens)
    with pytest.raises(ValueError):
        ops.paged_cache_read(cache.k_pages, cache.v_pages, cache.table, cache.lens, -1)
    with pytest.raises(TypeError):
        ops.paged_cache_read(cache.k_pages, cache.v_pages, cache.table, cache.lens, 4,
                             dtype=torch.float16)
    with pytest.raises(RuntimeError, match="v_pages"):
        v = torch.zeros(4, 2, 16, 64, dtype=BF, device=DEV)
        ops.paged_cache_read(v, v.clone().requires_grad_(), cache.table, cache.lens, 4)
    with pytest.raises(TypeError):
        v = torch.zeros(4, 2, 16, 64, dtype=BF, device=DEV)
        ops.paged_cache_read(v, v, cache.table, cache.lens, 4, dtype=F32)
    for d in (0, 16, 48, 160):
        with pytest.raises(ValueError):
            ops.fp4_row_bytes(d)


@pytest.mark.parametrize("bits", [4, 16])
def test_nothing(bits):
    """No sequences, no tokens, no pages, no room in the table."""
    cache = Cache4([40], 2, 64, 16, 1) if bits == 4 else Cache([40], 2, 64, 16, BF, 1)
    cos, sin = _tables(48, 64, BF)
    kp, vp = _pages(cache)
    e = torch.zeros(0, 4, 2, 64, dtype=BF, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert _ops().paged_rotary_append(e, e, e, cos, sin, kp, vp, cache.table, cache.lens,
                                      slots=none).shape == e.shape
    t = torch.zeros(1, 0, 2, 64, dtype=BF, device=DEV)
    assert _ops().paged_rotary_append(t, t, t, cos, sin, kp, vp, cache.table, cache.lens).numel() == 0
    x = cache.rand(1, 4, 2, 64, dtype=BF)
    y = _ops().paged_rotary_append(x, x, x, cos, sin, kp[:0], vp[:0], cache.table, cache.lens)
    _near(y[0], rotated64(x[0], cos, sin, torch.arange(36, 40, device=DEV), None), BF)
    k, v = _ops().paged_cache_read(kp[:0], vp[:0], cache.table, cache.lens, 4)
    assert k.shape == (1, 4, 2, 64) and not k.any() and not v.any()
    y = _ops().paged_rotary_append(x, x, x, cos[:0], sin[:0], kp, vp, cache.table[:, :0], cache.lens)
    assert not y.any()
    k, v = _ops().paged_cache_read(kp, vp, cache.table, cache.lens, 5,
                                   starts=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert k.shape == (5, 2, 64) and not k.any() and not v.any()
