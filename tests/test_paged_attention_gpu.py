"""Attention of new tokens over the paged cache against float64, element by element,
within the bound of its roundings."""

from __future__ import annotations

import math

import pytest
import torch

from paged_test_utils import DEV, Cache, attention64, attention_bound, lse_bound

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
    out, lse = _ops().paged_attention(x, cache.k, cache.v, cache.table, cache.lens, scale=scale,
                                      return_lse=True, **kw)
    assert out.shape == x.shape and out.dtype == x.dtype and lse.shape == x.shape[:-1]
    if packed:
        return list(zip(out.split(list(new)), lse.split(list(new))))
    return list(zip(out, lse))


def _check(got, want, dtype, D, lens):
    for i, ((out, lse), (o64, l64, mag, big)) in enumerate(zip(got, want)):
        bound = attention_bound(dtype, D, lens[i], mag, big)
        err = (out.double() - o64).abs()
        assert bool((err <= bound).all()), (
            i, float((err / bound).max()), float(err.max()))
        empty = l64 == -math.inf
        assert torch.equal(lse == -math.inf, empty), i
        assert bool((out[empty] == 0).all())
        e = (lse.double() - l64)[~empty].abs()
        assert bool((e <= lse_bound(D, lens[i], l64[~empty], big)).all()), (i, float(e.max()))


def _case(dtype, NH, NKVH, D, page, new, cached, packed, seed=0, slots=None, layout="head",
          qscale=1.0, **hints):
    lens = [a + b for a, b in zip(new, cached)]
    order = list(range(len(lens))) if slots is None else slots
    held = [0] * (max(order) + 1 if order else 0)
    for s, n in zip(order, lens):
        held[s] = n
    cache = Cache(held, NKVH, D, page, dtype, seed, layout=layout)
    q = [(cache.rand(n, NH, D) * qscale).to(dtype) for n in new]
    got = _run(cache, q, new, packed, slots, **hints)
    want = attention64(q, cache, order, new, D ** -0.5)
    _check(got, want, dtype, D, lens)


# heads, page size: groups of one to eight, widths of one to four tiles' quarters, pages
# that are no power of two, of one token and longer than the sequence
HEADS = [(6, 6, 128, 64), (8, 4, 128, 16), (10, 5, 64, 48), (8, 1, 96, 32), (3, 1, 8, 1),
         (2, 2, 72, 7), (16, 2, 128, 128), (6, 2, 40, 5), (32, 1, 64, 16), (5, 5, 120, 300)]


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
@pytest.mark.parametrize("T,cached", [(1, 3000), (3, 2049), (40, 1500), (257, 100), (512, 0)])
def test_longer(T, cached, dtype):
    _case(dtype, 4, 2, 128, 32, [T] * 2, [cached, cached // 3], packed=False, seed=2, qscale=3.0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_context_split_over_many(dtype):
    """Few rows, a long and a short context: the keys are split and joined."""
    _case(dtype, 4, 1, 64, 64, [1, 1, 2], [40000, 10, 9000], packed=True, seed=3, qscale=2.0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B", [257, 700])
def test_many_sequences(B, dtype):
    """More sequences than a workgroup has threads, most of them short, some in chunks."""
    new = [1 + (i % 97 == 5) * (i % 150) for i in range(B)]
    new[B // 2] = 0
    _case(dtype, 4, 2, 64, 16, new, [(i * 37) % 230 for i in range(B)], packed=True, seed=23)


@pytest.mark.parametrize("B,NH,NKVH,D,page", [(130, 12, 4, 128, 16), (90, 6, 6, 64, 7),
                                              (600, 2, 1, 96, 48), (70, 64, 8, 128, 64),
                                              (4500, 1, 1, 64, 16)])
@pytest.mark.parametrize("max_len", [None, 512])
@pytest.mark.parametrize("T", [1, 2])
def test_many_short_sequences(T, max_len, B, NH, NKVH, D, page):
    """Enough sequences and heads for the shape of one wavefront, where they are said to be
    short; a long one among them all the same."""
    cached = [(i * 53) % 140 for i in range(B)]
    cached[B // 3], cached[7], cached[8] = 3000, 0, -T  # (no token in the cache at all)
    _case(BF, NH, NKVH, D, page, [T] * B, cached, packed=False, seed=29, max_len=max_len)


@pytest.mark.parametrize("B", [140, 300])
def test_many_short_sequences_and_wrong_hints(B):
    """Hints that are too small for some of them: more rows, and keys, than were expected."""
    new = [1 + 49 * (i % 60 == 3) for i in range(B)]
    _case(BF, 8, 4, 128, 16, new, [(i * 29) % 300 for i in range(B)], packed=True, seed=31,
          max_new=1, max_len=16)


@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_many_short_sequences_with_poison(poison):
    """The same where masked places hold infinities and NaN, in keys and values."""
    B, lens = 140, [2 + (i * 31) % 90 for i in range(140)]
    cache = Cache(lens, 4, 64, 16, BF, 30, spare=4)
    used = torch.zeros(cache.P, 16, dtype=torch.bool, device=DEV)
    for i, n in enumerate(lens):
        pos = torch.arange(n, device=DEV)
        used[cache.table[i, pos // 16].long(), pos % 16] = True
    for x in (cache.k, cache.v):
        x.transpose(1, 2)[~used] = poison
    q = [cache.rand(1, 8, 64, dtype=BF) for _ in range(B)]
    _check(_run(cache, q, [1] * B, False), attention64(q, cache, list(range(B)), [1] * B, 64 ** -0.5),
           BF, 64, lens)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("NH,NKVH,D", [(8, 4, 128), (6, 6, 64), (3, 1, 128)])
def test_long_chunk_among_short_ones(NH, NKVH, D, dtype):
    """One sequence has nearly all the work: its row tiles are cut many times."""
    _case(dtype, NH, NKVH, D, 16, [1] * 9 + [200, 3, 70, 1], [5, 300] * 4 + [0, 5000, 9, 40, 2500],
          packed=True, seed=24, qscale=2.0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_many_rows_of_few_keys(page, dtype):
    """More new tokens than the table has room for: the first ones see nothing."""
    _case(dtype, 4, 2, 64, page, [700, 300, 40], [-690, -270, -8], packed=True, seed=25)
    _case(dtype, 4, 4, 64, page, [300, 300], [-287, -299], packed=False, seed=26)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_wide_table(dtype):
    """A table with room for 2^30 tokens of each sequence, hardly any of it used."""
    new, lens = [600, 1, 40], [700, 300, 41]
    cache = Cache(lens, 32, 8, 128, dtype, 27)
    wide = torch.full((3, 1 << 23), -1, dtype=torch.int32, device=DEV)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    q = [cache.rand(n, 32, 8, dtype=dtype) for n in new]
    got = _run(cache, q, new, True)
    _check(got, attention64(q, cache, [0, 1, 2], new, 8 ** -0.5), dtype, 8, lens)


@pytest.mark.parametrize("layout", ["token", "gaps"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_page_layouts(layout, dtype):
    _case(dtype, 6, 3, 64, 16, [4, 40], [50, 9], packed=True, seed=4, layout=layout)


def test_q_layouts_and_alignment():
    """Head-major q, q at an odd element, q without a contiguous last axis."""
    cache = Cache([90, 40], 2, 64, 16, BF, 5)
    q = cache.rand(2, 3, 4, 64, dtype=BF)
    ops = _ops()
    want = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.lens)
    _check(list(zip(*ops.paged_attention(q, cache.k, cache.v, cache.table, cache.lens,
                                         return_lse=True))),
           attention64(list(q), cache, [0, 1], [3, 3], 64 ** -0.5), BF, 64, [90, 40])
    head_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(q.numel() + 1, dtype=BF, device=DEV)[1:].view(q.shape).copy_(q)
    apart = torch.empty(*q.shape[:3], 128, dtype=BF, device=DEV)[..., ::2].copy_(q)
    for x in (head_major, odd, apart):
        got = ops.paged_attention(x, cache.k, cache.v, cache.table, cache.lens)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_slots(dtype):
    """A call for some of the cache's slots, in another order."""
    _case(dtype, 4, 2, 64, 16, [1, 7, 3], [20, 3, 45], packed=True, slots=[4, 0, 2], seed=6)
    _case(dtype, 4, 2, 64, 16, [2, 2], [20, 3], packed=False, slots=[3, 1], seed=7)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_keys(dtype):
    """Sequences shorter than their new tokens, empty ones, slots out of range: 0, -inf."""
    cache = Cache([3, 0, 20], 2, 64, 8, dtype, 8)
    new, slots = [5, 4, 2, 3, 1], [0, 1, 2, -1, 99]
    q = [cache.rand(n, 4, 64, dtype=dtype) for n in new]
    got = _run(cache, q, new, True, slots)
    want = attention64(q, cache, slots, new, 64 ** -0.5)
    assert bool((want[0][1][:2] == -math.inf).all()) and bool((want[3][1] == -math.inf).all())
    _check(got, want, dtype, 64, [3, 0, 20, 0, 0])


@pytest.mark.parametrize("T", [1, 4, 70])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_missing_pages(T, dtype):
    """Ids out of range hold no keys, the page of the row's own token among them."""
    cache = Cache([200, 150, 90], 2, 128, 16, dtype, 9)
    cache.table[0, 2] = -1
    cache.table[0, 5] = cache.P
    cache.table[1, :] = -1
    cache.table[2, 5] = 2 ** 30
    q = [cache.rand(T, 2, 128, dtype=dtype) for _ in range(3)]
    got = _run(cache, q, [T] * 3, False)
    _check(got, attention64(q, cache, [0, 1, 2], [T] * 3, 128 ** -0.5), dtype, 128,
           [200, 150, 90])


@pytest.mark.parametrize("cached", [20, 4000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_nan_query(dtype, cached):
    """A query that is NaN gives NaN, in one piece or many, and leaves the others alone."""
    cache = Cache([cached + 3, 50], 2, 64, 16, dtype, 28)
    q = [cache.rand(3, 4, 64, dtype=dtype), cache.rand(3, 4, 64, dtype=dtype)]
    want = attention64(q, cache, [0, 1], [3, 3], 64 ** -0.5)
    q[0][1, 2] = math.nan
    got = _run(cache, q, [3, 3], True)
    assert bool(got[0][0][1, 2].isnan().all()) and bool(got[0][1][1, 2].isnan())
    for (out, lse), (o64, l64, *_) in zip(got, want):
        out[out.isnan()] = o64[out.isnan()].to(dtype)
        lse[lse.isnan()] = l64[lse.isnan()].float()
    assert bool(got[0][0].isfinite().all())
    _check(got, want, dtype, 64, [cached + 3, 50])


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf, "lowest"])
@pytest.mark.parametrize("T", [1, 6, 48, 150])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_masked_places_may_hold_anything(T, dtype, poison):
    """Poison in free pages, behind the sequences' ends and at a late token: rows before
    it are what they are without it."""
    value = torch.finfo(dtype).min if poison == "lowest" else poison
    lens = [T + 45, T]
    cache = Cache(lens, 2, 64, 16, dtype, 10, spare=4)
    used = torch.zeros(cache.P, 16, dtype=torch.bool, device=DEV)
    for i, n in enumerate(lens):
        pos = torch.arange(n, device=DEV)
        used[cache.table[i, pos // 16].long(), pos % 16] = True
    for x in (cache.k, cache.v):
        x.transpose(1, 2)[~used] = value
    q = [cache.rand(T, 4, 64, dtype=dtype) for _ in range(2)]
    want = attention64(q, cache, [0, 1], [T, T], 64 ** -0.5)
    _check(_run(cache, q, [T, T], False), want, dtype, 64, lens)
    if T == 1:
        return
    # a token in the chunk: rows from it on see the poison
    late = T - 2
    for i, n in enumerate(lens):
        pos = n - T + late
        cache.v[cache.table[i, pos // 16].long(), :, pos % 16, ::3] = value
        cache.k[cache.table[i, pos // 16].long(), :, pos % 16] = value
    got = _run(cache, q, [T, T], False)
    _check([(o[:late], l[:late]) for o, l in got],
           [(o[:late], l[:late], m[:late], b) for o, l, m, b in want], dtype, 64, lens)
    # values alone: the rows that see them show them where they are, and nowhere else
    if poison != "lowest":
        for i, n in enumerate(lens):
            pos = n - T + late
            cache.k[cache.table[i, pos // 16].long(), :, pos % 16] = 0.5
        for out, _ in _run(cache, q, [T, T], False):
            assert not bool(out[late:, :, ::3].isfinite().any())
            rest = torch.ones(64, dtype=torch.bool, device=DEV)
            rest[::3] = False
            assert bool(out[:, :, rest].isfinite().all())
            assert bool(out[:late].isfinite().all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_scores(dtype):
    """Scores of some thousands, one key far above the others: no overflow."""
    cache = Cache([300, 60], 1, 64, 16, dtype, 11)
    q = [cache.rand(n, 2, 64, dtype=dtype) for n in (2, 40)]
    for i, n in enumerate((300, 60)):
        cache.k[cache.table[i, 1].long(), 0, 3] = 60.0 * q[i][0, 0].sign()
    q = [x * 8 for x in q]
    got = _run(cache, q, [2, 40], True)
    _check(got, attention64(q, cache, [0, 1], [2, 40], 0.125), dtype, 64, [300, 60])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("size", [1e6, 1e20])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_enormous_scores(dtype, size, T):
    """Scores of any finite size: the largest takes all, nothing overflows."""
    cache = Cache([T + 150], 1, 64, 16, dtype, 21)
    cache.k.mul_(size)
    q = [cache.rand(T, 2, 64, dtype=dtype)]
    want = attention64(q, cache, [0], [T], 0.125)
    # (a second key within 2^-10 of the largest would share: none does here)
    out = _run(cache, q, [T], False)[0][0]
    assert float((out.double() - want[0][0]).abs().max()) <= (2.0 ** -8 if dtype == BF else 1e-6) * float(
        cache.v.abs().max())


def test_scores_falling_and_rising_along_the_keys():
    """The running maximum changes in every tile, or never again after the first."""
    for sign in (1.0, -1.0):
        cache = Cache([2000], 1, 128, 64, BF, 12)
        ramp = torch.linspace(0, 40, 2000, device=DEV) * sign
        pos = torch.arange(2000, device=DEV)
        cache.k[cache.table[0, pos // 64].long(), 0, pos % 64, 0] = ramp.to(BF)
        q = cache.rand(100, 2, 128, dtype=BF)
        q[..., 0] = 6.0
        got = _run(cache, [q], [100], False)
        _check(got, attention64([q], cache, [0], [100], 128 ** -0.5), BF, 128, [2000])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new,cached", [([1, 1], [3000, 10]), ([70, 1], [900, 2500])])
def test_hints_do_not_change_results(new, cached, dtype):
    """max_new and max_len that are too small choose another split, within the bound."""
    for hints in ({"max_new": 1, "max_len": 1}, {"max_len": 64}, {"max_new": 40}, {}):
        _case(dtype, 4, 2, 64, 16, new, cached, packed=True, seed=13, **hints)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_offsets_past_32_bits(dtype):
    """Pages more than 2^32 elements into the cache."""
    P = 2 ** 32 // 1024 + 7
    k, v = (torch.empty(P, 1, 16, 64, dtype=dtype, device=DEV) for _ in range(2))
    cache = Cache([40], 1, 64, 16, dtype, 14)
    ids = torch.tensor([P - 1, 5, P - 3], device=DEV)
    k[ids], v[ids] = cache.k[cache.table[0].long()], cache.v[cache.table[0].long()]
    table = ids.int()[None]
    for T in (1, 40):
        q = cache.rand(1, T, 2, 64, dtype=dtype)
        want = _ops().paged_attention(q, cache.k, cache.v, cache.table, cache.lens)
        assert torch.equal(_ops().paged_attention(q, k, v, table, cache.lens), want)
    new = cache.rand(1, 3, 1, 64, dtype=dtype)
    _ops().paged_cache_append(new, new, k, v, table, cache.lens)
    assert torch.equal(k[P - 3, 0, 5:8], new[0, :, 0])


@pytest.mark.parametrize("T", [1, 80])
def test_repeats_are_bitwise_equal(T):
    cache = Cache([5000, 70 + T], 2, 128, 64, BF, 15)
    q = cache.rand(2, T, 4, 128, dtype=BF)
    first = _ops().paged_attention(q, cache.k, cache.v, cache.table, cache.lens)
    for _ in range(3):
        assert torch.equal(_ops().paged_attention(q, cache.k, cache.v, cache.table, cache.lens),
                           first)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_starts_out_of_order_stay_in_range(dtype):
    """Starts that fall, overlap or lie outside: the rows of one sequence only are its own."""
    cache = Cache([200, 30, 40, 500, 20], 4, 64, 16, dtype, 32)
    q = cache.rand(7, 8, 64, dtype=dtype)
    starts = torch.tensor([0, 3, 2, -5, 40, 7], dtype=torch.int32, device=DEV)
    out, lse = _ops().paged_attention(q, cache.k, cache.v, cache.table, cache.lens, starts=starts,
                                      return_lse=True)
    want = attention64([q], cache, [3], [7], 64 ** -0.5)  # (from -5 to 40: all seven rows)
    _check([(out[3:], lse[3:])], [(*(x[3:] for x in want[0][:3]), want[0][3])], dtype, 64, [500])


def test_no_tokens_and_no_sequences():
    cache = Cache([10], 2, 64, 16, BF, 16)
    ops = _ops()
    assert ops.paged_attention(cache.rand(1, 0, 4, 64, dtype=BF), cache.k, cache.v, cache.table,
                               cache.lens).shape == (1, 0, 4, 64)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = cache.rand(0, 4, 64, dtype=BF)
    assert ops.paged_attention(q, cache.k, cache.v, cache.table, cache.lens, starts=none,
                               ).shape == (0, 4, 64)
    # pages of a cache without any
    empty = cache.k[:0]
    q = cache.rand(1, 2, 4, 64, dtype=BF)
    out, lse = ops.paged_attention(q, empty, empty, cache.table, cache.lens, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_other_stream():
    cache = Cache([4000, 900], 2, 128, 64, BF, 17)
    q = cache.rand(2, 1, 4, 128, dtype=BF)
    want = _ops().paged_attention(q, cache.k, cache.v, cache.table, cache.lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _ops().paged_attention(q, cache.k, cache.v, cache.table, cache.lens)
    side.synchronize()
    assert torch.equal(got, want)


def test_step_replays_in_a_graph():
    """Append and attention captured once; lengths, table and tokens change between the
    replays, with eager steps in between."""
    ops = _ops()
    cache = Cache([900, 64, 10], 2, 64, 16, BF, 18, spare=20, width=70)
    q, k, v = (cache.rand(3, 1, n, 64, dtype=BF) for n in (4, 2, 2))

    def step(kp, vp):
        ops.paged_cache_append(k, v, kp, vp, cache.table, cache.lens)
        return ops.paged_attention(q, kp, vp, cache.table, cache.lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache.k, cache.v)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache.k, cache.v)
    for i in range(4):
        cache.lens += torch.tensor([-7, 1, -1], dtype=torch.int32, device=DEV)
        cache.table[1, 4] = cache.P - 1 - i
        for x in (q, k, v):
            x.copy_(cache.rand(*x.shape, dtype=BF))
        kp, vp = cache.k.clone(), cache.v.clone()
        want = step(kp, vp)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(cache.k, kp) and torch.equal(cache.v, vp)


def test_under_compile():
    ops = _ops()
    cache = Cache([30, 64], 2, 64, 16, BF, 19)

    def step(q, k, v, kp, vp, table, lens):
        ops.paged_cache_append(k, v, kp, vp, table, lens)
        return ops.paged_attention(q * 2.0, kp, vp, table, lens)

    q, k, v = (cache.rand(2, 1, n, 64, dtype=BF) for n in (4, 2, 2))
    kp, vp = cache.k.clone(), cache.v.clone()
    want = step(q, k, v, cache.k, cache.v, cache.table, cache.lens)
    got = torch.compile(step, backend="aot_eager")(q, k, v, kp, vp, cache.table, cache.lens)
    assert torch.equal(got, want) and torch.equal(kp, cache.k) and torch.equal(vp, cache.v)


def test_refusals():
    ops = _ops()
    cache = Cache([30, 64], 2, 64, 16, BF, 20)
    q = cache.rand(2, 1, 4, 64, dtype=BF)

    def call(q=q, k=cache.k, v=cache.v, t=cache.table, n=cache.lens, **kw):
        return ops.paged_attention(q, k, v, t, n, **kw)

    call()
    with pytest.raises(TypeError):
        call(q=q.half())
    with pytest.raises(TypeError):
        call(q=q.float())
    with pytest.raises(TypeError):
        call(t=cache.table.long())
    with pytest.raises(RuntimeError):
        call(q=q.cpu())
    with pytest.raises(RuntimeError):
        call(t=cache.table.cpu())
    for bad in (dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(n=cache.lens[:1]),
                dict(t=cache.table[0]), dict(v=cache.v[:1]), dict(k=cache.k[0], v=cache.v[0]),
                dict(slots=torch.zeros(1, dtype=torch.int32, device=DEV)),
                dict(starts=torch.zeros(3, dtype=torch.int32, device=DEV)),
                dict(q=q[0], starts=torch.zeros(0, dtype=torch.int32, device=DEV)),
                dict(max_new=2), dict(max_len=-1), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=math.nan), dict(q=q.repeat(2, 1, 1, 1)),
                dict(q=q[..., :60].contiguous(), k=cache.k[..., :60], v=cache.v[..., :60]),
                dict(k=cache.k[..., ::2].contiguous().expand(-1, -1, -1, 32), v=cache.v),
                dict(k=cache.k.transpose(2, 3), v=cache.v.transpose(2, 3))):
        with pytest.raises(ValueError):
            call(**bad)
    wide = torch.zeros(2, 2, 16, 136, dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        call(q=torch.zeros(2, 1, 4, 136, dtype=BF, device=DEV), k=wide, v=wide)
    with pytest.raises(RuntimeError, match="no_grad"):
        call(q=q.clone().requires_grad_(True))
    with torch.no_grad():
        call(q=q.clone().requires_grad_(True))
    odd = torch.zeros(cache.k.numel() + 1, dtype=BF, device=DEV)[1:].view(cache.k.shape)
    with pytest.raises(ValueError):
        call(k=odd, v=odd)
