"""The paged cache's bookkeeping against a host model that works entry after entry, and
its copies bit for bit."""

from __future__ import annotations

import random

import pytest
import torch

from paged_test_utils import DEV, Cache, PageModel

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class State:
    """A cache on the device beside its model; page p of the model holds the content
    number pages[p], as every element of the device's page does."""

    def __init__(self, S, W, P, page, layers=2, NKVH=2, D=8, dtype=BF, layout="head"):
        self.m = PageModel([[-1] * W] * S, [0] * S, [0] * P, page)
        self.table, self.lens, self.refs = _i(self.m.table), _i(self.m.lens), _i(self.m.refs)
        shape = (layers, P, NKVH, page, D) if layout == "head" else (layers, P, page, NKVH, D)
        content = (torch.arange(P, device=DEV) % 251).to(dtype).view(1, P, 1, 1, 1)
        self.k = content.expand(shape).contiguous()
        self.v = (-content).expand(shape).contiguous()
        if layout != "head":
            self.k, self.v = self.k.transpose(2, 3), self.v.transpose(2, 3)

    def reserve(self, slots, counts):
        status = _ops().paged_cache_reserve(self.table, self.lens, self.refs, _i(slots),
                                            _i(counts), self.k, self.v)
        assert int(status) == self.m.reserve(slots, counts)
        return int(status)

    def fork(self, src, dst):
        _ops().paged_cache_fork(self.table, self.lens, self.refs, _i(src), _i(dst))
        self.m.fork(src, dst)

    def free(self, slots):
        _ops().paged_cache_free(self.table, self.lens, self.refs, _i(slots))
        self.m.free(slots)

    def compact(self):
        live = _ops().paged_cache_compact(self.table, self.refs, self.k, self.v)
        assert int(live) == self.m.compact()

    def check(self):
        assert self.table.tolist() == self.m.table
        assert self.lens.tolist() == self.m.lens
        assert self.refs.tolist() == self.m.refs
        want = (_i(self.m.pages) % 251).to(self.k.dtype).view(1, -1, 1, 1, 1)
        assert torch.equal(self.k, want.expand(self.k.shape))
        assert torch.equal(self.v, (-want).expand(self.v.shape))
        held = [p for r in self.m.table for p in r if 0 <= p < len(self.m.refs)]
        assert [held.count(p) for p in range(len(self.m.refs))] == self.m.refs


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [1, 4, 16])
def test_random_operations(page, seed):
    rng = random.Random(seed * 10 + page)
    S, W = 12, 9
    s = State(S, W, rng.choice([20, 70, 130]), page, layout=rng.choice(["head", "token"]))
    for _ in range(40):
        what = rng.choice(["reserve"] * 4 + ["fork"] * 2 + ["free", "compact"])
        if what == "reserve":
            slots = rng.sample(range(S), rng.randint(1, S))
            s.reserve(slots, [rng.choice([0, 1, 1, 2, page, 2 * page + 1]) for _ in slots])
        elif what == "fork":
            n = rng.randint(1, S // 2)
            slots = rng.sample(range(S), S)
            dst = slots[:n]
            s.fork([rng.choice(slots[n:] + [d]) for d in dst], dst)
        elif what == "free":
            s.free(rng.sample(range(S), rng.randint(1, 4)))
        else:
            s.compact()
        s.check()


def test_shared_last_page_parts_in_order():
    """Five slots hold one partly filled page: four copies in the order of the entries,
    the last keeps the page; with a sixth holder outside, everyone copies."""
    s = State(8, 4, 30, 8)
    s.reserve([0], [13])
    s.fork([0] * 4, [1, 2, 3, 4])
    s.reserve([3, 0, 4, 2, 1], [1, 2, 1, 8, 1])
    s.check()
    assert s.m.table[1][1] == 1  # the last entry
    s = State(8, 4, 30, 8)
    s.reserve([0], [13])
    s.fork([0] * 5, [1, 2, 3, 4, 5])
    s.reserve([3, 4, 2, 1], [1, 1, 0, 1])
    s.check()
    assert s.m.table[0] == s.m.table[5] == s.m.table[2]


def test_missing_pages_change_nothing():
    s = State(4, 8, 10, 4)
    s.reserve([0, 1], [15, 9])
    s.fork([1], [2])
    before = (s.table.clone(), s.lens.clone(), s.refs.clone(), s.k.clone())
    # three pages free; a copy for slot 2 or 1 and more
    assert s.reserve([1, 2, 3], [1, 1, 12]) == 1
    assert s.reserve([3], [32]) == 5
    for a, b in zip(before, (s.table, s.lens, s.refs, s.k)):
        assert torch.equal(a, b)
    assert s.reserve([1, 2, 3], [1, 1, 8]) == 0
    s.check()


@pytest.mark.parametrize("slots,counts", [([0, 4], [1, 1]), ([-1], [1]), ([0], [-1]),
                                          ([0], [33]), ([0, 1], [1, 2 ** 31 - 1])])
def test_out_of_range_changes_nothing(slots, counts):
    s = State(4, 8, 40, 4)
    s.reserve([1], [3])
    assert s.reserve(slots, counts) == -1
    s.check()


def test_free_and_fork_of_what_is_not_there():
    """Empty slots, slots out of range, a slot named twice, its own fork."""
    s = State(5, 4, 20, 4)
    s.reserve([0, 1], [10, 3])
    s.free([3, -1, 7])
    s.check()
    s.fork([0, 9, 1, -2], [0, 2, 9, 3])
    s.check()
    _ops().paged_cache_free(s.table, s.lens, s.refs, _i([0, 0]))
    s.m.free([0])
    s.check()
    s.compact()
    s.check()


def test_a_slot_named_twice_stays_in_range():
    """Distinct slots are the caller's part; what comes of others is not defined, but the
    pages it gives are pages."""
    s = State(4, 3, 20, 4)
    s.reserve([0, 1], [10, 5])
    s.fork([0], [2])
    _ops().paged_cache_reserve(s.table, s.lens, s.refs, _i([0, 0, 0]), _i([1, 2, 2]), s.k, s.v)
    assert bool((s.table >= -1).all()) and bool((s.table < 20).all())
    assert bool((s.lens <= 12).all()) and bool((s.lens >= 0).all())


@pytest.mark.parametrize("P", [1, 63, 64, 1023, 1024, 1025, 5000])
def test_many_pages(P):
    """Scans over several rounds of the workgroup; every other page a hole."""
    S = 7
    W = -(-P // S)
    s = State(S, W, P, 1, layers=1, NKVH=1)
    s.reserve(list(range(S)), [P // S] * S)
    s.check()
    s.free([0, 2, 3])
    s.reserve([5], [W - P // S])
    s.compact()
    s.check()
    s.compact()
    s.check()


def test_many_entries():
    """More entries than the workgroup has threads."""
    n = 1500
    s = State(2 * n, 2, 3 * n, 4, layers=1, NKVH=1)
    s.reserve(list(range(n)), [i % 7 for i in range(n)])
    s.fork(list(range(n)), list(range(n, 2 * n)))
    s.check()
    s.reserve(list(range(n, 2 * n)), [1] * n)
    s.check()


def test_pages_with_holes_in_the_table():
    """Rows with ids that are no pages: they are left where they are."""
    s = State(3, 6, 20, 4)
    s.reserve([0, 1], [18, 24])
    for t in (s.table, ):
        t[0, 1] = -1
        t[1, 2] = 10 ** 9
    s.m.table[0][1] = -1
    s.m.table[1][2] = 10 ** 9
    s.fork([0], [2])
    s.free([1])
    s.compact()
    assert s.table.tolist() == s.m.table and s.refs.tolist() == s.m.refs


@pytest.mark.parametrize("dtype", [BF, F32, torch.float16, torch.uint8])
def test_copy(dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randint(0, 200, (3, 40, 2, 16, 72), generator=g, device=DEV).to(dtype)
            for _ in range(2))
    src, dst = [3, 5, -1, 7, 40, 9, 2 ** 31 - 1, 8], [0, 39, 1, -5, 2, 9, 4, 100]
    wk, wv = k.clone(), v.clone()
    for a, b in ((3, 0), (5, 39)):
        wk[:, b], wv[:, b] = wk[:, a], wv[:, a]
    _ops().paged_cache_copy(k, v, _i(src), _i(dst))
    assert torch.equal(k, wk) and torch.equal(v, wv)
    # one layer, ids as int64, a slice of a wider allocation
    both = torch.randn(10, 2, 4, 16, 64, generator=g, device=DEV)
    want = both.clone()
    want[7] = want[2]
    _ops().paged_cache_copy(both[:, 0], both[:, 1], torch.tensor([2], device=DEV),
                            torch.tensor([7], device=DEV))
    assert torch.equal(both, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,page,layout", [(64, 16, "head"), (128, 48, "token"), (72, 1, "gaps")])
@pytest.mark.parametrize("packed", [False, True])
def test_append(D, page, layout, packed, dtype):
    """Rows land where the table says; negative positions and missing pages are dropped."""
    new = [3, 3, 3, 3] if not packed else [1, 0, 50, 3]
    cache = Cache([40, 2, 90, 17], 3, D, page, dtype, 2, layout=layout)
    cache.table[0, -(-40 // page) - 1] = -1
    k, v = (cache.rand(sum(new), 3, D, dtype=dtype) for _ in range(2))
    wk, wv = cache.k.clone(), cache.v.clone()
    row = 0
    for i, n in enumerate(new):
        for t in range(n):
            pos = int(cache.lens[i]) - n + t
            if pos >= 0 and int(cache.table[i, pos // page]) >= 0:
                wk[int(cache.table[i, pos // page]), :, pos % page] = k[row]
                wv[int(cache.table[i, pos // page]), :, pos % page] = v[row]
            row += 1
    kw = {}
    if packed:
        kw = {"starts": _i([0, 1, 1, 51, 54])}
    else:
        # head-major, as the filter's outputs are, and v at an odd element
        k = k.view(4, 3, 3, D).transpose(1, 2).contiguous().transpose(1, 2)
        v = torch.empty(v.numel() + 1, dtype=dtype, device=DEV)[1:].view(4, 3, 3, D).copy_(
            v.view(4, 3, 3, D))
    _ops().paged_cache_append(k, v, cache.k, cache.v, cache.table, cache.lens, **kw)
    assert torch.equal(cache.k, wk) and torch.equal(cache.v, wv)


def test_starts_out_of_range_stay_in_range():
    """Starts past the rows, negative or descending: the rows there are, no others."""
    cache = Cache([40, 40], 1, 64, 16, F32, 3)
    before = cache.k.clone()
    k = cache.rand(5, 1, 64)
    _ops().paged_cache_append(k, k, cache.k, cache.v, cache.table, cache.lens,
                              starts=_i([3, 1000, 4]))
    # sequence 0: rows 3 .. 5 (the last two tokens); sequence 1: none
    want = before.clone()
    for j, pos in enumerate((38, 39)):
        want[int(cache.table[0, pos // 16]), :, pos % 16] = k[3 + j]
    assert torch.equal(cache.k, want)


def test_under_compile():
    a, b = State(4, 4, 20, 4), State(4, 4, 20, 4)

    def steps(t, n, r, k, v, one, two, counts):
        ops = _ops()
        status = ops.paged_cache_reserve(t, n, r, one, counts, k, v)
        ops.paged_cache_fork(t, n, r, one, two)
        ops.paged_cache_reserve(t, n, r, two, counts, k, v)
        ops.paged_cache_free(t, n, r, one)
        ops.paged_cache_copy(k, v, one, two)
        return status, ops.paged_cache_compact(t, r, k, v)

    args = (_i([0]), _i([2]), _i([6]))
    want = steps(a.table, a.lens, a.refs, a.k, a.v, *args)
    got = torch.compile(steps, backend="aot_eager")(b.table, b.lens, b.refs, b.k, b.v, *args)
    for x, y in zip((*want, a.table, a.lens, a.refs, a.k, a.v),
                    (*got, b.table, b.lens, b.refs, b.k, b.v)):
        assert torch.equal(x, y)


def test_refusals():
    ops = _ops()
    s = State(4, 4, 20, 4)
    one = _i([0])

    def reserve(t=s.table, n=s.lens, r=s.refs, a=one, c=one, k=s.k, v=s.v):
        return ops.paged_cache_reserve(t, n, r, a, c, k, v)

    for bad in (dict(t=s.table[0]), dict(n=s.lens[:2]), dict(r=s.refs[:5]), dict(a=_i([0, 1])),
                dict(a=_i([[0]])), dict(v=s.v[:1]), dict(k=s.k[0, 0], v=s.v[0, 0]),
                dict(k=s.k[..., :4], v=s.v[..., :4]), dict(t=s.table.t()),
                dict(k=s.k.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            reserve(**bad)
    for bad in (dict(t=s.table.long()), dict(a=one.float()), dict(v=s.v.float())):
        with pytest.raises(TypeError):
            reserve(**bad)
    for bad in (dict(t=s.table.cpu()), dict(a=one.cpu()), dict(k=s.k.cpu(), v=s.v.cpu())):
        with pytest.raises(RuntimeError):
            reserve(**bad)
    with pytest.raises(ValueError):
        ops.paged_cache_fork(s.table, s.lens, s.refs, one, _i([1, 2]))
    with pytest.raises(ValueError):
        ops.paged_cache_copy(s.k, s.v, one, _i([1, 2]))
    with pytest.raises(RuntimeError):  # pages of 6 bytes
        x = torch.zeros(4, 1, 1, 3, dtype=BF, device=DEV)
        ops.paged_cache_copy(x, x.clone(), one, _i([1]))
    k = torch.zeros(4, 1, 2, 8, dtype=BF, device=DEV)
    for bad in (k[:, :, :, :4], k[:, 0], torch.zeros(4, 1, 1, 8, dtype=BF, device=DEV)):
        with pytest.raises(ValueError):
            ops.paged_cache_append(bad, bad, s.k[0], s.v[0], s.table, s.lens)
    with pytest.raises(RuntimeError, match="no_grad"):
        x = k.clone().requires_grad_(True)
        ops.paged_cache_append(x, x, s.k[0], s.v[0], s.table, s.lens)
    # nothing to do
    none = _i([])
    assert int(reserve(a=none, c=none)) == 0
    ops.paged_cache_fork(s.table, s.lens, s.refs, none, none)
    ops.paged_cache_free(s.table, s.lens, s.refs, none)
    ops.paged_cache_copy(s.k, s.v, none, none)
    s.check()
