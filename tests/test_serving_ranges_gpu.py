"""The serving operators at the ends of their arguments' ranges, and with arguments in
unusual places of memory."""

from __future__ import annotations

import pytest
import torch

from paged_test_utils import DEV, Cache

pytestmark = pytest.mark.gpu


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_expanded_page_table():
    """Several sequences over one row of the table: read as that row, and not written."""
    c = Cache([70], 2, 64, 16, torch.bfloat16, 1)
    lens = _i([70, 33, 50])
    shared, own = c.table.expand(3, -1), c.table.repeat(3, 1)
    q = c.rand(3, 2, 4, 64, dtype=torch.bfloat16)
    assert torch.equal(_ops().paged_attention(q, c.k, c.v, shared, lens),
                       _ops().paged_attention(q, c.k, c.v, own, lens))
    refs = torch.zeros(c.P, dtype=torch.int32, device=DEV)
    one, two = _i([0]), _i([1])
    for call in (lambda: _ops().paged_cache_reserve(shared, lens, refs, one, one, c.k, c.v),
                 lambda: _ops().paged_cache_fork(shared, lens, refs, one, two),
                 lambda: _ops().paged_cache_free(shared, lens, refs, one),
                 lambda: _ops().paged_cache_compact(shared, refs, c.k, c.v)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    # one row may have any stride
    wide = torch.full((4, 9), -1, dtype=torch.int32, device=DEV)
    wide[0, :c.table.shape[1]] = c.table[0]
    x = c.rand(1, 2, 4, 64, dtype=torch.bfloat16)
    assert torch.equal(_ops().paged_attention(x, c.k, c.v, wide[:1], lens[:1]),
                       _ops().paged_attention(x, c.k, c.v, c.table, lens[:1]))


def test_ids_past_32_bits():
    """int64 slots, pages, counts and starts that 32 bits do not hold are out of range, not
    what is left of them."""
    ops, far = _ops(), 2 ** 32
    c = Cache([40, 20], 2, 64, 16, torch.bfloat16, 2, spare=4, width=6)
    refs = torch.bincount(c.table[c.table >= 0], minlength=c.P).int()

    def state():
        return [x.clone() for x in (c.table, c.lens, refs, c.k, c.v)]

    def same(a):
        return all(torch.equal(x, y) for x, y in zip(a, state()))

    before, l = state(), lambda *v: torch.tensor(v, device=DEV)
    ops.paged_cache_free(c.table, c.lens, refs, l(far, -far, far + 1))
    ops.paged_cache_fork(c.table, c.lens, refs, l(far, 1), l(1, far))
    ops.paged_cache_copy(c.k, c.v, l(far, 0, -far), l(1, far + 2, 3))
    assert same(before)
    for slots, counts in ((l(far), l(1)), (l(0), l(far + 1)), (l(0), l(-far))):
        assert int(ops.paged_cache_reserve(c.table, c.lens, refs, slots, counts, c.k, c.v)) == -1
    assert same(before)
    q = c.rand(3, 4, 64, dtype=torch.bfloat16)
    out, lse = ops.paged_attention(q, c.k, c.v, c.table, c.lens, slots=l(far, 1),
                                   starts=l(0, 2, far + 3), return_lse=True)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -float("inf")).all())
    want = ops.paged_attention(q[2:], c.k, c.v, c.table, c.lens, slots=l(1), starts=l(0, 1))
    assert torch.equal(out[2:], want)


@pytest.mark.parametrize("page,width,counts", [(1_500_000_000, 1, [1_400_000_000, 1, 1]),
                                               (2 ** 20, 2047, [2047 * 2 ** 20, 2 ** 20, 1]),
                                               (2 ** 31 - 1, 1, [2 ** 31 - 1, 0, 5])])
def test_reserve_of_very_long_sequences(page, width, counts):
    """Lengths whose rounding up to pages passes 31 bits (of a cache without layers: the
    bookkeeping alone)."""
    held = [-(-n // page) for n in counts]
    P = sum(held) + 1
    k = torch.empty(0, P, 1, page, 1, dtype=torch.uint8, device=DEV)
    table = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    lens, refs = _i([0, 0, 0]), torch.zeros(P, dtype=torch.int32, device=DEV)
    assert int(_ops().paged_cache_reserve(table, lens, refs, _i([0, 1, 2]), _i(counts), k, k)) == 0
    assert lens.tolist() == counts and refs.tolist() == [1] * (P - 1) + [0]
    rows, at = table.tolist(), 0
    for row, n in zip(rows, held):
        assert row == list(range(at, at + n)) + [-1] * (width - n)
        at += n


def test_reserve_of_more_pages_than_31_bits_count():
    """3,000 slots that want 2^20 pages each: missing, with nothing changed."""
    n, width = 3000, 2 ** 20
    k = torch.empty(0, 9, 1, 1, 8, dtype=torch.bfloat16, device=DEV)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    lens, refs = torch.zeros(n, dtype=torch.int32, device=DEV), _i([0] * 9)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    for many, missing in ((n, 2 ** 31 - 1), (2000, 2000 * width - 9), (4, 4 * width - 9)):
        counts = torch.full((many,), width, dtype=torch.int32, device=DEV)
        status = _ops().paged_cache_reserve(table, lens, refs, slots[:many], counts, k, k)
        assert int(status) == missing
        assert int(lens.abs().sum()) == int(refs.sum()) == 0 and int(table.max()) == -1


def test_numbers_that_float32_does_not_hold():
    c = Cache([40], 2, 64, 16, torch.bfloat16, 3)
    q = c.rand(1, 1, 4, 64, dtype=torch.bfloat16)
    for scale in (1e-60, 1e39, 3e38, 1e300):
        with pytest.raises(ValueError):
            _ops().paged_attention(q, c.k, c.v, c.table, c.lens, scale=scale)
    x, t = torch.randn(4, 50, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for cap in (1e-60, 1e39, 1e300):
        with pytest.raises(ValueError):
            _ops().token_logprobs(x, t, softcap=cap)


def test_strides_of_axes_of_one_element():
    """Pages that are laid out alike but for strides that say nothing."""
    g = torch.Generator(DEV).manual_seed(4)
    k = torch.randn(3, 10, 1, 16, 8, generator=g, device=DEV)
    v = torch.randn(3, 10, 16, 1, 8, generator=g, device=DEV).transpose(2, 3)
    assert k.stride(2) != v.stride(2)
    for a, b in ((k, v), (k[0], v[0])):
        wk, wv = a.clone(), b.clone()
        wk[..., 7, :, :, :], wv[..., 7, :, :, :] = wk[..., 2, :, :, :], wv[..., 2, :, :, :]
        _ops().paged_cache_copy(a, b, _i([2]), _i([7]))
        assert torch.equal(a, wk) and torch.equal(b, wv)
    # one page, one layer
    odd = torch.randn(2 * 16 * 8 + 1, generator=g, device=DEV)
    one = odd[:128].as_strided((1, 1, 1, 16, 8), (129, 129, 128, 8, 1))
    table, lens, refs = _i([[-1]]), _i([0]), _i([0])
    assert int(_ops().paged_cache_reserve(table, lens, refs, _i([0]), _i([3]), one, one)) == 0
    assert table.tolist() == [[0]] and refs.tolist() == [1]
    assert int(_ops().paged_cache_compact(table, refs, one, one)) == 1


@pytest.mark.parametrize("scale", [1.0, 2.0 ** 24, 1e12, 1e30])
def test_gradient_of_a_scaled_entropy(scale):
    """A loss scaled up: masked entries keep a gradient of 0."""
    g = torch.Generator(DEV).manual_seed(5)
    x = torch.randn(3, 300, generator=g, device=DEV)
    x[0, ::2], x[1, ::3] = -float("inf"), torch.finfo(torch.float32).min
    x.requires_grad_(True)
    t = torch.ones(3, dtype=torch.int64, device=DEV)
    (one,) = torch.autograd.grad(_ops().token_logprobs(x, t).entropy.sum(), [x])
    (got,) = torch.autograd.grad((_ops().token_logprobs(x, t).entropy * scale).sum(), [x])
    assert bool(got.isfinite().all())
    assert bool((got[0, ::2] == 0).all()) and bool((got[1, ::3] == 0).all())
    assert float((got / scale - one).abs().max()) <= 2.0 ** -20
