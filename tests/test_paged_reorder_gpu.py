"""Slots that exchange their sequences, against the bookkeeping done one after the other."""

from __future__ import annotations

import random

import pytest
import torch

from paged_test_utils import DEV, PageModel

pytestmark = pytest.mark.gpu


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _model(S, W, page, seed):
    """Slots with sequences of random lengths, some of them forks of others."""
    r = random.Random(seed)
    m = PageModel([[-1] * W for _ in range(S)], [0] * S, [0] * (S * W + 3), page)
    for s in range(S):
        if s and r.random() < 0.4:
            m.fork([r.randrange(s)], [s])
        else:
            assert m.reserve([s], [r.randint(0, W * page - 2)]) == 0
    return m


def _reorder(m, slots, src):
    """All at once, on the host."""
    S, P = len(m.lens), len(m.refs)
    pairs = [(a, b) for a, b in zip(slots, src) if 0 <= a < S and 0 <= b < S]
    rows = [(list(m.table[b]), m.lens[b]) for _, b in pairs]
    for (a, _), (row, n) in zip(pairs, rows):
        for p in m.table[a]:
            if 0 <= p < P:
                m.refs[p] -= 1
        m.table[a], m.lens[a] = row, n
        for p in row:
            if 0 <= p < P:
                m.refs[p] += 1


def _check(m, slots, src, stride=None):
    W = len(m.table[0])
    table = torch.full((len(m.lens), stride or W), -9, dtype=torch.int32, device=DEV)[:, :W]
    table.copy_(_ints(m.table))
    lens, refs = _ints(m.lens), _ints(m.refs)
    _ops().paged_cache_reorder(table, lens, refs, _ints(slots), _ints(src))
    _reorder(m, slots, src)
    assert table.tolist() == m.table and lens.tolist() == m.lens and refs.tolist() == m.refs
    assert all(r >= 0 for r in m.refs)


# (more than 2,048 entries go by way of memory; 4 to 64 columns to a workgroup)
@pytest.mark.parametrize("S,W,page", [(1, 1, 16), (2, 3, 1), (5, 7, 16), (64, 20, 16), (7, 700, 4),
                                      (300, 67, 16), (512, 33, 16), (513, 5, 16), (900, 18, 1), (2048, 5, 16), (2049, 5, 16), (2600, 9, 4)])
def test_selections(S, W, page):
    r = random.Random(S)
    for seed in range(4):
        m = _model(S, W, page, seed)
        slots = r.sample(range(S), r.randint(1, S))
        _check(m, slots, [r.randrange(S) for _ in slots])         # any
        _check(m, slots, [slots[i - 1] for i in range(len(slots))])  # a cycle
        _check(m, slots, slots)                                   # as they are
        _check(m, slots, [slots[0]] * len(slots), stride=W + 3)   # all alike


def test_out_of_range():
    m = _model(6, 5, 4, 1)
    _check(m, [0, 9, -1, 3, 2], [5, 1, 2, -4, 6])


def test_ids_of_no_page():
    """Table entries outside the pages move, and no count follows them."""
    m = _model(4, 5, 4, 2)
    m.table[1] = [99999, -7, m.table[1][2], -1, 2147483647]
    for p in range(len(m.refs)):
        m.refs[p] = sum(row.count(p) for row in m.table)
    _check(m, [0, 1, 2], [1, 2, 1])


def test_empty_and_64_bits():
    m = _model(4, 5, 4, 3)
    table, lens, refs = _ints(m.table), _ints(m.lens), _ints(m.refs)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    _ops().paged_cache_reorder(table, lens, refs, none, none)
    assert table.tolist() == m.table and refs.tolist() == m.refs
    far = torch.tensor([0, 1 << 32], device=DEV)
    _ops().paged_cache_reorder(table, lens, refs, torch.tensor([1, 2], device=DEV), far)
    _reorder(m, [1], [0])
    assert table.tolist() == m.table and lens.tolist() == m.lens and refs.tolist() == m.refs


def test_captured():
    m = _model(8, 6, 4, 4)
    table, lens, refs = _ints(m.table), _ints(m.lens), _ints(m.refs)
    slots, src = _ints(list(range(8))), _ints([0] * 8)
    first = [t.clone() for t in (table, lens, refs)]
    _ops().paged_cache_reorder(table, lens, refs, slots, slots)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _ops().paged_cache_reorder(table, lens, refs, slots, src)
    for t, w in zip((table, lens, refs), first):
        t.copy_(w)
    r = random.Random(5)
    for _ in range(5):
        pick = [r.randrange(8) for _ in range(8)]
        src.copy_(_ints(pick))
        graph.replay()
        torch.cuda.synchronize()
        _reorder(m, list(range(8)), pick)
        assert table.tolist() == m.table and lens.tolist() == m.lens and refs.tolist() == m.refs


def test_compiled():
    m = _model(8, 6, 4, 6)
    table, lens, refs = _ints(m.table), _ints(m.lens), _ints(m.refs)
    slots, src = _ints([0, 1, 2]), _ints([2, 0, 5])
    torch.compile(lambda: _ops().paged_cache_reorder(table, lens, refs, slots, src), fullgraph=True,
                  backend="eager")()
    _reorder(m, [0, 1, 2], [2, 0, 5])
    assert table.tolist() == m.table and lens.tolist() == m.lens and refs.tolist() == m.refs


def test_refusals():
    t, n, r = _ints([[0, 1], [2, -1]]), _ints([5, 3]), _ints([1, 1, 1, 0])
    f = _ops().paged_cache_reorder
    with pytest.raises(ValueError):
        f(t, n, r, _ints([0, 1]), _ints([0]))
    with pytest.raises(ValueError):
        f(t, n, r, _ints([[0]]), _ints([[0]]))
    with pytest.raises(ValueError):
        f(t[:1].expand(2, 2), n, r, _ints([0]), _ints([1]))
    with pytest.raises(ValueError):
        f(t, n[:1], r, _ints([0]), _ints([1]))
    with pytest.raises(TypeError):
        f(t, n, r, _ints([0]).float(), _ints([1]))
    with pytest.raises(TypeError):
        f(t.long(), n, r, _ints([0]), _ints([1]))
    with pytest.raises(RuntimeError):
        f(t.cpu(), n, r, _ints([0]), _ints([1]))
    with pytest.raises(RuntimeError):
        f(t, n, r, _ints([0]).cpu(), _ints([1]))
