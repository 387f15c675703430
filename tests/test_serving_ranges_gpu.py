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
