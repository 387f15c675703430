"""Steps of the paged cache that do not wait for their status."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
NH, NKVH, D, PAGE = 4, 2, 64, 16


def _cache(num_pages, max_seqs=6):
    from nanochat_amd.paged_kv_cache import PagedKVCache

    cache = PagedKVCache(2, NH, NKVH, D, num_pages=num_pages, max_seqs=max_seqs, max_len=256,
                         page_size=PAGE)
    cache.k_pages.zero_()
    cache.v_pages.zero_()
    return cache


def _layers(step, seed):
    """What a model's layers do with a step; the attention of both."""
    g = torch.Generator(DEV).manual_seed(seed)
    B, T = len(step.positions), step.n_new

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV).bfloat16()

    out = []
    for i in range(2):
        q, k, v = rand(B, T, NH, D), rand(B, T, NKVH, D), rand(B, T, NKVH, D)
        step.update_last_qkv(i, q[:, -1], k[:, -1], v[:, -1])
        out.append(step.attend(i, q, k, v))
    return out


def _state(cache):
    return [t.clone() for t in (cache.k_pages, cache.v_pages, cache.page_table, cache.seq_lens,
                                cache.ref_counts, *cache.rows)]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_step_without_room_changes_nothing():
    """Pages shared by forks, rows, lengths: bit for bit what they were, whatever the layers
    write; so after later steps that would fit, until the failure has been raised."""
    cache = _cache(5)
    _layers(cache.step([0], 40), 1)
    cache.fork([0, 0], [1, 2])
    before = _state(cache)
    bad = cache.step([0, 1, 2], 30, check=False)  # two copies and more pages than are free
    assert all(bool((o == 0).all()) for o in _layers(bad, 2))
    later = cache.step([1], 1, check=False)
    assert all(bool((o == 0).all()) for o in _layers(later, 3))
    assert _same(_state(cache), before)
    assert int(bad.status) == int(later.status) > 0
    with pytest.raises(RuntimeError, match="missing"):
        cache.check_steps()
    assert cache.lens == cache.seq_lens.tolist() == [40, 40, 40, 0, 0, 0]
    assert _same(_state(cache), before)
    # and then goes on as a cache in which nothing failed
    other = _cache(5)
    _layers(other.step([0], 40), 1)
    other.fork([0, 0], [1, 2])
    for a, b in zip(_layers(cache.step([1], 1, check=False), 4), _layers(other.step([1], 1), 4)):
        assert torch.equal(a, b) and bool((a != 0).any())
    cache.check_steps()
    assert _same(_state(cache), _state(other)) and cache.lens == other.lens


def test_a_checked_step_raises_for_those_before():
    cache = _cache(4)
    _layers(cache.step([0], 60), 5)
    before = _state(cache)
    _layers(cache.step([0], 10, check=False), 6)
    cache.fork([0], [1])
    cache.free([0])
    with pytest.raises(RuntimeError, match="missing"):
        cache.step([1], 1)
    assert cache.lens == cache.seq_lens.tolist() == [0, 60, 0, 0, 0, 0]
    assert _same(_state(cache)[:2], before[:2])
    a, b = _layers(cache.step([1], 4), 7)
    assert bool((a != 0).any()) and cache.lens[1] == int(cache.seq_lens[1]) == 64


def test_steps_with_room_are_those_that_wait():
    a, b = _cache(20), _cache(20)
    for cache, check in ((a, True), (b, False)):
        _layers(cache.step([0, 3], 33, check=check), 8)
        cache.fork([3], [1])
        for i in range(4):
            _layers(cache.step([0, 1, 3], 1 + i, check=check), 9 + i)
        cache.check_steps()
    assert _same(_state(a), _state(b)) and a.lens == b.lens == b.seq_lens.tolist()
