"""The GPT harness and the slots of a caller's cache: sequences that are there stay, and what
fails leaves nothing behind."""

from __future__ import annotations

import pytest
import torch

from test_engine_gpu import _tokens, model  # noqa: F401

pytestmark = pytest.mark.gpu


def _state(cache):
    return [t.clone() for t in (cache.k_pages, cache.v_pages, cache.page_table, cache.seq_lens,
                                cache.ref_counts)] + [torch.tensor(cache.lens)]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("slot", [0, 1])
def test_occupied_slots_are_refused(model, slot):  # noqa: F811
    from nanochat_amd import engine
    cache = engine.make_cache(model, num_pages=30, max_seqs=4, page_size=16)
    cache.k_pages.zero_()
    cache.v_pages.zero_()
    engine.prefill(model, cache, slot, _tokens(40))
    before = _state(cache)
    for call in (lambda: engine.prefill(model, cache, slot, _tokens(3)),
                 lambda: engine.generate(model, _tokens(5), 2, 4, cache=cache),
                 lambda: engine.score(model, _tokens(9), cache=cache, slot=slot)):
        with pytest.raises(ValueError, match="holds 40 tokens"):
            call()
        assert _same(_state(cache), before)
    # beside it there is room
    engine.score(model, _tokens(9), cache=cache, slot=3)
    assert cache.lens[slot] == 40 and sum(cache.lens) == 40


def test_what_fails_leaves_nothing_behind(model):  # noqa: F811
    """Pages that run out among the samples, in a prompt, in a text: the slots are empty
    again, a sequence beside them is what it was."""
    from nanochat_amd import engine
    cache = engine.make_cache(model, num_pages=9, max_seqs=4, page_size=16)
    engine.prefill(model, cache, 3, _tokens(30))
    held = [x[:, cache.page_table[3, :2].long()].clone() for x in (cache.k_pages, cache.v_pages)]
    for call in (lambda: engine.generate(model, _tokens(20), 3, 60, cache=cache),
                 lambda: engine.prefill(model, cache, 1, _tokens(150), chunk=50),
                 lambda: engine.score(model, _tokens(200), cache=cache, slot=2, chunk=64)):
        with pytest.raises(RuntimeError, match="missing"):
            call()
        assert cache.lens == cache.seq_lens.tolist() == [0, 0, 0, 30]
        assert int(cache.ref_counts.sum()) == 2
        for x, y in zip((cache.k_pages, cache.v_pages), held):
            assert torch.equal(x[:, cache.page_table[3, :2].long()], y)
    assert len(engine.generate(model, _tokens(20), 3, 5, cache=cache)) == 3
