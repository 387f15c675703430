"""CPU checks of what the GPT harness refuses before anything reaches the device."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


@pytest.fixture(scope="module")
def model():
    from nanochat_amd.gpt import GPT, GPTConfig
    return GPT(GPTConfig(sequence_len=64, vocab_size=50, n_layer=1, n_head=2, n_kv_head=1,
                         n_embd=32, ltv_r=16))


@pytest.mark.parametrize("positions,T", [([64], 1), ([0, 60], 5), ([0], 65)])
def test_positions_past_the_rotary_table(model, positions, T):
    """A cache may have room for more tokens than the model."""
    step = SimpleNamespace(positions=positions)
    with pytest.raises(ValueError, match="made for 64"):
        model.cached_features(torch.zeros(len(positions), T, dtype=torch.int64), step)


@pytest.mark.parametrize("tokens", [[3, 50], [-1, 3], [2 ** 40, 1]])
def test_tokens_outside_the_vocabulary(model, tokens):
    from nanochat_amd import engine

    cache = engine.make_cache(model, num_pages=4, max_seqs=2, page_size=16)
    for call in (lambda: engine.prefill(model, cache, 0, tokens),
                 lambda: engine.generate(model, tokens, 1, 3, cache=cache),
                 lambda: engine.score(model, tokens, cache=cache)):
        with pytest.raises(ValueError, match="tokens are 0 to 49"):
            call()


@pytest.mark.parametrize("kw", [dict(top_k=0), dict(top_k=51), dict(top_k=-3),
                                dict(max_tokens=63), dict(num_samples=3)])
def test_generate_refuses_before_it_begins(model, kw):
    """top_k outside the vocabulary, more tokens than there is room for, too few slots."""
    from nanochat_amd import engine

    cache = engine.make_cache(model, num_pages=4, max_seqs=2, page_size=16)
    args = dict(num_samples=2, max_tokens=3, top_k=5, cache=cache) | kw
    with pytest.raises(ValueError):
        engine.generate(model, [1, 2, 3], **args)
