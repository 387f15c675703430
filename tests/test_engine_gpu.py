"""The GPT harness over the paged cache: chunks, single tokens, forks and compaction
give what the whole-sequence forward gives."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 300


@pytest.fixture(scope="module")
def model():
    from nanochat_amd.gpt import GPT, GPTConfig
    torch.manual_seed(0)
    m = GPT(GPTConfig(sequence_len=512, vocab_size=VOCAB, n_layer=3, n_head=4, n_kv_head=2,
                      n_embd=256, ltv_r=64)).to(DEV)
    m.init_weights(randomise_output_projections=True)
    m.lm_head.weight.data.normal_(0.0, 0.05, generator=torch.Generator(DEV).manual_seed(1))
    m.wte.to(dtype=torch.bfloat16)
    return m


def _tokens(n, seed=0):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _whole(model, tokens):
    """The training forward's log probabilities of tokens[1:], (n - 1, vocabulary)."""
    idx = torch.tensor(tokens, device=DEV)[None]
    with torch.no_grad(), torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        return torch.log_softmax(model(idx)[0, :-1].float(), -1)


@pytest.mark.parametrize("chunk", [1000, 64, 7, 1])
def test_score_matches_the_whole_forward(model, chunk):
    """bf16 activations through three layers: the logits of the two dataflows differ by
    their roundings, about 2^-8 of their size at each; the capped logits are about 1."""
    from nanochat_amd import engine
    tokens = _tokens(200 if chunk > 1 else 40)
    want = _whole(model, tokens)
    got = engine.score(model, tokens, top_k=5, chunk=chunk)
    y = torch.tensor(tokens[1:], device=DEV)
    chosen = want.gather(1, y[:, None])[:, 0]
    assert float((got.logprobs - chosen).abs().max()) <= 0.1
    assert float((got.logprobs - chosen).abs().mean()) <= 0.02
    ent = -(want.exp() * want).sum(-1)
    assert float((got.entropy - ent).abs().max()) <= 0.1
    assert got.top_ids.shape == (len(y), 5)
    assert float((got.top_logprobs - want.gather(1, got.top_ids)).abs().max()) <= 0.1


def test_greedy_generation_continues_as_scoring_says(model):
    from nanochat_amd import engine
    prompt = _tokens(70, seed=2)
    samples = engine.generate(model, prompt, 3, 40, temperature=0.0, top_k=4, chunk=32)
    assert all(s == samples[0] for s in samples) and len(samples[0].tokens) == 40
    got = engine.score(model, prompt + samples[0].tokens, top_k=1)
    lp = got.logprobs[len(prompt) - 1:].tolist()
    assert max(abs(a - b) for a, b in zip(lp, samples[0].logprobs)) <= 0.1
    # each token is the most probable one, up to the dataflows' rounding
    best = got.top_logprobs[len(prompt) - 1:, 0].tolist()
    assert max(b - a for a, b in zip(lp, best)) <= 0.1


def test_samples_share_the_prompt_and_part_ways(model):
    from nanochat_amd import engine
    prompt = _tokens(100, seed=3)
    page = 16
    cache = engine.make_cache(model, num_pages=64, max_seqs=5, page_size=page)
    samples = engine.generate(model, prompt, 5, 30, top_k=20, seed=4, cache=cache, chunk=50)
    assert len({tuple(s.tokens) for s in samples}) > 1
    assert int(cache.ref_counts.sum()) == 0 and cache.lens == [0] * 5
    for s in samples[:2]:
        got = engine.score(model, prompt + s.tokens, cache=cache, slot=3)
        lp = got.logprobs[len(prompt) - 1:].tolist()
        assert max(abs(a - b) for a, b in zip(lp, s.logprobs)) <= 0.1
        assert all(p <= 0 and math.isfinite(p) for p in s.logprobs)


def test_stopped_samples_make_room(model):
    """A stop token ends a sample; the others' pages move down afterwards."""
    from nanochat_amd import engine
    prompt = _tokens(20, seed=5)
    free = engine.generate(model, prompt, 4, 25, top_k=8, seed=6)
    stop = free[1].tokens[3]
    got = engine.generate(model, prompt, 4, 25, top_k=8, seed=6, stop=stop)
    for a in got:
        assert stop not in a.tokens[:-1]
        assert len(a.tokens) == 25 or a.tokens[-1] == stop
    assert any(len(a.tokens) < 25 for a in got)


def test_cache_moves_sequences(model):
    """fork, free and compact between steps do not change what a sequence continues
    with, bit for bit."""
    from nanochat_amd import engine
    prompts = [_tokens(n, seed=7 + n) for n in (50, 33, 80)]
    nxt = torch.tensor([[5], [6], [7]], device=DEV)

    def run(move):
        cache = engine.make_cache(model, num_pages=40, max_seqs=8, page_size=8)
        for s, p in enumerate(prompts):
            engine.prefill(model, cache, s, p, chunk=40)
        slots = [0, 1, 2]
        if move:
            cache.fork([1, 0], [6, 7])
            cache.free([0, 1])
            cache.compact()
            assert int((cache.ref_counts > 0).nonzero().max()) + 1 == int(cache.compact())
            slots = [7, 6, 2]
        with torch.no_grad(), torch.autocast(device_type="cuda", dtype=torch.bfloat16):
            a = model.cached_features(nxt, cache.step(slots, 1))
            b = model.cached_features(nxt, cache.step(slots, 1))
        return a, b

    for x, y in zip(run(False), run(True)):
        assert torch.equal(x, y)


def test_policy_gradient_step(model):
    """Log probabilities with a gradient through the model's head: those of the capped
    float32 composition."""
    import torch.nn.functional as F

    from nanochat_amd.ops import token_logprobs
    h = torch.randn(64, 256, device=DEV, generator=torch.Generator(DEV).manual_seed(8))
    y = torch.tensor(_tokens(64, seed=9), device=DEV)
    w = model.lm_head.weight
    lp = token_logprobs(model.raw_logits(h), y, softcap=model.SOFTCAP)
    (got,) = torch.autograd.grad((lp.logprobs - 0.01 * lp.entropy).mean(), [w])
    z = 15 * torch.tanh(F.linear(h, w)[:, :VOCAB] / 15)
    ref = torch.log_softmax(z, -1)
    loss = ref.gather(1, y[:, None])[:, 0] + 0.01 * (ref.exp() * ref).sum(-1)
    (want,) = torch.autograd.grad(loss.mean(), [w])
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max()) + 1e-7


def test_refusals(model):
    from nanochat_amd import engine
    cache = engine.make_cache(model, num_pages=3, max_seqs=2, page_size=16)
    with pytest.raises(RuntimeError, match="missing"):
        engine.prefill(model, cache, 0, _tokens(60))
    assert cache.lens == [0, 0] and int(cache.seq_lens.sum()) == 0
    engine.prefill(model, cache, 0, _tokens(20))
    for call in (lambda: cache.step([2], 1), lambda: cache.step([0, 0], 1),
                 lambda: cache.step([0], 0), lambda: cache.step([0], 600),
                 lambda: cache.fork([0], [0]), lambda: cache.fork([0], [5]),
                 lambda: cache.fork([9], [1]), lambda: cache.fork([0], []),
                 lambda: cache.free([-1]), lambda: engine.score(model, [1]),
                 lambda: engine.prefill(model, cache, 1, []),
                 lambda: engine.generate(model, [1], 0, 5)):
        with pytest.raises(ValueError):
            call()
