"""A search over a cache in 4 bits with rotation on the way: the operators together, as the
engine runs them."""

from __future__ import annotations

import math

import pytest
import torch

from fp4_test_utils import held4, rotated64, values4

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 300


@pytest.fixture(scope="module")
def model():
    from nanochat_amd.gpt import GPT, GPTConfig
    torch.manual_seed(0)
    m = GPT(GPTConfig(sequence_len=500, vocab_size=VOCAB, n_layer=3, n_head=4, n_kv_head=2,
                      n_embd=256, ltv_r=64)).to(DEV)
    m.init_weights(randomise_output_projections=True)
    m.lm_head.weight.data.normal_(0.0, 0.05, generator=torch.Generator(DEV).manual_seed(1))
    m.wte.to(dtype=torch.bfloat16)
    return m


def _tokens(n, seed=0):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("chunk", [1000, 7])
def test_rotation_on_the_way_scores_as_before(model, chunk):
    """The same log probabilities but for the roundings of the model's own rotation and norm."""
    from nanochat_amd import engine
    tokens = _tokens(90)
    want = engine.score(model, tokens, chunk=chunk)
    cache = engine.make_cache(model, 8, 1, 16, rotate=True)
    got = engine.score(model, tokens, chunk=chunk, cache=cache)
    assert cache.k_pages.dtype == torch.bfloat16
    assert float((got.logprobs - want.logprobs).abs().max()) <= 0.1
    assert float((got.logprobs - want.logprobs).abs().mean()) <= 0.02


def test_pages_hold_rotated_keys(model):
    """After a prompt in chunks the first layer's pages hold, in 4 bits, what the filter gave."""
    from nanochat_amd import engine
    tokens = _tokens(70, seed=1)
    cache = engine.make_cache(model, 8, 2, 16, bits=4)
    seen = []
    attn = model.h[0].attn
    step_attend = type(cache.step([1], 1)).attend
    cache.free([1])

    def attend(self, layer, q, k, v, scale=None):
        if layer == 0:
            seen.append((k.clone(), v.clone()))
        return step_attend(self, layer, q, k, v, scale)

    cls = type(cache.step([1], 1))
    cache.free([1])
    cls.attend = attend
    try:
        engine.prefill(model, cache, 0, tokens, chunk=30)
    finally:
        cls.attend = step_attend
    k, v = (torch.cat(x, 1)[0].bfloat16() for x in zip(*seen))
    assert k.shape[0] == 70 and attn.head_dim == 64
    pos = torch.arange(70, device=DEV)
    want = held4(rotated64(k, model.cos[0, :, 0], model.sin[0, :, 0], pos, 2.0 ** -23))[0]
    pages = cache.page_table[0, (pos // 16).long()].long()
    assert torch.equal(values4(cache.k_pages[0])[pages, :, pos % 16], want)
    assert torch.equal(values4(cache.v_pages[0])[pages, :, pos % 16], held4(v)[0])


def test_four_bits_score_alike_in_any_chunks(model):
    """Every key and value goes through the pages, so that the log probabilities do not depend on
    the chunks but for the filter's and the products' roundings."""
    from nanochat_amd import engine
    tokens = _tokens(120, seed=2)
    a, b = (engine.score(model, tokens, chunk=c, cache=engine.make_cache(model, 8, 1, 16, bits=4))
            for c in (1000, 11))
    assert float((a.logprobs - b.logprobs).abs().mean()) <= 0.05
    whole = engine.score(model, tokens)
    # (4 bits move them, though not far: the logits are about 1)
    assert float((a.logprobs - whole.logprobs).abs().mean()) <= 0.3


def test_sampling_from_four_bits(model):
    """Samples share a prompt's pages and part ways in them."""
    from nanochat_amd import engine
    prompt = _tokens(70, seed=9)
    cache = engine.make_cache(model, num_pages=40, max_seqs=4, page_size=16, bits=4)
    samples = engine.generate(model, prompt, 4, 20, top_k=20, seed=4, cache=cache, chunk=50)
    assert len({tuple(s.tokens) for s in samples}) > 1
    assert int(cache.ref_counts.sum()) == 0 and cache.lens == [0] * 4
    for s in samples[:2]:
        got = engine.score(model, prompt + s.tokens, cache=cache, slot=3)
        lp = got.logprobs[len(prompt) - 1:].tolist()
        # (the chunks differ, and with them the keys' roundings to 4 bits here and there)
        assert sum(abs(a - b) for a, b in zip(lp, s.logprobs)) <= 0.1 * len(lp)


def _search64(model, prompt, n, steps, stop, make):
    """The same search with whole scorings: each continuation's log probabilities from a
    prefill of prompt and tokens; the widest difference between kept and dropped."""
    from nanochat_amd import engine
    beams = [([], 0.0)]
    gap = math.inf
    for _ in range(steps):
        cand = []
        for toks, s in beams:
            if toks and toks[-1] == stop:
                cand.append((s, toks))
                continue
            cache = make()
            logits = engine.prefill(model, cache, 0, prompt + toks, chunk=len(prompt))
            z = 15 * torch.tanh(logits[0].double() / 15)
            lp = torch.log_softmax(z, 0)
            top = lp.topk(n)
            cand += [(s + float(p), toks + [int(t)]) for p, t in zip(top.values, top.indices)]
        cand.sort(key=lambda c: -c[0])
        if len(cand) > n:
            gap = min(gap, cand[n - 1][0] - cand[n][0])
        beams = [(t, s) for s, t in cand[:n]]
        if all(t and t[-1] == stop for t, _ in beams):
            break
    return beams, gap


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("n", [1, 3, 8])
def test_beam_search(model, n, bits):
    """The search's beams have the log probabilities that scoring them gives, and are at least as
    good as those of a search that scores every candidate by itself, up to the roundings of the
    dataflows (0.1 for each token, as in the tests of scoring)."""
    from nanochat_amd import engine
    prompt, steps = _tokens(37, seed=3), 6
    cache = engine.make_cache(model, 60, n, 16, bits=bits)
    got = engine.beam_search(model, prompt, n, steps, cache=cache, length_penalty=0.0)
    assert cache.lens == [0] * n and int(cache.ref_counts.sum()) == 0
    assert len(got) == n and len({tuple(b.tokens) for b in got}) == n
    assert all(len(b.tokens) == steps for b in got)
    assert [b.score for b in got] == sorted((b.score for b in got), reverse=True)
    for b in got:
        assert b.score == b.logprob
        lp = engine.score(model, prompt + b.tokens, cache=engine.make_cache(model, 8, 1, 16, bits=bits))
        own = float(lp.logprobs[len(prompt) - 1:].sum())
        assert abs(own - b.logprob) <= 0.1 * steps
    want, _ = _search64(model, prompt, n, steps, None,
                        lambda: engine.make_cache(model, 8, 1, 16, bits=bits))
    assert abs(got[0].logprob - want[0][1]) <= 0.2 * steps


def test_beam_search_of_one_is_greedy(model):
    from nanochat_amd import engine
    prompt = _tokens(50, seed=4)
    greedy = engine.generate(model, prompt, 1, 20, temperature=0.0)[0]
    got = engine.beam_search(model, prompt, 1, 20, length_penalty=1.0)[0]
    assert got.tokens == greedy.tokens
    assert abs(got.logprob - sum(greedy.logprobs)) <= 1e-3
    assert got.score == got.logprob / 20


def test_stopped_beams_stay(model):
    """A beam that has ended keeps its tokens and its log probability."""
    from nanochat_amd import engine
    prompt = _tokens(30, seed=5)
    free = engine.beam_search(model, prompt, 4, 12, length_penalty=0.0)
    stop = free[0].tokens[2]
    got = engine.beam_search(model, prompt, 4, 12, stop=stop, length_penalty=0.0)
    assert any(b.tokens[-1] == stop and len(b.tokens) < 12 for b in got)
    for b in got:
        assert stop not in b.tokens[:-1]
        assert len(b.tokens) == 12 or b.tokens[-1] == stop
        lp = engine.score(model, prompt + b.tokens)
        own = float(lp.logprobs[len(prompt) - 1:].sum())
        assert abs(own - b.logprob) <= 0.1 * len(b.tokens)


def test_smallest_searches(model):
    """One token; one that ends it; a prompt of one; more beams than differ at first."""
    from nanochat_amd import engine
    one = engine.beam_search(model, _tokens(5), 4, 1)
    lp = engine.score(model, _tokens(5) + one[0].tokens, top_k=4)
    assert [b.tokens for b in one] == [[t] for t in lp.top_ids[-1].tolist()]
    for b in engine.beam_search(model, _tokens(5), 1, 6, stop=one[0].tokens[0]):
        assert b.tokens == one[0].tokens
    out = engine.beam_search(model, [7], 32, 3)
    assert len({tuple(b.tokens) for b in out}) == 32 and all(len(b.tokens) == 3 for b in out)
    assert [b.score for b in out] == sorted((b.score for b in out), reverse=True)


def test_reorder_of_nothing(model):
    from nanochat_amd import engine
    cache = engine.make_cache(model, num_pages=8, max_seqs=2, page_size=16, bits=4)
    engine.prefill(model, cache, 0, _tokens(20))
    was = [t.clone() for t in (cache.page_table, cache.seq_lens, cache.ref_counts)]
    cache.reorder([], [])
    cache.reorder([0], [0])
    assert all(torch.equal(a, b) for a, b in
               zip(was, (cache.page_table, cache.seq_lens, cache.ref_counts)))
    assert cache.lens == [20, 0]
    cache.reorder([0], [1])  # (an empty slot: the other is let go)
    assert cache.lens == [0, 0] and not cache.ref_counts.any() and not cache.seq_lens.any()


def test_failure_leaves_the_slots_empty(model):
    from nanochat_amd import engine
    cache = engine.make_cache(model, 4, 3, 16, bits=4)
    with pytest.raises(RuntimeError, match="missing"):
        engine.beam_search(model, _tokens(33, seed=6), 3, 40, cache=cache)
    assert cache.lens == [0] * 3 and int(cache.ref_counts.sum()) == 0
    assert len(engine.beam_search(model, _tokens(17, seed=6), 2, 3, cache=cache)) == 2


@pytest.mark.parametrize("bits", [None, 4])
def test_unchecked_step_without_room(model, bits):
    """It changes nothing, with rotation on the way too, and its attention is 0."""
    from nanochat_amd import engine
    cache = engine.make_cache(model, 2, 2, 16, bits=bits, rotate=True)
    engine.prefill(model, cache, 0, _tokens(30, seed=7))
    # (bytes: what was never written may be NaN)
    held = lambda: [p.view(torch.uint8).clone() for p in (cache.k_pages, cache.v_pages)]  # noqa: E731
    pages = held()
    q = torch.randn(1, 5, 4, 64, device=DEV)
    k = torch.randn(1, 5, 2, 64, device=DEV)
    step = cache.step([0], 5, check=False)
    y = step.attend(0, q, k, k)
    assert not y.any()
    assert all(torch.equal(a, b) for a, b in zip(held(), pages))
    with pytest.raises(RuntimeError, match="missing"):
        cache.check_steps()


def test_reorder_takes_the_filter_along(model):
    """Slots that exchange places continue as they would have, bit for bit."""
    from nanochat_amd import engine
    prompts = [_tokens(n, seed=8 + n) for n in (50, 33, 80)]
    nxt = torch.tensor([[5], [6], [7]], device=DEV)

    def run(order):
        cache = engine.make_cache(model, num_pages=60, max_seqs=4, page_size=16, bits=4)
        for s, p in enumerate(prompts):
            engine.prefill(model, cache, s, p, chunk=40)
        cache.reorder([0, 1, 2, 3], [*order, order[0]])
        assert cache.lens == cache.seq_lens.tolist()
        with torch.no_grad(), torch.autocast(device_type="cuda", dtype=torch.bfloat16):
            back = [order.index(i) for i in range(3)]
            a = model.cached_features(nxt, cache.step(back, 1))
            return a, model.cached_features(nxt, cache.step(back, 1))

    for x, y in zip(run([0, 1, 2]), run([2, 0, 1])):
        assert torch.equal(x, y)


def test_refusals(model):
    from nanochat_amd import engine
    from nanochat_amd.paged_kv_cache import PagedKVCache
    cache = engine.make_cache(model, num_pages=8, max_seqs=2, page_size=16, bits=4)
    engine.prefill(model, cache, 0, _tokens(20))
    for call in (lambda: cache.reorder([0], [2]), lambda: cache.reorder([0, 0], [1, 1]),
                 lambda: cache.reorder([0], [0, 1]), lambda: cache.reorder([-1], [0]),
                 lambda: engine.make_cache(model, 8, 2, 8, bits=4),
                 lambda: engine.make_cache(model, 8, 2, 16, bits=3),
                 lambda: engine.beam_search(model, [1], 0, 5),
                 lambda: engine.beam_search(model, [1], 33, 5),
                 lambda: engine.beam_search(model, [1], 2, 0),
                 lambda: engine.beam_search(model, [1], 2, 600),
                 lambda: engine.beam_search(model, [1], 2, 5, length_penalty=math.inf),
                 lambda: engine.beam_search(model, [1], 2, 5, length_penalty=math.nan),
                 lambda: engine.beam_search(model, [1], 2, 5, length_penalty=-1e6),
                 lambda: engine.beam_search(model, [1], 3, 5, cache=cache),
                 lambda: engine.beam_search(model, [1], 2, 5, cache=cache),  # slot 0 is in use
                 lambda: PagedKVCache(1, 2, 2, 40, num_pages=2, max_seqs=1, max_len=32, bits=4),
                 lambda: PagedKVCache(1, 2, 2, 64, num_pages=2, max_seqs=1, max_len=32, norm_eps=0.1),
                 lambda: PagedKVCache(1, 2, 2, 64, num_pages=2, max_seqs=1, max_len=32,
                                      rotary=(torch.zeros(31, 32), torch.zeros(31, 32)))):
        with pytest.raises(ValueError):
            call()
    assert cache.lens == [20, 0]


def test_cache_that_does_not_normalise(model):
    """A cache that rotates and leaves the norm out, which this model has: refused, and the slot is as it
    was."""
    from nanochat_amd import engine
    from nanochat_amd.paged_kv_cache import PagedKVCache
    tables = model.cos[0, :, 0], model.sin[0, :, 0]
    make = lambda **kw: PagedKVCache(3, 4, 2, 64, num_pages=8, max_seqs=1, max_len=128, page_size=16,  # noqa: E731
                                     rotary=tables, **kw)
    cache = make()
    assert cache.step([0], 1).rotates
    cache.free([0])
    with pytest.raises(ValueError, match="norm"):
        engine.prefill(model, cache, 0, _tokens(20))
    assert cache.lens == [0] and not cache.seq_lens.any() and not cache.ref_counts.any()
    want = engine.prefill(model, engine.make_cache(model, 8, 1, 16, rotate=True), 0, _tokens(20))
    assert torch.equal(engine.prefill(model, make(norm_eps=2.0 ** -23), 0, _tokens(20)), want)


@pytest.mark.parametrize("n", [2, 4])
def test_beam_search_keeps_the_best(n, monkeypatch):
    """In float32, where the dataflows differ by little: whenever the candidates that an independent
    search keeps and drops are further apart than that, the beams are the same, all of them.

    A log probability may be off by 2^-24 for each of 256 products' additions, some 20 such sums deep,
    of logits up to 15: 0.005 a token."""
    import contextlib

    from nanochat_amd import engine
    from nanochat_amd.gpt import GPT, GPTConfig
    from nanochat_amd.paged_kv_cache import PagedKVCache
    torch.manual_seed(2)
    model = GPT(GPTConfig(sequence_len=200, vocab_size=VOCAB, n_layer=2, n_head=4, n_kv_head=2,
                          n_embd=256, ltv_r=64)).to(DEV)
    model.init_weights(randomise_output_projections=True)
    model.lm_head.weight.data.normal_(0.0, 0.3, generator=torch.Generator(DEV).manual_seed(3))
    monkeypatch.setattr(engine, "_autocast", contextlib.nullcontext)
    make = lambda: PagedKVCache(2, 4, 2, 64, num_pages=8 * n, max_seqs=n, max_len=200, page_size=16,  # noqa: E731
                                dtype=torch.float32)
    steps, off, decided = 5, 0.005 * 5, 0
    for seed in range(8):
        prompt = _tokens(20 + seed, seed=40 + seed)
        want, gap = _search64(model, prompt, n, steps, None, make)
        got = engine.beam_search(model, prompt, n, steps, cache=make(), length_penalty=0.0)
        if gap <= 2 * off:
            continue
        decided += 1
        lp = {tuple(t): p for t, p in want}
        assert {tuple(b.tokens) for b in got} == set(lp), (seed, gap)
        for b in got:
            assert abs(b.logprob - lp[tuple(b.tokens)]) <= off, seed
    assert decided >= 2
