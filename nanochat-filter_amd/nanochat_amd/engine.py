"""Generation and scoring with the GPT harness over the paged cache: a prompt in
chunks, several samples from it (``generate``), and the log probabilities of given
texts (``score``).

The reference's ``nanochat/engine.py`` prefills a prompt once and copies the cache to
every sample; here the samples share the prompt's pages, a finished sample's pages are
free for the others, and log probabilities, entropy and alternatives come from one
pass over the logits.
"""

from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional, Sequence

import torch

from nanochat_amd.gpt import GPT
from nanochat_amd.ops.token_logprobs import TokenLogprobs, token_logprobs
from nanochat_amd.paged_kv_cache import PagedKVCache


class Sample(NamedTuple):
    tokens: list      # the continuation, a stop token included
    logprobs: list    # of each of its tokens


def make_cache(model: GPT, num_pages: int, max_seqs: int, page_size: int = 64) -> PagedKVCache:
    c = model.config
    return PagedKVCache(c.n_layer, c.n_head, c.n_kv_head, c.n_embd // c.n_head,
                        num_pages=num_pages, max_seqs=max_seqs, max_len=c.sequence_len,
                        page_size=page_size, device=model.wte.weight.device)


def _autocast():
    return torch.autocast(device_type="cuda", dtype=torch.bfloat16)


def _indices(model: GPT, tokens: Sequence[int], device) -> torch.Tensor:
    """The tokens on the device, where one outside the vocabulary would be a fault."""
    idx = torch.as_tensor(tokens, device="cpu")
    if not 0 <= int(idx.min()) <= int(idx.max()) < model.config.vocab_size:
        raise ValueError(f"tokens are 0 to {model.config.vocab_size - 1}, got {int(idx.min())} "
                         f"to {int(idx.max())}")
    return idx.to(device)


def _empty(cache: PagedKVCache, slots: Sequence[int]) -> None:
    for s in slots:
        if not 0 <= s < len(cache.lens):
            raise ValueError(f"slots are 0 to {len(cache.lens) - 1}, got {s}")
        if cache.lens[s]:
            raise ValueError(f"slot {s} holds {cache.lens[s]} tokens of another sequence")


@contextlib.contextmanager
def _freed_on_error(cache: PagedKVCache, slots: Sequence[int]):
    """Empties the slots, which were empty before, if what is done with them fails."""
    try:
        yield
    except BaseException:
        taken = [s for s in slots if cache.lens[s]]
        if taken:
            cache.free(taken)
        raise


@torch.no_grad()
def prefill(model: GPT, cache: PagedKVCache, slot: int, tokens: Sequence[int],
            chunk: int = 2048) -> torch.Tensor:
    """Feeds the prompt into an empty slot, ``chunk`` tokens at a time; the logits after
    its last token, (1, vocabulary), before the cap.  The slot is empty again if that fails."""
    if not len(tokens):
        raise ValueError("an empty prompt")
    _empty(cache, [slot])
    idx = _indices(model, tokens, cache.page_table.device)[None]
    with _freed_on_error(cache, [slot]), _autocast():
        for x in idx.split(chunk, dim=1):
            hidden = model.cached_features(x, cache.step([slot], x.size(1)))
        return model.raw_logits(hidden[:, -1])


@torch.no_grad()
def generate(model: GPT, prompt: Sequence[int], num_samples: int, max_tokens: int, *,
             top_k: int = 20, temperature: float = 1.0, stop: Optional[int] = None,
             seed: int = 0, cache: Optional[PagedKVCache] = None,
             chunk: int = 2048) -> list[Sample]:
    """``num_samples`` continuations of the prompt, sampled among the ``top_k`` most
    probable tokens (``temperature`` 0: the most probable).  The log probabilities are
    the model's own, of the whole vocabulary.  A given cache's slots 0 to
    ``num_samples`` - 1 are used, which are empty before and after."""
    if num_samples <= 0 or max_tokens <= 0 or temperature < 0:
        raise ValueError("at least one sample of one token, and no negative temperature")
    most = min(64, model.config.vocab_size)
    if not 0 < top_k <= most:
        raise ValueError(f"top_k must be 1 to {most}, got {top_k}")
    longest = len(prompt) + max_tokens - 1  # (the last token is not fed)
    if stop is None and longest > min(model.config.sequence_len, cache.max_len if cache else longest):
        raise ValueError(f"{longest} tokens, more than the model or the cache is made for")
    n = num_samples
    if cache is None:
        page = 64
        shared, own = -(-len(prompt) // page), -(-max_tokens // page) + 1
        cache = make_cache(model, shared + n * own, n, page)
    _empty(cache, range(n))
    with _freed_on_error(cache, range(n)):
        out = _sample(model, prompt, n, max_tokens, top_k, temperature, stop, seed, cache, chunk)
    cache.compact()
    return out


def _sample(model: GPT, prompt: Sequence[int], n: int, max_tokens: int, top_k: int,
            temperature: float, stop: Optional[int], seed: int, cache: PagedKVCache,
            chunk: int) -> list[Sample]:
    device = cache.page_table.device
    g = torch.Generator(device=device).manual_seed(seed)
    logits = prefill(model, cache, 0, prompt, chunk).expand(n, -1)
    if n > 1:
        cache.fork([0] * (n - 1), list(range(1, n)))
    out = [Sample([], []) for _ in range(n)]
    live = list(range(n))
    none = torch.full((n,), -1, device=device)
    for _ in range(max_tokens):
        lp = token_logprobs(logits, none[:len(live)], top_k=top_k, softcap=GPT.SOFTCAP)
        if temperature > 0:
            p = torch.softmax(lp.top_logprobs / temperature, dim=-1)
            pick = torch.multinomial(p, 1, generator=g)
        else:
            pick = torch.zeros(len(live), 1, dtype=torch.int64, device=device)
        tokens = lp.top_ids.gather(1, pick)
        probs = lp.top_logprobs.gather(1, pick)
        going = []
        for i, (s, t, p) in enumerate(zip(live, tokens[:, 0].tolist(), probs[:, 0].tolist())):
            out[s].tokens.append(t)
            out[s].logprobs.append(p)
            if t != stop and len(out[s].tokens) < max_tokens:
                going.append(i)
        ended = [s for i, s in enumerate(live) if i not in set(going)]
        if ended:
            cache.free(ended)
        live = [live[i] for i in going]
        if not live:
            break
        with _autocast():
            hidden = model.cached_features(tokens[torch.tensor(going, device=device)],
                                           cache.step(live, 1))
            logits = model.raw_logits(hidden[:, -1])
    return out


@torch.no_grad()
def score(model: GPT, tokens: Sequence[int], *, top_k: int = 0,
          cache: Optional[PagedKVCache] = None, slot: int = 0,
          chunk: int = 2048) -> TokenLogprobs:
    """Log probability, entropy and alternatives at each of ``tokens[1:]`` given what is
    before it, fed through an empty slot of the cache ``chunk`` tokens at a time."""
    if len(tokens) < 2:
        raise ValueError("at least two tokens")
    if cache is None:
        cache = make_cache(model, -(-len(tokens) // 64), slot + 1)
    _empty(cache, [slot])
    idx = _indices(model, tokens, cache.page_table.device)
    parts = []
    with _freed_on_error(cache, [slot]), _autocast():
        for x, y in zip(idx[:-1].split(chunk), idx[1:].split(chunk)):
            hidden = model.cached_features(x[None], cache.step([slot], len(x)))
            parts.append(token_logprobs(model.raw_logits(hidden[0]), y, top_k=top_k,
                                        softcap=GPT.SOFTCAP))
    cache.free([slot])
    return TokenLogprobs(*(None if p[0] is None else torch.cat(p) for p in zip(*parts)))
