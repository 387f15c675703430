"""The operators that serving and scoring with a paged cache are made of, as
workloads: what their speed is judged by.

Three sets of calls, each as a program makes them:

* attention of new tokens over a paged cache: the new keys and values are
  written into the cache's pages, then every new token attends to the cached
  tokens and the new ones up to itself.  A decode step has one token per
  sequence, a prompt's chunk many, a mixed batch some of each;
* the pages themselves: sequences that share a prompt's pages and part ways
  (free, fork, reserve with a copy of the pages they would write into), and
  sequences that move (reserve, copy, free, compact);
* log probabilities of given tokens with the entropy and the top alternatives
  of each row of soft-capped logits, and their gradient.

``listed`` gives the fixed cases, ``draw`` another one of the same ranges,
``prepare`` the tensors that exist before the call, ``run`` one call, ``work``
the bytes and operations it cannot do without and ``exact`` its results in
float64.  With ``own`` false ``run`` computes the plain form in elementary torch
operations in float32, with ``own`` true it calls the framework.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"


def _framework():
    """The framework's operators, found beside this folder."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "nanochat-filter_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nanochat_amd.ops as ops

    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# the d12 model's attention heads
_D12 = {"n_head": 6, "n_kv_head": 6, "head_dim": 128}


def _attn(name, seqs, ones, new, cached, lengths, dtype="bf16", heads=None, page=64, packed=True):
    """``seqs`` sequences, the last ``ones`` of them with one new token, the others
    with new[0] .. new[1]; cached[0] .. cached[1] tokens in the cache before.  The
    first has the most of both, the others spread over the logarithm (``lengths``
    seeds them).  packed: the new tokens in one row after the other, else (B, T)."""
    c = {"name": name, "kind": "attn", "seqs": seqs, "ones": ones, "new_lo": new[0],
         "new_hi": new[1], "cached_lo": cached[0], "cached_hi": cached[1], "lengths": lengths,
         "dtype": dtype, "page": page, "packed": packed}
    c.update(heads or _D12)
    return c


def _pages(name, kind, layers, parents, children, lens, lengths, dtype="bf16", heads=None,
           page=64):
    c = {"name": name, "kind": kind, "layers": layers, "parents": parents, "children": children,
         "len_lo": lens[0], "len_hi": lens[1], "lengths": lengths, "dtype": dtype, "page": page}
    c.update(heads or _D12)
    return c


def _logp(name, rows, vocab, dtype, top_k, softcap, grad, padded=0):
    return {"name": name, "kind": "logp", "rows": rows, "vocab": vocab,
            "padded": max(padded, vocab), "dtype": dtype, "top_k": top_k, "softcap": softcap,
            "grad": grad}


def listed():
    return [
        # one token of each of four chats: launches and latency
        _attn("decode_small", 4, 4, (1, 1), (200, 600), 1, packed=False),
        # a serving step of a batch with one very long context among ordinary ones
        _attn("decode_ragged", 16, 16, (1, 1), (300, 131071), 2, packed=False),
        # a step that decodes some sequences while the prompts of others come in chunks
        _attn("chunk_mixed", 16, 8, (37, 1024), (1, 8000), 3, page=16,
              heads={"n_head": 8, "n_kv_head": 4, "head_dim": 128}),
        # the last chunk of a long prompt
        _attn("prefill_long", 1, 0, (12289, 12289), (20000, 20000), 4, packed=False),
        # a float32 program, 64-channel heads in groups, pages that are no power of two
        _attn("chunk_fp32", 5, 2, (65, 129), (100, 1500), 5, dtype="fp32", page=48,
              heads={"n_head": 10, "n_kv_head": 5, "head_dim": 64}),
        # eight continuations of one prompt, drawn anew
        _pages("fork_small", "fork", 12, 1, 8, (500, 500), 6),
        # a sampling round: 24 prompts, eight continuations each
        _pages("fork_round", "fork", 12, 24, 8, (300, 2500), 7),
        # two short sequences move to other slots and the cache is closed up
        _pages("compact_small", "compact", 12, 2, 2, (100, 200), 8, page=16),
        # half of a cache moves and the cache is closed up
        _pages("compact_half", "compact", 12, 16, 16, (200, 1500), 9),
        # the alternatives shown beside a decode step's tokens
        _logp("logp_decode", 16, 65536, "fp32", 20, 15.0, False),
        # scoring documents
        _logp("logp_score", 4096, 65536, "bf16", 5, 15.0, False),
        # a policy gradient step with an entropy term; the vocabulary's padding is cut off
        _logp("logp_train", 4096, 50257, "bf16", 0, 15.0, True, padded=50304),
    ]


def _log_int(rng, lo, hi):
    if hi <= lo:
        return lo
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_heads(rng):
    nkv = rng.randint(1, 8)
    return {"n_head": nkv * rng.choice([1, 1, 1, 2, 3, 4, 8]), "n_kv_head": nkv,
            "head_dim": rng.choice([64, 96, 128, 128])}


def draw(rng):
    kind = rng.choice(["decode"] * 3 + ["chunk"] * 3 + ["prefill"] * 2 + ["fork"] * 2
                      + ["compact"] * 2 + ["logp"] * 3 + ["train"] * 3)
    lengths = rng.randrange(1 << 20)
    if kind in ("decode", "chunk", "prefill"):
        heads = _draw_heads(rng)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        page = rng.choice([16, 32, 48, 64, 128])
        if kind == "decode":
            seqs = _log_int(rng, 1, 128)
            hi = max(16, min(131071, 2_000_000 // seqs * 6 // max(6, heads["n_kv_head"])))
            cached = _log_int(rng, 16, hi)
            c = _attn("", seqs, seqs, (1, 1), (max(1, cached // 20), cached), lengths, dtype,
                      heads, page, packed=rng.random() < 0.5)
        else:
            seqs = _log_int(rng, 2, 32) if kind == "chunk" else 1
            most = (200_000_000 if dtype == "fp32" else 2_000_000_000) // heads["n_head"]
            new = _log_int(rng, 2, max(2, min(1500 if kind == "chunk" else 12289,
                                              math.isqrt(most // seqs))))
            cached = _log_int(rng, 1, max(1, min(32000, most // seqs // new - new)))
            ones = rng.randint(0, seqs - 1) if kind == "chunk" else 0
            c = _attn("", seqs, ones, (max(1, new // 20), new), (max(1, cached // 20), cached),
                      lengths, dtype, heads, page, packed=kind == "chunk")
    elif kind in ("fork", "compact"):
        heads = _draw_heads(rng)
        page = rng.choice([16, 32, 64])
        layers = rng.randint(1, 12)
        one = page * 2 * heads["n_kv_head"] * heads["head_dim"] * 2 * layers
        most = 2_200_000_000 // one  # pages of the cache
        parents = _log_int(rng, 1, 24)
        children = _log_int(rng, 1, max(1, min(8, most // parents // 4)))
        hi = max(2, min(2500, (most // parents // 3 - children) * page))
        length = _log_int(rng, 2, hi)
        c = _pages("", kind, layers, parents, parents if kind == "compact" else children,
                   (max(1, length // 5), length), lengths, "bf16", heads, page)
    else:
        dtype = rng.choice(["bf16", "fp32"])
        vocab = _log_int(rng, 1000, 131072)
        rows = _log_int(rng, 1, (100_000_000 if kind == "train" else 200_000_000) // vocab)
        pad = rng.choice([0, (vocab + 63) // 64 * 64])
        c = _logp("", rows, vocab, dtype, rng.choice([0, 1, 5, 20, 32]),
                  rng.choice([15.0, 15.0, 0.0]), kind == "train", pad)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# lengths and inputs
# ---------------------------------------------------------------------------
def _dtype(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _attn_lengths(case):
    """New and cached tokens of each sequence."""
    rng = random.Random(case["lengths"])
    n, new, cached = case["seqs"], [], []
    for i in range(n):
        if i >= n - case["ones"]:
            new.append(1)
        else:
            new.append(case["new_hi"] if i == 0 else _log_int(rng, case["new_lo"], case["new_hi"]))
        cached.append(case["cached_hi"] if i == 0 else
                      _log_int(rng, case["cached_lo"], case["cached_hi"]))
    return new, cached


def _page_lengths(case):
    """Lengths of the parents (or moving sequences) and of those that stay."""
    rng = random.Random(case["lengths"])
    lens = [case["len_hi"] if i == 0 else _log_int(rng, case["len_lo"], case["len_hi"])
            for i in range(case["parents"])]
    return lens, lens[::-1]


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _prepare_attn(case, seed):
    g, dt = _generator(seed), _dtype(case)
    new, cached = _attn_lengths(case)
    NH, NKVH, D, ps = case["n_head"], case["n_kv_head"], case["head_dim"], case["page"]
    lens = [a + b for a, b in zip(new, cached)]
    held = [-(-n // ps) for n in lens]
    P, W = sum(held) + 3, max(held) + 1
    order = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(new), W), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dt)

    s = {"kind": "attn", "k_pages": randn(P, NKVH, ps, D), "v_pages": randn(P, NKVH, ps, D),
         "page_table": table, "seq_lens": _ints(lens), "max_new": max(new), "max_len": max(lens),
         "starts": None}
    if case["packed"]:
        N = sum(new)
        s["q"], s["k"], s["v"] = randn(N, NH, D), randn(N, NKVH, D), randn(N, NKVH, D)
        s["starts"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
    else:
        # the filter's head-major outputs
        B, T = len(new), max(new)
        s["q"], s["k"], s["v"] = (randn(B, n, T, D).transpose(1, 2) for n in (NH, NKVH, NKVH))
    # trained attention has some keys far above the others
    s["q"].mul_(2.0)
    return s


def _prepare_pages(case, seed):
    """fork: slots [0, n) hold the parents, slots n + i * children + j child j of
    parent i, forked and grown by one token (the round before).  compact: slots
    [0, n) hold the sequences that move, [n, 2 n) those that stay, [2 n, 3 n) are
    empty; the movers' pages lie between the others'."""
    g, dt = _generator(seed), _dtype(case)
    NKVH, D, ps, L = case["n_kv_head"], case["head_dim"], case["page"], case["layers"]
    n, ch, fork = case["parents"], case["children"], case["kind"] == "fork"
    lens, stay = _page_lengths(case)
    held = [-(-m // ps) for m in lens]
    slots = n + n * ch if fork else 3 * n
    W = -(-(max(lens) + 1) // ps) + 1
    table, refs, seq_lens = [[-1] * W for _ in range(slots)], [], [0] * slots

    def take():
        refs.append(1)
        return len(refs) - 1

    if fork:
        for i in range(n):
            seq_lens[i] = lens[i]
            table[i][:held[i]] = [take() for _ in range(held[i])]
        for i in range(n):
            for j in range(ch):
                c = n + i * ch + j
                seq_lens[c] = lens[i] + 1
                full = lens[i] // ps
                table[c][:full + 1] = table[i][:full] + [take()]
                for p in table[i][:full]:
                    refs[p] += 1
        spare = 5
    else:
        for i in range(n):
            seq_lens[i], seq_lens[n + i] = lens[i], stay[i]
            theirs = -(-stay[i] // ps)
            for j in range(max(held[i], theirs)):
                if j < held[i]:
                    table[i][j] = take()
                if j < theirs:
                    table[n + i][j] = take()
        spare = sum(held) + 5
    refs += [0] * spare
    P = len(refs)
    s = {"kind": case["kind"], "page_table": _ints(table), "seq_lens": _ints(seq_lens),
         "ref_counts": _ints(refs),
         "k_pages": torch.randn(L, P, NKVH, ps, D, generator=g, device=DEV, dtype=dt),
         "v_pages": torch.randn(L, P, NKVH, ps, D, generator=g, device=DEV, dtype=dt)}
    if fork:
        s["src"] = _ints([i for i in range(n) for _ in range(ch)])
        s["dst"] = _ints(list(range(n, n + n * ch)))
        s["one"] = _ints([1] * (n * ch))
    else:
        s["here"], s["there"] = _ints(list(range(n))), _ints(list(range(2 * n, 3 * n)))
        s["counts"] = _ints(lens)
    return s


def _prepare_logp(case, seed):
    g, dt = _generator(seed), _dtype(case)
    N, V = case["rows"], case["vocab"]
    # a trained head's logits before the cap: most are low, some stand out
    logits = (torch.randn(N, case["padded"], generator=g, device=DEV) * 2.5 - 2.0).to(dt)[:, :V]
    targets = torch.randint(0, V, (N,), generator=g, device=DEV)
    logits.scatter_(1, targets[:, None],
                    (torch.randn(N, 1, generator=g, device=DEV) * 4 + 6).to(dt))
    s = {"kind": "logp", "logits": logits, "targets": targets, "top_k": case["top_k"],
         "softcap": case["softcap"] or None, "grad": case["grad"]}
    if case["grad"]:
        s["g_logp"] = torch.randn(N, generator=g, device=DEV) / N
        s["g_entropy"] = torch.full((N,), -0.01 / N, device=DEV)
        s["g_top"] = (torch.randn(N, case["top_k"], generator=g, device=DEV) / N
                      if case["top_k"] else None)
        s["logits"] = logits.detach().requires_grad_(True)
    return s


def prepare(case, seed):
    if case["kind"] == "attn":
        return _prepare_attn(case, seed)
    if case["kind"] == "logp":
        return _prepare_logp(case, seed)
    return _prepare_pages(case, seed)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_attn(s):
    kp, vp, table, lens, q = s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], s["q"]
    P, NKVH, ps, D = kp.shape
    B, W, T = table.shape[0], table.shape[1], s["max_new"]
    NH = q.shape[-2]
    step = torch.arange(T, device=DEV)
    if s["starts"] is None:
        n = torch.full((B,), T, device=DEV)
        rows = None
        qb, kb, vb = q, s["k"], s["v"]
    else:
        first, n = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
        rows = (first[:, None] + step).clamp(max=q.shape[0] - 1)
        qb, kb, vb = q[rows], s["k"][rows], s["v"][rows]
    at = (lens - n)[:, None] + step  # position of each new token
    real = step < n[:, None]
    page = table.gather(1, (at // ps).clamp(0, W - 1)).long()
    b, t = (real & (page >= 0)).nonzero(as_tuple=True)
    kp.transpose(1, 2)[page[b, t], at[b, t] % ps] = kb[b, t]
    vp.transpose(1, 2)[page[b, t], at[b, t] % ps] = vb[b, t]
    # the cache as (B, NKVH, L, D)
    pages = -(-s["max_len"] // ps)
    ids = table[:, :pages].clamp(min=0).long()
    L = pages * ps
    held = (torch.arange(L, device=DEV) < lens[:, None]) & (table[:, :pages] >= 0
                                                             ).repeat_interleave(ps, 1)

    def gathered(x):
        x = x[ids].transpose(1, 2).reshape(B, NKVH, L, D).float()
        return x.masked_fill_(~held[:, None, :, None], 0.0)

    scores = torch.matmul(
        qb.float().view(B, T, NKVH, NH // NKVH, D).permute(0, 2, 3, 1, 4).reshape(
            B, NKVH, NH // NKVH * T, D) * D ** -0.5, gathered(kp).transpose(2, 3).contiguous())
    seen = held[:, None, :] & (torch.arange(L, device=DEV) <= at[:, :, None])
    scores = scores.view(B, NKVH, NH // NKVH, T, L)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(B, NKVH, -1, L), gathered(vp)).view(
        B, NKVH, NH // NKVH, T, D) / total.clamp_(min=1e-38)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, T, NH, D).to(q.dtype)
    if rows is not None:
        b, t = real.nonzero(as_tuple=True)
        out = out[b, t]
    return [out, kp, vp]


def _plain_free(table, lens, refs, slots):
    slots = slots.long()
    rows = table[slots]
    refs.index_add_(0, rows[rows >= 0], refs.new_full((1,), -1).expand(int((rows >= 0).sum())))
    table[slots] = -1
    lens[slots] = 0


def _plain_fork(table, lens, refs, src, dst):
    rows = table[src.long()]
    refs.index_add_(0, rows[rows >= 0], refs.new_ones(1).expand(int((rows >= 0).sum())))
    table[dst.long()] = rows
    lens[dst.long()] = lens[src.long()]


def _plain_reserve(table, lens, refs, slots, counts, k_pages, v_pages):
    """The lowest free pages, slot after slot: one in the place of a shared last page
    that new tokens would be written into, then one for each page more."""
    ps, slots = k_pages.shape[3], slots.long()
    n, W = slots.shape[0], table.shape[1]
    old, new = lens[slots], lens[slots] + counts
    held, needed = (old + ps - 1) // ps, (new + ps - 1) // ps
    last = table[slots, ((old - 1) // ps).clamp(min=0).long()].long()
    writes = (old % ps != 0) & (counts > 0)
    same = (last[:, None] == last) & writes[:, None] & writes
    earlier = torch.tril(same, diagonal=-1).sum(1)
    part = writes & (refs[last.clamp(min=0)] - earlier > 1)
    wanted = part + (needed - held)
    first = wanted.cumsum(0) - wanted
    free = (refs == 0).nonzero()[:, 0].to(torch.int32)
    (who,) = part.nonzero(as_tuple=True)
    from_, to = last[who], free[first[who]].long()
    k_pages[:, to], v_pages[:, to] = k_pages[:, from_], v_pages[:, from_]
    refs.index_add_(0, from_, refs.new_full((1,), -1).expand(who.shape[0]))
    refs[to] = 1
    table[slots[who], ((old[who] - 1) // ps).long()] = to.int()
    col = torch.arange(W, device=DEV)
    i, c = ((col >= held[:, None]) & (col < needed[:, None])).nonzero(as_tuple=True)
    ids = free[first[i] + part[i] + c - held[i]]
    table[slots[i], c] = ids
    refs[ids.long()] = 1
    lens[slots] = new


def _plain_copy(k_pages, v_pages, src, dst):
    ok = (src >= 0) & (dst >= 0)
    src, dst = src[ok].long(), dst[ok].long()
    k_pages[:, dst], v_pages[:, dst] = k_pages[:, src], v_pages[:, src]


def _plain_compact(table, refs, k_pages, v_pages):
    """Live pages past the count of live ones move, in order, into the holes before."""
    live = refs > 0
    ids = torch.arange(refs.shape[0], device=DEV)
    n = live.sum()
    (movers,), (holes,) = (live & (ids >= n)).nonzero(as_tuple=True), (
        ~live & (ids < n)).nonzero(as_tuple=True)
    _plain_copy(k_pages, v_pages, movers, holes)
    refs[holes] = refs[movers]
    refs[movers] = 0
    place = ids.to(torch.int32)
    place[movers] = holes.int()
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], table))


def _plain_pages(s):
    t, n, r, k, v = (s[x] for x in ("page_table", "seq_lens", "ref_counts", "k_pages", "v_pages"))
    if s["kind"] == "fork":
        _plain_free(t, n, r, s["dst"])
        _plain_fork(t, n, r, s["src"], s["dst"])
        _plain_reserve(t, n, r, s["dst"], s["one"], k, v)
    else:
        _plain_move(t, n, r, k, v, s["here"], s["there"], s["counts"])
        _plain_move(t, n, r, k, v, s["there"], s["here"], s["counts"])
    return [t, n, r, k, v]


def _plain_move(t, n, r, k, v, here, there, counts):
    _plain_reserve(t, n, r, there, counts, k, v)
    _plain_copy(k, v, t[here.long()].view(-1), t[there.long()].view(-1))
    _plain_free(t, n, r, here)
    _plain_compact(t, r, k, v)


def _plain_logp(s):
    with torch.no_grad():
        raw = s["logits"].detach()
        x = raw.float()
        cap = s["softcap"]
        z = x if cap is None else cap * torch.tanh(x / cap)
        top = z.amax(1, keepdim=True)
        lp = z - (top + (z - top).exp().sum(1, keepdim=True).log())
        p = lp.exp()
        entropy = -(p * lp).sum(1)
        t = s["targets"][:, None]
        out = [lp.gather(1, t)[:, 0], entropy]
        ids = None
        if s["top_k"]:
            # by value, ties to the lowest index
            bits = (x + 0.0).view(torch.int32).long()
            key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32)
            key -= torch.arange(x.shape[1], device=DEV)
            ids = key.topk(s["top_k"], dim=1).indices
            out += [lp.gather(1, ids), ids]
        if s["grad"]:
            g = s["g_entropy"][:, None] * -p * (lp + entropy[:, None])
            total = s["g_logp"][:, None].clone()
            if ids is not None:
                total += s["g_top"].sum(1, keepdim=True)
            g -= p * total
            g.scatter_add_(1, t, s["g_logp"][:, None])
            if ids is not None:
                g.scatter_add_(1, ids, s["g_top"])
            if cap is not None:
                g *= 1.0 - (z / cap).square()
            out.append(g.to(raw.dtype))
        return out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_attn(s):
    ops = _framework()
    ops.paged_cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"],
                           s["seq_lens"], starts=s["starts"], max_new=s["max_new"])
    out = ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"],
                              starts=s["starts"], max_new=s["max_new"], max_len=s["max_len"])
    return [out, s["k_pages"], s["v_pages"]]


def _own_pages(s):
    ops = _framework()
    t, n, r, k, v = (s[x] for x in ("page_table", "seq_lens", "ref_counts", "k_pages", "v_pages"))
    if s["kind"] == "fork":
        ops.paged_cache_free(t, n, r, s["dst"])
        ops.paged_cache_fork(t, n, r, s["src"], s["dst"])
        ops.paged_cache_reserve(t, n, r, s["dst"], s["one"], k, v)
    else:
        for here, there in ((s["here"], s["there"]), (s["there"], s["here"])):
            ops.paged_cache_reserve(t, n, r, there, s["counts"], k, v)
            ops.paged_cache_copy(k, v, t[here].view(-1), t[there].view(-1))
            ops.paged_cache_free(t, n, r, here)
            ops.paged_cache_compact(t, r, k, v)
    return [t, n, r, k, v]


def _own_logp(s):
    ops = _framework()
    if not s["grad"]:
        return [x for x in ops.token_logprobs(s["logits"], s["targets"], top_k=s["top_k"],
                                              softcap=s["softcap"]) if x is not None]
    lp, entropy, top, ids = ops.token_logprobs(s["logits"], s["targets"], top_k=s["top_k"],
                                               softcap=s["softcap"])
    outs, grads = [lp, entropy], [s["g_logp"], s["g_entropy"]]
    if s["top_k"]:
        outs, grads = outs + [top], grads + [s["g_top"]]
    (grad,) = torch.autograd.grad(outs, [s["logits"]], grads)
    return [x.detach() for x in ([lp, entropy, top, ids] if s["top_k"] else outs)] + [grad]


def run(state):
    """attention: the new tokens' outputs and the cache's pages; pages: page table,
    lengths, reference counts and pages; log probabilities: those of the targets, the
    entropies, the alternatives' log probabilities and indices (with top_k), and the
    logits' gradient (a training step)."""
    kind = state["kind"]
    if kind == "attn":
        return _own_attn(state) if own else _plain_attn(state)
    if kind == "logp":
        return _own_logp(state) if own else _plain_logp(state)
    return _own_pages(state) if own else _plain_pages(state)


# ---------------------------------------------------------------------------
# the least a call has to do
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "logp":
        one = case["rows"] * case["vocab"] * e
        top = case["rows"] * case["top_k"]
        # (the training step has to read the logits twice: the gradient needs the sums)
        return {"bytes": one * (3 if case["grad"] else 1) + case["rows"] * 16 + top * 12,
                "flops": case["rows"] * case["vocab"] * (12 if case["grad"] else 6)}
    row = case["n_kv_head"] * case["head_dim"] * e
    if case["kind"] == "attn":
        new, cached = _attn_lengths(case)
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
        q = sum(new) * case["n_head"] * case["head_dim"] * e
        return {"bytes": 2 * q + 4 * sum(new) * row + 2 * sum(cached) * row,
                "flops": 4 * pairs * case["n_head"] * case["head_dim"]}
    lens, _ = _page_lengths(case)
    page = 2 * case["layers"] * case["page"] * row
    held = [-(-n // case["page"]) for n in lens]
    if case["kind"] == "fork":
        parting = case["children"] * sum(n % case["page"] != 0 for n in lens)
        # table rows: the children's read and cleared, the parents' read and written to them
        ids = 4 * sum(held) * 4 * case["children"]
        return {"bytes": 2 * parting * page + ids, "flops": 0}
    # twice: each page of the movers is copied, then moved into the hole
    return {"bytes": 2 * 2 * 2 * sum(held) * page, "flops": 0}


# ---------------------------------------------------------------------------
# the same results in float64
# ---------------------------------------------------------------------------
def _exact_attn(case, seed):
    s = _prepare_attn(case, seed)
    new, cached = _attn_lengths(case)
    g = case["n_head"] // case["n_kv_head"]
    outs, at = [], 0
    for i, (n, c) in enumerate(zip(new, cached)):
        pages = s["page_table"][i, :-(-(n + c) // case["page"])].long()

        def mine(x, add):
            x = x[pages].transpose(0, 1).flatten(1, 2)[:, :c]
            add = add[at:at + n] if case["packed"] else add[i, :n]
            return torch.cat([x, add.transpose(0, 1)], 1).double()

        k, v = mine(s["k_pages"], s["k"]), mine(s["v_pages"], s["v"])
        q = (s["q"][at:at + n] if case["packed"] else s["q"][i, :n]).double()
        ahead = (torch.arange(n + c, device=DEV) > c + torch.arange(n, device=DEV)[:, None])
        heads = []
        for h in range(case["n_head"]):
            w = (q[:, h] @ k[h // g].t() / math.sqrt(case["head_dim"])).masked_fill_(
                ahead, -math.inf).softmax(1)
            heads.append(w @ v[h // g])
        outs.append(torch.stack(heads, 1))
        at += n
    return [torch.cat(outs) if case["packed"] else torch.stack(outs), None, None]


def _exact_logp(case, seed):
    s = _prepare_logp(case, seed)
    raw = s["logits"].detach().double().requires_grad_(case["grad"])
    cap = case["softcap"]
    z = cap * torch.tanh(raw / cap) if cap else raw
    lp = torch.log_softmax(z, 1)
    entropy = -(lp.exp() * lp).sum(1)
    out = [lp.gather(1, s["targets"][:, None])[:, 0], entropy]
    ids = None
    if case["top_k"]:
        ids = raw.detach().sort(dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
        out += [lp.gather(1, ids)]
    if case["grad"]:
        grads = [s["g_logp"].double(), s["g_entropy"].double()]
        if ids is not None:
            grads.append(s["g_top"].double())
        out += list(torch.autograd.grad(out, [raw], grads))
    out = [x.detach() for x in out]
    return out[:3] + [ids] + out[3:] if ids is not None else out


def exact(case, seed):
    if case["kind"] == "attn":
        return _exact_attn(case, seed)
    if case["kind"] == "logp":
        return _exact_logp(case, seed)
    return None  # page numbers and copies: nothing is computed
