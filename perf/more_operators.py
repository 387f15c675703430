"""The operators that a decoding step of a search over a cache in 4 bits is made of,
as workloads: what their speed is judged by.

Four sets of calls, each as a program makes them:

* new tokens' queries and keys are rotated by their positions and normalised, and the
  keys and values written into the cache's pages on the way, in 16, 32 or 4 bits;
* attention of new tokens over a paged cache held in 4 bits, which takes the new keys
  and values first.  What it stored of them is read back;
* a search's selection: the k best continuations over all beams of a prompt and the
  vocabulary, by cumulative log probabilities of soft-capped logits;
* the beams' sequences in the cache follow that selection.

A 4-bit page holds, for each head, the codes of its tokens (head_dim / 2 bytes each, the
even channel in the low bits) and then head_dim / 32 rows of one scale byte per token,
of 32 channels each: value = code * 2^(byte - 127), the codes' low three bits standing for
0, 0.5, 1, 1.5, 2, 3, 4, 6 and the fourth for the sign.  The byte is that of the smallest
power of two by which no channel is larger than 7.

``listed`` gives the fixed cases, ``draw`` another one of the same ranges,
``prepare`` the tensors that exist before the call, ``run`` one call, ``work``
the bytes and operations it cannot do without and ``exact`` its results in
float64.  With ``own`` false ``run`` computes the plain form in elementary torch
operations in float32 (float64 where a value's side of a border, or the order of
scores, is decided), with ``own`` true it calls the framework.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 2.0 ** -23  # of the norm


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


def _tokens(name, kind, seqs, ones, new, cached, lengths, dtype="bf16", bits=16, heads=None,
            page=64, packed=True, tables="bf16"):
    """``seqs`` sequences, the last ``ones`` of them with one new token, the others
    with new[0] .. new[1]; cached[0] .. cached[1] tokens in the cache before.  The
    first has the most of both, the others spread over the logarithm (``lengths``
    seeds them).  packed: the new tokens in one row after the other, else (B, T)."""
    c = {"name": name, "kind": kind, "seqs": seqs, "ones": ones, "new_lo": new[0],
         "new_hi": new[1], "cached_lo": cached[0], "cached_hi": cached[1], "lengths": lengths,
         "dtype": dtype, "bits": bits, "page": page, "packed": packed, "tables": tables}
    c.update(heads or _D12)
    return c


def _beams(name, prompts, beams, k, vocab, dtype, softcap, padded=0):
    return {"name": name, "kind": "beams", "prompts": prompts, "beams": beams, "k": k,
            "vocab": vocab, "padded": max(padded, vocab), "dtype": dtype, "softcap": softcap}


def _reorder(name, prompts, beams, lens, lengths, page=64):
    return {"name": name, "kind": "reorder", "prompts": prompts, "beams": beams,
            "len_lo": lens[0], "len_hi": lens[1], "lengths": lengths, "page": page}


def listed():
    return [
        # the step of a batch of chats: one token each, into 16-bit pages
        _tokens("rotate_decode", "rotate", 64, 64, (1, 1), (200, 1000), 1, packed=False),
        # a long prompt's chunk, with shared key heads, into 4-bit pages
        _tokens("rotate_prompt4", "rotate", 1, 0, (12289, 12289), (4000, 4000), 2, bits=4,
                heads={"n_head": 12, "n_kv_head": 4, "head_dim": 128}),
        # chunks among decoding sequences of a float32 program
        _tokens("rotate_fp32", "rotate", 9, 4, (65, 700), (1, 900), 3, dtype="fp32",
                heads={"n_head": 10, "n_kv_head": 5, "head_dim": 64}, page=48, tables="fp32"),
        # one token of each of four chats: launches and latency
        _tokens("decode4_small", "attn4", 4, 4, (1, 1), (200, 600), 4, bits=4, packed=False),
        # a serving step of a batch with one very long context among ordinary ones
        _tokens("decode4_ragged", "attn4", 16, 16, (1, 1), (300, 131071), 5, bits=4,
                packed=False),
        # many sequences whose query heads share a key head
        _tokens("decode4_groups", "attn4", 96, 96, (1, 1), (500, 6000), 6, bits=4,
                heads={"n_head": 32, "n_kv_head": 4, "head_dim": 64}, page=32),
        # a float32 program: a step that decodes some and takes the prompts of others
        _tokens("chunk4_fp32", "attn4", 6, 3, (33, 257), (50, 1500), 7, dtype="fp32", bits=4,
                heads={"n_head": 8, "n_kv_head": 4, "head_dim": 96}, page=16),
        # the last chunk of a long prompt
        _tokens("prefill4_long", "attn4", 1, 0, (8193, 8193), (16000, 16000), 8, bits=4,
                packed=False),
        # one question with four beams
        _beams("beams_small", 1, 4, 8, 65536, "fp32", 15.0),
        # a batch of questions; the vocabulary's padding is cut off
        _beams("beams_batch", 48, 8, 16, 50257, "bf16", 15.0, padded=50304),
        # the beams of one question, and of a batch
        _reorder("reorder_small", 1, 4, (500, 500), 9),
        _reorder("reorder_batch", 48, 8, (300, 8000), 10, page=16),
    ]


def _log_int(rng, lo, hi):
    if hi <= lo:
        return lo
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["rotate"] * 3 + ["decode"] * 3 + ["chunk"] * 2 + ["prefill"] * 2
                      + ["beams"] * 3 + ["reorder"] * 2)
    lengths = rng.randrange(1 << 20)
    if kind in ("rotate", "decode", "chunk", "prefill"):
        nkv = rng.randint(1, 8)
        bits = 4 if kind != "rotate" else rng.choice([4, 16])
        dims = [32, 64, 96, 128, 128] if bits == 4 else [16, 40, 64, 96, 128, 128]
        heads = {"n_head": nkv * rng.choice([1, 1, 2, 3, 4, 8]), "n_kv_head": nkv,
                 "head_dim": rng.choice(dims)}
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        page = rng.choice([16, 32, 48, 64, 128])
        tables = rng.choice(["bf16", "fp32"])
        seqs = 1 if kind == "prefill" else _log_int(rng, 1, 128 if kind == "decode" else 48)
        if kind == "rotate":
            new = _log_int(rng, 1, max(1, 49000 // seqs // heads["n_head"]))
            cached = _log_int(rng, 1, max(1, 80000 // seqs))
            ones = rng.randint(0, seqs)
        elif kind == "decode":
            new, ones = 1, seqs
            cached = _log_int(rng, 16, max(16, min(131071, 2_000_000 // seqs * 6
                                                   // max(6, heads["n_kv_head"]))))
        else:
            most = (200_000_000 if dtype == "fp32" else 900_000_000) // heads["n_head"]
            new = _log_int(rng, 2, max(2, min(1500 if kind == "chunk" else 8193,
                                              math.isqrt(most // seqs))))
            cached = _log_int(rng, 1, max(1, min(20000, most // seqs // new - new)))
            ones = rng.randint(0, seqs - 1)
        packed = kind == "chunk" or (kind != "prefill" and rng.random() < 0.5)
        if not packed and 0 < ones < seqs:
            ones = seqs
        c = _tokens("", "rotate" if kind == "rotate" else "attn4", seqs, ones,
                    (max(1, new // 20) if packed else new, new),
                    (max(1, cached // 20), cached), lengths, dtype, bits, heads, page, packed,
                    tables)
        if not packed and ones == seqs:
            c["new_lo"] = c["new_hi"] = 1
    elif kind == "beams":
        dtype = rng.choice(["bf16", "fp32"])
        vocab = _log_int(rng, 1000, 131072)
        beams = rng.randint(1, 16)
        prompts = _log_int(rng, 1, max(1, min(64, 20_000_000 // vocab // beams)))
        pad = rng.choice([0, (vocab + 63) // 64 * 64])
        c = _beams("", prompts, beams, min(64, beams * rng.choice([1, 2])), vocab, dtype,
                   rng.choice([15.0, 15.0, 0.0]), pad)
    else:
        length = _log_int(rng, 20, 8000)
        c = _reorder("", _log_int(rng, 1, 48), rng.randint(2, 16), (max(1, length // 10), length),
                     lengths, rng.choice([16, 32, 64]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# lengths and inputs
# ---------------------------------------------------------------------------
def _dtype(name):
    return torch.float32 if name == "fp32" else torch.bfloat16


def _lengths(case):
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


def _reorder_lengths(case):
    rng = random.Random(case["lengths"])
    return [case["len_hi"] if i == 0 else _log_int(rng, case["len_lo"], case["len_hi"])
            for i in range(case["prompts"])]


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _prepare_tokens(case, seed):
    g, dt = _generator(seed), _dtype(case["dtype"])
    new, cached = _lengths(case)
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

    def pages():
        if case["bits"] != 4:
            return randn(P, NKVH, ps, D)
        out = torch.empty(P, NKVH, ps, D // 2 + D // 32, dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // (NKVH * ps * D))
        for p in range(0, P, step):
            n = min(step, P - p)
            x = torch.randn(n, NKVH, ps, D, generator=g, device=DEV)
            _store4(out[p:p + n], *_codes4(x))
        return out

    s = {"kind": case["kind"], "k_pages": pages(), "v_pages": pages(), "bits": case["bits"],
         "page_table": table, "seq_lens": _ints(lens), "max_new": max(new), "max_len": max(lens),
         "starts": None, "tokens": sum(new) if case["packed"] else max(new)}
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
    if case["kind"] == "rotate":
        angles = torch.arange(W * ps, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        s["cos"], s["sin"] = (x.to(_dtype(case["tables"])) for x in (angles.cos(), angles.sin()))
    return s


def _prepare_beams(case, seed):
    g, dt = _generator(seed), _dtype(case["dtype"])
    G, B, V = case["prompts"], case["beams"], case["vocab"]
    # a trained head's logits before the cap: most are low, some stand out
    x = torch.randn(G * B, case["padded"], generator=g, device=DEV) * 2.5 - 2.0
    x.scatter_(1, torch.randint(0, V, (G * B, 8), generator=g, device=DEV),
               torch.randn(G * B, 8, generator=g, device=DEV) * 3 + 8)
    scores = -3.0 * torch.rand(G, B, generator=g, device=DEV).cumsum(1)
    return {"kind": "beams", "logits": x.to(dt).view(G, B, -1)[..., :V], "scores": scores,
            "k": case["k"], "softcap": case["softcap"] or None,
            "finished": torch.rand(G, B, generator=g, device=DEV) < 0.1}


def _prepare_reorder(case, seed):
    """Slots i * beams .. of prompt i: its beams share the prompt's full pages and hold a
    last one each."""
    G, B, ps = case["prompts"], case["beams"], case["page"]
    rng, lens = random.Random(seed), _reorder_lengths(case)
    W = -(-(max(lens) + 1) // ps) + 1
    table, refs, seq_lens, src = [], [], [], []
    for i in range(G):
        full = lens[i] // ps
        shared = list(range(len(refs), len(refs) + full))
        refs += [B] * full
        for _ in range(B):
            table.append(shared + [len(refs)] + [-1] * (W - full - 1))
            refs.append(1)
            seq_lens.append(lens[i] + 1)
            # (the best beams have most of the continuations)
            src.append(i * B + min(rng.randrange(B), rng.randrange(B)))
    place = list(range(len(refs) + 5))
    rng.shuffle(place)
    counts = [0] * len(place)
    for p, r in enumerate(refs):
        counts[place[p]] = r
    return {"kind": "reorder", "page_table": _ints([[place[p] if p >= 0 else -1 for p in r]
                                                    for r in table]),
            "seq_lens": _ints(seq_lens), "ref_counts": _ints(counts),
            "slots": _ints(list(range(G * B))), "src": _ints(src)}


def prepare(case, seed):
    if case["kind"] == "beams":
        return _prepare_beams(case, seed)
    if case["kind"] == "reorder":
        return _prepare_reorder(case, seed)
    return _prepare_tokens(case, seed)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _codes4(x):
    """Codes (0 to 15) and scale bytes (one per 32) of values x (..., D), computed in
    x's own precision, in which the steps below are exact."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1
    byte = (e - 3 + (m > 0.875) + 127).clamp_(2, 252)
    byte = torch.where(top == 0, 2, byte)
    a = b.abs() * ((254 - byte) << 23).view(torch.float32)  # 2^(127 - byte)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0))
    code += (b < 0).to(torch.uint8) << 3
    return code.flatten(-2), byte.squeeze(-1).to(torch.uint8)


def _parts4(pages):
    """The codes' bytes (P, NKVH, page, D / 2) and the scales (P, NKVH, D / 32, page) of 4-bit
    pages, as views."""
    P, NKVH, ps, row = pages.shape
    D = row * 32 // 17
    flat = pages.view(P, NKVH, -1)
    return (flat[..., :ps * D // 2].view(P, NKVH, ps, D // 2),
            flat[..., ps * D // 2:].view(P, NKVH, D // 32, ps))


def _store4(pages, code, byte):
    """Codes and scales of all tokens of some pages, (P, NKVH, page, ..)."""
    c, s = _parts4(pages)
    c.copy_(code[..., 0::2] | code[..., 1::2] << 4)
    s.copy_(byte.transpose(2, 3))


def _values4(codes, scales):
    """Values (float32) of code bytes (..., D / 2) and scale bytes (..., D / 32)."""
    one = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    one = torch.cat([one, -one])
    two = torch.stack([one.repeat(16), one.repeat_interleave(16)], -1)
    x = two[codes.int()].flatten(-2).unflatten(-1, (-1, 32))
    return x.mul_((scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _plain_rows(s):
    """Of a call's tokens (B, T): positions, which are real, their pages and places in
    them, and the rows of the packed tensors (None: they are (B, T) already)."""
    table, lens, T = s["page_table"], s["seq_lens"], s["max_new"]
    ps = s["k_pages"].shape[2]
    step = torch.arange(T, device=DEV)
    if s["starts"] is None:
        n, rows = torch.full((table.shape[0],), T, device=DEV), None
    else:
        first, n = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
        rows = (first[:, None] + step).clamp(max=s["q"].shape[0] - 1)
    at = (lens - n)[:, None] + step
    page = table.gather(1, (at // ps).clamp(0, table.shape[1] - 1)).long()
    return at, step < n[:, None], page, rows


def _plain_write(s, k, v, at, real, page):
    """k, v (B, T, NKVH, D) float32 or float64 into the pages."""
    ps = s["k_pages"].shape[2]
    b, t = (real & (page >= 0)).nonzero(as_tuple=True)
    p, i = page[b, t], at[b, t] % ps
    if s["bits"] != 4:
        s["k_pages"].transpose(1, 2)[p, i] = k[b, t].to(s["k_pages"].dtype)
        s["v_pages"].transpose(1, 2)[p, i] = v[b, t].to(s["v_pages"].dtype)
        return
    for pages, x in ((s["k_pages"], k), (s["v_pages"], v)):
        code, byte = _codes4(x[b, t])
        c, m = _parts4(pages)
        c.transpose(1, 2)[p, i] = code[..., 0::2] | code[..., 1::2] << 4
        m.permute(0, 3, 1, 2)[p, i] = byte


def _plain_read(s, at, real, page, rows):
    """What the 4-bit pages hold of the tokens, in bfloat16."""
    ps, out = s["k_pages"].shape[2], []
    p, i = page.clamp(min=0), at % ps
    if rows is not None:
        b, t = real.nonzero(as_tuple=True)
        p, i = p[b, t], i[b, t]
    for pages in (s["k_pages"], s["v_pages"]):
        c, m = _parts4(pages)
        out.append(_values4(c.transpose(1, 2)[p, i], m.permute(0, 3, 1, 2)[p, i]).bfloat16())
    return out


def _plain_rotate(s):
    at, real, page, rows = _plain_rows(s)
    cos, sin = (x[at.clamp(min=0)][:, :, None] for x in (s["cos"], s["sin"]))

    def rotated(x, real_type):
        x = (x if rows is None else x[rows]).to(real_type)
        c, n = cos.to(real_type), sin.to(real_type)
        a, b = x.chunk(2, -1)
        y = torch.cat([a * c + b * n, b * c - a * n], -1)
        return y / (y.square().mean(-1, keepdim=True) + EPS).sqrt()

    q = rotated(s["q"], torch.float32).to(s["q"].dtype)
    if rows is not None:
        q = q[real]
    v = s["v"] if rows is None else s["v"][rows]
    # (which code a key gets is decided in float64)
    k = rotated(s["k"], torch.float64 if s["bits"] == 4 else torch.float32)
    _plain_write(s, k, v.float(), at, real, page)
    if s["bits"] == 4:
        return [q, *_plain_read(s, at, real, page, rows)]
    return [q, s["k_pages"], s["v_pages"]]


def _plain_attn4(s):
    at, real, page, rows = _plain_rows(s)
    table, lens, q = s["page_table"], s["seq_lens"], s["q"]
    P, NKVH, ps, _ = s["k_pages"].shape
    D, NH, B, T = q.shape[-1], q.shape[-2], table.shape[0], s["max_new"]
    qb, kb, vb = (x if rows is None else x[rows] for x in (q, s["k"], s["v"]))
    _plain_write(s, kb.float(), vb.float(), at, real, page)
    # the cache as (B, NKVH, L, D)
    pages = -(-s["max_len"] // ps)
    ids = table[:, :pages].clamp(min=0).long()
    L = pages * ps
    held = (torch.arange(L, device=DEV) < lens[:, None]) & (table[:, :pages] >= 0
                                                             ).repeat_interleave(ps, 1)

    def gathered(x):
        c, m = _parts4(x)
        x = _values4(c[ids], m[ids].transpose(3, 4)).transpose(1, 2).reshape(B, NKVH, L, D)
        return x.masked_fill_(~held[:, None, :, None], 0.0)

    scores = torch.matmul(
        qb.float().view(B, T, NKVH, NH // NKVH, D).permute(0, 2, 3, 1, 4).reshape(
            B, NKVH, NH // NKVH * T, D) * D ** -0.5,
        gathered(s["k_pages"]).transpose(2, 3).contiguous())
    seen = held[:, None, :] & (torch.arange(L, device=DEV) <= at[:, :, None])
    scores = scores.view(B, NKVH, NH // NKVH, T, L)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(B, NKVH, -1, L), gathered(s["v_pages"])).view(
        B, NKVH, NH // NKVH, T, D) / total.clamp_(min=1e-38)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, T, NH, D).to(q.dtype)
    if rows is not None:
        out = out[real]
    return [out, *_plain_read(s, at, real, page, rows)]


def _plain_beams(s):
    """By score; equal ones by beam, and in a beam by logit, then token."""
    x = s["logits"].double()
    G, B, V = x.shape
    k, done = s["k"], s["finished"]
    cap = s["softcap"]
    z = x if cap is None else cap * torch.tanh(x / cap)
    top = z.amax(-1, keepdim=True)
    lp = z - (top + (z - top).exp().sum(-1, keepdim=True).log())
    n = min(k, V)
    # in a beam by logit, ties to the lowest index
    bits = (s["logits"].float() + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32)
    ids = (key - torch.arange(V, device=DEV)).topk(n, dim=-1).indices
    total = s["scores"].double()[..., None] + lp.gather(2, ids)
    # a finished beam has one continuation: itself
    total = torch.where(done[..., None], -math.inf, total)
    total[..., 0] = torch.where(done, s["scores"].double(), total[..., 0])
    ids = torch.where(done[..., None], -1, ids)
    total, at = total.view(G, -1).sort(dim=1, descending=True, stable=True)
    at = at[:, :k]
    return [total[:, :k].float(), at // n, ids.view(G, -1).gather(1, at)]


def _plain_reorder(s):
    table, lens, refs = s["page_table"], s["seq_lens"], s["ref_counts"]
    slots, src = s["slots"].long(), s["src"].long()
    old, rows = table[slots], table[src]
    refs.index_add_(0, rows[rows >= 0], refs.new_ones(1).expand(int((rows >= 0).sum())))
    refs.index_add_(0, old[old >= 0], refs.new_full((1,), -1).expand(int((old >= 0).sum())))
    n = lens[src]
    table[slots] = rows
    lens[slots] = n
    return [table, lens, refs]


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_read(ops, s):
    return ops.paged_cache_read(s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"],
                                s["tokens"], starts=s["starts"], max_new=s["max_new"])


def _own_rotate(s):
    ops = _framework()
    q = ops.paged_rotary_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_pages"],
                                s["v_pages"], s["page_table"], s["seq_lens"], starts=s["starts"],
                                max_new=s["max_new"], norm_eps=EPS)
    return [q, *(_own_read(ops, s) if s["bits"] == 4 else (s["k_pages"], s["v_pages"]))]


def _own_attn4(s):
    ops = _framework()
    ops.paged_cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"],
                           s["seq_lens"], starts=s["starts"], max_new=s["max_new"])
    out = ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"],
                              starts=s["starts"], max_new=s["max_new"], max_len=s["max_len"])
    return [out, *_own_read(ops, s)]


def _own_beams(s):
    return list(_framework().beam_select(s["logits"], s["scores"], s["k"], softcap=s["softcap"],
                                         finished=s["finished"]))


def _own_reorder(s):
    _framework().paged_cache_reorder(s["page_table"], s["seq_lens"], s["ref_counts"], s["slots"],
                                     s["src"])
    return [s["page_table"], s["seq_lens"], s["ref_counts"]]


def run(state):
    """rotate: the queries, and the pages or, of 4-bit ones, the new tokens' values in them;
    attn4: the new tokens' outputs, and their values in the pages; beams: scores, beams and
    tokens of the best continuations; reorder: page table, lengths and reference counts."""
    kind = state["kind"]
    if kind == "rotate":
        return _own_rotate(state) if own else _plain_rotate(state)
    if kind == "attn4":
        return _own_attn4(state) if own else _plain_attn4(state)
    if kind == "beams":
        return _own_beams(state) if own else _plain_beams(state)
    return _own_reorder(state) if own else _plain_reorder(state)


# ---------------------------------------------------------------------------
# the least a call has to do
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "beams":
        rows = case["prompts"] * case["beams"]
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": rows * (case["vocab"] * e + 5) + case["prompts"] * case["k"] * 20,
                "flops": rows * case["vocab"] * 6}
    if kind == "reorder":
        # table rows read and written, the counts of what they hold
        held = sum(-(-(n + 1) // case["page"]) for n in _reorder_lengths(case))
        return {"bytes": case["beams"] * held * 4 * 4 + case["prompts"] * case["beams"] * 16,
                "flops": 0}
    e = 4 if case["dtype"] == "fp32" else 2
    NH, NKVH, D = case["n_head"], case["n_kv_head"], case["head_dim"]
    new, cached = _lengths(case)
    N = sum(new)
    held = NKVH * (D // 2 + D // 32 if case["bits"] == 4 else D * e)  # of a token's k or v
    bytes_ = N * (2 * NH + 2 * NKVH) * D * e + 2 * N * held
    if case["bits"] == 4:
        bytes_ += 2 * N * NKVH * D * 2  # (what was stored, read back)
    if kind == "rotate":
        at = max(a + b for a, b in zip(new, cached)) - min(cached)
        return {"bytes": bytes_ + min(N, at) * D * (4 if case["tables"] == "fp32" else 2),
                "flops": N * (NH + NKVH) * D * 7}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
    return {"bytes": bytes_ + 2 * sum(cached) * held, "flops": 4 * pairs * NH * D}


# ---------------------------------------------------------------------------
# the same results in float64
# ---------------------------------------------------------------------------
_STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e of whole numbers -200 to 200 (a device's pow may be a rounding off)."""
    table = torch.tensor([math.ldexp(1.0, n) for n in range(-200, 201)], dtype=torch.float64,
                         device=e.device)
    return table[e.long() + 200]


def _held4(x):
    """What 4-bit pages hold of x (..., D), float64."""
    shape = x.shape
    x = x.double().reshape(-1, 32)
    big = x.abs().max(1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(big > 0, big, 1.0)))
    # (log2 may be a rounding off)
    e = e + (big >= _power(e + 1)).double() - (big < _power(e)).double()
    e = torch.where(big > 0, e - 2, -125.0)
    e = torch.where(big > 7.0 * _power(e), e + 1, e).clamp(-125, 125)
    a = x.abs() * _power(-e)
    steps = torch.tensor(_STEPS, dtype=torch.float64, device=x.device)
    far = (a[..., None] - steps).abs()
    # (a tie goes to the even place)
    odd = torch.tensor([0.0, 1e-12] * 4, dtype=torch.float64, device=x.device)
    at = (far + odd).argmin(-1)
    return (steps[at] * x.sign() * _power(e)).reshape(shape)


def _cached4(pages, ids, n):
    """Values of the first n tokens of a sequence's pages, (NKVH, n, D) float64."""
    P, NKVH, ps, row = pages.shape
    D = row * 32 // 17
    raw = pages[ids].reshape(len(ids), NKVH, -1)
    codes = raw[..., :ps * D // 2].reshape(len(ids), NKVH, ps, D // 2).long()
    nibble = torch.stack([codes % 16, codes // 16], -1).flatten(-2)
    steps = torch.tensor(_STEPS, dtype=torch.float64, device=pages.device)
    value = steps[nibble % 8] * (1.0 - 2.0 * (nibble // 8))
    byte = raw[..., ps * D // 2:].reshape(len(ids), NKVH, D // 32, ps).transpose(2, 3)
    value = value * _power(byte.long() - 127).repeat_interleave(32, -1)
    return value.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_tokens(case, seed):
    s = _prepare_tokens(case, seed)
    new, cached = _lengths(case)
    NH, NKVH, D, ps = case["n_head"], case["n_kv_head"], case["head_dim"], case["page"]
    rotate, four = case["kind"] == "rotate", case["bits"] == 4
    outs, at = [], 0
    for i, (n, c) in enumerate(zip(new, cached)):
        q, k, v = ((x[at:at + n] if case["packed"] else x[i, :n]).double()
                   for x in (s["q"], s["k"], s["v"]))
        at += n
        if rotate:
            turn = torch.complex(s["cos"][c:c + n].double(), -s["sin"][c:c + n].double())[:, None]

            def turned(x):
                y = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
                y = torch.cat([y.real, y.imag], -1)
                return y * (y.pow(2).sum(-1, keepdim=True) / D + EPS).rsqrt()

            q, k = turned(q), turned(k)
        if four:
            k, v = _held4(k), _held4(v)
        if rotate:
            outs.append([q, k, v])
            if not four:
                pos = torch.arange(c, c + n, device=DEV)
                for pages, x in ((s["k_pages"], k), (s["v_pages"], v)):
                    pages[s["page_table"][i, pos // ps].long(), :, pos % ps] = x.to(pages.dtype)
            continue
        ids = s["page_table"][i, :-(-(n + c) // ps)].long()
        kk, vv = (torch.cat([_cached4(pages, ids, c), x.transpose(0, 1)], 1)
                  for pages, x in ((s["k_pages"], k), (s["v_pages"], v)))
        ahead = (torch.arange(n + c, device=DEV) > c + torch.arange(n, device=DEV)[:, None])
        heads = []
        for h in range(NH):
            w = (q[:, h] @ kk[h * NKVH // NH].t() / math.sqrt(D)).masked_fill_(
                ahead, -math.inf).softmax(1)
            heads.append(w @ vv[h * NKVH // NH])
        outs.append([torch.stack(heads, 1), k, v])
    outs = [torch.cat(x) if case["packed"] else torch.stack(x) for x in zip(*outs)]
    # (16 and 32 bit pages: what was there, and copies of the new values in their type)
    return outs if four else [outs[0], s["k_pages"].double(), s["v_pages"].double()]


def _exact_beams(case, seed):
    s = _prepare_beams(case, seed)
    z = s["logits"].double()
    if s["softcap"]:
        z = s["softcap"] * torch.tanh(z / s["softcap"])
    G, B, V = z.shape
    total = torch.log_softmax(z, 2) + s["scores"].double()[..., None]
    only = torch.full_like(total, -math.inf)
    only[..., 0] = s["scores"].double()
    total = torch.where(s["finished"][..., None], only, total).view(G, -1)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :case["k"]], at[:, :case["k"]]
    beam = at // V
    token = torch.where(s["finished"].gather(1, beam), -1, at % V)
    return [best, beam, token]


def exact(case, seed):
    if case["kind"] == "beams":
        return _exact_beams(case, seed)
    if case["kind"] == "reorder":
        return None  # page numbers: nothing is computed
    return _exact_tokens(case, seed)
