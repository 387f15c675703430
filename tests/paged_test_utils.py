"""Plain float64 forms of the paged cache's operators, for their tests."""

from __future__ import annotations

import math

import torch

DEV = "cuda"


class Cache:
    """Random pages and a page table for sequences of given lengths, pages dealt in
    random order; ``spare`` free pages."""

    def __init__(self, lens, NKVH, D, page, dtype, seed, spare=2, width=None, layout="head"):
        g = torch.Generator(device=DEV).manual_seed(seed)
        held = [-(-n // page) for n in lens]
        self.P, W = sum(held) + spare, width or max([1, *held])
        order = torch.randperm(self.P, generator=g, device=DEV).tolist()
        rows, at = [], 0
        for n in held:
            rows.append(order[at:at + n] + [-1] * (W - n))
            at += n
        self.table = torch.tensor(rows, dtype=torch.int32, device=DEV).view(len(lens), W)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.page, self.g = page, g

        def rand(*shape):
            return torch.randn(*shape, generator=g, device=DEV).to(dtype)

        if layout == "head":      # (P, NKVH, page, D)
            self.k, self.v = rand(self.P, NKVH, page, D), rand(self.P, NKVH, page, D)
        elif layout == "token":   # (P, page, NKVH, D)
            self.k, self.v = (rand(self.P, page, NKVH, D).transpose(1, 2) for _ in range(2))
        else:                     # one allocation, k and v of a page side by side, rows with gaps
            both = rand(self.P, 2, NKVH, page, D + 8)
            self.k, self.v = both[:, 0, :, :, :D], both[:, 1, :, :, :D]

    def rand(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device=DEV).to(dtype)


def keys_of(cache, slot, length):
    """(positions that hold a token, k rows, v rows) of a sequence, float64: rows (n,
    NKVH, D)."""
    pos = torch.arange(length, device=DEV)
    W = cache.table.shape[1]
    pos = pos[pos < W * cache.page]
    pages = cache.table[slot, (pos // cache.page).long()].long()
    ok = (pages >= 0) & (pages < cache.k.shape[0])
    pos, pages = pos[ok], pages[ok]
    at = (pos % cache.page).long()
    return pos, cache.k[pages, :, at].double(), cache.v[pages, :, at].double()


def attention64(q, cache, slots, new, scale):
    """q: list of (n_i, NH, D) tensors.  For each sequence (out, lse, sum p |v|, largest
    scale sum |q| |k|), float64.  A row attends only to the keys that it sees, by
    indexing: nothing else can reach it."""
    res = []
    for i, n in enumerate(new):
        qi = q[i].double()
        NH, D = qi.shape[1:]
        slot = slots[i]
        length = int(cache.lens[slot]) if 0 <= slot < len(cache.lens) else 0
        pos, k, v = keys_of(cache, slot, length) if length else (
            torch.zeros(0, device=DEV), *(torch.zeros(0, cache.k.shape[1], D, device=DEV,
                                                      dtype=torch.float64) for _ in range(2)))
        g = NH // cache.k.shape[1]
        out, lse, mag = torch.zeros_like(qi), torch.full(qi.shape[:2], -math.inf, device=DEV,
                                                         dtype=torch.float64), torch.zeros_like(qi)
        big = 0.0
        for t in range(n):
            m = int((pos <= length - n + t).sum())
            if m == 0:
                continue
            kk, vv = (x[:m].repeat_interleave(g, 1) for x in (k, v))
            s = (qi[t][None] * kk).sum(-1) * scale  # (m, NH)
            p = s.softmax(0)
            out[t] = (p[..., None] * vv).sum(0)
            mag[t] = (p[..., None] * vv.abs()).sum(0)
            lse[t] = s.logsumexp(0)
            b = float(((qi[t].abs()[None] * kk.abs()).sum(-1) * scale).max())
            big = max(big, b) if math.isfinite(b) else big
        res.append((out, lse, mag, big))
    return res


def attention_bound(dtype, D, length, mag, big):
    """How far a correct kernel's output may be from the exact one, element by element.

    float32 sums: a score is off by at most (D + 4) 2^-24 of sum |q k|, its
    exponential's argument by as much again in rounding; a sum of L terms by L 2^-24.
    bfloat16 adds one rounding (2^-9) of each probability and one of the output."""
    u = 2.0 ** -24
    rel = u * (4 * (D + 8) * (1 + big) + 2 * length + 64)
    if dtype == torch.bfloat16:
        rel = rel + 2 * 2.0 ** -9 + 2.0 ** -12
    return rel * mag + 1e-30


def lse_bound(D, length, lse, big):
    u = 2.0 ** -24
    return u * (4 * (D + 8) * (1 + big) + 2 * length + 64) + 4 * u * lse.abs()


class PageModel:
    """The bookkeeping of the paged cache, one entry after the other, on the host."""

    def __init__(self, table, lens, refs, page, pages=None):
        self.table = [list(r) for r in table]
        self.lens, self.refs, self.page = list(lens), list(refs), page
        self.pages = list(range(len(refs))) if pages is None else list(pages)  # contents

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, slots, counts):
        """0, or what is missing with nothing changed, or -1."""
        W, ps = len(self.table[0]), self.page
        for s, c in zip(slots, counts):
            if not 0 <= s < len(self.lens) or c < 0 or self.lens[s] + c > W * ps:
                return -1
        saved = ([list(r) for r in self.table], list(self.lens), list(self.refs),
                 list(self.pages))
        missing = 0
        for s, c in zip(slots, counts):
            old, new = self.lens[s], self.lens[s] + c
            ids = []
            if c > 0 and old % ps:
                last = self.table[s][old // ps]
                if 0 <= last < len(self.refs) and self.refs[last] > 1:
                    ids.append(old // ps)
            ids += range(-(-old // ps), -(-new // ps))
            for col in ids:
                if 0 not in self.refs:
                    missing += 1
                    if col == old // ps and old % ps:
                        self.refs[self.table[s][col]] -= 1
                    continue
                p = self._take()
                if col == old // ps and old % ps:
                    last = self.table[s][col]
                    self.pages[p] = self.pages[last]
                    self.refs[last] -= 1
                self.table[s][col] = p
            self.lens[s] = new
        if missing:
            self.table, self.lens, self.refs, self.pages = saved
        return missing

    def free(self, slots):
        for s in slots:
            if 0 <= s < len(self.lens):
                for p in self.table[s]:
                    if 0 <= p < len(self.refs):
                        self.refs[p] -= 1
                self.table[s] = [-1] * len(self.table[s])
                self.lens[s] = 0

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            if a == b or not (0 <= a < len(self.lens) and 0 <= b < len(self.lens)):
                continue
            self.free([b])
            self.table[b], self.lens[b] = list(self.table[a]), self.lens[a]
            for p in self.table[b]:
                if 0 <= p < len(self.refs):
                    self.refs[p] += 1

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        movers = [p for p, r in enumerate(self.refs) if r > 0 and p >= live]
        holes = [p for p, r in enumerate(self.refs) if r <= 0 and p < live]
        place = dict(zip(movers, holes))
        for a, b in place.items():
            self.pages[b] = self.pages[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[place.get(p, p) for p in r] for r in self.table]
        return live
