"""The best continuations of beams against float64."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _select(*a, **kw):
    from nanochat_amd.ops import beam_select

    return beam_select(*a, **kw)


def _all64(logits, scores, k, cap, finished):
    """Of each group the candidates (score, beam, place, token), all of each beam up to k, in
    the order of the definition; float64, on the host."""
    x = logits.double().cpu()
    z = x if cap is None else cap * torch.tanh(x / cap)
    lse = torch.logsumexp(z, -1, keepdim=True)
    G, B, V = x.shape
    n = min(k, V)
    out = []
    for g in range(G):
        c = []
        for b in range(B):
            s = float(scores[g, b])
            if finished is not None and bool(finished[g, b]):
                c += [(s if r == 0 else -math.inf, b, r, -1) for r in range(n)]
                continue
            row = x[g, b] + 0.0
            key = torch.where(row.isnan(), math.inf, row)
            # NaN before infinity, then by logit, ties to the lowest index
            ids = sorted(range(V), key=lambda v: (not bool(row[v].isnan()), -float(key[v]), v))[:n] \
                if V <= 300 else key.sort(descending=True, stable=True).indices[:n].tolist()
            for r, v in enumerate(ids):
                lp = float(z[g, b, v] - lse[g, b])
                t = -math.inf if s == -math.inf or float(z[g, b, v]) == -math.inf else s + lp
                c.append((t, b, r, v))
        c.sort(key=lambda e: (not math.isnan(e[0]), -e[0] if not math.isnan(e[0]) else 0.0, e[1], e[2]))
        out.append(c)
    return out


def _check(logits, scores, k, cap=None, finished=None):
    """Scores within a float32 rounding and what the sums may be off; the order wherever two
    candidates differ by more than that.

    A row's sum of exponentials has terms that are each off by some roundings: of z (by the cap, at
    most 6 half steps of it) and of the exponential's argument and value (2^-24 of |z| and some
    2^-23); and it is added up in float32, 2^-24 for each term that a thread adds (at most 16,384)."""
    got = _select(logits, scores, k, softcap=cap, finished=finished)
    assert got.scores.shape == got.parents.shape == got.tokens.shape == (*scores.shape[:-1], k)
    assert got.scores.dtype == F32 and got.parents.dtype == got.tokens.dtype == torch.int64
    B, V = logits.shape[-2:]
    flat = [t.reshape(-1, B, *t.shape[scores.dim():]) for t in (logits, scores)]
    fin = None if finished is None else finished.reshape(-1, B)
    want = _all64(flat[0], flat[1], k, cap, fin)
    u = 2.0 ** -24
    size = cap or float(logits[logits.isfinite()].abs().max())
    off = u * (12 * size + 8 + min(16384, V // 256 + 64))
    for g, c in enumerate(want):
        rows = list(zip(*(t.reshape(len(want), k)[g].tolist() for t in got)))
        by_place = {(b, r): (t, v) for t, b, r, v in c}
        place = {}
        seen = []
        for i, (t, b, v) in enumerate(rows):
            r = place.get(b, 0)  # the next of its beam
            place[b] = r + 1
            w, token = by_place[b, r]
            assert v == token, (g, i, rows[i], c[i])
            if math.isfinite(w):
                assert abs(t - w) <= u * abs(w) + off, (g, i, t, w)
            else:
                assert t == w or (math.isnan(t) and math.isnan(w)), (g, i, t, w)
            # not after one that is better by more than the two may be off
            best = c[i][0]
            if math.isfinite(w):
                assert abs(w - best) <= 2 * off, (g, i, w, best)
            else:
                assert (b, r, v) == c[i][1:], (g, i)
            seen.append((b, r))
        assert len(set(seen)) == k


def _rand(G, B, V, dtype, seed=0, pad=0, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(G, B, V + pad, generator=g, device=DEV) * scale).to(dtype)[..., :V]
    s = -2.0 * torch.rand(G, B, generator=g, device=DEV).cumsum(1)
    return x, s, torch.rand(G, B, generator=g, device=DEV) < 0.2


@pytest.mark.parametrize("cap", [None, 15.0, 100.0])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("G,B,V,k", [(1, 1, 5, 5), (1, 4, 65536, 8), (3, 2, 1000, 64), (2, 16, 50257, 64),
                                     (5, 7, 4099, 9), (1, 3, 7, 21), (600, 1, 2000, 3), (70, 8, 8193, 16),
                                     (2, 64, 300, 16), (1, 1, 1, 1), (1, 5, 131072, 10)])
def test_selections(G, B, V, k, dtype, cap):
    x, s, fin = _rand(G, B, V, dtype, seed=V + k)
    _check(x, s, k, cap)
    _check(x, s, k, cap, fin)


@pytest.mark.parametrize("G,B,V,k", [(2, 3, 900, 5), (1, 4, 70000, 8)])
def test_caps_of_any_size(G, B, V, k):
    """A cap far above the logits changes nothing; one far below leaves all tokens alike."""
    x, s, fin = _rand(G, B, V, F32)
    plain = _select(x, s, k, finished=fin)
    for cap in (1e6, 1e30, 3e38):
        got = _select(x, s, k, softcap=cap, finished=fin)
        # (1 - (x / c)^2 / 3 of x is left, and the sums of two passes)
        assert bool(((got.scores - plain.scores).abs() <= 1e-5).all())
        assert torch.equal(got.parents, plain.parents) and torch.equal(got.tokens, plain.tokens)
    for cap in (1e-3, 63.9, 64.1):
        _check(x, s, k, cap, fin)
    got = _select(x, s, k, softcap=1e-30)
    assert bool(torch.isfinite(got.scores).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding_and_strides(dtype):
    x, s, fin = _rand(3, 4, 1000, dtype, pad=24)
    _check(x, s, 8, 15.0, fin)
    want = _select(x.contiguous(), s, 8, softcap=15.0)
    for y in (x, x.transpose(1, 2).contiguous().transpose(1, 2), x.transpose(0, 1).contiguous().transpose(0, 1)):
        got = _select(y, s.t().contiguous().t(), 8, softcap=15.0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = _select(x[0], s[0], 8, softcap=15.0)
    assert all(torch.equal(a, b[0]) for a, b in zip(got, want))


@pytest.mark.parametrize("V", [50, 9000])
def test_ties(V):
    """Equal logits and equal beams: the lowest beam, then the lowest token."""
    x = torch.zeros(2, 3, V, dtype=BF, device=DEV)
    s = torch.zeros(2, 3, device=DEV)
    got = _select(x, s, 5)
    assert got.parents.tolist() == [[0] * 5] * 2 and got.tokens.tolist() == [list(range(5))] * 2
    x[:, :, 7] = 1.0
    got = _select(x, s, 5, softcap=15.0)
    assert got.parents.tolist() == [[0, 1, 2, 0, 0]] * 2
    assert got.tokens.tolist() == [[7, 7, 7, 0, 1]] * 2


@pytest.mark.parametrize("V", [40, 9000])
@pytest.mark.parametrize("cap", [None, 15.0])
def test_first_step(V, cap):
    """All beams alike, of which one counts: its continuations only."""
    x, _, _ = _rand(2, 1, V, F32)
    x = x.expand(2, 4, V)
    s = torch.full((2, 4), -math.inf, device=DEV)
    s[:, 0] = 0.0
    _check(x, s, 8, cap)
    assert not _select(x, s, 8, softcap=cap).parents.any()


@pytest.mark.parametrize("V", [40, 9000])
def test_masked_vocabulary(V):
    """-inf logits; rows of nothing else; fewer candidates than k."""
    x, s, fin = _rand(3, 4, V, F32)
    x[:, :, ::2] = -math.inf
    x[0, 1] = -math.inf
    x[1] = -math.inf
    x[1, 2, 5] = 1.0
    _check(x, s, 8, None)
    _check(x, s, 8, None, fin)
    s[2] = -math.inf
    _check(x, s, 8, None)


@pytest.mark.parametrize("V", [40, 9000])
@pytest.mark.parametrize("cap", [None, 15.0])
def test_not_finite(V, cap):
    """NaN in a row, and in a score, comes first; an infinity makes its row NaN without a cap."""
    x, s, _ = _rand(4, 3, V, F32)
    x[0, 1, 3] = math.nan
    s[1, 2] = math.nan
    x[2, 0, 5] = math.inf
    got = _select(x, s, 4, softcap=cap)
    assert got.parents[0].tolist() == [1] * 4 and bool(got.scores[0].isnan().all())
    assert int(got.tokens[0, 0]) == 3
    assert got.parents[1].tolist() == [2] * 4 and bool(got.scores[1].isnan().all())
    if cap is None:
        assert got.parents[2].tolist() == [0] * 4 and bool(got.scores[2].isnan().all())
    else:
        _check(x[2:], s[2:], 4, cap)
    _check(x[3:], s[3:], 4, cap)


@pytest.mark.parametrize("cap", [None, 15.0])
def test_one_token_has_most(cap):
    """Rows whose sum is one term's but for a few millionths: that decides."""
    V = 5000
    x = torch.full((1, 2, V), -30.0, device=DEV)
    x[0, 0, 10] = 12.0
    x[0, 1, 20] = 12.0
    x[0, 0, 21] = -1.1  # a little less for the first of beam 0
    s = torch.zeros(1, 2, device=DEV)
    want = _all64(x, s, 2, cap, None)[0]
    got = _select(x, s, 2, softcap=cap)
    assert got.parents[0].tolist() == [e[1] for e in want[:2]] == [1, 0]


@pytest.mark.parametrize("rows", ["one", "near", "spread"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [65.0, 100.0, 1000.0, 3e4, 2.0 ** 20, 3e6])
def test_large_caps_are_as_exact_as_none(cap, dtype, rows):
    """Logits as large as the cap, of which a float32 z is off by more than a likely token's log
    probability: one token near the cap, many near each other, or ordinary ones.

    What a row's sum may be off, in units of 2^-24 of it: a term's argument d by two roundings (2 |d| in
    binary digits, over the terms by their weights at most 2 log2 V), its exponential by 4, a thread's
    additions by one each (4 here) and the joins of 64 lanes, 4 wavefronts and two pieces' sums by 3 each,
    the candidates that are taken out and put back by 8 more; the score by its own rounding."""
    G, B, V, k = 32, 2, 300, 4
    g = torch.Generator(device=DEV).manual_seed(int(cap))
    x = torch.randn(G, B, V, generator=g, device=DEV)
    u01 = torch.rand(G, B, 1, generator=g, device=DEV)
    if rows == "one":
        x = x * cap * 0.01
        x[..., 7:8] = cap * (0.8 + u01)
        # (the next one from some millionths to some hundredths as likely)
        z = cap * torch.tanh(x[..., 7:8].double() / cap) - 3.0 - 10.0 * u01.flip(0)
        x[..., 8:9] = cap * torch.atanh(z / cap)
    elif rows == "near":
        x = cap * (0.3 + 0.6 * u01) + 2.0 * x
    else:
        x = 3.0 * x
    x = x.to(dtype)
    s = torch.zeros(G, B, device=DEV)
    got = _select(x, s, k, softcap=cap)
    u = 2.0 ** -24
    off = u * (2 * math.log2(V) + 4 + 4 + 3 * (6 + 4 + 1) + 8)
    for i, c in enumerate(_all64(x, s, k, cap, None)):
        place = {(b, v): t for t, b, _, v in c}
        for j in range(k):
            t, e = float(got.scores[i, j]), (int(got.parents[i, j]), int(got.tokens[i, j]))
            assert abs(t - place[e]) <= off + u * abs(place[e]), (i, j, t, place[e])
            # not after one that is better by more than the two may be off
            assert place[e] >= c[j][0] - 2 * off, (i, j, place[e], c[j])


def test_all_finished():
    x, s, _ = _rand(2, 3, 1000, BF)
    fin = torch.ones(2, 3, dtype=torch.bool, device=DEV)
    got = _select(x, s, 3, finished=fin)
    assert torch.equal(got.scores, s) and got.tokens.tolist() == [[-1] * 3] * 2
    assert got.parents.tolist() == [[0, 1, 2]] * 2
    # logits of finished beams are not looked at
    x.fill_(math.nan)
    assert torch.equal(_select(x, s, 3, finished=fin).scores, s)


def test_captured():
    x, s, fin = _rand(2, 4, 20000, BF)
    call = lambda: _select(x, s, 8, softcap=15.0, finished=fin)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in range(4):
        y, t, f = _rand(2, 4, 20000, BF, seed=seed + 5)
        x.copy_(y), s.copy_(t), fin.copy_(f)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_stream_and_compiled():
    x, s, fin = _rand(2, 4, 20000, BF)
    want = _select(x, s, 8, softcap=15.0, finished=fin)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = _select(x, s, 8, softcap=15.0, finished=fin)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    f = torch.compile(lambda x, s: _select(x, s, 8, softcap=15.0, finished=fin), fullgraph=True,
                      backend="eager")
    assert all(torch.equal(a, b) for a, b in zip(f(x, s), want))


def test_no_groups():
    got = _select(torch.zeros(0, 4, 100, device=DEV), torch.zeros(0, 4, device=DEV), 8)
    assert got.scores.shape == (0, 8) and got.parents.shape == (0, 8)


def test_refusals():
    x, s, fin = _rand(2, 4, 100, F32)
    for bad in (0, -1, 65, 401):
        with pytest.raises(ValueError):
            _select(x, s, bad)
    with pytest.raises(ValueError):
        _select(torch.zeros(1, 17, 100, device=DEV), torch.zeros(1, 17, device=DEV), 64)
    with pytest.raises(ValueError):
        _select(x, s[:, :3], 4)
    with pytest.raises(ValueError):
        _select(x[0, 0], s[0, 0], 4)
    with pytest.raises(ValueError):
        _select(x[..., :0], s, 4)
    with pytest.raises(ValueError):
        _select(x, s, 4, finished=fin[:, :3])
    for cap in (0.0, -1.0, math.inf, math.nan, 1e-60):
        with pytest.raises(ValueError):
            _select(x, s, 4, softcap=cap)
    with pytest.raises(TypeError):
        _select(x.half(), s, 4)
    with pytest.raises(TypeError):
        _select(x, s.double(), 4)
    with pytest.raises(TypeError):
        _select(x, s, 4, finished=fin.int())
    with pytest.raises(RuntimeError):
        _select(x.cpu(), s.cpu(), 4)
    with pytest.raises(RuntimeError):
        _select(x, s.cpu(), 4)
    with pytest.raises(RuntimeError, match="grad"):
        _select(x.requires_grad_(), s, 4)
