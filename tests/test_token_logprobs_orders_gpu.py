"""Alternatives of rows whose order is against the search: the results, and that the time
stays that of a few readings."""

from __future__ import annotations

import pytest
import torch

from test_token_logprobs_gpu import BF, DEV, F32, _check_forward, _ops, _targets

pytestmark = pytest.mark.gpu

ROWS = 512  # (not cut into pieces)


def _rising(V, kind):
    i = torch.arange(V, device=DEV).double()
    if kind == "linear":
        x = i / V * 40 - 20
    elif kind == "steps":         # runs of equal ones, each above the last
        x = (i / 3000).floor()
    elif kind == "last bits":     # all in one power of two, apart by their last bits
        x = 8 + i * 2.0 ** -20
    elif kind == "exponents":
        x = 2.0 ** (i / V * 200 - 100)
    else:                         # low ones first, then many of the largest
        x = (i > 9000).double() * 3
    return x.float()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["linear", "steps", "last bits", "exponents", "plateau"])
@pytest.mark.parametrize("V", [9101, 70001])
def test_rising_rows(V, kind, dtype):
    x = _rising(V, kind).to(dtype).repeat(ROWS, 1)
    x[1::2] = -x[1::2].flip(1)    # rising, too, below 0
    x[2, V // 2] = float("nan")
    t = _targets(ROWS, V)
    for k in (1, 20, 64):
        out = _ops().token_logprobs(x, t, top_k=k, softcap=15.0)
        rows = torch.tensor([0, 1, ROWS - 2, ROWS - 1], device=DEV)
        _check_forward(x[rows], t[rows], 15.0, k,
                       type(out)(*(None if o is None else o[rows] for o in out)))
        assert int(out.top_ids[2, 0]) == V // 2
        want = torch.sort(x[3].float(), descending=True, stable=True).indices[:k]
        assert bool((out.top_ids[3::2] == want).all())


@pytest.mark.parametrize("kind", ["linear", "last bits", "plateau"])
def test_rising_rows_take_a_few_readings(kind):
    """At most nine readings in place of one; 120 were to be expected of a search that drops
    a thousand elements in each."""
    V = 131072
    x = _rising(V, kind).repeat(ROWS, 1)
    mixed = x[:, torch.randperm(V, device=DEV)].contiguous()
    t = _targets(ROWS, V)

    def time(x):
        best = 1e9
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            _ops().token_logprobs(x, t, top_k=20)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    usual, rising = time(mixed), time(x)
    print(f"{kind}: {usual * 1e3:.0f} us shuffled, {rising * 1e3:.0f} us")
    assert rising <= 30 * usual
