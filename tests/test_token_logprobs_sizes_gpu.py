"""Log probabilities of very many rows, and of the widest one."""

from __future__ import annotations

import math

import pytest
import torch

from test_token_logprobs_gpu import BF, DEV, U, _exact, _noise, _ops, _targets

pytestmark = pytest.mark.gpu


def _mixed(N, V, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(N, V, generator=g, device=DEV) * 3).to(BF), _targets(N, V, seed)


def test_more_rows_than_a_launch_takes():
    N, V = 2 ** 24 + 5, 8
    x, t = _mixed(N, V, 1)
    out = _ops().token_logprobs(x, t, top_k=2, softcap=15.0)
    for a in (0, 2 ** 23 - 4, 2 ** 23, 2 ** 24 - 3):
        rows = slice(a, a + 8)
        z, lp, chosen, ent, top, ids = _exact(x[rows], t[rows], 15.0, 2)
        e = _noise(V, 15.0) + 8 * U * (z.abs().amax(-1) + chosen.abs())
        assert bool(((out.logprobs[rows].double() - chosen).abs() <= e).all())
        assert float((out.entropy[rows].double() - ent).abs().max()) <= 1e-4
        assert torch.equal(out.top_ids[rows], ids)
        assert float((out.top_logprobs[rows].double() - top).abs().max()) <= 1e-4
    # every row: those of one launch at a time
    for a in range(0, N, 2 ** 22):
        rows = slice(a, a + 2 ** 22)
        part = _ops().token_logprobs(x[rows], t[rows], top_k=2, softcap=15.0)
        assert all(torch.equal(o[rows], p) for o, p in zip(out, part))


@pytest.mark.parametrize("N,V,k", [(65535 * 2 + 3, 9, 3), (65536, 40, 0)])
def test_gradient_of_more_rows_than_a_launch_takes(N, V, k):
    """The gradient's launches end at 65,535 rows."""
    x, t = _mixed(N, V, 2)
    t[::7] = -1
    x.requires_grad_(True)
    gs = [torch.randn(N, device=DEV), torch.randn(N, device=DEV) * 0.3]
    out = _ops().token_logprobs(x, t, top_k=k, softcap=15.0)
    outs = list(out[:2])
    if k:
        outs.append(out.top_logprobs)
        gs.append(torch.randn(N, k, device=DEV))
    (got,) = torch.autograd.grad(outs, [x], gs)
    y = x.detach().double().requires_grad_(True)
    z, lp, chosen, ent, top, ids = _exact(y, t, 15.0, k)
    (want,) = torch.autograd.grad([chosen, ent] + ([top] if k else []), [y],
                                  [g.double() for g in gs])
    size = sum(g.double().abs().view(N, -1).sum(1, keepdim=True) for g in gs) * (
        1 + z.abs().amax(1, keepdim=True))
    # a rounding of the result, and float32's of each of its terms
    bound = 2.0 ** -8 * want.abs() + 1e-5 * size
    assert bool(((got.double() - want).abs() <= bound).all())


def test_the_widest_row():
    """2^31 - 1 logits: indices end where 32 bits do."""
    V = 2 ** 31 - 1
    at = torch.tensor([5, 2 ** 30 + 1, V - 1], device=DEV)
    x = torch.full((1, V), -60.0, dtype=BF, device=DEV)
    x[0, at] = torch.tensor([20.0, 19.0, 21.0], dtype=BF, device=DEV)
    x.requires_grad_(True)
    out = _ops().token_logprobs(x, torch.tensor([V - 1], device=DEV), top_k=4)
    want = torch.log_softmax(torch.tensor([20.0, 19.0, 21.0], dtype=torch.float64, device=DEV), 0)
    assert out.top_ids[0].tolist() == [V - 1, 5, 2 ** 30 + 1, 0]
    # (the others' part is 2^31 e^-81)
    assert abs(float(out.logprobs.detach()) - float(want[2])) <= 1e-5
    assert float((out.top_logprobs[0, :3].double() - want[[2, 0, 1]]).abs().max()) <= 1e-5
    (g,) = torch.autograd.grad(out.logprobs.sum(), [x])
    exact = torch.tensor([0.0, 0.0, 1.0], device=DEV).double() - want.exp()
    assert float((g[0, at].double() - exact).abs().max()) <= 2.0 ** -8
    # everywhere else -e^(-60 - lse), which bfloat16 holds
    other = math.exp(-60.0 - 21.0 + float(want[2]))
    off = sum(int(((c.float() / -other - 1).abs() > 2.0 ** -7).sum()) for c in g[0].split(2 ** 28))
    assert off == 3
