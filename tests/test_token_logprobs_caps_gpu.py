"""Log probabilities and their gradient with soft caps of any size, against float64."""

from __future__ import annotations

import math

import pytest
import torch

from test_token_logprobs_gpu import BF, DEV, F32, U, _exact, _grads, _noise, _ops, _randn, _targets

pytestmark = pytest.mark.gpu

# at which the way of the evaluation changes, and around the range of float32's exponent
CAPS = [1e-40, 1e-3, 1.0, 30.0, 44.0, 50.0, 64.0, 64.5, 85.0, 100.0, 300.0, 1e3, 1e6, 1e30, 3e38]


def _rows(V, dtype):
    """Ordinary logits, all far below 0, all far above, both ends, one above all others."""
    x = _randn(6, V, seed=41, scale=2.5)
    x[0] -= 2.0
    x[1] -= 60.0
    x[2] += 70.0
    x[3, ::2] = -1e4
    x[4] = -90.0
    x[4, V // 2] = 90.0
    x[5] *= 1e-3
    return x.to(dtype), _targets(6, V)


def _errors(cap, V, zmax):
    """Of a sum's logarithm.  Up to 64 z is off by some roundings of the cap, above that by
    some of its own: a division, a tanh of about an ulp, a product."""
    return _noise(V, cap) + 0.0 * zmax if cap <= 64 else _noise(V, 0.0) + 8 * U * zmax


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [37, 9001, 50257])
@pytest.mark.parametrize("cap", CAPS)
def test_forward(cap, V, dtype):
    x, t = _rows(V, dtype)
    out = _ops().token_logprobs(x, t, top_k=5, softcap=cap)
    z, lp, chosen, ent, top, ids = _exact(x, t, cap, 5)
    zmax = z.abs().amax(-1)
    e = _errors(cap, V, zmax)
    err = (out.logprobs.double() - chosen).abs()
    bound = e + 8 * U * (zmax + chosen.abs())
    assert bool((err <= bound).all()), (err / bound).tolist()
    spread = (lp.exp() * (z - z.amax(-1, keepdim=True)).abs()).sum(-1)
    err = (out.entropy.double() - ent).abs()
    bound = (2 * e + 16 * U) * (1 + spread) + 8 * U * zmax
    assert bool((err <= bound).all()), (err / bound).tolist()
    assert torch.equal(out.top_ids, ids)
    err = (out.top_logprobs.double() - top).abs()
    assert bool((err <= e[:, None] + 8 * U * (zmax[:, None] + top.abs())).all())


@pytest.mark.parametrize("cap", [50.0, 100.0, 1e4])
def test_many_rows(cap):
    """Rows that are not cut into pieces."""
    x, t = _randn(1500, 3001, seed=42), _targets(1500, 3001)
    x[::3] -= 3 * cap
    out = _ops().token_logprobs(x, t, softcap=cap)
    z, lp, chosen, ent, _, _ = _exact(x, t, cap, 0)
    zmax = z.abs().amax(-1)
    e = _errors(cap, 3001, zmax)
    assert bool(((out.logprobs.double() - chosen).abs()
                 <= e + 8 * U * (zmax + chosen.abs())).all())
    spread = (lp.exp() * (z - z.amax(-1, keepdim=True)).abs()).sum(-1)
    assert bool(((out.entropy.double() - ent).abs()
                 <= (2 * e + 16 * U) * (1 + spread) + 8 * U * zmax).all())


@pytest.mark.parametrize("cap", [1.0, 50.0, 100.0, 1e3])
def test_infinite_logits(cap):
    """The cap brings them back into range; NaN stays."""
    x, t = _randn(4, 200, seed=43), torch.tensor([3, 3, 4, 5], device=DEV)
    x[0, 3], x[1, 3], x[2] = math.inf, -math.inf, -math.inf
    x[3, 9] = math.nan
    out = _ops().token_logprobs(x, t, softcap=cap)
    z, lp, chosen, ent, _, _ = _exact(x, t, cap, 0)
    e = _errors(cap, 200, z.abs().amax(-1)) + 16 * U * cap
    assert bool(((out.logprobs.double() - chosen).abs() <= e)[:3].all())
    assert bool(out.logprobs[3].isnan()) and bool(out.entropy[3].isnan())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [37, 50257])
@pytest.mark.parametrize("cap", CAPS[1:])
def test_gradient(cap, V, dtype):
    x, t = _rows(V, dtype)
    x.requires_grad_(True)
    g_lp, g_ent, g_top = _grads(6, 3, 44)
    out = _ops().token_logprobs(x, t, top_k=3, softcap=cap)
    (got,) = torch.autograd.grad(list(out[:3]), [x], [g_lp, g_ent, g_top])
    y = x.detach().double().requires_grad_(True)
    z, lp, chosen, ent, top, ids = _exact(y, t, cap, 3)
    (want,) = torch.autograd.grad([chosen, ent, top], [y], [g.double() for g in
                                                            (g_lp, g_ent, g_top)])
    with torch.no_grad():
        p = lp.exp()
        total = g_lp.double().abs() + g_top.double().abs().sum(1)
        size = p * (total[:, None] + g_ent.double().abs()[:, None] * (
            lp.abs() + ent.abs()[:, None] + 1))
        hit = torch.zeros_like(size).scatter_(1, t[:, None], g_lp.double().abs()[:, None])
        hit.scatter_add_(1, ids, g_top.double().abs())
        zmax = z.abs().amax(1, keepdim=True)
        rel = _errors(cap, V, zmax) * 4 + 16 * U * (zmax + 1)
        bound = rel * (size + hit) + (2.0 ** -8 * want.abs() if dtype == BF else 0) + 1e-37
        err = (got.double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


def test_gradient_against_differences():
    """Central differences of the float32 forward with a cap of 100: a step's own error is
    eps^2 of a third derivative of order one, and some roundings of z over eps."""
    N, V, k, eps = 4, 30, 2, 0.02
    x, t = _randn(N, V, seed=45, scale=1.5), _targets(N, V)
    x[:, 5], x[:, 6] = 9.0, 10.0  # alternatives that no step reorders
    g = _grads(N, k, 46)

    def f(y):
        o = _ops().token_logprobs(y, t, top_k=k, softcap=100.0)
        return sum((a.double() * b.double()).sum() for a, b in zip(o[:3], g))

    y = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(f(y), [y])
    for i in range(4):
        d = _randn(N, V, seed=50 + i, scale=1.0)
        d /= d.norm()
        diff = (f(x + eps * d) - f(x - eps * d)) / (2 * eps)
        assert abs(float(diff) - float((grad.double() * d.double()).sum())) <= 4 * eps ** 2 + 1e-3
