"""Log probabilities of given tokens, entropy, alternatives and the logits' gradient
against float64, element by element."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _randn(*shape, seed=0, scale=3.0, dtype=F32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _targets(N, V, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000)
    return torch.randint(0, V, (N,), generator=g, device=DEV)


def _exact(x, targets, cap, k):
    """float64 (z, lp of every token, logprobs, entropy, alternatives' lp, their ids)."""
    x = x.double()
    z = cap * torch.tanh(x / cap) if cap else x
    lp = z - torch.logsumexp(z, -1, keepdim=True)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    ok = (targets >= 0) & (targets < x.shape[-1])
    t = targets.clamp(0, x.shape[-1] - 1)
    chosen = torch.where(ok, lp.gather(-1, t[..., None])[..., 0], torch.zeros_like(ent))
    key = torch.where(x.isnan(), torch.full_like(x, math.inf), x)
    # (a NaN goes before +inf: sorted by itself, stably, first)
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    nan_first = torch.argsort(x.isnan().gather(-1, order).int(), dim=-1, descending=True,
                              stable=True)
    ids = order.gather(-1, nan_first)[..., :k]
    return z, lp, chosen, ent, lp.gather(-1, ids), ids


def _noise(V, cap):
    """Relative error of a sum over the vocabulary by at least 64 partial sums, each
    term's exponential with an argument off by a few roundings; a cap's tanh is off by
    a few roundings of the cap."""
    return U * (V / 64 + 64) + 4 * U * cap


def _check_forward(x, targets, cap, k, out):
    V = x.shape[-1]
    z, lp, chosen, ent, top, ids = _exact(x, targets, cap, k)
    e = _noise(V, cap)
    zmax = z.abs().amax(-1)
    err = (out.logprobs.double() - chosen).abs()
    bound = e + 8 * U * (zmax + chosen.abs())
    assert bool((err <= bound).all()), float((err / bound).max())
    spread = (lp.exp() * (z - z.amax(-1, keepdim=True)).abs()).sum(-1)
    err = (out.entropy.double() - ent).abs()
    bound = (2 * e + 16 * U) * (1 + spread) + 8 * U * zmax
    assert bool((err <= bound).all()), float((err / bound).max())
    if k == 0:
        assert out.top_logprobs is None and out.top_ids is None
        return
    assert torch.equal(out.top_ids, ids)
    err = (out.top_logprobs.double() - top).abs()
    assert bool((err <= e + 8 * U * (zmax[..., None] + top.abs())).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [None, 15.0])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 2, 2), (5, 63, 5), (4, 64, 64), (7, 65, 1),
                                   (2, 1000, 20), (3, 4097, 64), (33, 8191, 0), (1, 50257, 20),
                                   (2, 65536, 5), (2, 131072, 32), (1, 300001, 64)])
def test_forward(N, V, k, cap, dtype):
    x, t = _randn(N, V, seed=N + V, dtype=dtype), _targets(N, V)
    _check_forward(x, t, cap or 0.0, k, _ops().token_logprobs(x, t, top_k=k, softcap=cap))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_rows(dtype):
    x, t = _randn(3001, 777, seed=1, dtype=dtype), _targets(3001, 777)
    _check_forward(x, t, 15.0, 5, _ops().token_logprobs(x, t, top_k=5, softcap=15.0))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_shapes_strides_and_alignment(dtype):
    """(B, T, V), a cut-off padded vocabulary, a row in the middle of an allocation, rows
    at odd elements, no contiguous last axis; int32 targets."""
    x = _randn(2, 5, 130, seed=2, dtype=dtype)
    t = _targets(10, 101).view(2, 5)
    want = _ops().token_logprobs(x[..., :101].contiguous(), t, top_k=3, softcap=15.0)
    assert want.logprobs.shape == (2, 5) and want.top_ids.shape == (2, 5, 3)
    odd = torch.empty(2 * 5 * 101 + 1, dtype=dtype, device=DEV)[1:].view(2, 5, 101)
    odd.copy_(x[..., :101])
    last = torch.empty(2, 5, 202, dtype=dtype, device=DEV)[..., ::2].copy_(x[..., :101])
    for y, tt in ((x[..., :101], t), (odd, t), (last, t), (x[..., :101], t.int()),
                  (x[..., :101].transpose(0, 1).contiguous().transpose(0, 1), t)):
        got = _ops().token_logprobs(y, tt, top_k=3, softcap=15.0)
        assert torch.equal(got.top_ids, want.top_ids)
        # (a row's terms may be summed in another order where it starts elsewhere)
        for a, b in zip(got[:3], want[:3]):
            assert float((a - b).abs().max()) <= 4e-6
    one = _ops().token_logprobs(x[0, 0], t[0, 0])
    assert one.logprobs.shape == () and one.entropy.shape == ()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties_and_orders(dtype):
    """Equal logits by index; rows that rise, fall, are constant, or have their largest
    entries side by side."""
    V = 70001
    up = torch.linspace(-20, 20, V, device=DEV)
    const = torch.full((V,), 1.5, device=DEV)
    few = (torch.arange(V, device=DEV) % 7).float()
    block = torch.zeros(V, device=DEV)
    block[40000:40100] = torch.arange(100, device=DEV).float()
    zeros = torch.zeros(V, device=DEV)
    zeros[::2] = -0.0
    tail = torch.zeros(V, device=DEV)
    tail[-40:] = 3.0
    x = torch.stack([up, up.flip(0), const, few, block, zeros, tail]).to(dtype)
    t = _targets(len(x), V)
    for k in (1, 5, 64):
        _check_forward(x, t, 0.0, k, _ops().token_logprobs(x, t, top_k=k))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_infinite_and_lowest_logits(dtype):
    """Masked vocabulary entries (-inf, the type's lowest), all but one masked, a masked
    target, +inf and NaN rows."""
    V = 5000
    x = _randn(7, V, seed=3, dtype=dtype)
    x[0, ::3] = -math.inf
    x[1, :] = -math.inf
    x[1, 77] = 2.0
    x[2, 1:] = torch.finfo(dtype).min
    x[3, 100:4000] = torch.finfo(dtype).min
    x[4, 10] = math.inf
    x[5, 20] = math.nan
    x[6, :] = -math.inf
    t = torch.tensor([0, 77, 0, 200, 4, 4, 4], device=DEV)
    out = _ops().token_logprobs(x, t, top_k=4)
    assert float(out.logprobs[0]) == -math.inf
    assert float(out.logprobs[1]) == 0.0 and float(out.entropy[1]) == 0.0
    assert float(out.logprobs[2]) == 0.0 and float(out.entropy[2]) == 0.0
    keep = torch.tensor([0, 2, 3], device=DEV)
    z, lp, chosen, ent, top, ids = _exact(x, t, 0.0, 4)
    assert bool((out.entropy[keep].double() - ent[keep]).abs().max() <= 1e-5)
    assert torch.equal(out.top_ids, ids)
    assert bool(out.logprobs[4:].isnan().all()) and bool(out.entropy[4:].isnan().all())
    # the cap brings infinities back into range
    _check_forward(x[:5], t[:5], 15.0, 4, _ops().token_logprobs(x[:5], t[:5], top_k=4,
                                                                softcap=15.0))
    assert bool(_ops().token_logprobs(x[5:6], t[5:6], softcap=15.0).logprobs.isnan().all())


@pytest.mark.parametrize("cap", [None, 15.0])
def test_large_logits(cap):
    """Sums do not overflow, whatever the rows' scale and offset."""
    x = _randn(6, 3000, seed=4) * torch.tensor([1e-6, 1.0, 30.0, 1e3, 1e30, 1.0],
                                               device=DEV)[:, None]
    x[5] += 1e4
    t = _targets(6, 3000)
    _check_forward(x, t, cap or 0.0, 0, _ops().token_logprobs(x, t, softcap=cap))


def test_targets_outside_the_vocabulary():
    x = _randn(5, 100, seed=5).requires_grad_(True)
    t = torch.tensor([-1, 100, 3, -100, 2 ** 40], device=DEV)
    out = _ops().token_logprobs(x, t)
    assert out.logprobs[[0, 1, 3, 4]].tolist() == [0.0] * 4 and float(out.logprobs[2].detach()) < 0
    (g,) = torch.autograd.grad(out.logprobs.sum(), [x])
    assert bool((g[[0, 1, 3, 4]] == 0).all()) and bool((g[2] != 0).any())


def _grads(N, k, seed):
    return (_randn(N, seed=seed, scale=1.0), _randn(N, seed=seed + 1, scale=0.3),
            _randn(N, k, seed=seed + 2, scale=0.5) if k else None)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [None, 15.0])
@pytest.mark.parametrize("N,V,pad,k", [(1, 1, 1, 1), (5, 63, 64, 5), (4, 100, 100, 64),
                                       (3, 4097, 4160, 20), (2, 50257, 50304, 0),
                                       (2, 65536, 65536, 3), (700, 333, 333, 2)])
def test_gradient(N, V, pad, k, cap, dtype):
    x = _randn(N, pad, seed=N + V, dtype=dtype)[:, :V].detach().requires_grad_(True)
    t = _targets(N, V)
    if N > 2:
        t[1] = -1
    if k:  # an alternative that is the target, too
        t[0] = int(x[0].float().argmax())
    g_lp, g_ent, g_top = _grads(N, k, 7)
    out = _ops().token_logprobs(x, t, top_k=k, softcap=cap)
    outs, gs = list(out[:2]) + ([out.top_logprobs] if k else []), [g_lp, g_ent] + (
        [g_top] if k else [])
    (got,) = torch.autograd.grad(outs, [x], gs)
    assert got.shape == x.shape and got.dtype == x.dtype
    x64 = x.detach().double().requires_grad_(True)
    z, lp, chosen, ent, top, ids = _exact(x64, t, cap or 0.0, k)
    (want,) = torch.autograd.grad([chosen, ent] + ([top] if k else []), [x64],
                                  [v.double() for v in gs])
    # every term's relative error; the cap's factor 1 - (z / cap)^2 has an absolute one
    with torch.no_grad():
        p = lp.exp()
        total = g_lp.double().abs() + (g_top.double().abs().sum(1) if k else 0)
        size = p * (total[:, None] + g_ent.double().abs()[:, None] * (
            lp.abs() + ent.abs()[:, None] + 1))
        hit = torch.zeros_like(size).scatter_(1, t.clamp(min=0)[:, None],
                                              g_lp.double().abs()[:, None])
        if k:
            hit.scatter_add_(1, ids, g_top.double().abs())
        rel = _noise(V, cap or 0.0) * 4 + 16 * U * (z.abs().amax(1, keepdim=True) + 1)
        bound = rel * (size + hit) + (2.0 ** -8 * want.abs() if dtype == BF else 0) + 1e-37
        err = (got.double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("cap,dtype", [(15.0, BF), (None, F32)])
def test_gradient_of_many_long_rows(cap, dtype):
    """Rows of more than 64 KiB that are not cut into pieces."""
    test_gradient(4097, 33001, 33024, 2, cap, dtype)


def test_gradient_against_differences():
    """Directional derivatives by central differences of the float32 forward; their own
    error is eps^2 of a third derivative of order one, and 10 roundings over eps."""
    N, V, k, eps = 6, 40, 3, 0.02
    x, t = _randn(N, V, seed=8, scale=1.5), _targets(N, V)
    x[:, 5:8] += 6.0  # alternatives that no step reorders
    x += torch.arange(V, device=DEV) * 0.0
    x[:, 5], x[:, 6], x[:, 7] = 8.0, 9.0, 10.0
    g = _grads(N, k, 9)

    def f(y):
        o = _ops().token_logprobs(y, t, top_k=k, softcap=15.0)
        return sum((a.double() * b.double()).sum() for a, b in zip(o[:3], g))

    y = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(f(y), [y])
    for i in range(4):
        d = _randn(N, V, seed=20 + i, scale=1.0)
        d /= d.norm()
        diff = (f(x + eps * d) - f(x - eps * d)) / (2 * eps)
        assert abs(float(diff) - float((grad.double() * d.double()).sum())) <= 4 * eps ** 2 + 1e-3


def test_gradient_of_some_outputs():
    """Only one output used, the others without a gradient; a scalar expanded."""
    x, t = _randn(4, 500, seed=10).requires_grad_(True), _targets(4, 500)
    y = x.detach().double().requires_grad_(True)
    z, lp, chosen, ent, top, ids = _exact(y, t, 0.0, 2)
    out = _ops().token_logprobs(x, t, top_k=2)
    for a, b in ((out.logprobs, chosen), (out.entropy, ent), (out.top_logprobs, top)):
        (got,) = torch.autograd.grad(a.sum(), [x], retain_graph=True)
        (want,) = torch.autograd.grad(b.sum(), [y], retain_graph=True)
        assert float((got.double() - want).abs().max()) <= 1e-5
    assert not out.top_ids.requires_grad


def test_second_gradient_is_refused():
    x, t = _randn(3, 40, seed=11).requires_grad_(True), _targets(3, 40)
    lp = _ops().token_logprobs(x, t).logprobs.sum()
    (want,) = torch.autograd.grad(lp, [x], retain_graph=True)
    (got,) = torch.autograd.grad(lp, [x], create_graph=True)
    assert torch.equal(got.detach(), want)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(got.square().sum(), [x])


def test_gradient_with_masked_entries():
    """-inf and lowest entries have probability 0 and gradient 0, not NaN."""
    for dtype in (BF, F32):
        x = _randn(2, 300, seed=11, dtype=dtype)
        x[0, ::2] = -math.inf
        x[1, ::2] = torch.finfo(dtype).min
        x.requires_grad_(True)
        out = _ops().token_logprobs(x, torch.tensor([1, 3], device=DEV), top_k=3)
        (g,) = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum()
                                   + out.top_logprobs.sum(), [x])
        assert bool(g.isfinite().all()) and bool((g[:, ::2] == 0).all())


def test_training_step_through_a_head():
    """The loss of the GPT harness from these log probabilities: cross entropy."""
    import torch.nn.functional as F

    w = _randn(200, 64, seed=12, scale=0.2).requires_grad_(True)
    h, t = _randn(32, 64, seed=13, scale=1.0), _targets(32, 200)
    t[3] = -1
    logits = h @ w.t()
    loss = -_ops().token_logprobs(logits, t, softcap=15.0).logprobs.sum() / (t >= 0).sum()
    (got,) = torch.autograd.grad(loss, [w])
    w64 = w.detach().double().requires_grad_(True)
    z = 15 * torch.tanh(h.double() @ w64.t() / 15)
    ref = F.cross_entropy(z, t, ignore_index=-1)
    (want,) = torch.autograd.grad(ref, [w64])
    assert abs(float(loss) - float(ref)) <= 1e-5
    assert float((got.double() - want).abs().max()) <= 1e-5


@pytest.mark.parametrize("grad", [False, True])
def test_repeats_are_bitwise_equal(grad):
    x, t = _randn(9, 50257, seed=14, dtype=BF).requires_grad_(grad), _targets(9, 50257)

    def call():
        o = _ops().token_logprobs(x, t, top_k=10, softcap=15.0)
        if not grad:
            return o
        return [*o, *torch.autograd.grad(o.logprobs.sum() + o.entropy.sum(), [x])]

    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))


def test_other_stream():
    x, t = _randn(64, 10000, seed=15), _targets(64, 10000)
    want = _ops().token_logprobs(x, t, top_k=4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _ops().token_logprobs(x, t, top_k=4)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_replays_in_a_graph():
    x, t = _randn(8, 5000, seed=16), _targets(8, 5000)

    def call():
        return _ops().token_logprobs(x, t, top_k=4, softcap=15.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        x.copy_(_randn(8, 5000, seed=30 + i))
        t.copy_(_targets(8, 5000, seed=i))
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_under_compile():
    def f(x, t):
        o = _ops().token_logprobs(x * 1.0, t, top_k=3, softcap=15.0)
        return o.logprobs.sum() + 0.1 * o.entropy.sum() + o.top_logprobs.sum(), o.top_ids

    x, t = _randn(6, 300, seed=17).requires_grad_(True), _targets(6, 300)
    a, ids = f(x, t)
    b, jds = torch.compile(f, backend="aot_eager")(x, t)
    assert torch.equal(ids, jds) and torch.equal(a, b)
    (ga,), (gb,) = torch.autograd.grad(a, [x]), torch.autograd.grad(b, [x])
    assert torch.equal(ga, gb)


def test_no_rows():
    x = torch.zeros(0, 50, device=DEV, requires_grad=True)
    out = _ops().token_logprobs(x, torch.zeros(0, dtype=torch.int64, device=DEV), top_k=3)
    assert out.logprobs.shape == (0,) and out.top_ids.shape == (0, 3)
    (g,) = torch.autograd.grad(out.logprobs.sum(), [x])
    assert g.shape == (0, 50)


def test_refusals():
    ops = _ops()
    x, t = _randn(4, 50), _targets(4, 50)
    for bad in (dict(top_k=51), dict(top_k=65), dict(top_k=-1), dict(softcap=0.0),
                dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=math.nan)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, t, **bad)
    wide = _randn(2, 100)
    with pytest.raises(ValueError):
        ops.token_logprobs(wide, t[:2], top_k=65)
    for a, b in ((x, t[:3]), (x, t[:, None]), (x[:, :0], t), (x[0, 0], t[0])):
        with pytest.raises(ValueError):
            ops.token_logprobs(a, b)
    for a, b in ((x.half(), t), (x.double(), t), (x, t.float())):
        with pytest.raises(TypeError):
            ops.token_logprobs(a, b)
    for a, b in ((x.cpu(), t), (x, t.cpu())):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(a, b)
