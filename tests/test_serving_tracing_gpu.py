"""The serving operators where something looks on: tracers, dispatch modes, fake tensors,
transforms, tangents, tensors that are views of a negation."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from paged_test_utils import Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    import nanochat_amd.ops as ops

    return ops


def _rows(seed, *shape):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * 3,
            torch.randint(0, shape[-1], shape[:-1], generator=g, device=DEV))


def _logprobs(x, t):
    o = _ops().token_logprobs(x, t, top_k=3, softcap=15.0)
    return o.logprobs, o.entropy, o.top_logprobs, o.top_ids


def _equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


class _Step:
    """A step of a cache as a function of its new tokens."""

    def __init__(self):
        self.c = Cache([40, 17], 2, 64, 16, torch.bfloat16, 3)

    def tokens(self, seed):
        g = torch.Generator(DEV).manual_seed(seed)
        return tuple(torch.randn(2, 1, n, 64, generator=g, device=DEV).bfloat16()
                     for n in (4, 2, 2))

    def __call__(self, q, k, v):
        c = self.c
        _ops().paged_cache_append(k, v, c.k, c.v, c.table, c.lens)
        return _ops().paged_attention(q, c.k, c.v, c.table, c.lens)


def test_jit_trace():
    x, t = _rows(1, 6, 300)
    traced = torch.jit.trace(_logprobs, (x, t), check_trace=False)
    for seed in (1, 2):
        x, t = _rows(seed, 6, 300)
        assert _equal(traced(x, t), _logprobs(x, t))
    step = _Step()
    traced = torch.jit.trace(lambda q, k, v: step(q, k, v), step.tokens(1), check_trace=False)
    got = traced(*step.tokens(2))
    pages = step.c.k.clone(), step.c.v.clone()
    step(*step.tokens(3))
    assert not torch.equal(step.c.k, pages[0])
    assert torch.equal(got, step(*step.tokens(2)))
    assert torch.equal(step.c.k, pages[0]) and torch.equal(step.c.v, pages[1])


def test_jit_trace_of_the_pages():
    c = Cache([40, 17], 2, 64, 16, torch.bfloat16, 4, spare=6, width=6)
    refs = torch.bincount(c.table[c.table >= 0], minlength=c.P).int()
    one, two = (torch.tensor([i], dtype=torch.int32, device=DEV) for i in (0, 1))

    def steps(table, lens, refs, k, v):
        ops = _ops()
        ops.paged_cache_free(table, lens, refs, two)
        ops.paged_cache_fork(table, lens, refs, one, two)
        status = ops.paged_cache_reserve(table, lens, refs, two, one + 5, k, v)
        ops.paged_cache_copy(k, v, one + 2, two + 2)
        return status, ops.paged_cache_compact(table, refs, k, v)

    def state():
        return [x.clone() for x in (c.table, c.lens, refs, c.k, c.v)]

    a, b, unused = state(), state(), state()
    traced = torch.jit.trace(steps, tuple(unused), check_trace=False)
    want, got = steps(*a), traced(*b)
    assert _equal(want, got) and _equal(a, b)


def test_make_fx():
    from torch.fx.experimental.proxy_tensor import make_fx

    graph = make_fx(_logprobs)(*_rows(1, 6, 300))
    assert any("token_logprobs" in str(n.target) for n in graph.graph.nodes)
    x, t = _rows(2, 6, 300)
    assert _equal(graph(x, t), _logprobs(x, t))


def test_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    step = _Step()
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        x, t = (mode.from_tensor(v) for v in _rows(1, 6, 300))
        lp, ent, top, ids = _logprobs(x, t)
        assert lp.shape == ent.shape == (6,) and top.shape == ids.shape == (6, 3)
        q = mode.from_tensor(step.tokens(1)[0])
        assert step(*(mode.from_tensor(v) for v in step.tokens(1))).shape == q.shape


def test_dispatch_mode():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x, t = _rows(1, 6, 300)
    want = _logprobs(x, t)
    step = _Step()
    out = step(*step.tokens(1))
    tokens = step.tokens(1)
    with Names() as names:
        lp, y = _logprobs(x, t), step(*tokens)
    assert _equal(lp, want) and torch.equal(y, out)
    for op in ("token_logprobs", "paged_cache_append", "paged_attention"):
        assert any(f"nanochat_amd.{op}" in n for n in names.seen), names.seen


def test_vmap():
    x, t = _rows(1, 4, 6, 300)
    assert _equal(torch.vmap(_logprobs)(x, t), _logprobs(x, t))


def test_negated_views():
    x, t = _rows(1, 6, 300)
    assert _equal(_logprobs(torch._neg_view(x), t), _logprobs(-x, t))
    step = _Step()
    q, k, v = step.tokens(1)
    assert torch.equal(step(torch._neg_view(q), torch._neg_view(k), v), step(-q, -k, v))


def test_tangents_are_refused():
    x, t = _rows(1, 6, 300)
    step = _Step()
    with fwAD.dual_level():
        for y in (x, x.clone().requires_grad_(True)):
            with pytest.raises(RuntimeError):
                _logprobs(fwAD.make_dual(y, torch.ones_like(x)), t)
        for i in range(3):
            new = list(step.tokens(1))
            new[i] = fwAD.make_dual(new[i], torch.ones_like(new[i]))
            with pytest.raises(RuntimeError, match="tangent"):
                step(*new)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda y: _logprobs(y, t)[0], (x,), (torch.ones_like(x),))
    # a gradient with a tangent, too
    y = x.clone().requires_grad_(True)
    lp = _logprobs(y, t)[0]
    with fwAD.dual_level():
        g = fwAD.make_dual(torch.ones_like(lp), torch.ones_like(lp))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(lp, [y], [g])


def test_traced_gradient():
    """Of a traced function of logits that require one."""
    x, t = _rows(1, 6, 300)

    def loss(x):
        return _ops().token_logprobs(x * 1.0, t, softcap=15.0).logprobs.sum()

    traced = torch.jit.trace(loss, (x.clone().requires_grad_(True),), check_trace=False)
    y, z = (_rows(2, 6, 300)[0].requires_grad_(True) for _ in range(2))
    (a,), (b,) = torch.autograd.grad(traced(y), [y]), torch.autograd.grad(loss(z), [z])
    assert torch.equal(a, b)
