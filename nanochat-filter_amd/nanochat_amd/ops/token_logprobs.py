"""Log probabilities of given tokens, with entropy and top alternatives, and their
gradient for the logits.

What scoring, sampling displays and policy gradients take from a model's logits;
composed of ``tanh``, ``log_softmax``, ``gather`` and ``topk`` it reads and writes the
(rows, vocabulary) array many times in float32.  Here the logits are read once (once
more for the gradient) in their own dtype.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from nanochat_amd import _native as N


class TokenLogprobs(NamedTuple):
    logprobs: Tensor                # (...) fp32
    entropy: Tensor                 # (...) fp32, in nats
    top_logprobs: Optional[Tensor]  # (..., top_k) fp32, descending; None for top_k = 0
    top_ids: Optional[Tensor]       # (..., top_k) int64


def token_logprobs(logits: Tensor, targets: Tensor, *, top_k: int = 0,
                   softcap: Optional[float] = None) -> TokenLogprobs:
    """logits (..., V) float32 or bfloat16 (rows may be strided, as a slice that cuts off
    a padded vocabulary is), targets (...) integers.  With ``softcap`` c the
    distribution is that of c tanh(logits / c) (the model's capped logits).

    A target outside [0, V) (-1, the ignored index of the training loss) has log
    probability 0 and no gradient.  The alternatives are the ``top_k`` <= 64 largest
    logits in descending order, equal ones by ascending index, NaN above all.  Sums are
    in float32.  Differentiable once: logprobs, entropy and top_logprobs."""
    cap = 0.0 if softcap is None else float(softcap)
    if softcap is not None and not cap > 0.0:
        raise ValueError(f"softcap must be positive and finite, got {softcap}")
    got = None if torch.compiler.is_compiling() else N.torch_ext().token_logprobs(
        logits, targets, top_k, cap)
    if got is None:  # (as the cache's functions)
        got = _logprobs_op(logits, targets, top_k, cap)[:4]
    lp, ent, top, ids = got
    if top_k == 0:
        return TokenLogprobs(lp, ent, None, None)
    return TokenLogprobs(lp, ent, top, ids)


# ---------------------------------------------------------------------------
# library ops (torch.compile, tracing, modes, transforms)
# ---------------------------------------------------------------------------
@torch.library.custom_op("nanochat_amd::token_logprobs", mutates_args=())
def _logprobs_op(logits: Tensor, targets: Tensor, top_k: int,
                 softcap: float) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    return N.done(N.torch_ext().token_logprobs_forward(logits, targets, top_k, softcap))


@_logprobs_op.register_fake
def _(logits, targets, top_k, softcap):
    def f(*shape, dtype=torch.float32):
        return torch.empty(*targets.shape, *shape, dtype=dtype, device=logits.device)

    return f(), f(), f(top_k), f(top_k, dtype=torch.int64), f()


@torch.library.custom_op("nanochat_amd::token_logprobs_backward", mutates_args=())
def _logprobs_backward_op(logits: Tensor, targets: Tensor, lse: Tensor, entropy: Tensor,
                          top_ids: Tensor, g_logprobs: Optional[Tensor],
                          g_entropy: Optional[Tensor], g_top: Optional[Tensor],
                          softcap: float) -> Tensor:
    return N.done(N.torch_ext().token_logprobs_backward(logits, targets, lse, entropy, top_ids,
                                                        g_logprobs, g_entropy, g_top, softcap))


@_logprobs_backward_op.register_fake
def _(logits, targets, lse, entropy, top_ids, g_logprobs, g_entropy, g_top, softcap):
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _setup(ctx, inputs, output):
    logits, targets, _, ctx.softcap = inputs
    _, entropy, _, ids, lse = output
    ctx.save_for_backward(logits, targets, lse, entropy, ids)
    ctx.mark_non_differentiable(ids, lse)
    ctx.set_materialize_grads(False)


def _backward(ctx, g_lp, g_ent, g_top, _g_ids, _g_lse):
    if g_lp is None and g_ent is None and g_top is None:
        return None, None, None, None
    logits, targets, lse, entropy, ids = ctx.saved_tensors
    return (_logprobs_backward_op(logits, targets, lse, entropy, ids, g_lp, g_ent, g_top,
                                  ctx.softcap), None, None, None)


_logprobs_op.register_autograd(_backward, setup_context=_setup)
