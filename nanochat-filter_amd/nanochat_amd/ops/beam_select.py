"""A search's selection: the best continuations of a prompt's beams.

Composed of ``tanh``, ``log_softmax``, an addition and ``topk`` over beams times
vocabulary it reads and writes the logits many times in float32.  Here they are read
once in their own dtype.  The reference only samples (``nanochat/engine.py``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from nanochat_amd import _native as N


class BeamSelection(NamedTuple):
    scores: Tensor   # (..., k) fp32, descending
    parents: Tensor  # (..., k) int64: the beam that is continued
    tokens: Tensor   # (..., k) int64: by this token; -1 of a finished beam


def beam_select(logits: Tensor, scores: Tensor, k: int, *, softcap: Optional[float] = None,
                finished: Optional[Tensor] = None) -> BeamSelection:
    """The ``k`` best of scores[b] + log_softmax(z[b])[v] over the beams b and tokens v of
    logits (..., beams, V), float32 or bfloat16 (rows may be strided, as a slice that cuts
    off a padded vocabulary is), and scores (..., beams) float32; with ``softcap`` c, z is
    c tanh(logits / c).  In descending order, NaN above all; equal ones by beam, in a beam
    by logit and then token.  Where a beam's score or z is -inf so is the continuation's.

    A beam that is ``finished`` ((..., beams) bool) has one continuation, itself: its score,
    and the token -1.  (Where there are fewer than k, others of score -inf follow; such of
    finished beams have the token -1.)  k is at most 64, or the vocabulary where that is less,
    which times the beams is at most 1,024.  No gradient.

    Scores are compared in float64, with rows' sums of exponentials that were added up in float32:
    off by some 2^-24 of them, of caps up to 64 also by some 2^-23 of the cap.  Continuations
    nearer to each other than that may change places."""
    cap = 0.0 if softcap is None else float(softcap)
    if softcap is not None and not cap > 0.0:
        raise ValueError(f"softcap must be positive and finite, got {softcap}")
    args = (logits, scores, k, cap, finished)
    got = None if torch.compiler.is_compiling() else N.torch_ext().beam_select(*args)
    return BeamSelection(*(_select_op(*args) if got is None else got))


# (torch.compile, tracing, modes, transforms)
@torch.library.custom_op("nanochat_amd::beam_select", mutates_args=())
def _select_op(logits: Tensor, scores: Tensor, k: int, softcap: float,
               finished: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    return N.done(N.torch_ext().beam_select(logits, scores, k, softcap, finished))


@_select_op.register_fake
def _(logits, scores, k, softcap, finished):
    shape = (*scores.shape[:-1], k)
    return (scores.new_empty(shape), scores.new_empty(shape, dtype=torch.int64),
            scores.new_empty(shape, dtype=torch.int64))
