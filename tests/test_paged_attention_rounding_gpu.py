"""bfloat16 attention of many keys of like weight: the outputs are off by their own rounding,
not by that of the probabilities."""

from __future__ import annotations

import pytest
import torch

from paged_test_utils import DEV, Cache, attention64

pytestmark = pytest.mark.gpu


def _relative(x, want):
    return float((x.double() - want).norm() / want.norm())


@pytest.mark.parametrize("B,T,NH,NKVH,D,length", [(4, 1, 8, 4, 128, 3000), (2, 3, 6, 6, 64, 5000),
                                                  (1, 40, 4, 2, 128, 2000), (300, 1, 4, 4, 96, 400),
                                                  (1, 200, 2, 2, 72, 900)])
def test_error_is_that_of_the_output(B, T, NH, NKVH, D, length):
    """Values around 0 make an output as small as the sum of its terms' roundings: rounded
    probabilities alone would give an error like the output's own, sqrt(2) of it together.
    Sums in float32 add some 1e-6."""
    import nanochat_amd.ops as ops

    cache = Cache([length] * B, NKVH, D, 16, torch.bfloat16, 50)
    q = (cache.rand(B, T, NH, D) * 0.3).bfloat16()
    got = ops.paged_attention(q, cache.k, cache.v, cache.table, cache.lens, max_len=length)
    some = list(range(0, B, max(1, B // 8)))
    want = torch.stack([o for o, *_ in attention64([q[i] for i in some], cache, some,
                                                   [T] * len(some), D ** -0.5)])
    own = _relative(want.bfloat16(), want)
    assert _relative(got[some], want) <= 1.01 * own + 1e-5
