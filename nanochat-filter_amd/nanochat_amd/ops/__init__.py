"""Op registrations of the LTV path (reference: ``nanochat/ops/__init__.py``).

Importing this package defines the ``nanochat_cuda`` ops of the reference path
and the ``nanochat_amd`` fast-path and serving ops.  The native library is loaded lazily on
the first call, so importing works on a machine without a GPU.
"""

from nanochat_amd.ops import ltv_cuda_ops  # noqa: F401
from nanochat_amd.ops import ltv_hm_fast  # noqa: F401
from nanochat_amd.ops.beam_select import BeamSelection, beam_select  # noqa: F401
from nanochat_amd.ops.paged_cache import (  # noqa: F401
    fp4_row_bytes,
    paged_attention,
    paged_cache_append,
    paged_cache_compact,
    paged_cache_copy,
    paged_cache_fork,
    paged_cache_free,
    paged_cache_read,
    paged_cache_reorder,
    paged_cache_reserve,
    paged_rotary_append,
)
from nanochat_amd.ops.token_logprobs import TokenLogprobs, token_logprobs  # noqa: F401
