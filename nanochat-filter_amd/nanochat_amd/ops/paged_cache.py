"""Attention over a paged cache, and the cache's pages.

One layer's cache is a pair of page arrays ``k_pages``, ``v_pages``
(P, kv heads, page size, head_dim); the layers of a model share the bookkeeping:

  page_table (S, W) int32 -- the pages of slot s in the order of its tokens, -1
                             (or any id outside [0, P)) where there is none
  seq_lens   (S)    int32 -- tokens of each slot, the ones being computed included
  ref_counts (P)    int32 -- how many slots hold a page; 0: free

All of it lives on the GPU and is read and written there in stream order: no call
waits for the device, and a step can be captured in a HIP graph.  A step of a
serving loop is

    paged_cache_reserve(...)                 # once: room for the new tokens
    for each layer:
        paged_cache_append(k, v, ...)        # their keys and values into the pages
        y = paged_attention(q, ...)          # what they attend to

``PagedKVCache`` (``nanochat_amd.paged_kv_cache``) keeps these tensors for a model.

New tokens come as (B, T, heads, head_dim) tensors, T for each sequence, or with
``starts`` (B + 1 ascending ints) as (N, heads, head_dim) tensors with sequence i's
tokens in rows starts[i] .. starts[i + 1], so that one call takes a batch in which
some sequences decode and the prompts of others come in chunks.  Sequence i is slot
``slots[i]`` (default: slot i).  ``max_new`` and ``max_len`` are what the caller knows
of the longest chunk and sequence; they choose launch shapes, and past 10^11 operations
how probabilities are rounded, not which keys are read.

The reference's cache is contiguous (``nanochat/kv_cache.py`` ``insert_kv``) and is
copied whole to start several samples from one prompt (``prefill``).

In eager mode the functions go straight to the native host path; under
``torch.compile``, and for what that path leaves (tensor subclasses, tracing, modes,
transforms), to the ``nanochat_amd`` library ops of the same names.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from nanochat_amd import _native as N


def paged_cache_append(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
                       seq_lens: Tensor, *, slots: Optional[Tensor] = None,
                       starts: Optional[Tensor] = None, max_new: Optional[int] = None) -> None:
    """Write the new tokens' keys and values, the last n tokens of each sequence's
    ``seq_lens``, into their pages.  Tokens at negative positions or of pages that the
    table does not hold are dropped."""
    args = (k, v, k_pages, v_pages, page_table, seq_lens, slots, starts, max_new)
    if torch.compiler.is_compiling() or not N.torch_ext().paged_cache_append(*args):
        _append_op(*args)


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
                    seq_lens: Tensor, *, slots: Optional[Tensor] = None,
                    starts: Optional[Tensor] = None, max_new: Optional[int] = None,
                    max_len: Optional[int] = None, scale: Optional[float] = None,
                    return_lse: bool = False):
    """softmax(scale q k) v of each new token over its sequence's cached tokens up to
    itself: q's shape, contiguous.  Query heads share the kv heads in equal groups;
    ``scale`` > 0 defaults to 1 / sqrt(head_dim).  A token that has nothing to attend to
    gives 0.  With ``return_lse`` also the log of the softmax's denominators (fp32, q's
    shape without head_dim; -inf where there is nothing), which joins attention over
    several caches.  float32 or bfloat16, head_dim a multiple of 8 up to 128; inference
    only."""
    args = (q, k_pages, v_pages, page_table, seq_lens, slots, starts, max_new, max_len, scale)
    got = None if torch.compiler.is_compiling() else N.torch_ext().paged_attention(*args,
                                                                                   return_lse)
    out, lse = _attention_op(*args) if got is None else got
    return (out, lse) if return_lse else out


def paged_cache_reserve(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, slots: Tensor,
                        counts: Tensor, k_pages: Tensor, v_pages: Tensor) -> Tensor:
    """Make room for counts[i] more tokens in slot slots[i]: ``seq_lens`` grows and free
    pages, the lowest first, are put into the table.  A slot whose partly filled last
    page is shared gets a copy of it first (in every layer: the pages are
    ([layers,] P, kv heads, page size, head_dim)).  Slots are distinct.

    Returns an int32 tensor of one element: 0; or, with nothing changed, how many pages
    are missing; or -1 for a slot or count out of range or a sequence longer than its
    table row.  Where it is not 0 there are no new tokens: appending some would overwrite
    the last ones there are.  A caller that does not wait for it passes on
    ``torch.where(status == 0, slots, -1)`` as the slots, which are no sequences then."""
    args = (page_table, seq_lens, ref_counts, slots, counts, k_pages, v_pages)
    got = None if torch.compiler.is_compiling() else N.torch_ext().paged_cache_reserve(*args)
    return _reserve_op(*args) if got is None else got


def paged_cache_fork(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, src: Tensor,
                     dst: Tensor) -> None:
    """Slot dst[i] becomes slot src[i], sharing its pages; what dst held is let go.  No
    dst is another dst or a src (src[i] == dst[i] does nothing)."""
    args = (page_table, seq_lens, ref_counts, src, dst)
    if torch.compiler.is_compiling() or not N.torch_ext().paged_cache_fork(*args):
        _fork_op(*args)


def paged_cache_free(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor,
                     slots: Tensor) -> None:
    """Empty the slots; pages that no other slot holds become free."""
    args = (page_table, seq_lens, ref_counts, slots)
    if torch.compiler.is_compiling() or not N.torch_ext().paged_cache_free(*args):
        _free_op(*args)


def paged_cache_copy(k_pages: Tensor, v_pages: Tensor, src: Tensor, dst: Tensor) -> None:
    """Copy page src[i] to page dst[i], in every layer; entries with an id outside
    [0, P) are skipped.  No dst is another dst or a src."""
    args = (k_pages, v_pages, src, dst)
    if torch.compiler.is_compiling() or not N.torch_ext().paged_cache_copy(*args):
        _copy_op(*args)


def paged_cache_compact(page_table: Tensor, ref_counts: Tensor, k_pages: Tensor,
                        v_pages: Tensor) -> Tensor:
    """Move the pages in use to the lowest ids (those past their number, in order, into
    the holes below it); the table and counts follow.  Returns their number, an int32
    tensor of one element."""
    args = (page_table, ref_counts, k_pages, v_pages)
    got = None if torch.compiler.is_compiling() else N.torch_ext().paged_cache_compact(*args)
    return _compact_op(*args) if got is None else got


# ---------------------------------------------------------------------------
# library ops (torch.compile, tracing, modes, transforms)
# ---------------------------------------------------------------------------
@torch.library.custom_op("nanochat_amd::paged_cache_append", mutates_args=("k_pages", "v_pages"))
def _append_op(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
               seq_lens: Tensor, slots: Optional[Tensor], starts: Optional[Tensor],
               max_new: Optional[int]) -> None:
    N.done(N.torch_ext().paged_cache_append(k, v, k_pages, v_pages, page_table, seq_lens, slots,
                                            starts, max_new))


@_append_op.register_fake
def _(k, v, k_pages, v_pages, page_table, seq_lens, slots, starts, max_new):
    return None


@torch.library.custom_op("nanochat_amd::paged_attention", mutates_args=())
def _attention_op(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
                  seq_lens: Tensor, slots: Optional[Tensor], starts: Optional[Tensor],
                  max_new: Optional[int], max_len: Optional[int],
                  scale: Optional[float]) -> Tuple[Tensor, Tensor]:
    out, lse = N.done(N.torch_ext().paged_attention(q, k_pages, v_pages, page_table, seq_lens,
                                                    slots, starts, max_new, max_len, scale, True))
    return out, lse


@_attention_op.register_fake
def _(q, k_pages, v_pages, page_table, seq_lens, slots, starts, max_new, max_len, scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32)


_STATE = ("page_table", "seq_lens", "ref_counts")


@torch.library.custom_op("nanochat_amd::paged_cache_reserve",
                         mutates_args=(*_STATE, "k_pages", "v_pages"))
def _reserve_op(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, slots: Tensor,
                counts: Tensor, k_pages: Tensor, v_pages: Tensor) -> Tensor:
    return N.done(N.torch_ext().paged_cache_reserve(page_table, seq_lens, ref_counts, slots,
                                                    counts, k_pages, v_pages))


@_reserve_op.register_fake
def _(page_table, seq_lens, ref_counts, slots, counts, k_pages, v_pages):
    return seq_lens.new_empty(1)


@torch.library.custom_op("nanochat_amd::paged_cache_fork", mutates_args=_STATE)
def _fork_op(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, src: Tensor,
             dst: Tensor) -> None:
    N.done(N.torch_ext().paged_cache_fork(page_table, seq_lens, ref_counts, src, dst))


@_fork_op.register_fake
def _(page_table, seq_lens, ref_counts, src, dst):
    return None


@torch.library.custom_op("nanochat_amd::paged_cache_free", mutates_args=_STATE)
def _free_op(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, slots: Tensor) -> None:
    N.done(N.torch_ext().paged_cache_free(page_table, seq_lens, ref_counts, slots))


@_free_op.register_fake
def _(page_table, seq_lens, ref_counts, slots):
    return None


@torch.library.custom_op("nanochat_amd::paged_cache_copy", mutates_args=("k_pages", "v_pages"))
def _copy_op(k_pages: Tensor, v_pages: Tensor, src: Tensor, dst: Tensor) -> None:
    N.done(N.torch_ext().paged_cache_copy(k_pages, v_pages, src, dst))


@_copy_op.register_fake
def _(k_pages, v_pages, src, dst):
    return None


@torch.library.custom_op("nanochat_amd::paged_cache_compact",
                         mutates_args=("page_table", "ref_counts", "k_pages", "v_pages"))
def _compact_op(page_table: Tensor, ref_counts: Tensor, k_pages: Tensor,
                v_pages: Tensor) -> Tensor:
    return N.done(N.torch_ext().paged_cache_compact(page_table, ref_counts, k_pages, v_pages))


@_compact_op.register_fake
def _(page_table, ref_counts, k_pages, v_pages):
    return page_table.new_empty(1)
