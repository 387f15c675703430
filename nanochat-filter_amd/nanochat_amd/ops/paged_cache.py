"""Attention over a paged cache, and the cache's pages.

One layer's cache is a pair of page arrays ``k_pages``, ``v_pages``
(P, kv heads, page size, head_dim); the layers of a model share the bookkeeping:

  page_table (S, W) int32 -- the pages of slot s in the order of its tokens, -1
                             (or any id outside [0, P)) where there is none
  seq_lens   (S)    int32 -- tokens of each slot, the ones being computed included
  ref_counts (P)    int32 -- how many slots hold a page; 0: free

Pages may be held in 4 bits: uint8 arrays (P, kv heads, page size,
``fp4_row_bytes(head_dim)``), head_dim 32, 64, 96 or 128 and the page size a multiple of
16, each page and head a dense block.  Of a block the codes come first (page size,
head_dim / 2), the even channel in the low half of a byte, then the scales (head_dim / 32,
page size), one byte for 32 channels of a token.  They stand for code * 2^(scale - 127),
the code's low three bits for 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the fourth for the sign; the
scale 255 for 32 times NaN.  ``paged_cache_append`` and ``paged_rotary_append`` round to
the nearest such value (ties to the even code) with the smallest scale by which no channel
is larger than 7 (6 is the largest code); ``paged_attention`` computes with the values and
``paged_cache_read`` gives them back.  What moves pages moves these as any others.

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
how probabilities are rounded (not over 4-bit pages), not which keys are read.

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


def fp4_row_bytes(head_dim: int) -> int:
    """Bytes that a token's head takes in 4-bit pages: the last size of their arrays."""
    if head_dim not in (32, 64, 96, 128):
        raise ValueError(f"4-bit pages have head_dim 32, 64, 96 or 128, got {head_dim}")
    return head_dim // 2 + head_dim // 32


def paged_rotary_append(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor,
                        k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seq_lens: Tensor,
                        *, slots: Optional[Tensor] = None, starts: Optional[Tensor] = None,
                        max_new: Optional[int] = None,
                        norm_eps: Optional[float] = None) -> Tensor:
    """Rotate the new tokens' queries and keys by their positions, with ``norm_eps`` divide
    each head by sqrt(mean of squares + norm_eps), write keys and values into their pages
    (as ``paged_cache_append``), and return the queries: q's shape, contiguous.

    ``cos`` and ``sin`` (positions, head_dim / 2), float32 or bfloat16, have a row for every
    position that the page table has room for.  The halves of a head are rotated as pairs:
    (x1 cos + x2 sin, x2 cos - x1 sin) at the token's row.  Computed in float64, and only
    then rounded, to q's dtype or to 4 bits.  A token at a negative position gives 0; with
    ``starts``, rows of no sequence are not written.  Inference only.

    The reference rotates and normalises q and k in a dozen launches
    (``nanochat/gpt.py:101-109, 231-236``) before its cache takes them."""
    args = (q, k, v, cos, sin, k_pages, v_pages, page_table, seq_lens, slots, starts, max_new,
            norm_eps)
    got = None if torch.compiler.is_compiling() else N.torch_ext().paged_rotary_append(*args)
    return _rotary_append_op(*args) if got is None else got


def paged_cache_read(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seq_lens: Tensor,
                     tokens: int, *, slots: Optional[Tensor] = None,
                     starts: Optional[Tensor] = None, max_new: Optional[int] = None,
                     dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """What the pages hold of the last ``tokens`` tokens of each sequence, (B, tokens, kv
    heads, head_dim), or, with ``starts``, of as many as it says, (tokens, kv heads,
    head_dim) with ``tokens`` rows in all: what ``paged_cache_append`` was given, rounded if
    the pages have 4 bits.  A token at a negative position or of no page, and a row of no
    sequence, is 0.  ``dtype`` of 4-bit pages is bfloat16 or float32 (both hold the values
    exactly; default bfloat16), else that of the pages."""
    if dtype is None:
        dtype = torch.bfloat16 if k_pages.dtype == torch.uint8 else k_pages.dtype
    args = (k_pages, v_pages, page_table, seq_lens, tokens, slots, starts, max_new, dtype)
    got = None if torch.compiler.is_compiling() else N.torch_ext().paged_cache_read(*args)
    return _read_op(*args) if got is None else got


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
    several caches.  float32 or bfloat16, head_dim a multiple of 8 up to 128, pages of
    that dtype or in 4 bits; inference only."""
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


def paged_cache_reorder(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, slots: Tensor,
                        src: Tensor) -> None:
    """Slot slots[i] becomes what slot src[i] holds before the call, all at once: a search's
    beams follow its selection, in whatever exchange.  A slot may be a src several times, and
    both; pages are shared as by fork, and what no slot holds any more is free.  ``slots`` are
    distinct.

    The reference copies a contiguous cache row by row."""
    args = (page_table, seq_lens, ref_counts, slots, src)
    if torch.compiler.is_compiling() or not N.torch_ext().paged_cache_reorder(*args):
        _reorder_op(*args)


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


@torch.library.custom_op("nanochat_amd::paged_rotary_append", mutates_args=("k_pages", "v_pages"))
def _rotary_append_op(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor, k_pages: Tensor,
                      v_pages: Tensor, page_table: Tensor, seq_lens: Tensor,
                      slots: Optional[Tensor], starts: Optional[Tensor], max_new: Optional[int],
                      norm_eps: Optional[float]) -> Tensor:
    return N.done(N.torch_ext().paged_rotary_append(q, k, v, cos, sin, k_pages, v_pages,
                                                    page_table, seq_lens, slots, starts, max_new,
                                                    norm_eps))


@_rotary_append_op.register_fake
def _(q, k, v, cos, sin, k_pages, v_pages, page_table, seq_lens, slots, starts, max_new, norm_eps):
    return q.new_empty(q.shape)


@torch.library.custom_op("nanochat_amd::paged_cache_read", mutates_args=())
def _read_op(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seq_lens: Tensor, tokens: int,
             slots: Optional[Tensor], starts: Optional[Tensor], max_new: Optional[int],
             dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    return N.done(N.torch_ext().paged_cache_read(k_pages, v_pages, page_table, seq_lens, tokens,
                                                 slots, starts, max_new, dtype))


@_read_op.register_fake
def _(k_pages, v_pages, page_table, seq_lens, tokens, slots, starts, max_new, dtype):
    D = k_pages.shape[3] // 17 * 32 if k_pages.dtype == torch.uint8 else k_pages.shape[3]
    rows = [] if starts is not None else [(page_table if slots is None else slots).shape[0]]
    shape = (*rows, tokens, k_pages.shape[1], D)
    return k_pages.new_empty(shape, dtype=dtype), k_pages.new_empty(shape, dtype=dtype)


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


@torch.library.custom_op("nanochat_amd::paged_cache_reorder", mutates_args=_STATE)
def _reorder_op(page_table: Tensor, seq_lens: Tensor, ref_counts: Tensor, slots: Tensor,
                src: Tensor) -> None:
    N.done(N.torch_ext().paged_cache_reorder(page_table, seq_lens, ref_counts, slots, src))


@_reorder_op.register_fake
def _(page_table, seq_lens, ref_counts, slots, src):
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
