"""The inference cache of a model over pages: attention keys and values of many
sequences in fixed-size pages, shared between sequences that began alike, beside the
LTV filter's last rows of each.

What ``KVCache`` (reference ``nanochat/kv_cache.py``) holds for one contiguous batch
is kept here per slot, so that sequences come and go, prompts come in chunks, and
several samples continue one prompt without copying it (``fork``; the reference's
``prefill`` copies the whole cache).  The operators are those of
``nanochat_amd.ops.paged_cache``; page table, lengths and counts stay on the GPU.

    cache = PagedKVCache(n_layer, n_head, n_kv_head, head_dim, num_pages=..., max_seqs=...,
                         max_len=...)
    step = cache.step([0], T)          # room for T new tokens of slot 0
    for i, layer in enumerate(layers):
        q, k, v = layer.qkv_computer(x, step)   # the filter continues the slot's rows
        y = step.attend(i, q, k, v)
    cache.fork([0, 0, 0], [1, 2, 3])   # three more samples of slot 0's prompt
    cache.reorder([0, 1, 2, 3], [2, 2, 0, 1])   # a search's beams after its selection

The pages hold the layers' dtype, or 4 bits (``bits=4``: 17 of 64 bytes); with ``rotary``
tables the cache rotates and normalises queries and keys on their way.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from nanochat_amd.ops.paged_cache import (
    fp4_row_bytes,
    paged_attention,
    paged_cache_append,
    paged_cache_compact,
    paged_cache_fork,
    paged_cache_free,
    paged_cache_reorder,
    paged_cache_reserve,
    paged_rotary_append,
)


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` tokens in each of ``n_layer`` layers, for at
    most ``max_seqs`` sequences (slots) of ``max_len`` tokens.

    ``bits=4`` holds keys and values in 4 bits (head_dim 32, 64, 96 or 128, the page size a
    multiple of 16), else in ``dtype``; queries and attention are ``dtype`` either way.
    ``rotary`` (cos, sin), (at least max_len, head_dim / 2) each: ``attend`` takes queries and
    keys as they come from the projection, rotates them by their positions and, with
    ``norm_eps``, divides each head by sqrt(mean of squares + norm_eps)."""

    def __init__(self, n_layer: int, n_head: int, n_kv_head: int, head_dim: int, *,
                 num_pages: int, max_seqs: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", bits: Optional[int] = None,
                 rotary: Optional[tuple] = None, norm_eps: Optional[float] = None):
        if n_kv_head <= 0 or n_head % n_kv_head:
            raise ValueError(f"{n_kv_head} k/v heads do not divide {n_head} heads")
        if min(n_layer, num_pages, max_seqs, max_len, page_size) <= 0:
            raise ValueError("a cache needs layers, pages, sequences and room for tokens")
        if bits not in (None, 4):
            raise ValueError(f"pages hold the cache's dtype or 4 bits, got {bits}")
        if bits == 4 and page_size % 16:
            raise ValueError(f"a 4-bit page must hold a multiple of 16 tokens, got {page_size}")
        if norm_eps is not None and rotary is None:
            raise ValueError("norm_eps without rotary tables")
        self.n_layer, self.page_size, self.max_len = n_layer, page_size, max_len
        self.dtype, self.norm_eps = dtype, norm_eps
        width = -(-max_len // page_size)

        def ints(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        row = fp4_row_bytes(head_dim) if bits == 4 else head_dim
        shape = (n_layer, num_pages, n_kv_head, page_size, row)
        held = torch.uint8 if bits == 4 else dtype
        self.k_pages = torch.empty(shape, dtype=held, device=device)
        self.v_pages = torch.empty(shape, dtype=held, device=device)
        self.rotary = None
        if rotary is not None:
            self.rotary = tuple(self._table(t, max_len, head_dim, width * page_size)
                                for t in rotary)
        self.page_table = ints(max_seqs, width, value=-1)
        self.seq_lens = ints(max_seqs)
        self.ref_counts = ints(num_pages)
        # the filter's last output rows of each slot
        self.rows = tuple(torch.zeros(n_layer, max_seqs, n, head_dim, dtype=dtype, device=device)
                          for n in (n_head, n_kv_head, n_kv_head))
        self.lens = [0] * max_seqs  # what seq_lens holds, known on the host
        # on the device: 0, or the status of the first of the steps not yet looked at that
        # found no room; None where there are no such steps
        self._status = None

    def _table(self, t: torch.Tensor, max_len: int, head_dim: int, rows: int) -> torch.Tensor:
        """A table with a row for each position that the page table has room for (those from
        max_len on are not reached)."""
        if t.dim() != 2 or t.size(0) < max_len or t.size(1) != head_dim // 2:
            raise ValueError(f"rotary tables are (at least {max_len}, {head_dim // 2}), got "
                             f"{tuple(t.shape)}")
        t = t.detach().to(self.k_pages.device)[:rows]
        return torch.cat([t, t[-1:].expand(rows - len(t), -1)]).contiguous()

    def _slots(self, slots: Sequence[int]) -> torch.Tensor:
        if len(set(slots)) != len(slots):
            raise ValueError(f"a slot is named twice: {list(slots)}")
        if any(not 0 <= s < len(self.lens) for s in slots):
            raise ValueError(f"slots are 0 to {len(self.lens) - 1}, got {list(slots)}")
        return torch.tensor(slots, dtype=torch.int32, device=self.page_table.device)

    def step(self, slots: Sequence[int], n_new: int, check: bool = True) -> "PagedStep":
        """Room for ``n_new`` more tokens in each of the slots, and the view of them that
        a model's layers take.  Raises if the pages run out, with nothing changed.

        With ``check`` off it does not wait for the device to say so.  If they ran out, this
        step and those that follow it change nothing in the cache (their attention is 0),
        until ``check_steps`` or a step with ``check`` on has raised; ``status`` of a step is
        0, or how many pages were missing at the first of them."""
        if check:
            self.check_steps()
        index = self._slots(slots)
        if n_new <= 0:
            raise ValueError(f"a step has new tokens, got {n_new}")
        longest = max((self.lens[s] for s in slots), default=0) + n_new
        if longest > self.max_len:
            raise ValueError(f"{longest} tokens, but the cache is made for {self.max_len}")
        fresh = [self.lens[s] == 0 for s in slots]
        if any(fresh) and not all(fresh):
            raise ValueError("a step's sequences are all new or all continued")
        counts = torch.full_like(index, n_new)
        if not check and self._status is not None:
            counts = torch.where(self._status == 0, counts, 0)
        status = paged_cache_reserve(self.page_table, self.seq_lens, self.ref_counts, index,
                                     counts, self.k_pages, self.v_pages)
        room = None
        if check:
            self._raise_for(int(status))
        else:
            if self._status is not None:
                status = torch.where(self._status == 0, status, self._status)
            self._status, room = status, status == 0
        positions = [self.lens[s] for s in slots]
        for s in slots:
            self.lens[s] += n_new
        return PagedStep(self, index, positions, n_new, status, room)

    def check_steps(self) -> None:
        """Wait for the steps that were made with ``check`` off, and raise if one of them
        found no room: it and the steps after it are undone, ``lens`` is what it was."""
        if self._status is None:
            return
        status, self._status = int(self._status), None
        if status:
            self.lens[:] = self.seq_lens.tolist()
        self._raise_for(status)

    @staticmethod
    def _raise_for(status: int) -> None:
        if status < 0:
            raise RuntimeError("the cache's lengths are not those of its steps")
        if status:
            raise RuntimeError(f"the paged cache is full: {status} pages are missing")

    def fork(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Slots dst continue from slots src (one src may be named several times)."""
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} source slots, {len(dst)} new ones")
        if set(src) & set(dst):
            raise ValueError("a slot is both forked and overwritten")
        to = self._slots(dst)
        from_ = torch.tensor(src, dtype=torch.int32, device=to.device)
        if any(not 0 <= s < len(self.lens) for s in src):
            raise ValueError(f"slots are 0 to {len(self.lens) - 1}, got {list(src)}")
        paged_cache_fork(self.page_table, self.seq_lens, self.ref_counts, from_, to)
        for rows in self.rows:
            rows.index_copy_(1, to.long(), rows.index_select(1, from_))
        for a, b in zip(src, dst):
            self.lens[b] = self.lens[a]

    def reorder(self, slots: Sequence[int], src: Sequence[int]) -> None:
        """Slot slots[i] becomes what slot src[i] holds, all at once (a slot may be a source
        several times, and both)."""
        if len(slots) != len(src):
            raise ValueError(f"{len(slots)} slots, {len(src)} sources")
        if any(not 0 <= s < len(self.lens) for s in src):
            raise ValueError(f"slots are 0 to {len(self.lens) - 1}, got {list(src)}")
        to = self._slots(slots)
        from_ = torch.tensor(src, dtype=torch.int32, device=to.device)
        paged_cache_reorder(self.page_table, self.seq_lens, self.ref_counts, to, from_)
        for rows in self.rows:
            rows.index_copy_(1, to.long(), rows.index_select(1, from_))
        lens = [self.lens[s] for s in src]
        for s, n in zip(slots, lens):
            self.lens[s] = n

    def free(self, slots: Sequence[int]) -> None:
        paged_cache_free(self.page_table, self.seq_lens, self.ref_counts, self._slots(slots))
        for s in slots:
            self.lens[s] = 0

    def compact(self) -> torch.Tensor:
        """Close up the pages in use; their number (int32, one element)."""
        return paged_cache_compact(self.page_table, self.ref_counts, self.k_pages, self.v_pages)


class _Rows:
    """``special[layer]``: a step's rows of one of q, k, v."""

    def __init__(self, rows: torch.Tensor, index: torch.Tensor):
        self._rows, self._index = rows, index

    @property
    def special(self):
        return self

    def __getitem__(self, layer: int) -> torch.Tensor:
        return self._rows[layer].index_select(0, self._index)


class PagedStep:
    """One step of some slots: the KV cache protocol of the filter's computer module
    (``has_last_qkv``, ``last_qkv``, ``update_last_qkv``), and attention."""

    def __init__(self, cache: PagedKVCache, slots: torch.Tensor, positions: list, n_new: int,
                 status: torch.Tensor, room: Optional[torch.Tensor] = None):
        self.cache, self.positions, self.n_new = cache, positions, n_new
        self.status = status
        # whether there was room (None: there was), known on the device; without it the
        # step is one of no slots, or the tokens would go where the last ones before are
        self._room = room
        self.slots = slots if room is None else torch.where(room, slots, -1)
        self._index = slots.long()
        self.q, self.k, self.v = (_Rows(r, self._index) for r in cache.rows)

    @property
    def rotates(self) -> bool:
        """Whether ``attend`` rotates queries and keys."""
        return self.cache.rotary is not None

    @property
    def normalises(self) -> bool:
        """Whether it divides their heads by their size, too."""
        return self.cache.norm_eps is not None

    @property
    def last_qkv(self) -> "PagedStep":
        return self

    def has_last_qkv(self, layer_idx: int) -> bool:
        return self.positions[0] > 0

    def update_last_qkv(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor,
                        v: torch.Tensor) -> None:
        for rows, t in zip(self.cache.rows, (q, k, v)):
            t = t.to(rows.dtype)
            if self._room is not None:
                t = torch.where(self._room, t, rows[layer_idx].index_select(0, self._index))
            rows[layer_idx].index_copy_(0, self._index, t)

    def attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               scale: Optional[float] = None) -> torch.Tensor:
        """q (B, T, n_head, head_dim), k and v (B, T, n_kv_head, head_dim), B the step's
        slots and T its new tokens: writes k and v into the pages and returns the
        attention of q over each sequence up to itself, (B, T, n_head, head_dim); q and k
        rotated, and normalised, first where the cache does that."""
        c = self.cache
        dt = c.dtype
        kp, vp = c.k_pages[layer_idx], c.v_pages[layer_idx]
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
        if c.rotary is not None:
            q = paged_rotary_append(q, k, v, *c.rotary, kp, vp, c.page_table, c.seq_lens,
                                    slots=self.slots, norm_eps=c.norm_eps)
        else:
            paged_cache_append(k, v, kp, vp, c.page_table, c.seq_lens, slots=self.slots)
        return paged_attention(q, kp, vp, c.page_table, c.seq_lens, slots=self.slots,
                               max_len=max(self.positions) + self.n_new, scale=scale)
