"""A paged key-value cache and the attention that decodes from it (trellis_kv_append,
trellis_paged_attention, trellis_kv_evict): what a decoder block runs between its q/k/v and its o linear
(the reference's QKNORM, ROPE, cache copy and ATTN dispatches over one contiguous sequence,
within web/model.js:77-102). For serving: forward only. Arguments are checked in csrc/bind.cpp.

append_kv, paged_attention and evict_kv work on tensors that the caller owns; PagedKVCache owns them.

  k_pages, v_pages: [pages, heads, page_size, head_dim] float16 or bfloat16; alike in strides, unit last
  table: int32 [rows, width], row b's token j in slot j % page_size of page table[b, j // page_size]; an
         id outside the pool is no page (nothing is written, its tokens count as absent)
  lens:  int32 [rows], tokens per row
  scores: float32 and pos: int32, [pages, heads, page_size]: each token's accumulated attention weight
          and its position
"""
from __future__ import annotations

import torch

from . import _capi


def _result(r):
    """A call's result, or the error that its status names."""
    if r.__class__ is int:
        _capi.check(r)
    return r


def append_kv(q, k, v, k_pages, v_pages, table, lens, *, starts=None, positions=None, q_norm=None, k_norm=None,
              eps: float = 1e-6, cos=None, sin=None, scores=None, pos=None, q_dtype=None):
    """New tokens into the cache; returns the queries that attend to it.

    q [tokens, q_heads, d], k and v [tokens, heads, d] (one dtype, any token and head strides):
        q' = rot(norm(q)) returned as q_dtype (q's if None); rot(norm(k)) and v into the token's slot
    norm: x * rsqrt(mean(x^2) + eps) * w per head, with float32 q_norm and k_norm [d] (both or neither)
    rot:  pairs (x_i, x_{i + r/2}), i < r/2, turned by float32 cos and sin [positions, r/2] at the token's
          position (both or neither; dims from r on stay; a position outside the table gives NaN)
    lens counts these tokens already: the i-th of a row's n goes to slot lens[b] - n + i.
    starts: int32 [rows + 1], tokens starts[b] .. starts[b+1]-1 are row b's; None: one token for each row.
    positions: int32 [tokens]; None: the slots (as long as nothing has been evicted).
    scores, pos: the new tokens' entries are set to 0 and to their positions.
    A token of no row, or whose slot the table does not hold (padding), is not stored and its q' is 0."""
    return _result(_capi.serve().append_kv(q, k, v, k_pages, v_pages, table, lens, starts, positions, q_norm, k_norm, eps,
                                           cos, sin, scores, pos, q_dtype))


def paged_attention(q, k_pages, v_pages, table, lens, *, scale: float | None = None, max_len: int | None = None,
                    scores=None, out=None, out_dtype=None, workspace=None):
    """Attention of one new token per row over the cache: q [rows, q_heads, d] (any row and head strides),
    query head i over key-value head i // (q_heads // heads); softmax(scale * q.k) v over the row's
    tokens, scale d**-0.5 if None. A row without tokens gives zeros. Returns [rows, q_heads, d] of
    out_dtype (q's if None), or fills a contiguous `out`.

    max_len: the longest row the call has to expect; it plans the split over the length, and tokens past
        it are not seen. None: all that the table can hold. Give the batch's own bound where one is known: a
        single row is split for it (4000 tokens take 9.6 us under 8192, 13.9 under 32768, 31 under 131072),
        and `scores` need scratch for it, 4 bytes per row, query head and token.
    scores: each token's entry grows by the sum of its weights over the query heads of its head.
    Keys and values of a row's tokens have to be finite (another makes the row's heads NaN); what the pages hold
    past them is not looked at.
    workspace: scratch for a caller that keeps its own, any contiguous tensor on the device (too small a one raises
        TRELLIS_ERR_WORKSPACE); None: taken from torch's allocator for the call."""
    return _result(_capi.serve().paged_attention(q, k_pages, v_pages, table, lens, scale, max_len, scores, out, out_dtype,
                                                 workspace))


def evict_kv(k_pages, v_pages, scores, pos, table, lens, keep: int, recent: int, *, next_pos=None, out_table=None,
             max_len: int | None = None, workspace=None):
    """Evict by accumulated attention weight: of each row's tokens, per key-value head, `keep` stay: those of
    the last `recent` positions (pos >= next_pos[b] - recent), then those of the largest scores, equal
    scores by the lowest slot. A kept token below slot `keep` stays in its slot; the freed slots below take
    the kept tokens from above, both in ascending order. Key, value, score and position move together.

    next_pos: int32 [rows], positions each row has seen; None: its length (nothing evicted before).
    out_table: int32 [rows, width]: the kept tokens are copied to these pages instead (none of them in
        `table`), whose own stay as they are; None: in place, where no page may be in two rows' tables.
        It needs a page for every slot below the new lengths; one with fewer slots than `keep` keeps what
        it has slots for.
    Tokens on pages that do not exist are absent. In place their slots stay empty, and as many tokens are
    kept as there are slots below `keep` on pages that exist; into an out_table only the present tokens go,
    without gaps, and the new lengths count them alone.
    Returns the new lengths min(lens, keep) as a new tensor; `lens` itself stays, for a model's other
    layers. Rows of up to `keep` tokens stay as they are."""
    return _result(_capi.serve().evict_kv(k_pages, v_pages, scores, pos, table, lens, keep, recent, next_pos, out_table,
                                          max_len, workspace))


class PagedKVCache:
    """The key-value cache of a model's layers for up to `rows` sequences of up to `max_len` cached tokens,
    in pages that the rows take from one pool as they grow.

    A step calls grow() once, then append() and attend() for each layer; evict() once after a step keeps
    the rows within a budget. The page tables, lengths and positions are shared by the layers. Calls are
    ordered on the current stream; use the cache on one stream at a time. A grow(), evict() or release() that
    changes a row's pages sends the table anew and waits for the stream (a budget that is a multiple of
    page_size takes and frees a page each step)."""

    def __init__(self, layers: int, heads: int, head_dim: int, *, rows: int, max_len: int, pages: int | None = None,
                 page_size: int = 64, dtype: torch.dtype = torch.float16, device="cuda", evictable: bool = False):
        width = -(-max_len // page_size)
        pages = rows * width if pages is None else pages
        if min(layers, heads, rows, max_len, pages) < 1:
            raise ValueError("layers, heads, rows, max_len and pages must be positive")
        shape = (pages, heads, page_size, head_dim)
        self.page_size, self.max_len, self.device = page_size, max_len, torch.device(device)
        # idle slots are never read as values: no fill
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.scores = [torch.zeros(shape[:3], dtype=torch.float32, device=device) if evictable else None for _ in range(layers)]
        self.pos = [torch.zeros(shape[:3], dtype=torch.int32, device=device) if evictable else None for _ in range(layers)]
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.next_pos = torch.zeros(rows, dtype=torch.int32, device=device)
        self.lengths, self.seen = [0] * rows, [0] * rows     # the host's copies of lens and next_pos
        self._free = list(range(pages - 1, -1, -1))
        self._owned: list[list[int]] = [[] for _ in range(rows)]
        self._starts = self._positions = None
        # rows that the last grow() gave tokens, on the device (None: all); lens of these and of the others
        self._fed: torch.Tensor | None = None
        self._lens_of: tuple[torch.Tensor, torch.Tensor] | None = None

    def _upload(self, dst: torch.Tensor, values) -> None:
        dst.copy_(torch.tensor(values, dtype=torch.int32))

    def _upload_table(self) -> None:
        width = self.table.shape[1]
        self._upload(self.table, [own + [-1] * (width - len(own)) for own in self._owned])

    def grow(self, counts) -> None:
        """Room for counts[b] new tokens in each row b (an int: in every row); the next append() calls fill it.
        Raises ValueError, and changes nothing, where a row would pass max_len or the pool has too few pages."""
        rows = len(self.lengths)
        counts = [counts] * rows if isinstance(counts, int) else list(counts)
        if len(counts) != rows or min(counts) < 0:
            raise ValueError(f"counts must be {rows} numbers >= 0")
        lengths = [n + c for n, c in zip(self.lengths, counts)]
        if max(lengths) > self.max_len:
            raise ValueError(f"a row of {max(lengths)} tokens passes max_len={self.max_len}")
        need = [-(-n // self.page_size) - len(own) for n, own in zip(lengths, self._owned)]
        if sum(need) > len(self._free):
            raise ValueError(f"{sum(need)} pages needed, {len(self._free)} free")
        for own, k in zip(self._owned, need):
            own.extend(self._free.pop() for _ in range(k))
        if any(need):
            self._upload_table()
        self.lengths = lengths
        self.seen = [p + c for p, c in zip(self.seen, counts)]
        self._fed, self._lens_of = None, None
        if self.scores[0] is not None and not all(counts):
            self._fed = torch.tensor([c > 0 for c in counts]).to(self.device)
        if all(c == 1 for c in counts):
            # a decode step: but for the table, where a row takes a page, nothing comes from the host
            self.lens += 1
            self._starts, self._positions = None, self.next_pos.clone()
            self.next_pos += 1
        else:
            self._upload(self.lens, self.lengths)
            self._upload(self.next_pos, self.seen)
            starts = [0]
            for c in counts:
                starts.append(starts[-1] + c)
            where = [i for p, c in zip(self.seen, counts) for i in range(p - c, p)]
            self._starts = torch.tensor(starts, dtype=torch.int32).to(self.device)
            self._positions = torch.tensor(where, dtype=torch.int32).to(self.device)

    def append(self, layer: int, q, k, v, **rotary):
        """append_kv of the tokens that grow() made room for (row by row), at their positions in the sequences."""
        if self._positions is None:
            raise ValueError("grow() first")
        return append_kv(q, k, v, self.k[layer], self.v[layer], self.table, self.lens, starts=self._starts,
                         positions=self._positions, scores=self.scores[layer], pos=self.pos[layer], **rotary)

    def attend(self, layer: int, q, *, scale: float | None = None, out_dtype=None):
        """paged_attention of one query token per row (a row without tokens gives zeros). An evictable cache adds the
        weights to its scores, of the rows that the last grow() gave tokens: the others wait, and what is asked of
        them meanwhile does not count."""
        def ask(lens, scores):
            return paged_attention(q, self.k[layer], self.v[layer], self.table, lens, scale=scale,
                                   max_len=max(self.lengths), scores=scores, out_dtype=out_dtype)

        if self._fed is None:
            return ask(self.lens, self.scores[layer])
        if self._lens_of is None:
            self._lens_of = self.lens * self._fed, self.lens * ~self._fed
        fed, waiting = self._lens_of
        return ask(fed, self.scores[layer]).add_(ask(waiting, None))     # each row is empty in one of them

    def evict(self, keep: int, recent: int) -> None:
        """evict_kv of every layer, in place; the pages that the rows no longer fill go back to the pool."""
        if self.scores[0] is None:
            raise ValueError("the cache was not made evictable")
        new_lens = None
        for k, v, scores, pos in zip(self.k, self.v, self.scores, self.pos):
            new_lens = evict_kv(k, v, scores, pos, self.table, self.lens, keep, recent, next_pos=self.next_pos,
                                max_len=max(self.lengths))
        self.lens.copy_(new_lens)
        self._set_lengths([min(n, keep) for n in self.lengths])

    def release(self, row: int) -> None:
        """The row's sequence has ended: its pages go back to the pool, the row is empty."""
        if not 0 <= row < len(self.lengths):
            raise ValueError(f"row must be in 0 .. {len(self.lengths) - 1}")
        self.seen[row] = 0
        self._upload(self.next_pos, self.seen)
        self._set_lengths([0 if b == row else n for b, n in enumerate(self.lengths)])
        self._upload(self.lens, self.lengths)

    def _set_lengths(self, lengths) -> None:
        self._starts = self._positions = self._lens_of = None
        self.lengths, freed = lengths, False
        for own, n in zip(self._owned, lengths):
            while len(own) > -(-n // self.page_size):
                self._free.append(own.pop())
                freed = True
        if freed:
            self._upload_table()
