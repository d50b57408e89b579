"""A paged key-value cache and the attention that decodes from it (trellis_kv_append,
trellis_paged_attention, trellis_kv_evict): what a decoder block runs between its q/k/v and its o linear
(the reference's QKNORM, ROPE, cache copy and ATTN dispatches over one contiguous sequence,
within web/model.js:77-102); and beyond the reference, several new tokens a row (prompts, drafted tokens in a
tree: trellis_tree_attention, trellis_kv_keep) and sequences that fork (trellis_kv_copy_pages). For serving:
forward only. Arguments are checked in csrc/bind.cpp.

append_kv, paged_attention, tree_attention, evict_kv, copy_pages and keep_kv work on tensors that the caller owns;
PagedKVCache owns them.

  k_pages, v_pages: [pages, heads, page_size, head_dim] float16 or bfloat16; alike in strides, unit last; bfloat16
         values up to 2^124 / (a row's tokens) in size (the attention's sums of up to 16 times them are fp32)
  table: int32 [rows, width], row b's token j in slot j % page_size of page table[b, j // page_size]; an
         id outside the pool is no page (nothing is written, its tokens count as absent)
  lens:  int32 [rows], tokens per row
  scores: float32 and pos: int32, [pages, heads, page_size]: each token's accumulated attention weight
          and its position
"""
from __future__ import annotations

from collections import Counter

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


def tree_attention(q, k_pages, v_pages, table, lens, *, starts=None, parents=None, scale: float | None = None,
                   max_len: int | None = None, out=None, out_dtype=None, workspace=None):
    """Attention of several new tokens per row: drafted tokens in a tree, or a prompt. Row b's n = starts[b+1] - starts[b]
    tokens are the newest of its lens[b] (append_kv has put their keys and values there, in its last n slots); the i-th
    sees the tokens before them, itself and its ancestors: softmax(scale * q.k) v over these, scale d**-0.5 if None.

    q: [tokens, q_heads, d], any token and head strides; query head i over key-value head i // (q_heads // heads)
    starts: int32 [rows + 1], ascending, row by row as for append_kv; None: the same number of tokens for each row
    parents: int32 [tokens], the number within its row of the token that each one continues; one that is not below the
        token's own (-1) is none: it continues the cached tokens. None: each continues the one before it, so that it
        sees them all (a prompt, or part of one).
    Returns [tokens, q_heads, d] of out_dtype (q's if None), or fills a contiguous `out`. Zeros for a token of no row
    (padding), for one whose slot the table or max_len does not hold, and where every page it could see is missing.
    max_len, workspace: as for paged_attention. Keys and values of a row's tokens have to be finite, those that a token
        does not see among them."""
    return _result(_capi.serve().tree_attention(q, k_pages, v_pages, table, lens, starts, parents, scale, max_len, out,
                                                out_dtype, workspace))


def copy_pages(k_pages, v_pages, src, dst, *, counts=None, scores=None, pos=None) -> None:
    """Page dst[i] becomes page src[i], its first counts[i] tokens if given (int32 [n] each), in one launch for up to 32
    layers: k_pages and v_pages (scores, pos) are one layer's tensor, a list with one for each layer, or one tensor with the
    layers as its first dim.
    No page may be in dst twice, or in src and dst; src[i] == dst[i], and ids outside the pool, copy nothing."""
    return _result(_capi.serve().copy_pages(k_pages, v_pages, src, dst, counts, scores, pos))


def keep_kv(k_pages, v_pages, table, lens, starts, path, *, scores=None, pos=None):
    """After a check of drafted tokens: of each row's n = starts[b+1] - starts[b] newest tokens those on its path stay.
    Token path[b, i] moves to slot lens[b] - n + i, in place, key, value, score and position together, in one launch for
    up to 32 layers (given as for copy_pages).

    path: int32 [rows, width], ascending numbers below n; it ends at the first entry that is not one (-1)
    Returns the new lengths lens - n + the paths' as a new tensor. No page that holds new tokens may be in two rows'
    tables; a token whose old or new slot is on no page is not moved."""
    return _result(_capi.serve().keep_kv(k_pages, v_pages, table, lens, starts, path, scores, pos))


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

    A step calls grow() once, then append() and attend() for each layer (attend_new() where it gave rows several
    tokens: prompts, drafts); evict() once after a step keeps the rows within a budget, by the weights that attend()
    has added up (attend_new() adds none: of a prompt that came in one pass, all of score 0 until later tokens' attend()
    weighs it, evict() keeps the last positions and the lowest slots; one fed a token at a time through attend() has its
    scores); keep() the drafted tokens that a check has accepted; reorder() lets rows go on from others' sequences, as
    beams do. The page tables, lengths and positions are shared by the layers, full pages by rows that have forked (but
    for an evictable cache, whose rows change all of theirs). Calls are ordered on the current stream; use the cache on
    one stream at a time. A grow(), evict(), keep(), reorder() or release() that changes a row's pages sends the table
    anew and waits for the stream (a budget that is a multiple of page_size takes and frees a page each step)."""

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
        self._refs = [0] * pages     # rows that have the page
        self._starts = self._positions = None
        self._drafts: tuple[list[int], list[int]] | None = None     # the last grow()'s counts, and seen before it
        # rows that the last grow() gave tokens, on the device (None: all); lens of these and of the others
        self._fed: torch.Tensor | None = None
        self._lens_of: tuple[torch.Tensor, torch.Tensor] | None = None

    def _upload(self, dst: torch.Tensor, values) -> None:
        dst.copy_(torch.tensor(values, dtype=torch.int32))

    def _upload_table(self) -> None:
        width = self.table.shape[1]
        self._upload(self.table, [own + [-1] * (width - len(own)) for own in self._owned])

    def _take(self) -> int:
        page = self._free.pop()
        self._refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def grow(self, counts, depths=None) -> None:
        """Room for counts[b] new tokens in each row b (an int: in every row); the next append() calls fill it.
        depths: for drafted tokens in a tree, each token's depth below its row's sequence (0: next after it), row by
            row; its position is that far on. None: the tokens follow each other.
        Raises ValueError, and changes nothing, where a row would pass max_len or the pool has too few pages."""
        rows = len(self.lengths)
        counts = [counts] * rows if isinstance(counts, int) else list(counts)
        if len(counts) != rows or min(counts) < 0:
            raise ValueError(f"counts must be {rows} numbers >= 0")
        if depths is not None:
            depths = list(depths)
            if len(depths) != sum(counts) or min(depths, default=0) < 0:
                raise ValueError(f"depths must be {sum(counts)} numbers >= 0")
        lengths = [n + c for n, c in zip(self.lengths, counts)]
        if max(lengths) > self.max_len:
            raise ValueError(f"a row of {max(lengths)} tokens passes max_len={self.max_len}")
        need = [-(-n // self.page_size) - len(own) for n, own in zip(lengths, self._owned)]
        if sum(need) > len(self._free):
            raise ValueError(f"{sum(need)} pages needed, {len(self._free)} free")
        for own, k in zip(self._owned, need):
            own.extend(self._take() for _ in range(k))
        if any(need):
            self._upload_table()
        self.lengths = lengths
        before, at = self.seen, 0
        self._drafts = counts, before
        steps = []          # positions that each row advances by
        for c in counts:
            steps.append(c if depths is None else max(depths[at:at + c], default=-1) + 1)
            at += c
        self.seen = [p + c for p, c in zip(before, steps)]
        self._fed, self._lens_of = None, None
        if self.scores[0] is not None and not all(counts):
            self._fed = torch.tensor([c > 0 for c in counts]).to(self.device)
        if depths is None and all(c == 1 for c in counts):
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
            if depths is None:
                where = [p + i for p, c in zip(before, counts) for i in range(c)]
            else:
                where = [p + d for p, d in zip([p for p, c in zip(before, counts) for _ in range(c)], depths)]
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

    def attend_new(self, layer: int, q, *, parents=None, scale: float | None = None, out_dtype=None):
        """tree_attention of the tokens that grow() made room for, row by row: q has a query for each. parents: int32 on
        the device, the number within its row of the token that each one continues (-1: the row's sequence); None: each
        continues the one before it. An evictable cache's scores stay as they are: a later evict() knows nothing of these
        tokens' attention."""
        if self._positions is None:
            raise ValueError("grow() first")
        new = self._positions.shape[0]
        if q.dim() != 3 or q.shape[0] != new:
            raise ValueError(f"q must be [{new}, q_heads, head_dim], a query for each token that grow() made room for")
        return tree_attention(q, self.k[layer], self.v[layer], self.table, self.lens, starts=self._starts, parents=parents,
                              scale=scale, max_len=max(self.lengths), out_dtype=out_dtype)

    def keep(self, paths) -> None:
        """keep_kv in every layer: of the tokens that the last grow() gave row b those numbered paths[b] stay (ascending, a
        line of the tree from its root), closed up; the pages that the rows no longer fill go back to the pool. The rows'
        sequences have then grown by their paths. Raises ValueError, and changes nothing, where a path does not fit."""
        if self._drafts is None:
            raise ValueError("grow() first")
        counts, before = self._drafts
        paths = [list(p) for p in paths]
        if len(paths) != len(counts) or any(p != sorted(set(p)) or (p and not 0 <= p[0] <= p[-1] < c) for p, c in zip(paths, counts)):
            raise ValueError("each row's path must be ascending numbers below its count of new tokens")
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        starts = self._starts if self._starts is not None else torch.tensor(starts, dtype=torch.int32).to(self.device)
        width = max(len(p) for p in paths)
        path = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32).view(len(paths), width).to(self.device)
        self.lens.copy_(keep_kv(self.k, self.v, self.table, self.lens, starts, path, scores=self.scores, pos=self.pos))
        self.seen = [p + len(k) for p, k in zip(before, paths)]
        self._upload(self.next_pos, self.seen)
        self._set_lengths([n - c + len(p) for n, c, p in zip(self.lengths, counts, paths)])

    def reorder(self, parents) -> None:
        """Row b goes on from what row parents[b] holds (several rows may from one; what no row goes on from is dropped): the
        rows share the pages that are full and copy the one that they will fill further (an evictable cache's rows copy
        all). Raises ValueError, and changes nothing, where the pool has too few pages."""
        rows = len(self.lengths)
        parents = [int(p) for p in parents]
        if len(parents) != rows or min(parents) < 0 or max(parents) >= rows:
            raise ValueError(f"parents must be {rows} numbers in 0 .. {rows - 1}")
        share = self.scores[0] is None
        # of the rows that go on from one, the row itself keeps its pages as they are, or else the first
        heir: dict[int, int] = {}
        for b, p in enumerate(parents):
            if p == b or p not in heir:
                heir[p] = b
        full = [n // self.page_size if share else 0 for n in self.lengths]
        want = sum(len(self._owned[p]) - full[p] for b, p in enumerate(parents) if heir[p] != b)
        gone = [page for p in range(rows) if p not in heir for page in self._owned[p]]
        back = sum(self._refs[page] == n for page, n in Counter(gone).items())
        if want > len(self._free) + back:
            raise ValueError(f"{want} pages needed, {len(self._free) + back} free")
        old = self._owned
        for page in gone:
            self._drop(page)
        src, dst, counts = [], [], []
        self._owned = []
        for b, p in enumerate(parents):
            own = list(old[p])
            if heir[p] != b:
                for i, page in enumerate(own):
                    if i < full[p]:
                        self._refs[page] += 1
                    else:
                        own[i] = self._take()
                        src.append(page)
                        dst.append(own[i])
                        counts.append(min(self.page_size, self.lengths[p] - i * self.page_size))
            self._owned.append(own)
        if src:
            ints = [torch.tensor(t, dtype=torch.int32).to(self.device) for t in (src, dst, counts)]
            copy_pages(self.k, self.v, ints[0], ints[1], counts=ints[2], scores=self.scores, pos=self.pos)
        if parents != list(range(rows)):
            self._upload_table()
            if self._fed is not None:
                self._fed = self._fed[torch.tensor(parents, device=self.device)]
        self.seen = [self.seen[p] for p in parents]
        self._upload(self.next_pos, self.seen)
        self._set_lengths([self.lengths[p] for p in parents])
        self._upload(self.lens, self.lengths)

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
        self._starts = self._positions = self._lens_of = self._drafts = None
        self.lengths, freed = lengths, False
        for own, n in zip(self._owned, lengths):
            while len(own) > -(-n // self.page_size):
                self._drop(own.pop())
                freed = True
        if freed:
            self._upload_table()
