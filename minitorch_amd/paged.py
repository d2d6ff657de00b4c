"""A key-value cache in pages, for generation.

The reference recomputes the whole context for every new token (GPT.generate,
transformer.py:93-104); GPT.generate_greedy keeps (B, Tmax, C) caches instead,
sized for the longest sequence.  A ``PagedKVCache`` holds keys and values in
pages of a fixed number of rows that sequences take as they grow and give back
when they end, in fp32 or bf16, and can be bounded: with ``keep``, each layer
and head remembers how much attention every row received, and when a sequence
has grown past ``keep + slack`` rows it is cut back to its last ``recent`` rows
and the ``keep - recent`` others that received the most.

All layers and heads of a sequence hold the same number of rows, so they share
one page table; which tokens' rows they hold differs once rows were evicted
(attention does not depend on their order).  Lengths and the table live in
device memory; a step of one token per sequence changes them without a copy
from the host unless a sequence enters a new page.
"""
from __future__ import annotations

import numpy as np

from . import device as dev
from . import kernels as K


class PagedKVCache:
    """Keys and values of n_layer layers with n_head K/V heads of head_dim for
    `batch` sequences of up to max_tokens cached rows each.

    page: rows a page; dtype: "float32" or "bfloat16"; pages: pages in the pool
    (default: enough for every sequence at its longest, and for an eviction).
    keep, recent, slack bound the cache as the module says (recent defaults to
    keep // 8, slack to one page); observe: how many of a prompt's last
    positions count its rows' attention (one-token steps always do)."""

    def __init__(self, n_layer, n_head, head_dim, batch, max_tokens, page=16, dtype="float32", pages=None, keep=None,
                 recent=None, slack=None, observe=8):
        if min(n_layer, n_head, head_dim, batch, max_tokens, page) < 1:
            raise ValueError("sizes must be at least 1")
        if head_dim not in (16, 32, 64, 128):
            raise ValueError(f"head_dim {head_dim} not in (16, 32, 64, 128)")
        if dtype not in ("float32", "bfloat16"):
            raise ValueError(f"unsupported dtype {dtype!r} (float32 or bfloat16)")
        self.n_layer, self.n_head, self.head_dim, self.batch = n_layer, n_head, head_dim, batch
        self.page, self.dtype, self.max_tokens = page, dtype, max_tokens
        self.width = -(-max_tokens // page)
        self.keep = keep
        spare = 0
        if keep is not None:
            self.recent = keep // 8 if recent is None else recent
            self.slack = page if slack is None else slack
            if not (1 <= keep and 0 <= self.recent <= keep and self.slack >= 0 and observe >= 0):
                raise ValueError("needs keep >= 1, 0 <= recent <= keep, slack >= 0 and observe >= 0")
            if keep + self.slack + 1 > max_tokens:
                raise ValueError(f"keep + slack + 1 = {keep + self.slack + 1} rows exceed max_tokens {max_tokens}")
            spare = batch * -(-keep // page)
        elif recent is not None or slack is not None:
            raise ValueError("recent and slack bound a cache that has keep")
        self.observed = observe
        self.n_pages = batch * self.width + spare if pages is None else pages
        if self.n_pages < 1:
            raise ValueError("the pool needs at least one page")
        # stored by heads: a head's rows of a page are adjacent
        shape = (self.n_pages, n_head, page, head_dim)
        self.k = [dev.empty_buf(shape, dtype) for _ in range(n_layer)]
        self.v = [dev.empty_buf(shape, dtype) for _ in range(n_layer)]
        self.table = dev.full((batch, self.width), -1, "int32").t
        self.lengths = dev.zeros((batch,), "int32").t
        self.counts = None  # rows of the append under way, where they differ
        self.weights = None
        if keep is not None:
            w = (batch, n_head, self.width * page)
            self.weights = [dev.zeros(w).t for _ in range(n_layer)]
            self._weights_to = dev.empty_buf(w)
            self._lengths_to = dev.empty_buf((batch,), "int32")
        # the host's copies
        self._len = np.zeros(batch, np.int32)
        self._tab = np.full((batch, self.width), -1, np.int32)
        self._free = list(range(self.n_pages - 1, -1, -1))
        # of the rows being appended
        self._rows = 0  # how many, of the sequence that gets most
        self._prompt = False  # whether they are their sequences' first
        self._ragged = False  # whether sequences that get some get different numbers
        self._active = None  # the lengths, 0 where none is new, if that is anywhere
        self._got = np.zeros(batch, bool)  # which sequences get some
        self._new = np.zeros(batch, np.int32)  # how many of each sequence undo can take back
        self._written = set()  # the layers that have them

    # -- what it holds ---------------------------------------------------------
    def length(self, b: int) -> int:
        """Cached rows of sequence b."""
        return int(self._len[b])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _check_room(self, prompt, steps):
        """Raises, as reserve or trim would on the way, unless prompts of that
        many rows in every sequence, and steps of one row after them, each followed
        by trim, fit the empty cache."""
        rows, spare = prompt + steps, 0
        if self.keep is not None and rows > self.keep + self.slack:
            rows, spare = max(prompt, self.keep + self.slack + 1), -(-self.keep // self.page)
        if rows > self.width * self.page:
            raise ValueError(f"{rows} rows exceed the {self.width * self.page} a sequence may hold")
        need = self.batch * -(-rows // self.page) + spare
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} free")

    # -- growing and shrinking ---------------------------------------------------
    def reserve(self, n=1):
        """Make room for n new rows in every sequence (an int, or one per
        sequence; 0 leaves it as it is, its queries see nothing): the rows that
        the layers' append then write.  Nothing has changed when it raises.  The
        sequences count the rows from here on: a step that is not carried out
        takes them back with undo; append and forward_paged do so before they
        raise, unless all layers have the rows."""
        n, most = np.broadcast_to(np.asarray(n, np.int64), (self.batch,)), self.width * self.page
        if n.min() < 0 or n.max() < 1:
            raise ValueError("reserve: at least one new row, none negative")
        if (n > most - self._len).any():
            rows = max(int(x) + int(y) for x, y in zip(self._len, n))
            raise ValueError(f"reserve: {rows} rows exceed the {most} a sequence may hold")
        n = n.astype(np.int32)
        grown = self._len + n
        have, need = -(-self._len // self.page), -(-grown // self.page)
        if (need - have).sum() > len(self._free):
            raise RuntimeError(f"reserve: {int((need - have).sum())} pages needed, {len(self._free)} free")
        for b in np.flatnonzero(need > have):
            for i in range(have[b], need[b]):
                self._tab[b, i] = self._free.pop()
        if (need > have).any():
            self.table.copy_(self._tab)
        self._prompt = not self._len[n > 0].any()
        self._ragged = n[n > 0].min() != n.max()
        if n.min() == n.max() == 1:
            K.decode_advance(self.lengths)
            self.counts = None
        else:
            self.lengths.copy_(grown)
            self.counts = None if n.min() == n.max() else dev.from_host(n, np.int32).t
        self._rows = int(n.max())
        self._active = None if n.min() else dev.from_host(np.where(n > 0, grown, 0), np.int32).t
        # rows reserved before that no layer has yet go with these
        self._len, self._new, self._got = grown, n if self._written else n + self._new, n > 0
        self._written.clear()

    def undo(self):
        """Take back the rows reserved last, in all layers (and those reserved
        before them if no layer had written any): lengths, table and free pages
        are what they were, the rows' weights 0.  (What a layer's attend has added
        to other rows' weights stays.)  Nothing happens if there are none, or trim
        has cut the sequences since."""
        if not self._new.any():
            return
        grown, self._len = self._len, self._len - self._new
        for b in np.flatnonzero(self._new)[::-1]:
            for i in range(-(-grown[b] // self.page) - 1, -(-self._len[b] // self.page) - 1, -1):
                self._free.append(int(self._tab[b, i]))
                self._tab[b, i] = -1
            for w in self.weights or ():
                w[b, :, int(self._len[b]):int(grown[b])].fill_(0.0)
        self._settle()
        self._rows, self._prompt, self.counts = 0, False, None
        self.table.copy_(self._tab)
        self.lengths.copy_(self._len)

    def _abandon(self):
        """What a layer does before it raises: a step that has not come through
        all layers leaves no rows."""
        if len(self._written) < self.n_layer:
            self.undo()

    def _settle(self):
        self._active = None
        self._new = np.zeros(self.batch, np.int32)

    def release(self, b: int):
        """Give back a sequence's pages; it is empty afterwards."""
        self._give_back(b, self._tab[b])
        self._len[b] = self._new[b] = 0
        self._active = None
        self.table.copy_(self._tab)
        self.lengths.copy_(self._len)
        if self.weights is not None:
            for w in self.weights:
                w[b].fill_(0.0)

    def _give_back(self, b, ids):
        self._free += [int(i) for i in ids if i >= 0]
        self._tab[b] = -1

    def trim(self) -> bool:
        """With keep: if a sequence holds more than keep + slack rows, cut all
        that hold more than keep back to keep, as many at a time as there are
        free pages for; the others stay where they are.  Returns whether it did;
        nothing has changed when there is not room for one."""
        if self.keep is None or self._len.max() <= self.keep + self.slack:
            return False
        cut, need = np.flatnonzero(self._len > self.keep), -(-self.keep // self.page)
        if need > len(self._free):
            raise RuntimeError(f"trim: {need} pages needed, {len(self._free)} free")
        first = 0
        while len(cut):  # a sequence that is cut gives back as many pages as it takes, or more
            n = min(len(cut), len(self._free) // need)
            end = int(cut[n]) if n < len(cut) else self.batch
            self._cut(cut[:n], first, end, need)
            first, cut = end, cut[n:]
        self.lengths, self._lengths_to = self._lengths_to, self.lengths
        self._settle()
        self.table.copy_(self._tab)
        return True

    def _cut(self, cut, first, end, need):
        """Cut the sequences `cut` of [first, end), `need` new pages each."""
        to = np.full((end - first, need), -1, np.int32)  # a sequence that has no new pages is not copied
        for b in cut:
            to[b - first] = [self._free.pop() for _ in range(need)]
        to_dev = dev.from_host(to, np.int32).t
        part = slice(first, end)
        for i in range(self.n_layer):
            K.kv_evict_paged(self.k[i], self.v[i], self.table[part], self.lengths[part], self.weights[i][part], to_dev,
                             self.keep, self.recent, lengths_out=self._lengths_to[part],
                             weights_out=self._weights_to[part])
            if end - first == self.batch:
                self.weights[i], self._weights_to = self._weights_to, self.weights[i]
            else:
                self.weights[i][part].copy_(self._weights_to[part])
        for b in cut:
            self._give_back(b, self._tab[b])
            self._tab[b, :need] = to[b - first]
            self._len[b] = self.keep

    # -- a layer's work ----------------------------------------------------------
    def append(self, layer, k, v):
        """Write the rows reserved last: k and v (B, n_head, T, head_dim), T the
        most that a sequence gets."""
        try:
            if k.shape[2] != self._rows:
                raise ValueError(f"append: {k.shape[2]} rows, {self._rows} reserved")
            K.kv_append_paged(k, v, self.k[layer], self.v[layer], self.table, self.lengths, counts=self.counts)
        except BaseException:
            self._abandon()
            raise
        self._written.add(layer)

    def attend(self, layer, q, scale, out=None):
        """Attention of one new token per sequence, q (B, H, 1, head_dim) with H
        a multiple of n_head, over the cached rows, whose weights it counts."""
        w = None if self.weights is None else self.weights[layer]
        lengths = self.lengths if self._active is None else self._active
        return K.attn_decode_paged(q, self.k[layer], self.v[layer], self.table, lengths, scale, out=out,
                                   weights=w, weights_in=w)[0]

    def observe(self, layer, q, scale):
        """Count the attention that a prompt's last positions, q
        (B, H, T, head_dim), pay its rows (with keep), in the sequences that got
        rows last."""
        if self.weights is None:
            return
        if self._ragged:
            raise ValueError("observe: prompts of one length")
        T = q.shape[2]
        n = min(self.observed, T)
        if layer == 0:  # the rows that each of those positions sees
            back = np.arange(n - 1, -1, -1, dtype=np.int32)[:, None]
            lengths = np.where(self._got, self._len, 0)
            self._seen = dev.from_host(np.maximum(lengths - back, 0), np.int32).t
        w = self.weights[layer]
        for i in range(n):
            t = T - n + i
            K.attn_decode_paged(q[:, :, t:t + 1], self.k[layer], self.v[layer], self.table, self._seen[i], scale,
                                weights=w, weights_in=w)
