"""Host side of the paged key-value cache: which pages each sequence has, and how long it is.

The pools, the page table and the lengths lie on the device, where wgpt_paged_append / _attention / _evict read them; this
class keeps the free pages and a mirror of table and lengths, and hands out the descriptors. All layers share one table.
A step is: advance() by the new tokens, append and attend per layer, retreat() by the drafts that were not accepted.
With weights, attention adds those of all new tokens up, of drafts too: a retreat clears those of the positions that it drops, not
what the dropped tokens gave to others.
"""
import ctypes as C

import numpy as np

from . import _lib

_TYPES = {"f32": (_lib.TYPE_F32, 4), "f16": (_lib.TYPE_F16, 2), "bf16": (_lib.TYPE_BF16, 2)}


class Layer:
    """One layer's cache as the operator calls take it (`ptr`: the descriptor's address, read during each call)."""

    def __init__(self, owner, descriptor):
        self._owner = owner  # its buffers have to outlive the descriptor
        self.descriptor = descriptor
        self.ptr = C.byref(descriptor)
        self.head_size, self.n_kv_head = descriptor.head_size, descriptor.n_kv_head
        self.n_seq, self.max_length = descriptor.n_seq, descriptor.max_length


class PagedCache:
    def __init__(self, device, n_seq, n_kv_head, head_size, n_pages, page_size=16, type="f16", n_layer=1, max_length=None,
                 weights=False):
        """n_pages pages of page_size positions for all sequences together, per layer; no sequence longer than max_length
        (default: what all pages hold). weights: keep each position's accumulated attention weight, which evict() goes by."""
        if type not in _TYPES:
            raise ValueError(f"unknown cache type {type!r}: one of {', '.join(_TYPES)}")
        self.type, elem = _TYPES[type]
        self.device, self.n_seq, self.n_layer = device, n_seq, n_layer
        self.n_pages, self.page_size = n_pages, page_size
        self.max_length = n_pages * page_size if max_length is None else max_length
        self.width = -(-self.max_length // page_size)
        self.lengths = np.zeros(n_seq, np.int32)
        self.pages = [[] for _ in range(n_seq)]
        self.free = list(range(n_pages - 1, -1, -1))
        self._shape = (n_kv_head, head_size)
        nbytes = n_pages * page_size * n_kv_head * head_size * elem
        # every buffer once more for evict(): a table and lengths to write to beside those that are read
        self._tables = [device.buffer(n_seq * self.width * 4) for _ in range(2)]
        self._lengths = [device.buffer(n_seq * 4) for _ in range(2)]
        self._pools = [(device.buffer(nbytes), device.buffer(nbytes)) for _ in range(n_layer)]
        self._weights = [device.buffer(n_seq * self.max_length * 4) for _ in range(n_layer)] if weights else None
        for b in self._weights or []:
            b.write(np.zeros(n_seq * self.max_length, np.float32))
        self._take_over(self.pages, self.lengths)

    # ------------------------------------------------------------------ what the calls take
    def layer(self, i=0, which=0, first=0, count=None):
        """The descriptor of layer i's cache (which = 1: the one that evict() writes to), of `count` sequences from `first` on."""
        k, v = self._pools[i]
        n_kv, hs = self._shape
        count = self.n_seq - first if count is None else count
        return Layer(self, _lib.PagedCache(k.ptr, v.ptr, self._tables[which].ptr + first * self.width * 4,
                                           self._lengths[which].ptr + first * 4, self.page_size * n_kv * hs, n_kv * hs, hs,
                                           self.type, self.n_pages, self.page_size, n_kv, hs, count, self.width, self.max_length))

    def weights(self, i=0):
        """Layer i's accumulated weights, [n_seq, max_length]."""
        return self._weights[i]

    # ------------------------------------------------------------------ lengths
    def advance(self, new):
        """Makes room for new[s] more tokens of each sequence (a number: as many for each). Changes nothing if a sequence
        would grow past max_length or there are too few pages."""
        new = self._each(new)
        want = self.lengths + new
        if (want > self.max_length).any():
            raise ValueError(f"a sequence would hold {int(want.max())} positions, more than max_length {self.max_length}")
        need = [-(-int(L) // self.page_size) - len(p) for L, p in zip(want, self.pages)]
        if sum(need) > len(self.free):
            raise MemoryError(f"{sum(need)} pages are needed, {len(self.free)} are free")
        free = list(self.free)
        self._take_over([p + [free.pop() for _ in range(n)] for p, n in zip(self.pages, need)], want)
        self.free = free

    def retreat(self, by):
        """Drops the by[s] newest positions of each sequence (a number: as many of each)."""
        by = np.broadcast_to(np.asarray(by, np.int64), (self.n_seq,))
        if (by < 0).any() or (by > self.lengths).any():
            raise ValueError("a sequence cannot retreat by a negative number of positions or past its beginning")
        want = self.lengths - by
        for s in np.flatnonzero(by):
            for w in self._weights or []:
                w.write(np.zeros(int(by[s]), np.float32), offset=int(s * self.max_length + want[s]) * 4)
        held = [-(-int(L) // self.page_size) for L in want]
        gone = [x for p, n in zip(self.pages, held) for x in p[n:]]
        # the table stays: what lies behind a sequence's last page is not read
        self._take_over([p[:n] for p, n in zip(self.pages, held)], want, table=False)
        self.free += gone

    def release(self, s):
        """Ends sequence s: its pages are free again."""
        by = np.zeros(self.n_seq, np.int64)
        by[s] = self.lengths[s]
        self.retreat(by)

    def starts(self, new):
        """The starts array of a step of new[s] tokens per sequence (a number: as many for each), on the device."""
        return self.device.tensor(np.concatenate([[0], np.cumsum(self._each(new))]).astype(np.int32))

    # ------------------------------------------------------------------ eviction
    def evict(self, keep, recent):
        """Thins out the sequences that hold more than keep positions, in every layer by its own weights; returns the
        positions that stayed, [n_layer, n_seq, min(keep, max_length)], -1 behind them. Sequences of up to keep positions
        stay as they are. What stays of the others goes to free pages: needs as many as one sequence of keep positions
        has. As many sequences as there are pages for are thinned out together; a failure leaves those whole whose turn
        had not come."""
        if self._weights is None:
            raise ValueError("the cache keeps no weights: create it with weights=True")
        keep, recent = int(keep), int(recent)
        if keep < 1 or not 0 <= recent <= keep:
            raise ValueError(f"keep {keep} and recent {recent}: 0 <= recent <= keep, keep >= 1")
        keep = min(keep, self.max_length)  # no sequence is longer
        each = -(-keep // self.page_size)
        long = [int(s) for s in np.flatnonzero(self.lengths > keep)]
        if long and each > len(self.free):
            raise MemoryError(f"{each} pages are needed, {len(self.free)} are free")
        stayed = np.where(np.arange(keep) < self.lengths[:, None], np.arange(keep), -1).astype(np.int32)
        stayed = np.tile(stayed, (self.n_layer, 1, 1))
        while long:  # each sequence gives back as many pages as it takes, or more
            n = len(self.free) // each
            self._thin_out(long[:n], keep, recent, stayed)
            long = long[n:]
        return stayed

    def _thin_out(self, sequences, keep, recent, stayed):
        """evict() of these, all longer than keep; free pages are enough. Nothing changes unless all layers' calls go through."""
        free = list(self.free)
        pages = [list(p) for p in self.pages]
        for s in sequences:
            pages[s] = [free.pop() for _ in range(-(-keep // self.page_size))]
        # consecutive sequences share a call: (where they begin among `sequences`, the first, how many)
        runs = []
        for at, s in enumerate(sequences):
            if runs and s == runs[-1][1] + runs[-1][2]:
                runs[-1][2] += 1
            else:
                runs.append([at, s, 1])
        row = self.max_length * 4
        self._tables[1].write(self._table_of(pages))  # first: where it is refused, so is giving buffers back
        got, moved, kept = [], [], None
        try:
            kept = self.device.buffer(len(sequences) * keep * 4)
            for _ in range(self.n_layer):  # the weights that stay, zeros behind them
                moved.append(self.device.buffer(len(sequences) * row))
                moved[-1].write(np.zeros(len(sequences) * self.max_length, np.float32))
            for i in range(self.n_layer):
                for at, s, n in runs:
                    _lib.call("wgpt_paged_evict", self.device.handle, self.layer(i, 0, s, n).ptr, self.layer(i, 1, s, n).ptr, keep, recent,
                              self._weights[i].ptr + s * row, self.max_length, moved[i].ptr + at * row, self.max_length,
                              kept.ptr + at * keep * 4)
                got.append(kept.read(np.int32, len(sequences) * keep).reshape(-1, keep))
            lengths = self.lengths.copy()
            lengths[sequences] = keep
            old = [x for s in sequences for x in self.pages[s]]
            self._take_over(pages, lengths)
            self.free = free + old
            stayed[:, sequences] = np.stack(got)
            for w, m in zip(self._weights, moved):
                for at, s, n in runs:
                    self.device.copy(m, at * row, w, s * row, n * row)
        finally:
            for b in [kept] * (kept is not None) + moved:
                b.destroy()

    # ------------------------------------------------------------------ inside
    def _each(self, new):
        new = np.broadcast_to(np.asarray(new, np.int64), (self.n_seq,))
        if (new < 0).any():
            raise ValueError("a sequence cannot advance by a negative number of tokens: use retreat()")
        return new

    def _table_of(self, pages):
        table = np.zeros((self.n_seq, self.width), np.uint32)
        for s, p in enumerate(pages):
            table[s, :len(p)] = p
        return table

    def _take_over(self, pages, lengths, table=True):
        """Makes these the cache's pages and lengths, on the device and here; a write that fails leaves the old ones."""
        lengths = np.asarray(lengths, np.int32)
        try:
            if table:
                self._tables[0].write(self._table_of(pages))
            self._lengths[0].write(lengths)
        except Exception:
            if table:
                self._tables[0].write(self._table_of(self.pages))
            raise
        self.pages = pages
        self.lengths[:] = lengths

    def destroy(self):
        for b in self._tables + self._lengths + [x for p in self._pools for x in p] + (self._weights or []):
            b.destroy()
