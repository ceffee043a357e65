"""CPU checks of PagedCache's steps over a fake device: what they hand to the kernels, and what is left when one of them fails."""
import numpy as np
import pytest

from test_paged import FakeBuffer, FakeDevice, check, state  # noqa: F401
from webgpt_b200.paged import PagedCache


def test_starts_has_a_number_for_every_sequence():
    """The kernels read n_seq + 1 numbers: a number of tokens stands for all sequences, as in advance(), and nothing else fits."""
    c = PagedCache(FakeDevice(), 3, 1, 8, n_pages=12, page_size=4)
    for new in (2, np.int64(2), [2, 2, 2], np.array([2, 2, 2], np.int32)):
        assert list(c.starts(new).data.view(np.int32)) == [0, 2, 4, 6]
    assert list(c.starts([2]).data.view(np.int32)) == [0, 2, 4, 6]
    assert list(c.starts(0).data.view(np.int32)) == [0, 0, 0, 0]
    for new in ([1, 2], [1, 2, 3, 4], [[1, 2, 3], [1, 2, 3]], [1, -1, 1], -1):
        with pytest.raises(ValueError):
            c.starts(new)


class Failing(FakeDevice):
    """A device whose n-th allocation or write from now on fails, and no other."""
    left = None

    def step(self):
        if self.left is not None:
            self.left -= 1
            if self.left < 0:
                self.left = None
                raise OSError("no")

    def buffer(self, nbytes, dims=None):
        self.step()
        device = self

        class Buffer(FakeBuffer):
            def write(self, array, offset=0):
                device.step()
                return super().write(array, offset)

            def read(self, dtype, count, offset=0):
                return self.data[offset:offset + count * np.dtype(dtype).itemsize].view(dtype).copy()

        b = Buffer(nbytes)
        b.nbytes = nbytes
        self.made = getattr(self, "made", []) + [b]
        return b


    def copy(self, src, src_offset, dst, dst_offset, size):  # only enqueues
        assert not src.gone and not dst.gone
        dst.data[dst_offset:dst_offset + size] = src.data[src_offset:src_offset + size]


def attempts(c, call, untouched):
    """Lets each allocation and write of the call fail in turn: the cache stays what it was. Then the call is made."""
    for n in range(100):
        before = list(c.free), [list(p) for p in c.pages], list(c.lengths)
        c.device.left = n
        try:
            call()
        except OSError:
            c.device.left = None
            assert (list(c.free), c.pages, list(c.lengths)) == before
            check(c)
            untouched()
            continue
        c.device.left = None
        check(c)
        return n
    raise AssertionError("too many steps")


def test_steps_that_fail_change_nothing():
    c = PagedCache(Failing(), 3, 1, 8, n_pages=20, page_size=4, max_length=30, weights=True)
    assert attempts(c, lambda: c.advance([9, 1, 17]), lambda: None) >= 2
    assert attempts(c, lambda: c.retreat([0, 1, 9]), lambda: None) >= 2
    assert attempts(c, lambda: c.release(0), lambda: None) >= 2
    assert list(c.lengths) == [0, 0, 8]


def keeper(monkeypatch, c, calls=None):
    """Stands in for wgpt_paged_evict on the fake device: the first keep - recent positions and the newest stay."""
    from webgpt_b200 import _lib
    buffers = lambda: {b.ptr: b for b in c.device.made}  # noqa: E731

    def find(ptr):
        for base, b in buffers().items():
            if base <= ptr < base + max(1, b.data.size):
                return b.data[ptr - base:]
        raise AssertionError("an address of no buffer")

    def call(name, handle, src, dst, keep, recent, w, ld, wt, ld_to, kept):
        c.device.step()
        assert name == "wgpt_paged_evict"
        a, b = src._obj, dst._obj
        if calls is not None:
            calls.append((a.n_seq, a.k))
        assert (a.max_length, a.table_stride, a.page_size, a.k) == (b.max_length, b.table_stride, b.page_size, b.k) and a.table != b.table
        lengths, to = find(a.lengths).view(np.int32)[:a.n_seq], find(b.lengths).view(np.int32)[:a.n_seq]
        pages = [find(x.table).view(np.uint32)[:a.n_seq * x.table_stride].reshape(a.n_seq, -1) for x in (a, b)]
        old, new = set(), set()
        for s, L in enumerate(lengths):
            n = min(L, keep)
            stay = list(range(L)) if L <= keep else list(range(keep - recent)) + list(range(L - recent, L))
            row = find(kept).view(np.int32)[s * keep:(s + 1) * keep]
            row[:n], row[n:] = stay, -1
            x, y = find(w).view(np.float32)[s * ld:], find(wt).view(np.float32)[s * ld_to:]
            y[:n], y[n:keep] = x[stay], 0
            old |= set(pages[0][s, :-(-int(L) // a.page_size)])
            new |= set(pages[1][s, :-(-int(n) // a.page_size)])
            to[s] = n
        assert not old & new and new <= set(c.free) and max(new) < c.n_pages  # nothing is moved in place

    monkeypatch.setattr(_lib, "call", call)


class Addresses(Failing):
    """Buffers with addresses far apart."""

    def buffer(self, nbytes, dims=None):
        b = super().buffer(nbytes, dims)
        b.ptr = len(self.made) << 32
        return b


def test_eviction_that_fails_anywhere_loses_no_page(monkeypatch):
    c = PagedCache(Addresses(), 3, 1, 8, n_pages=30, page_size=4, max_length=30, n_layer=2, weights=True)
    keeper(monkeypatch, c)
    c.advance([25, 3, 18])
    for i in range(2):
        c.weights(i).write(np.arange(90, dtype=np.float32) + i)
    made = len(c.device.made)
    before = [w.data.copy() for w in c._weights]

    def untouched():
        assert all(np.array_equal(w.data, x) for w, x in zip(c._weights, before))

    assert attempts(c, lambda: c.evict(8, 3), untouched) >= 7
    assert all(b.gone for b in c.device.made[made:])  # what the call allocated is given back, failed or not
    assert list(c.lengths) == [8, 3, 8] and len(c.free) == 30 - 5
    for i in range(2):
        w = c.weights(i).data.view(np.float32).reshape(3, 30)
        assert list(w[0]) == [x + i for x in (0, 1, 2, 3, 4, 22, 23, 24)] + [0] * 22
        assert list(w[1][:3]) == [30 + i, 31 + i, 32 + i]
        assert list(w[2]) == [60 + x + i for x in (0, 1, 2, 3, 4, 15, 16, 17)] + [0] * 22


def test_a_full_cache_is_thinned_out(monkeypatch):
    """Sequences that stay whole keep their pages and are not copied; the others go some at a time where few pages are free."""
    calls = []
    c = PagedCache(Addresses(), 6, 1, 8, n_pages=40, page_size=4, max_length=60, n_layer=2, weights=True)
    keeper(monkeypatch, c, calls)
    c.advance([7, 40, 33, 8, 28, 29])  # 2 + 10 + 9 + 2 + 7 + 8 pages: two are free
    for i in range(2):
        c.weights(i).write(np.arange(360, dtype=np.float32) + 1000 * i)
    assert len(c.free) == 2
    short = [list(c.pages[0]), list(c.pages[3])]
    kept = c.evict(8, 2)
    check(c)
    assert list(c.lengths) == [7, 8, 8, 8, 8, 8] and [c.pages[0], c.pages[3]] == short and len(c.free) == 40 - 12
    assert [n for n, _ in calls] == [1, 1, 1, 2, 1, 2]  # in both layers one sequence at first, then all that is left, run by run
    assert kept.shape == (2, 6, 8)
    for i in range(2):
        assert kept[i].tolist() == [[0, 1, 2, 3, 4, 5, 6, -1], [0, 1, 2, 3, 4, 5, 38, 39], [0, 1, 2, 3, 4, 5, 31, 32], list(range(8)),
                                    [0, 1, 2, 3, 4, 5, 26, 27], [0, 1, 2, 3, 4, 5, 27, 28]]
        w = c.weights(i).data.view(np.float32).reshape(6, 60)
        assert list(w[0]) == list(np.arange(60) + 1000 * i)  # untouched
        assert list(w[5]) == [300 + x + 1000 * i for x in kept[i, 5]] + [0] * 52
    # nothing longer than keep: no call, no page needed
    c.advance([0, 0, 0, 0, 0, 52])
    c.advance([0, 0, 52, 0, 0, 0])
    del calls[:]
    assert len(c.free) == 2
    assert c.evict(60, 0).shape == (2, 6, 60) and not calls
    # no room for a single one
    with pytest.raises(MemoryError):
        c.evict(12, 0)
    check(c)
    assert not calls and list(c.lengths) == [7, 8, 60, 8, 8, 60]


def test_keep_past_the_longest_sequence(monkeypatch):
    """0 <= recent <= keep is all that is asked: a keep that no sequence can pass thins nothing out, whatever recent is."""
    c = PagedCache(Addresses(), 2, 1, 8, n_pages=8, page_size=4, max_length=16, weights=True)
    c.advance([9, 3])
    for keep, recent in ((100, 100), (100, 17), (17, 16), (16, 16)):
        kept = c.evict(keep, recent)
        assert kept.shape == (1, 2, 16) and kept[0].tolist() == [list(range(9)) + [-1] * 7, list(range(3)) + [-1] * 13]
    for keep, recent in ((100, 101), (0, 0), (5, -1)):
        with pytest.raises(ValueError):
            c.evict(keep, recent)


def test_an_eviction_that_is_refused_allocates_nothing(monkeypatch):
    """While a pass list is being recorded writes are refused, and so is giving buffers back: none may have been made by then."""
    c = PagedCache(Addresses(), 1, 1, 8, n_pages=8, page_size=4, max_length=16, weights=True)
    keeper(monkeypatch, c)
    c.advance(12)

    def refused(self, array, offset=0):
        raise OSError("recording")

    made = len(c.device.made)
    monkeypatch.setattr(FakeBuffer, "write", refused)
    with pytest.raises(OSError):
        c.evict(4, 1)
    assert len(c.device.made) == made
