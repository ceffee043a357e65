"""CPU checks: the host side of the paged cache over a fake device, and the plain implementations that the GPU tests compare with."""
import numpy as np
import pytest

import serving_reference as ref
from webgpt_b200 import _lib
from webgpt_b200.paged import PagedCache


class FakeBuffer:
    def __init__(self, nbytes):
        self.data, self.ptr, self.gone = np.zeros(nbytes, np.uint8), id(self), False

    def write(self, array, offset=0):
        raw = np.frombuffer(np.ascontiguousarray(array).tobytes(), np.uint8)
        assert offset + raw.size <= self.data.size
        self.data[offset:offset + raw.size] = raw
        return self

    def destroy(self):
        self.gone = True


class FakeDevice:
    handle = None

    def buffer(self, nbytes, dims=None):
        return FakeBuffer(nbytes)

    def tensor(self, array):
        return FakeBuffer(array.nbytes).write(array)


def state(c):
    table = c._tables[0].data.view(np.uint32).reshape(c.n_seq, c.width)
    return table, c._lengths[0].data.view(np.int32)


def check(c):
    """No page is lost or given out twice, and the device's table and lengths are the host's."""
    assert sorted(c.free + [p for s in c.pages for p in s]) == list(range(c.n_pages))
    table, lengths = state(c)
    assert np.array_equal(lengths, c.lengths)
    for s, p in enumerate(c.pages):
        assert len(p) == -(-int(c.lengths[s]) // c.page_size)
        assert list(table[s, :len(p)]) == p


def test_advance_retreat_release():
    c = PagedCache(FakeDevice(), 3, 2, 8, n_pages=10, page_size=4, max_length=24)
    check(c)
    c.advance([5, 0, 4])
    assert [len(p) for p in c.pages] == [2, 0, 1]
    c.advance(1)
    check(c)
    assert list(c.lengths) == [6, 1, 5]
    c.retreat([2, 1, 0])
    check(c)
    assert [len(p) for p in c.pages] == [1, 0, 2]
    c.release(2)
    check(c)
    assert list(c.lengths) == [4, 0, 0] and len(c.free) == 9
    starts = c.starts([2, 0, 3]).data.view(np.int32)
    assert list(starts) == [0, 2, 2, 5]


def test_refusals_change_nothing():
    c = PagedCache(FakeDevice(), 2, 1, 8, n_pages=4, page_size=4, max_length=12)
    c.advance([12, 1])
    for call, error in ((lambda: c.advance([1, 0]), ValueError), (lambda: c.advance([0, 4]), MemoryError),
                        (lambda: c.advance([0, -1]), ValueError), (lambda: c.retreat([13, 0]), ValueError),
                        (lambda: c.retreat(-1), ValueError), (lambda: c.evict(4, 1), ValueError)):
        with pytest.raises(error):
            call()
        check(c)
        assert list(c.lengths) == [12, 1]
    with pytest.raises(ValueError):
        PagedCache(FakeDevice(), 1, 1, 8, 4, type="f64")


def test_descriptor():
    c = PagedCache(FakeDevice(), 2, 3, 16, n_pages=4, page_size=5, type="f16", n_layer=2)
    d = c.layer(1).descriptor
    assert (d.page_stride, d.position_stride, d.head_stride) == (5 * 48, 48, 16)
    assert (d.type, d.n_pages, d.page_size, d.n_kv_head, d.head_size, d.n_seq) == (_lib.TYPE_F16, 4, 5, 3, 16, 2)
    assert d.table_stride * d.page_size >= d.max_length == 20
    assert c.layer(1, 1).descriptor.table != d.table and c.layer(1, 1).descriptor.k == d.k
    assert c._pools[0][0].data.size == 4 * 5 * 48 * 2
    c.destroy()
    assert all(b.gone for b in c._tables + c._lengths)


def test_descriptor_matches_the_header():
    import os
    import re
    from conftest import ROOT
    text = open(os.path.join(ROOT, "include", "webgpt_b200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct wgpt_paged_cache \{(.*?)\}", text, re.S).group(1), flags=re.S)
    names = [n.strip(" *") for line in body.split(";") for n in re.sub(r"^\s*(const\s+)?\w+", "", line).split(",") if n.strip(" *\n")]
    assert [n.strip() for n in names] == [f[0] for f in _lib.PagedCache._fields_]


# ------------------------------------------------------------------ the plain implementations
def test_reference_attention_against_a_whole_matrix():
    rng = np.random.default_rng(3)
    pages = ref.Pages(rng, [9, 0, 4], 3, 2, 8)
    pages.fill(rng, lambda x: x)
    q = rng.standard_normal((9, 4, 8)).astype(np.float32)
    starts = [1, 6, 6, 8]  # a row before and one behind the sequences
    out, weights, _, _ = ref.attend(pages, starts, 4, 0.5, 0, q)
    assert np.isnan(out[0]).all() and np.isnan(out[8]).all() and np.isfinite(out[1:8]).all()
    k, v = pages.rows("k", 0).astype(float), pages.rows("v", 0).astype(float)
    mask = np.tril(np.ones((9, 9)))[4:]
    for h in range(4):
        e = np.exp(0.5 * q[1:6, h].astype(float) @ k[:, h // 2].T) * mask
        assert np.allclose(out[1:6, h], e @ v[:, h // 2] / e.sum(1, keepdims=True))
    assert weights.sum() == pytest.approx(7 * 4) and weights[1].sum() == 0


def test_reference_attention_rows_that_see_nothing():
    rng = np.random.default_rng(4)
    pages = ref.Pages(rng, [2], 4, 1, 8)
    pages.fill(rng, lambda x: x)
    q = rng.standard_normal((4, 1, 8)).astype(np.float32)
    out = ref.attend(pages, [0, 4], 1, 1.0, 0, q)[0]
    assert (out[:2] == 0).all() and np.allclose(out[2, 0], pages.rows("v", 0)[0, 0])


def test_reference_verification_leaves_the_targets_distribution():
    """Whatever the draft proposes, the token that comes out has the target's probabilities: q(x) min(1, p(x) / q(x)) accepted,
    and the rest from max(p - q, 0)."""
    rng = np.random.default_rng(5)
    target, draft = rng.standard_normal((2, 5)) * 2, rng.standard_normal((1, 5)) * 2
    p, q = ref.distribution(target[0], 0, 0.7)[1], ref.distribution(draft[0], 0, 0.7)[1]
    got = np.zeros(5)
    grid = (np.arange(400) + 0.5) / 400
    for x in range(5):
        for a in grid[::4]:
            accepted, _ = ref.verify(target, draft, [x], 1, 0, 0.7, np.array([a, 0.5]))
            if accepted:
                got[x] += q[x] / 100
            else:
                for b in grid[::4]:
                    got[ref.verify(target, draft, [x], 1, 0, 0.7, np.array([a, b]))[1]] += q[x] / 10000
    assert np.abs(got - p).max() < 0.02


def test_reference_verification_known_answers():
    t = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]]))
    d = np.log(np.array([[0.25, 0.5, 0.25]]))
    assert ref.verify(t, d, [0], 1, 0, 1.0, np.array([0.999, 0.95])) == (1, 2)     # p > q: always accepted
    assert ref.verify(t, d, [1], 1, 0, 1.0, np.array([0.49, 0.15])) == (1, 1)      # accepted below p / q = 1/2
    assert ref.verify(t, d, [1], 1, 0, 1.0, np.array([0.51, 0.999])) == (0, 0)     # else only id 0 has p > q
    assert ref.verify(t, None, [2], 1, 0, 1.0, np.array([0.3, 0.7])) == (0, 1)     # q is one at the drafted id: p without it
    assert ref.verify(t, d, [1], 1, 1, 1.0, np.array([0.0, 0.0])) == (0, 0)        # greedy: the draft is not the best
    assert ref.verify(t, None, [0], 1, 1, 1.0, np.array([0.9, 0.0])) == (1, 2)
    bad = np.full((1, 3), -np.inf)
    assert ref.verify(np.vstack([bad, t[:1]]), d, [0], 1, 0, 1.0, np.array([0.0, 0.9])) == (0, 0)
    assert ref.verify(t, bad, [0], 1, 0, 1.0, np.array([0.0, 0.6])) == (0, 1)      # no draft distribution: drawn from p
    assert ref.verify(t, d, [7], 1, 0, 1.0, np.array([0.0, 0.0])) == (0, 0)


def test_reference_eviction():
    w = np.array([3.0, 1.0, np.nan, 1.0, 2.0, 0.0, 9.0], np.float32)
    assert ref.keep(w, 7, 4, 1) == [0, 2, 4, 6]
    assert ref.keep(w, 7, 5, 1) == [0, 1, 2, 4, 6]   # of the two ones, the first
    assert ref.keep(w, 7, 3, 3) == [4, 5, 6]
    assert ref.keep(w, 7, 2, 0) == [2, 6]
    assert ref.keep(w, 3, 3, 0) == [0, 1, 2]


def test_eviction_that_fails_changes_nothing(monkeypatch):
    """A call that fails in a later layer leaves pages, lengths and every layer's weights as they were."""
    class Readable(FakeBuffer):
        def read(self, dtype, count):
            return self.data.view(dtype)[:count]

    monkeypatch.setattr(FakeDevice, "buffer", lambda self, nbytes, dims=None: Readable(nbytes))
    c = PagedCache(FakeDevice(), 2, 1, 8, n_pages=12, page_size=4, max_length=16, n_layer=2, weights=True)
    c.advance([13, 5])
    for i in range(2):
        c.weights(i).write(np.arange(32, dtype=np.float32))
    calls = []

    def call(name, *args):
        calls.append(name)
        if len(calls) == 2:
            raise _lib.WgptError(_lib.ERR_SHAPE, "no")

    monkeypatch.setattr(_lib, "call", call)
    pages, weights = [list(p) for p in c.pages], [w.data.copy() for w in c._weights]
    with pytest.raises(_lib.WgptError):
        c.evict(4, 2)
    assert c.pages == pages and list(c.lengths) == [13, 5] and len(calls) == 2
    assert all(np.array_equal(w.data, before) for w, before in zip(c._weights, weights))
    check(c)
    for keep, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            c.evict(keep, recent)
    check(c)
