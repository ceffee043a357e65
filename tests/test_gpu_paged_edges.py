"""The paged cache's operators where the other tests do not look: full pools, offsets that make no sense, row tiles beside one another,
values that are not finite in long sequences, workspaces larger than memory."""
import ctypes as C
import math

import numpy as np
import pytest

import serving_reference as ref
from test_gpu_paged import OnDevice, attend, cast, check_attention, dev, make, reported, to_bits, to_f32  # noqa: F401 (dev: a fixture)
from webgpt_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["f32", "f16"])
def test_a_full_cache_is_thinned_out(dev, type):  # noqa: F811
    """One free page: the long sequences go one after the other, those that stay whole keep their pages."""
    from webgpt_b200.paged import PagedCache
    rng = np.random.default_rng(1)
    lengths, n_kv, hs, page, keep, recent = [5, 40, 37, 8, 64, 23, 8], 2, 16, 8, 8, 3
    used = sum(-(-L // page) for L in lengths)
    cache = PagedCache(dev, 7, n_kv, hs, n_pages=used + 1, page_size=page, type=type, n_layer=2, max_length=70, weights=True)
    cache.advance(lengths)
    width = n_kv * hs
    rows = [rng.standard_normal((sum(lengths), 2 * width)).astype(np.float32) for _ in range(2)]
    w = rng.integers(0, 30, (2, 7, 70)).astype(np.float32)
    for s, L in enumerate(lengths):
        w[:, s, L:] = 0
    starts = cache.starts(lengths)
    for i in range(2):
        b = dev.tensor(rows[i])
        _lib.call("wgpt_paged_append", dev.handle, cache.layer(i).ptr, sum(lengths), starts.ptr, b.ptr, b.ptr + 4 * width, 2 * width)
        cache.weights(i).write(w[i])
        dev.synchronize()
    kept = cache.evict(keep, recent)
    assert list(cache.lengths) == [min(L, keep) for L in lengths] and len(cache.free) == used + 1 - 7
    table = cache._tables[0].read(np.uint32).reshape(7, -1)
    assert list(cache._lengths[0].read(np.int32)) == list(cache.lengths)
    first = np.cumsum([0] + lengths)
    for i in range(2):
        pools = [to_f32(b.read(np.uint32 if type == "f32" else np.uint16), type).reshape(-1, page, width) for b in cache._pools[i]]
        got = cache.weights(i).read().reshape(7, 70)
        for s, L in enumerate(lengths):
            stay = ref.keep(w[i, s], L, keep, recent)
            assert list(kept[i, s]) == stay + [-1] * (keep - len(stay))
            assert list(got[s]) == list(w[i, s, stay]) + [0] * (70 - len(stay))
            at = np.arange(len(stay))
            for x, pool in enumerate(pools):
                want = cast(type)(rows[i][first[s] + np.array(stay), x * width:(x + 1) * width])
                assert np.array_equal(pool[table[s, at // page], at % page], want)
    _lib.call("wgpt_device_check", dev.handle)
    cache.destroy()


@pytest.mark.parametrize("type,n_head", [("f32", 1), ("f16", 1), ("bf16", 12)])
def test_windows_past_every_length(dev, type, n_head):  # noqa: F811
    """A window that no sequence fills is none, up to the largest number, also for sequences shorter than their new tokens."""
    rng = np.random.default_rng(2)
    pages = make(rng, [300, 200, 3], 16, 1, 64, type)
    for window in (301, 1 << 30, (1 << 31) - 1):
        check_attention(dev, pages, type, "positions", [303, 205, 9], n_head, window=window, weights=True)


@pytest.mark.parametrize("type,n_head,n_seq", [("f32", 1, 3), ("f16", 1, 20), ("f16", 12, 20), ("f32", 1, 1024), ("f16", 1, 1024), ("bf16", 16, 1024)])
def test_offsets_that_decrease(dev, type, n_head, n_seq):  # noqa: F811
    """Sequences that would share rows: nothing is computed, nothing out of range is touched, and the call is reported. The rows
    of all of them together times their tiles do not fit 32 bits at 1024 sequences: 512 x 1024 rows of 8192 units and more."""
    rng = np.random.default_rng(3)
    pages = make(rng, [17] * n_seq, 16, 1, 64, type, max_length=1 << 20)
    c = OnDevice(dev, pages, type)
    c.lengths.write(np.full(n_seq, 1 << 20, np.int32))  # pages that are not there are not seen
    q = rng.standard_normal((n_seq, n_head, 64)).astype(np.float32)
    alternating = [0, n_seq] * (n_seq // 2 + 1)
    for starts in (alternating[:n_seq + 1], [n_seq - i for i in range(n_seq + 1)], list(range(n_seq)) + [n_seq - 2]):
        got, _ = attend(dev, c, starts, n_seq, n_head, 0.125, 0, q)
        assert (got == 7.0).all()
        reported(dev)
    small = OnDevice(dev, make(rng, [9] * n_seq, 16, 1, 64, type), type)
    w0 = rng.random((n_seq, 9)).astype(np.float32)
    got, w = attend(dev, small, alternating[:n_seq + 1], n_seq, n_head, 0.125, 0, q, w0)
    assert (got == 7.0).all() and np.array_equal(w, w0)
    reported(dev)
    attend(dev, small, list(range(n_seq + 1)), n_seq, n_head, 0.125, 0, q, w0)
    _lib.call("wgpt_device_check", dev.handle)


@pytest.mark.parametrize("type,n_kv,group,hs,new", [("f16", 2, 12, 64, 1), ("f16", 2, 4, 128, 6), ("bf16", 2, 16, 64, 1), ("bf16", 1, 3, 128, 9), ("f16", 2, 1, 64, 1),
                                                    ("bf16", 1, 8, 128, 1), ("f32", 2, 2, 64, 1), ("f16", 1, 4, 256, 2)])
def test_values_that_are_not_finite_in_long_sequences(dev, type, n_kv, group, hs, new):  # noqa: F811
    """Sequences of thousands of positions beside many short ones, each of the long ones with a value that is not finite: rows that
    see it get it, rows that do not and other sequences stay as good as ever, and no wait runs out meanwhile."""
    rng = np.random.default_rng(4)
    lengths = [6000, 9000] + [int(x) for x in rng.integers(new, 300, 90)] + [7001]
    pages = make(rng, lengths, 16, n_kv, hs, type)
    n_head = n_kv * group
    starts = [new * s for s in range(len(lengths) + 1)]
    q = (rng.standard_normal((starts[-1], n_head, hs)) * 1.5).astype(np.float32)
    want, _, size, top = ref.attend(pages, starts, n_head, 0.125, 2500, q)
    pages.v[pages.place(0, 5990)][0, 3] = np.inf        # in every row's window
    pages.v[pages.place(1, 100)] = np.nan               # in no row's window nor tiles
    pages.v[pages.place(1, 9000 - 2500 - new)] = -np.inf  # just before the first row's
    pages.k[pages.place(92, 7001 - 2500 + 1 - new)] = np.nan  # in the first row's alone
    cache = OnDevice(dev, pages, type)
    got, _ = attend(dev, cache, starts, starts[-1], n_head, 0.125, 2500, q)
    _lib.call("wgpt_device_check", dev.handle)
    assert (got[:new, :group, 3] == np.inf).all()
    got[:new, :group, 3] = want[:new, :group, 3]
    first = starts[92]
    assert np.isnan(got[first]).all()
    got[first] = want[first]
    assert (np.abs(got - want) <= ref.attend_tolerance(pages, size, top)).all()


@pytest.mark.parametrize("type,group", [("f16", 12), ("f16", 1), ("f32", 1)])
def test_many_sequences_without_new_tokens(dev, type, group):  # noqa: F811
    """Two sequences with new tokens and tens of thousands without between them: a CTA that has a part of both looks for its next one
    for a long time."""
    n_seq, hs = 65535, 64
    rng = np.random.default_rng(5)
    lengths = [150] + [0] * (n_seq - 2) + [170]
    pages = make(rng, lengths, 16, 1, hs, type)
    starts = [0] + [1] * (n_seq - 1) + [2]
    q = rng.standard_normal((2, group, hs)).astype(np.float32)
    c = OnDevice(dev, pages, type)
    for _ in range(2):
        got, _ = attend(dev, c, starts, 2, group, 0.125, 0, q)
    few = ref.Pages(rng, [150, 170], 16, 1, hs)
    for which in ("k", "v"):
        for at, s in enumerate((0, n_seq - 1)):
            for j in range(lengths[s]):
                getattr(few, which)[few.place(at, j)] = getattr(pages, which)[pages.place(s, j)]
    want, _, size, top = ref.attend(few, [0, 1, 2], group, 0.125, 0, q)
    assert (np.abs(got - want) <= ref.attend_tolerance(few, size, top)).all()
    _lib.call("wgpt_device_check", dev.handle)


@pytest.mark.parametrize("type,n_kv,group,hs,window", [("f32", 8, 1, 64, 0), ("f16", 2, 4, 64, 30), ("bf16", 1, 12, 128, 0), ("f16", 1, 8, 256, 0), ("f16", 1, 16, 64, 17)])
def test_scores_of_more_than_the_workspace_holds(dev, type, n_kv, group, hs, window):  # noqa: F811
    """2^20 positions a sequence at most: 32 rows of eight heads take a gigabyte. A call of more rows is cut, inside sequences too."""
    rng = np.random.default_rng(6)
    lengths, new = [40, 3, 90, 0, 300, 61], [20, 9, 1, 2, 33, 30]
    pages = make(rng, lengths, 16, n_kv, hs, type, max_length=1 << 20)
    free = dev.mem_info()[0]
    check_attention(dev, pages, type, "positions", new, n_kv * group, window=window, weights=True, before=1, behind=3)
    assert free - dev.mem_info()[0] < 3 << 29  # 95 rows whole: 3 GB
    check_attention(dev, pages, type, "positions", [1, 1, 1, 0, 1, 1], n_kv * group, window=window, weights=True)
    _lib.call("wgpt_device_check", dev.handle)


@pytest.mark.parametrize("type,n_kv,group,hs", [("f16", 2, 3, 64), ("bf16", 1, 5, 128), ("f16", 1, 20, 40), ("bf16", 2, 1, 72), ("f32", 1, 3, 64), ("f16", 1, 2, 256)])
@pytest.mark.parametrize("window", [0, 200])
def test_prompts_behind_contexts(dev, type, n_kv, group, hs, window):  # noqa: F811
    """Many row tiles over many key tiles each: tiles that begin and end at different units, parts without any, joins of unequal parts."""
    rng = np.random.default_rng(7)
    pages = make(rng, [1500, 260, 700, 129], 32, n_kv, hs, type)
    check_attention(dev, pages, type, "heads", [170, 260, 90, 1], n_kv * group, window=window, weights=True, before=1, behind=1)


@pytest.mark.parametrize("type,group,hs", [("f32", 1, 64), ("f32", 8, 64), ("f16", 1, 64), ("f16", 8, 128), ("f16", 12, 64), ("f16", 20, 128), ("bf16", 1, 64),
                                           ("bf16", 8, 128), ("bf16", 12, 64), ("bf16", 20, 128), ("f16", 9, 256), ("bf16", 9, 256)])
def test_queries_and_probabilities_are_as_good_as_f32(dev, type, group, hs):  # noqa: F811
    """Keys and values of the unit vectors and a scale of one: the output is the softmax of the query itself, whose products and
    sums of values are exact. What is left, in halves of an f32 step: a score s is the query's value times log2 e in f32 (two roundings), the
    difference to a maximum (one), all times s; an exponential (four: 2^-22); a probability and the sum it is divided by have these
    (twice); additions of the sum over lanes, tiles and key groups, rescalings, the quotient: up to 28. Half-precision queries are two
    values, good to 2^-22 of the row's largest, four steps of it. Third terms of bfloat16 queries that are left out are 2^-18 of the query:
    64 steps times s; of probabilities likewise 64, on average 37, of which the root of the mean square shows more than a tenth."""
    rng = np.random.default_rng(8)
    pages = ref.Pages(rng, [hs], 16, 1, hs)
    for j in range(hs):
        for pool in (pages.k, pages.v):
            pool[pages.place(0, j)] = np.eye(hs, dtype=np.float32)[j]
    cache = OnDevice(dev, pages, type)
    for low, high in ((12.0, 16.0), (-1.0, 1.0)):
        q = rng.uniform(low, high, (1, group, hs)).astype(np.float32)
        got, _ = attend(dev, cache, None, 1, group, 1.0, 0, q)
        e = np.exp(q.astype(np.float64) - q.max(-1, keepdims=True))
        want = e / e.sum(-1, keepdims=True)
        off = np.abs(got / want - 1) / ref.U32
        most = 2 * (6 * max(abs(low), high) + 4) + 28 + (2 * 4 * 16 if type == "f16" and high > 2 else 8 if type == "f16" else 0)
        assert off.max() <= most
        if high < 2:
            # some 50 roundings, each of a mean square of a third of a half step's: four steps, three times over
            assert math.sqrt((off ** 2).mean()) <= 12


def test_a_step_while_a_pass_list_is_recorded(dev):  # noqa: F811
    """What waits for the device is refused there, and the cache stays as it was."""
    from webgpt_b200.paged import PagedCache
    cache = PagedCache(dev, 2, 1, 8, n_pages=8, page_size=4, n_layer=1, weights=True)
    cache.advance([5, 9])
    before = [list(p) for p in cache.pages], list(cache.free), list(cache.lengths)
    g = C.c_void_p()
    _lib.call("wgpt_graph_begin", dev.handle)
    for step in (lambda: cache.advance(1), lambda: cache.retreat([1, 0]), lambda: cache.release(1), lambda: cache.evict(4, 1)):
        with pytest.raises(_lib.WgptError) as e:
            step()
        assert e.value.code == _lib.ERR_STATE
        assert (cache.pages, cache.free, list(cache.lengths)) == before
    _lib.call("wgpt_graph_end", dev.handle, C.byref(g))
    _lib.call("wgpt_graph_destroy", dev.handle, g)
    cache.retreat([1, 2])
    assert list(cache._lengths[0].read(np.int32)) == [4, 7]
    cache.destroy()
