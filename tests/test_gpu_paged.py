"""The paged cache's operators through the C ABI: append, attention and eviction against plain 64-bit implementations."""
import ctypes as C
import math

import numpy as np
import pytest

import serving_reference as ref
from webgpt_b200 import _lib

pytestmark = pytest.mark.gpu

TYPE = {"f32": _lib.TYPE_F32, "f16": _lib.TYPE_F16, "bf16": _lib.TYPE_BF16}


@pytest.fixture(scope="module")
def dev():
    from webgpt_b200 import Device
    d = Device(0)
    yield d
    d.destroy()


def to_bits(x, type):
    """f32 values as the bits of the cache's type, rounded to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if type == "f32":
        return x.view(np.uint32)
    if type == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def to_f32(bits, type):
    if type == "f32":
        return bits.view(np.float32)
    return bits.view(np.float16).astype(np.float32) if type == "f16" else (bits.astype(np.uint32) << 16).view(np.float32)


def cast(type):
    return lambda x: to_f32(to_bits(x, type), type)


class OnDevice:
    """A reference cache's pools, table and lengths on the device, and the descriptor."""

    def __init__(self, dev, pages, type, layout="positions"):
        self.type, self.layout, self.pages = type, layout, pages
        swap = (lambda x: x) if layout == "positions" else (lambda x: x.transpose(0, 2, 1, 3))
        self.shape = swap(pages.k).shape
        self.k, self.v = (dev.tensor(to_bits(swap(p), type)) for p in (pages.k, pages.v))
        self.table, self.lengths = dev.tensor(pages.table), dev.tensor(np.array(pages.lengths, np.int32))
        P, kv, hs = pages.page_size, pages.n_kv, pages.hs
        strides = (P * kv * hs, kv * hs, hs) if layout == "positions" else (P * kv * hs, hs, P * hs)
        self.d = _lib.PagedCache(self.k.ptr, self.v.ptr, self.table.ptr, self.lengths.ptr, *strides, TYPE[type], pages.n_pages, P, kv, hs,
                                 len(pages.lengths), pages.width, pages.max_length)
        self.ptr = C.byref(self.d)

    def pools(self):
        got = []
        for b in (self.k, self.v):
            x = to_f32(b.read(np.uint32 if self.type == "f32" else np.uint16), self.type).reshape(self.shape)
            got.append(x if self.layout == "positions" else x.transpose(0, 2, 1, 3))
        return got


def attend(dev, cache, starts, n_rows, n_head, scale, window, q, weights=None, ld_q=None, ld_out=None, untouched=7.0):
    hs = cache.pages.hs
    E = n_head * hs
    ld_q, ld_out = ld_q or E, ld_out or E
    rows = np.zeros((n_rows, ld_q), np.float32)
    rows[:, :E] = q.reshape(n_rows, E)
    qb, ob = dev.tensor(rows), dev.tensor(np.full((n_rows, ld_out), untouched, np.float32))
    sb = dev.tensor(np.array(starts, np.int32)) if starts is not None else None
    wb = dev.tensor(weights) if weights is not None else None
    _lib.call("wgpt_paged_attention", dev.handle, cache.ptr, n_rows, sb.ptr if sb else None, n_head, scale, window, qb.ptr, ld_q, ob.ptr,
              ld_out, wb.ptr if wb else None, weights.shape[1] if wb else 0)
    out = ob.read().reshape(n_rows, ld_out)
    assert (out[:, E:] == untouched).all()
    return out[:, :E].reshape(n_rows, n_head, hs), (wb.read().reshape(weights.shape) if wb else None)


def check_attention(dev, pages, type, layout, new, n_head, window=0, weights=False, seed=0, before=0, behind=0, q=None, scale=None,
                    **kw):
    """One call against the 64-bit result, every row at its own tolerance."""
    rng = np.random.default_rng(seed + 1)
    starts = [before] + list(before + np.cumsum(new))
    n_rows = starts[-1] + behind
    if q is None:
        q = (rng.standard_normal((n_rows, n_head, pages.hs)) * 1.5).astype(np.float32)
    scale = 1 / math.sqrt(pages.hs) if scale is None else scale
    cache = OnDevice(dev, pages, type, layout)
    w0 = rng.random((len(pages.lengths), pages.max_length)).astype(np.float32) if weights else None
    got, w = attend(dev, cache, starts, n_rows, n_head, scale, window, q, w0, **kw)
    want, dw, size, top = ref.attend(pages, starts, n_head, np.float32(scale).astype(np.float64), window, q)
    mine = ~np.isnan(want)
    assert (got[~mine] == 7.0).all()
    tol = ref.attend_tolerance(pages, size, top)
    off = np.abs(got - want)
    assert (off[mine] <= tol[mine]).all(), (off[mine] / tol[mine]).max()
    if weights:
        # each probability is off as in the output's tolerance, one rounding for each of the terms, and one of the sum
        L, terms = max(pages.lengths), max(new) * n_head
        rel = 4 * (pages.hs + 10) * ref.U32 * np.nanmax(top) + (2 * L + 16 + terms) * ref.U32
        assert (np.abs(w - (w0 + dw)) <= dw * rel + (w0 + dw) * 2 * ref.U32).all()
    return got, w


def make(rng, lengths, page, n_kv, hs, type, **kw):
    pages = ref.Pages(rng, lengths, page, n_kv, hs, **kw)
    pages.fill(rng, cast(type))
    return pages


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,n_kv,hs,layout", [(16, 2, 64, "positions"), (1, 3, 8, "positions"), (7, 1, 40, "heads"), (33, 2, 256, "heads")])
def test_append(dev, type, page, n_kv, hs, layout):
    rng = np.random.default_rng(page)
    lengths, new, before, behind = [20, 0, 1, 37, 5], [3, 0, 1, 37, 5], 2, 3
    pages = make(rng, lengths, page, n_kv, hs, type, fill=-7.0)
    cache = OnDevice(dev, pages, type, layout)
    starts = [before] + list(before + np.cumsum(new))
    n_rows, width = starts[-1] + behind, n_kv * hs
    rows = (rng.standard_normal((n_rows, 3 * width)) * 10.0 ** rng.integers(-6, 4, (n_rows, 1))).astype(np.float32)
    rows[3, :5] = [1e6, -np.inf, np.nan, 65519.9, 3e-8]  # past the largest half, not a number, below the smallest
    buf, sb = dev.tensor(rows), dev.tensor(np.array(starts, np.int32))
    _lib.call("wgpt_paged_append", dev.handle, cache.ptr, n_rows, sb.ptr, buf.ptr + 4 * width, buf.ptr + 8 * width, 3 * width)
    want = [pages.k.copy(), pages.v.copy()]
    for s, L in enumerate(lengths):
        for i in range(new[s]):
            for x, pool in enumerate(want):
                pool[pages.place(s, L - new[s] + i)] = cast(type)(rows[starts[s] + i, (1 + x) * width:(2 + x) * width]).reshape(n_kv, hs)
    for got, w in zip(cache.pools(), want):
        assert np.array_equal(got, w, equal_nan=True)


def test_append_without_starts_and_tokens_without_a_position(dev):
    rng = np.random.default_rng(2)
    pages = make(rng, [1, 9], 4, 1, 16, "f32")  # the first of the two rows of a sequence of length one has no position
    cache = OnDevice(dev, pages, "f32")
    rows = dev.tensor(rng.standard_normal((4, 16)).astype(np.float32))
    _lib.call("wgpt_paged_append", dev.handle, cache.ptr, 4, None, rows.ptr, rows.ptr, 16)
    x = rows.read().reshape(4, 1, 16)
    pages.k[pages.place(0, 0)] = x[1]
    for i in range(2):
        pages.k[pages.place(1, 7 + i)] = x[2 + i]
    assert np.array_equal(cache.pools()[0], pages.k, equal_nan=True)
    _lib.call("wgpt_device_check", dev.handle)


# ------------------------------------------------------------------ attention
HEADS = [(2, 1, 64), (1, 8, 128), (3, 1, 8), (2, 3, 80), (1, 2, 256), (2, 4, 32), (1, 20, 72)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,group,hs", HEADS)
def test_attention_single_tokens(dev, type, n_kv, group, hs):
    rng = np.random.default_rng(hs)
    lengths = [1, 200, 15, 16, 17, 64, 333, 0, 65]
    for page, layout in ((16, "positions"), (5, "heads")):
        pages = make(rng, lengths, page, n_kv, hs, type)
        check_attention(dev, pages, type, layout, [1] * len(lengths), n_kv * group, weights=page == 5)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,group,hs", [(2, 1, 64), (1, 8, 128), (2, 3, 40), (1, 4, 256)])
def test_attention_several_tokens(dev, type, n_kv, group, hs):
    """Drafts of different numbers, rows before and behind the sequences, sequences shorter than their new tokens, windows."""
    rng = np.random.default_rng(hs + 1)
    lengths, new = [3, 120, 64, 2, 0, 50, 17], [3, 5, 1, 4, 2, 0, 9]
    for window in (0, 1, 4, 33):
        pages = make(rng, lengths, 7, n_kv, hs, type)
        check_attention(dev, pages, type, "positions", new, n_kv * group, window=window, weights=window != 4, before=2, behind=2)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_attention_prompt_through_the_cache(dev, type):
    rng = np.random.default_rng(8)
    pages = make(rng, [90, 41], 16, 2, 64, type)
    check_attention(dev, pages, type, "positions", [90, 30], 4)
    check_attention(dev, pages, type, "heads", [70, 41], 4, window=20)


@pytest.mark.parametrize("type,n_kv,group,hs", [("f32", 1, 1, 64), ("f16", 1, 4, 128), ("bf16", 2, 5, 64)])
def test_attention_long(dev, type, n_kv, group, hs):
    """Lengths that are split over many CTAs and joined again, beside short ones."""
    rng = np.random.default_rng(10)
    pages = make(rng, [9001, 3, 1200], 64, n_kv, hs, type)
    check_attention(dev, pages, type, "positions", [1, 1, 2], n_kv * group, weights=True)
    check_attention(dev, pages, type, "heads", [2, 0, 1], n_kv * group, window=4000)


def test_attention_many_sequences(dev):
    rng = np.random.default_rng(11)
    lengths = [int(x) for x in rng.integers(0, 40, 700)]
    pages = make(rng, lengths, 8, 1, 16, "f16")
    check_attention(dev, pages, "f16", "positions", [1] * 700, 2, weights=True)


def test_attention_without_starts_and_with_row_strides(dev):
    rng = np.random.default_rng(12)
    pages = make(rng, [30, 55], 16, 2, 64, "f32")
    cache = OnDevice(dev, pages, "f32")
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    want, _, size, top = ref.attend(pages, [0, 2, 4], 4, 0.125, 0, q)
    for ld in ((256, 256), (260, 300)):
        got, _ = attend(dev, cache, None, 4, 4, 0.125, 0, q, ld_q=ld[0], ld_out=ld[1])
        assert (np.abs(got - want) <= ref.attend_tolerance(pages, size, top)).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_attention_masked_positions_may_hold_anything(dev, type):
    """What a row does not see is not to reach it: later drafts and positions before its window that are infinite or NaN."""
    rng = np.random.default_rng(13)
    lengths, new = [40, 70, 33], [4, 3, 1]
    pages = make(rng, lengths, 16, 1, 64, type)
    q = (np.random.default_rng(1).standard_normal((8, 2, 64)) * 1.5).astype(np.float32)
    want, _, size, top = ref.attend(pages, [0, 4, 7, 8], 2, 0.125, 20, q)
    pages.k[pages.place(0, 39)] = np.nan      # the last draft: its own row alone sees it
    pages.v[pages.place(0, 39)] = np.inf
    pages.k[pages.place(1, 47)] = -np.inf     # in the window of the first row alone
    pages.v[pages.place(1, 48)] = np.nan      # in those of the first two (48 .. 67, 49 .. 68, 50 .. 69: the first alone)
    pages.v[pages.place(2, 3)] = np.nan       # behind every window
    cache = OnDevice(dev, pages, type)
    got, _ = attend(dev, cache, [0, 4, 7, 8], 8, 2, 0.125, 20, q)
    assert np.isnan(got[3]).all()
    assert np.isnan(got[4]).all()
    # The other rows are what they are without those positions, each within its own tolerance: two results of f32 arithmetic
    # in different orders (rows beside one that sees such a value are added up apart) lie that near to the same 64-bit value,
    # though not at the same bits.
    rows = [0, 1, 2, 5, 6, 7]
    assert (np.abs(got[rows] - want[rows]) <= ref.attend_tolerance(pages, size, top)[rows]).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_attention_infinities_that_are_seen(dev, type):
    """An infinite value goes into the rows that see it, with its sign; a key that makes a score -infinity counts nothing;
    keys that make all scores -infinity leave zeros."""
    pages = ref.Pages(np.random.default_rng(14), [20, 3], 16, 1, 64)
    pages.fill(np.random.default_rng(15), cast(type))
    q = np.abs(np.random.default_rng(16).standard_normal((2, 1, 64))).astype(np.float32)
    pages.v[pages.place(0, 5)][0, 3], pages.v[pages.place(0, 6)][0, 4] = np.inf, -np.inf
    pages.k[pages.place(0, 7)] = -np.inf
    pages.v[pages.place(0, 7)] = 99.0
    for j in range(3):
        pages.k[pages.place(1, j)] = -np.inf
    got, _ = attend(dev, OnDevice(dev, pages, type), None, 2, 1, 0.125, 0, q)
    assert got[0, 0, 3] == np.inf and got[0, 0, 4] == -np.inf and np.isfinite(got[0, 0, 5:]).all() and np.abs(got[0, 0, 5:]).max() < 50
    assert (got[1] == 0).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_attention_large_and_small_values(dev, type):
    """Scores of several hundred, values near the ends of the half-precision range, rows of tiny and of mixed queries."""
    rng = np.random.default_rng(17)
    pages = ref.Pages(rng, [100, 100, 100], 16, 1, 128)
    pages.fill(rng, cast(type), scale=100.0)
    q = (rng.standard_normal((3, 1, 128)) * np.array([3.0, 1e-20, 1.0])[:, None, None]).astype(np.float32)
    q[2, 0, ::2] *= 1e-6
    check_attention(dev, pages, type, "positions", [1, 1, 1], 1, q=q)
    pages.v *= 2.0 ** -20 if type == "f16" else 1e-30
    pages.v = cast(type)(pages.v)
    check_attention(dev, pages, type, "positions", [1, 1, 1], 1, q=q)


def test_attention_same_bits_twice_and_in_a_replay(dev):
    rng = np.random.default_rng(18)
    pages = make(rng, [3000, 10, 500], 16, 2, 64, "f16")
    cache = OnDevice(dev, pages, "f16")
    q = dev.tensor(rng.standard_normal((5, 4 * 64)).astype(np.float32))
    starts = dev.tensor(np.array([0, 3, 4, 5], np.int32))
    outs = [dev.buffer(5 * 256 * 4) for _ in range(2)]
    w = [dev.tensor(np.zeros((3, 3000), np.float32)) for _ in range(2)]

    def call(i):
        _lib.call("wgpt_paged_attention", dev.handle, cache.ptr, 5, starts.ptr, 4, 0.125, 0, q.ptr, 256, outs[i].ptr, 256, w[i].ptr, 3000)

    call(0)
    g = C.c_void_p()
    _lib.call("wgpt_graph_begin", dev.handle)
    call(1)
    _lib.call("wgpt_graph_end", dev.handle, C.byref(g))
    for n in range(1, 3):
        _lib.call("wgpt_graph_launch", dev.handle, g)
        a, b = outs[0].read(), outs[1].read()
        assert np.array_equal(a, b)
        call(0)
        assert np.array_equal(outs[0].read(), b)
        # the replay reads lengths and table when it runs
    cache.lengths.write(np.array([1500, 10, 0], np.int32))
    _lib.call("wgpt_graph_launch", dev.handle, g)
    call(0)
    assert np.array_equal(outs[0].read(), outs[1].read()) and not np.array_equal(outs[1].read(), b)
    assert (outs[1].read()[4 * 256:] == 0).all()
    _lib.call("wgpt_graph_destroy", dev.handle, g)


def test_two_devices_handles_at_once(dev):
    """Two handles on one GPU have workspaces of their own."""
    from webgpt_b200 import Device
    rng = np.random.default_rng(19)
    pages = make(rng, [5000], 16, 1, 64, "bf16")
    q = rng.standard_normal((1, 8, 64)).astype(np.float32)
    want = attend(dev, OnDevice(dev, pages, "bf16"), None, 1, 8, 0.125, 0, q)[0]
    other = Device(0)
    try:
        made = []
        for d in (dev, other) * 10:
            c = OnDevice(d, pages, "bf16")
            made.append((d, c, d.tensor(q), d.buffer(8 * 64 * 4)))
        for d, c, qb, ob in made:
            _lib.call("wgpt_paged_attention", d.handle, c.ptr, 1, None, 8, 0.125, 0, qb.ptr, 512, ob.ptr, 512, None, 0)
        for _, _, _, ob in made:
            assert np.array_equal(ob.read().reshape(1, 8, 64), want)
        for _, c, qb, ob in made:
            for b in (c.k, c.v, c.table, c.lengths, qb, ob):
                b.destroy()
    finally:
        other.destroy()


def test_offsets_past_32_bits(dev):
    """Pages whose elements lie more than 2^32 bytes and 2^31 elements into a pool."""
    hs, page = 64, 16
    stride = 1 << 26  # elements from page to page: 40 pages of 256 MB
    free, _ = dev.mem_info()
    if free < 40 * stride * 4 + (1 << 31):
        pytest.skip("not enough memory")
    pool = dev.buffer(40 * stride * 4)
    rng = np.random.default_rng(20)
    pages = ref.Pages(rng, [3 * page], page, 1, hs, spare=37)
    pages.table[0, :3] = [39, 1, 33]
    pages.fill(rng, lambda x: x)
    for p in (39, 1, 33):
        pool.write(pages.k[p], offset=p * stride * 4)
        pool.write(pages.v[p], offset=(p * stride + page * hs) * 4)
    cache = OnDevice(dev, pages, "f32")
    d = cache.d
    d.k, d.v, d.page_stride = pool.ptr, pool.ptr + page * hs * 4, stride
    q = rng.standard_normal((1, 1, hs)).astype(np.float32)
    got, _ = attend(dev, cache, None, 1, 1, 0.125, 0, q)
    want, _, size, top = ref.attend(pages, [0, 1], 1, 0.125, 0, q)
    assert (np.abs(got - want) <= ref.attend_tolerance(pages, size, top)).all()
    rows = dev.tensor(rng.standard_normal((1, 2 * hs)).astype(np.float32))
    _lib.call("wgpt_paged_append", dev.handle, C.byref(d), 1, None, rows.ptr, rows.ptr + 4 * hs, 2 * hs)
    got = pool.read(np.float32, hs, offset=(33 * stride + 15 * hs) * 4)
    assert np.array_equal(got, rows.read()[:hs])
    pool.destroy()


# ------------------------------------------------------------------ eviction
@pytest.mark.parametrize("type,page,n_kv,hs,layout", [("f32", 16, 2, 64, "positions"), ("f16", 5, 3, 40, "heads"), ("bf16", 64, 1, 256, "positions"),
                                                      ("f16", 1, 1, 8, "positions")])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (10, 3), (64, 64), (100, 0), (101, 30), (5000, 7)])
def test_evict(dev, type, page, n_kv, hs, layout, keep, recent):
    rng = np.random.default_rng(keep)
    lengths = [101, 0, 1, 100, 10, 11, 1200, 2500]
    pages = make(rng, lengths, page, n_kv, hs, type, max_length=2600)
    w = np.round(rng.random((8, 2700)) ** 4 * 50).astype(np.float32)  # few values: many equal
    w[0, ::7] = -0.0
    w[6] = 1.0
    w[7, 100:110] = [np.nan, np.inf, -np.inf, -3.0, 1e-40, 0.0, -0.0, 1e38, np.nan, 2.0]
    n = [min(L, keep) for L in lengths]
    to = ref.Pages(rng, n, page, n_kv, hs, max_length=min(keep, 2600), fill=5.0)
    src, dst = OnDevice(dev, pages, type, layout), OnDevice(dev, to, type, layout)
    dst.lengths.write(np.full(8, -1, np.int32))
    wb, wt, kept = dev.tensor(w), dev.tensor(np.full((8, keep + 3), 9.0, np.float32)), dev.buffer(8 * keep * 4)
    _lib.call("wgpt_paged_evict", dev.handle, src.ptr, dst.ptr, keep, recent, wb.ptr, 2700, wt.ptr, keep + 3, kept.ptr)
    got, gw = kept.read(np.int32).reshape(8, keep), wt.read().reshape(8, keep + 3)
    assert list(dst.lengths.read(np.int32)) == n
    want_k, want_v = to.k.copy(), to.v.copy()
    for s, L in enumerate(lengths):
        stay = ref.keep(w[s], L, keep, recent)
        assert list(got[s, :n[s]]) == stay and (got[s, n[s]:] == -1).all()
        assert np.array_equal(gw[s, :n[s]], w[s, stay], equal_nan=True) and (gw[s, n[s]:keep] == 0).all() and (gw[s, keep:] == 9.0).all()
        for i, j in enumerate(stay):
            want_k[to.place(s, i)], want_v[to.place(s, i)] = pages.k[pages.place(s, j)], pages.v[pages.place(s, j)]
    for x, y in zip(dst.pools(), (want_k, want_v)):
        assert np.array_equal(x, y, equal_nan=True)
    for x, y in zip(src.pools(), (pages.k, pages.v)):
        assert np.array_equal(x, y, equal_nan=True)
    wt.write(np.zeros(1, np.float32))
    _lib.call("wgpt_paged_evict", dev.handle, src.ptr, dst.ptr, keep, recent, wb.ptr, 2700, None, 0, kept.ptr)
    assert np.array_equal(kept.read(np.int32).reshape(8, keep), got)
    _lib.call("wgpt_device_check", dev.handle)


@pytest.mark.parametrize("L,keep,recent", [(40000, 12345, 100), (140001, 70000, 1), (70000, 69999, 0)])
def test_evict_long(dev, L, keep, recent):
    rng = np.random.default_rng(L)
    lengths = [L, L // 2, L - 17]
    pages = ref.Pages(rng, lengths, 64, 1, 8)
    pages.k = rng.standard_normal(pages.k.shape).astype(np.float32)
    pages.v = rng.standard_normal(pages.v.shape).astype(np.float32)
    w = (rng.random((3, L)) ** 8 * 100).astype(np.float32)
    w[1] = np.round(w[1])
    n = [min(x, keep) for x in lengths]
    to = ref.Pages(rng, n, 64, 1, 8, fill=0.0)
    src, dst = OnDevice(dev, pages, "f32"), OnDevice(dev, to, "f32")
    wb, kept = dev.tensor(w), dev.buffer(3 * keep * 4)
    _lib.call("wgpt_paged_evict", dev.handle, src.ptr, dst.ptr, keep, recent, wb.ptr, L, None, 0, kept.ptr)
    got, pool = kept.read(np.int32).reshape(3, keep), dst.pools()[1]
    for s in range(3):
        stay = np.array(ref.keep(w[s], lengths[s], keep, recent))
        assert np.array_equal(got[s, :n[s]], stay)
        i = np.arange(n[s])
        assert np.array_equal(pool[to.table[s, i // 64], i % 64], pages.v[pages.table[s, stay // 64], stay % 64])


# ------------------------------------------------------------------ refusals and what the kernels find
def cache_of(dev, **kw):
    pages = make(np.random.default_rng(0), [20, 10], 16, 2, 64, "f32")
    c = OnDevice(dev, pages, "f32")
    for name, value in kw.items():
        setattr(c.d, name, value)
    return c


@pytest.mark.parametrize("change,code", [
    (dict(k=None), _lib.ERR_ARG), (dict(v=None), _lib.ERR_ARG), (dict(table=None), _lib.ERR_ARG), (dict(lengths=None), _lib.ERR_ARG),
    (dict(type=3), _lib.ERR_ARG), (dict(type=-1), _lib.ERR_ARG), (dict(n_pages=0), _lib.ERR_SHAPE), (dict(page_size=0), _lib.ERR_SHAPE),
    (dict(n_kv_head=0), _lib.ERR_SHAPE), (dict(n_seq=0), _lib.ERR_SHAPE), (dict(max_length=0), _lib.ERR_SHAPE), (dict(head_size=4), _lib.ERR_SHAPE),
    (dict(head_size=60), _lib.ERR_SHAPE), (dict(head_size=264), _lib.ERR_SHAPE), (dict(max_length=33), _lib.ERR_SHAPE),
    (dict(page_stride=-4), _lib.ERR_SHAPE), (dict(position_stride=130), _lib.ERR_ALIGN), (dict(head_stride=66), _lib.ERR_ALIGN)])
def test_cache_refusals(dev, change, code):
    c = cache_of(dev, **change)
    x, w = dev.buffer(4096), dev.buffer(4096)
    ok = cache_of(dev)
    for name, args in (("wgpt_paged_append", (c.ptr, 2, None, x.ptr, x.ptr, 128)),
                       ("wgpt_paged_attention", (c.ptr, 2, None, 2, 0.125, 0, x.ptr, 128, w.ptr, 128, None, 0)),
                       ("wgpt_paged_evict", (c.ptr, ok.ptr, 4, 1, x.ptr, 64, None, 0, w.ptr)),
                       ("wgpt_paged_evict", (ok.ptr, c.ptr, 4, 1, x.ptr, 64, None, 0, w.ptr))):
        with pytest.raises(_lib.WgptError) as e:
            _lib.call(name, dev.handle, *args)
        assert e.value.code == code


def test_call_refusals(dev):
    c, x = cache_of(dev), dev.buffer(1 << 16)
    p = x.ptr

    def refused(code, name, *args):
        with pytest.raises(_lib.WgptError) as e:
            _lib.call(name, dev.handle, *args)
        assert e.value.code == code, e.value

    S, A, G = _lib.ERR_SHAPE, _lib.ERR_ALIGN, _lib.ERR_ARG
    refused(G, "wgpt_paged_append", None, 2, None, p, p, 128)
    for args, code in (((0, None, p, p, 128), S), ((3, None, p, p, 128), S), ((2, None, None, p, 128), G), ((2, None, p, None, 128), G),
                       ((2, None, p, p, 124), S), ((2, None, p, p, 130), A), ((2, None, p + 4, p, 128), A)):
        refused(code, "wgpt_paged_append", c.ptr, *args)
    good = [2, None, 4, 0.125, 0, p, 256, p + 4096, 256, None, 0]
    for at, value, code in ((0, 0, S), (0, 5, S), (2, 3, S), (2, 0, S), (4, -1, S), (5, None, G), (5, p + 8, A), (6, 252, S), (6, 258, A),
                            (7, None, G), (8, 128, S), (9, p, S)):
        refused(code, "wgpt_paged_attention", c.ptr, *(good[:at] + [value] + good[at + 1:]))
    to = cache_of(dev)
    good = [4, 1, p, 20, p + 4096, 4, p + 8192]
    for at, value, code in ((0, 0, S), (1, -1, S), (1, 5, S), (2, None, G), (3, 19, S), (5, 3, S), (6, None, G)):
        refused(code, "wgpt_paged_evict", c.ptr, to.ptr, *(good[:at] + [value] + good[at + 1:]))
    for change in (dict(type=_lib.TYPE_F16), dict(head_size=32), dict(n_kv_head=1), dict(n_seq=1), dict(max_length=3)):
        refused(S, "wgpt_paged_evict", c.ptr, cache_of(dev, **change).ptr, *good)
    for name in ("wgpt_paged_append", "wgpt_paged_attention", "wgpt_paged_evict"):
        assert getattr(_lib.load(), name)(None, *([c.ptr] + [0] * (len(_lib.SIGNATURES[name]) - 2) if name != "wgpt_paged_evict"
                                                  else [c.ptr, c.ptr] + [0] * 8)) == G


def reported(dev):
    with pytest.raises(_lib.WgptError) as e:
        _lib.call("wgpt_device_check", dev.handle)
    assert e.value.code == _lib.ERR_ARG and "paged cache" in e.value.message
    _lib.call("wgpt_device_check", dev.handle)  # reported once


def test_bad_pages_lengths_and_offsets_are_reported(dev):
    rng = np.random.default_rng(21)
    pages = make(rng, [40, 30], 16, 1, 64, "f16")
    q = rng.standard_normal((2, 1, 64)).astype(np.float32)
    # a page id out of range: its positions are not seen
    c = OnDevice(dev, pages, "f16")
    table = pages.table.copy()
    table[0, 1] = pages.n_pages
    c.table.write(table)
    got, _ = attend(dev, c, None, 2, 1, 0.125, 0, q)
    reported(dev)
    gone = ref.Pages(rng, [24, 30], 16, 1, 64)
    for which in ("k", "v"):
        a, b = getattr(gone, which), getattr(pages, which)
        for i, j in enumerate(list(range(16)) + list(range(32, 40))):
            a[gone.place(0, i)] = b[pages.place(0, j)]
        for j in range(30):
            a[gone.place(1, j)] = b[pages.place(1, j)]
    want, _, size, top = ref.attend(gone, [0, 1, 2], 1, 0.125, 0, q)
    assert (np.abs(got - want) <= ref.attend_tolerance(pages, size, top)).all()
    table[0] = 0xFFFFFFFF  # no page at all: zeros
    c.table.write(table)
    got, _ = attend(dev, c, None, 2, 1, 0.125, 0, q)
    assert (got[0] == 0).all() and (np.abs(got[1] - want[1]) <= ref.attend_tolerance(pages, size, top)[1]).all()
    reported(dev)
    rows = dev.tensor(np.zeros((2, 64), np.float32))
    _lib.call("wgpt_paged_append", dev.handle, c.ptr, 2, None, rows.ptr, rows.ptr, 64)  # the first has no page to go to
    reported(dev)
    # lengths out of range
    c = OnDevice(dev, pages, "f16")
    c.lengths.write(np.array([41, -5], np.int32))
    got, _ = attend(dev, c, None, 2, 1, 0.125, 0, q)
    reported(dev)
    want = ref.attend(pages, [0, 1, 2], 1, 0.125, 0, q)[0]
    assert np.abs(got[0] - want[0]).max() < 1e-4 and (got[1] == 0).all()
    # offsets that go back, or past the rows
    c = OnDevice(dev, pages, "f16")
    for starts in ([0, 2, 1], [0, 1, 9], [-4, 1, 2], [5, 6, 7]):
        attend(dev, c, starts, 2, 1, 0.125, 0, q, np.zeros((2, 40), np.float32))
        reported(dev)
    # eviction from and to pages that are not there
    to = OnDevice(dev, ref.Pages(rng, [20, 20], 16, 1, 64, fill=0.0), "f16")
    to.table.write(np.full_like(to.pages.table, 0xFFFFFFFF))
    w, kept = dev.tensor(rng.random((2, 40)).astype(np.float32)), dev.buffer(160)
    _lib.call("wgpt_paged_evict", dev.handle, c.ptr, to.ptr, 20, 4, w.ptr, 40, None, 0, kept.ptr)
    reported(dev)
    assert (to.pools()[0] == 0).all()


def test_workspace_is_not_grown_while_recording():
    from webgpt_b200 import Device
    d = Device(0)
    try:
        pages = make(np.random.default_rng(22), [400], 16, 1, 64, "f32")
        c, x = OnDevice(d, pages, "f32"), d.buffer(1 << 16)
        args = (c.ptr, 1, None, 64, 0.125, 0, x.ptr, 4096, x.ptr + (1 << 15), 4096, x.ptr + (3 << 14), 400)
        _lib.call("wgpt_graph_begin", d.handle)
        with pytest.raises(_lib.WgptError) as e:
            _lib.call("wgpt_paged_attention", d.handle, *args)
        assert e.value.code == _lib.ERR_STATE
        g = C.c_void_p()
        _lib.call("wgpt_graph_end", d.handle, C.byref(g))
        _lib.call("wgpt_graph_destroy", d.handle, g)
    finally:
        d.destroy()


def test_workspace_that_cannot_be_had(dev):
    """Weights of more rows and positions than memory holds: refused, and the next call works."""
    rng = np.random.default_rng(24)
    small = make(rng, [30], 16, 1, 8, "f16")
    c = OnDevice(dev, small, "f16")
    c.d.max_length, c.d.table_stride = 1 << 30, 1 << 26
    x = dev.buffer(1 << 20)
    with pytest.raises(_lib.WgptError) as e:
        _lib.call("wgpt_paged_attention", dev.handle, c.ptr, 64, None, 64, 0.125, 0, x.ptr, 512, x.ptr + (1 << 19), 512, x.ptr, 1 << 30)
    assert e.value.code == _lib.ERR_OOM
    check_attention(dev, small, "f16", "positions", [1], 4, weights=True)
