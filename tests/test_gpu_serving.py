"""The serving operators together, through PagedCache and the instruction classes: steps of several users with drafts, two layers,
projections ahead of the cache, verification, retreat and eviction, enqueued call by call and as a replayed graph."""
import ctypes as C
import math

import numpy as np
import pytest

import serving_reference as ref
from test_gpu_paged import OnDevice, cast, check_attention, make
from webgpt_b200 import _lib

pytestmark = pytest.mark.gpu

N_SEQ, N_DRAFT, V, LAYERS = 3, 2, 1000, 2


class Host:
    """What one layer's cache should hold: each sequence's keys, values (as ref.Pages has them) and weights with their error."""

    def __init__(self, n_kv, hs, max_length):
        self.n_kv, self.hs, self.max_length = n_kv, hs, max_length
        self.k = [np.zeros((0, n_kv, hs), np.float32) for _ in range(N_SEQ)]
        self.v = [x.copy() for x in self.k]
        self.w, self.off = np.zeros((N_SEQ, max_length)), np.zeros((N_SEQ, max_length))

    @property
    def lengths(self):
        return [len(k) for k in self.k]

    def rows(self, which, s):
        return getattr(self, which)[s]

    def cut(self, by):
        for s, n in enumerate(by):
            L = len(self.k[s]) - n
            self.k[s], self.v[s] = self.k[s][:L], self.v[s][:L]
            self.w[s, L:] = self.off[s, L:] = 0


@pytest.fixture(scope="module")
def blocks():
    from webgpt_b200 import Device, globals as g
    d = Device(0)
    g.initializeOperations(d)
    yield d, g
    for b in g.operations:
        b.destroy()
    d.destroy()


def run(passes):
    for p in passes:
        p["run"]()


@pytest.mark.parametrize("type,n_head,n_kv,hs,window,replayed", [
    ("f32", 4, 4, 64, 0, False), ("f16", 4, 2, 64, 0, True), ("bf16", 8, 2, 128, 40, True), ("f16", 12, 2, 64, 0, True), ("f32", 4, 1, 40, 0, True)])
def test_steps_of_several_users(blocks, type, n_head, n_kv, hs, window, replayed):
    """After prompts of different lengths: steps of three tokens each, of which the verification keeps some. Every step's results
    are compared with those of 64-bit arithmetic on what the host says is in the cache; the projections' own results are read back."""
    from webgpt_b200.paged import PagedCache
    dev, g = blocks
    rng = np.random.default_rng(n_head * 100 + hs)
    E, KV = n_head * hs, n_kv * hs
    width = E + 2 * KV
    shared = 64
    scale = 1 / math.sqrt(hs)
    cache = PagedCache(dev, N_SEQ, n_kv, hs, n_pages=60, page_size=8, type=type, n_layer=LAYERS, max_length=150, weights=True)
    host = [Host(n_kv, hs, 150) for _ in range(LAYERS)]
    proj = [dev.tensor((rng.standard_normal((shared, width)) / 6).astype(np.float32)) for _ in range(LAYERS)]
    bias = [dev.tensor((rng.standard_normal(width) / 6).astype(np.float32)) for _ in range(LAYERS)]

    def layers(n_rows, starts, x):
        passes, outs = [], []
        for i in range(LAYERS):
            qkv = g.FastMatMulBlock.newInstance(n_rows, width, shared, x, proj[i], bias[i])
            b = qkv["resultBuffer"]
            k, v = (Part(b, 4 * at) for at in (E, E + KV))
            app = g.PagedAppendBlock.newInstance(cache.layer(i), n_rows, starts, k, v, width)
            att = g.PagedAttentionBlock.newInstance(cache.layer(i), n_rows, starts, n_head, scale, b, width, window, cache.weights(i))
            passes += qkv["passes"] + app["passes"] + att["passes"]
            outs.append((b, att["resultBuffer"]))
        return passes, outs

    def check(outs, n_rows, new):
        starts = [0] + list(np.cumsum(new))
        for h, (qkv, out), w in zip(host, outs, (cache.weights(i) for i in range(LAYERS))):
            rows = qkv.read(np.float32, n_rows * width).reshape(n_rows, width)
            for s in range(N_SEQ):
                mine = rows[starts[s]:starts[s + 1]]
                h.k[s] = np.concatenate([h.k[s], cast(type)(mine[:, E:E + KV]).reshape(-1, n_kv, hs)])
                h.v[s] = np.concatenate([h.v[s], cast(type)(mine[:, E + KV:]).reshape(-1, n_kv, hs)])
            q = np.ascontiguousarray(rows[:, :E]).reshape(n_rows, n_head, hs)
            want, dw, size, top = ref.attend(h, starts, n_head, np.float64(np.float32(scale)), window, q)
            got = out.read(np.float32, n_rows * E).reshape(n_rows, n_head, hs)
            assert (np.abs(got - want) <= ref.attend_tolerance(h, size, top)).all()
            # as in the test of one call; what earlier steps were off by stays
            L, terms = max(h.lengths), max(new) * n_head
            rel = 4 * (hs + 10) * ref.U32 * top.max() + (2 * L + 16 + terms) * ref.U32
            h.w += dw
            h.off += dw * rel + h.w * 2 * ref.U32 + 1e-30
            got = w.read(np.float32).reshape(N_SEQ, 150)
            assert (np.abs(got - h.w) <= h.off).all()
            h.w = np.where(h.w > 0, got, 0).astype(np.float64)  # what the cache goes by from here on
            h.off[:] = 0

    # prompts
    new = np.array([37, 1, 64])
    cache.advance(new)
    starts = cache.starts(new)
    n_rows = int(new.sum())
    x = dev.tensor(rng.standard_normal((n_rows, shared)).astype(np.float32))
    passes, outs = layers(n_rows, starts, x)
    run(passes)
    check(outs, n_rows, new)

    # steps of N_DRAFT + 1 tokens each: the last token and the drafts behind it
    n_rows = N_SEQ * (N_DRAFT + 1)
    x = dev.buffer(n_rows * shared * 4)
    target, draft, ids, u = dev.buffer(n_rows * V * 4), dev.buffer(N_SEQ * N_DRAFT * V * 4), dev.buffer(N_SEQ * N_DRAFT * 4), dev.buffer(n_rows * 8)
    passes, outs = layers(n_rows, None, x)
    ver = g.VerifyDraftsBlock.newInstance(N_SEQ, N_DRAFT, V, target, draft, ids, None, 0, 0.9, u)
    passes += ver["passes"]
    graph = None
    kept_some = [0] * (N_DRAFT + 1)
    for step in range(9):
        cache.advance(N_DRAFT + 1)
        t = (rng.standard_normal((N_SEQ, N_DRAFT + 1, V)) * 2.5).astype(np.float32)
        d = (t[:, :N_DRAFT] + rng.standard_normal((N_SEQ, N_DRAFT, V)) * 0.7).astype(np.float32)
        drafted = np.zeros((N_SEQ, N_DRAFT), np.uint32)
        for s in range(N_SEQ):
            for i in range(N_DRAFT):
                of, p = ref.distribution(d[s, i], 0, 0.9)
                drafted[s, i] = rng.choice(of, p=p)
        numbers = rng.random((N_SEQ, N_DRAFT + 1))
        for b, a in ((x, rng.standard_normal((n_rows, shared)).astype(np.float32)), (target, t), (draft, d), (ids, drafted), (u, numbers)):
            b.write(a)
        if step == 0 or not replayed:
            run(passes)
        else:
            if graph is None:
                graph = C.c_void_p()
                _lib.call("wgpt_graph_begin", dev.handle)
                run(passes)
                _lib.call("wgpt_graph_end", dev.handle, C.byref(graph))
            _lib.call("wgpt_graph_launch", dev.handle, graph)
        check(outs, n_rows, [N_DRAFT + 1] * N_SEQ)
        accepted = ver["acceptedBuffer"].read(np.int32, N_SEQ)
        got = ver["resultBuffer"].read(np.uint32, n_rows).reshape(N_SEQ, N_DRAFT + 1)
        for s in range(N_SEQ):
            a, drawn = ref.verify(t[s], d[s], drafted[s], N_DRAFT, 0, 0.9, numbers[s])
            assert accepted[s] == a and list(got[s][:a + 1]) == list(drafted[s][:a]) + [drawn]
            kept_some[a] += 1
        cache.retreat(N_DRAFT - accepted)
        for h in host:
            h.cut(N_DRAFT - accepted)
            assert h.lengths == list(cache.lengths)
        if step == 3:
            cache.release(1)  # a user leaves: its pages go to others
            for h in host:
                h.cut([0, h.lengths[1], 0])
        if step % 3 == 2:
            keep, recent = 24, 6
            stayed = cache.evict(keep, recent)
            for h, k in zip(host, stayed):
                for s, L in enumerate(h.lengths):
                    want = ref.keep(h.w[s], L, keep, recent)
                    assert list(k[s]) == want + [-1] * (keep - len(want))
                    h.k[s], h.v[s] = h.k[s][want], h.v[s][want]
                    h.w[s] = np.concatenate([h.w[s, want], np.zeros(150 - len(want))])
                assert h.lengths == list(cache.lengths)
    assert all(kept_some)  # every number of accepted drafts came up
    if graph is not None:
        _lib.call("wgpt_graph_destroy", dev.handle, graph)
    dev.synchronize()
    _lib.call("wgpt_device_check", dev.handle)
    for b in g.operations:
        b.clearBufferCache()
    cache.destroy()


@pytest.mark.parametrize("type,group,new,hs,L", [("f16", 8, 4, 64, 17920), ("f16", 8, 4, 64, 9000), ("bf16", 4, 1, 128, 9000), ("f16", 8, 1, 64, 70000),
                                                 ("f32", 8, 1, 40, 50000)])
def test_one_sequence_over_all_ctas(blocks, type, group, new, hs, L):
    """One head's positions spread over the GPU: joins of many parts, also of more than their factors have places for."""
    dev, _ = blocks
    pages = make(np.random.default_rng(L), [L], 64, 1, hs, type)
    check_attention(dev, pages, type, "positions", [new], group, weights=True)


@pytest.mark.parametrize("type,group,hs,window", [("f16", 6, 64, 0), ("bf16", 6, 128, 50), ("f16", 1, 128, 0), ("f32", 2, 64, 50), ("f16", 12, 256, 0)])
def test_seventy_sequences_of_all_lengths(blocks, type, group, hs, window):
    """More sequences than a warp has lanes, some empty, some without new tokens, for each of the kernels."""
    dev, _ = blocks
    rng = np.random.default_rng(group * hs)
    lengths = [int(x) for x in rng.integers(0, 400, 70)]
    lengths[3], lengths[40], lengths[41], lengths[69] = 0, 1, 0, 1500
    new = [int(min(L, n)) for L, n in zip(lengths, rng.integers(0, 5, 70))]
    new[69] = 4
    pages = make(rng, lengths, 16, 2, hs, type)
    check_attention(dev, pages, type, "heads", new, 2 * group, window=window, weights=True, before=1, behind=2)


def test_eviction_replayed(blocks):
    """A recorded eviction goes by the lengths and weights of the time it is replayed, and may share the lengths of its two caches."""
    dev, g = blocks
    rng = np.random.default_rng(5)
    pages = make(rng, [40, 25, 5000], 8, 2, 16, "f16")
    src, dst = OnDevice(dev, pages, "f16"), OnDevice(dev, make(rng, [5000] * 3, 8, 2, 16, "f16", fill=-7.0), "f16")
    src.d.lengths = dst.d.lengths  # one array
    lengths = dst.lengths
    lengths.write(np.array([40, 25, 5000], np.int32))
    w = rng.random((3, 5000)).astype(np.float32)
    wb = dev.tensor(w)
    wt = dev.buffer(3 * 30 * 4)
    graph = C.c_void_p()
    passes = g.PagedEvictBlock.newInstance(Described(src), Described(dst), 30, 7, wb, wt)
    _lib.call("wgpt_graph_begin", dev.handle)
    run(passes["passes"])
    _lib.call("wgpt_graph_end", dev.handle, C.byref(graph))
    for L in ([40, 25, 5000], [31, 0, 4096], [30, 29, 31]):
        L = [min(a, b) for a, b in zip(L, [40, 25, 5000])]
        lengths.write(np.array(L, np.int32))
        w = rng.integers(0, 50, w.shape).astype(np.float32)  # many equal ones
        wb.write(w)
        _lib.call("wgpt_graph_launch", dev.handle, graph)
        kept, moved = passes["resultBuffer"].read(np.int32, 90).reshape(3, 30), wt.read(np.float32, 90).reshape(3, 30)
        for s in range(3):
            want = ref.keep(w[s], L[s], 30, 7)
            assert list(kept[s]) == want + [-1] * (30 - len(want))
            assert list(moved[s]) == list(w[s, want]) + [0] * (30 - len(want))
            assert lengths.read(np.int32, 3)[s] == len(want)
    _lib.call("wgpt_graph_destroy", dev.handle, graph)


def test_limits(blocks):
    """Counts past what the kernels' grids and positions hold, and evictions that would write what they read, are refused."""
    dev, _ = blocks
    pages = make(np.random.default_rng(0), [20, 10], 16, 2, 64, "f32")
    x = dev.buffer(1 << 16)

    def refused(code, name, *args):
        with pytest.raises(_lib.WgptError) as e:
            _lib.call(name, dev.handle, *args)
        assert e.value.code == code, e.value

    for change in (dict(n_seq=65536), dict(max_length=(1 << 30) + 1, page_size=1 << 30)):
        c = OnDevice(dev, pages, "f32")
        for name, value in change.items():
            setattr(c.d, name, value)
        refused(_lib.ERR_SHAPE, "wgpt_paged_append", c.ptr, 65536, None, x.ptr, x.ptr, 128)
        refused(_lib.ERR_SHAPE, "wgpt_paged_attention", c.ptr, 65536, None, 2, 0.125, 0, x.ptr, 128, x.ptr, 128, None, 0)
        refused(_lib.ERR_SHAPE, "wgpt_paged_evict", c.ptr, c.ptr, 4, 1, x.ptr, 1 << 30, None, 0, x.ptr)
    refused(_lib.ERR_SHAPE, "wgpt_verify_drafts", 1, 0, (1 << 30) + 1, x.ptr, (1 << 30) + 1, None, 0, None, None, 0, 1.0, x.ptr, x.ptr, x.ptr)
    refused(_lib.ERR_SHAPE, "wgpt_verify_drafts", 65536, 0, 8, x.ptr, 8, None, 0, None, None, 0, 1.0, x.ptr, x.ptr, x.ptr)
    c, to = OnDevice(dev, pages, "f32"), OnDevice(dev, pages, "f32")
    refused(_lib.ERR_ARG, "wgpt_paged_evict", c.ptr, c.ptr, 4, 1, x.ptr, 20, None, 0, x.ptr + 4096)
    for at in (0, 39 * 4, -4 * 7):  # weights are 20 + 20 values, weights_to 4 + 4
        refused(_lib.ERR_ARG, "wgpt_paged_evict", c.ptr, to.ptr, 4, 1, x.ptr + 2048, 20, x.ptr + 2048 + at, 4, x.ptr + 4096)
    _lib.call("wgpt_paged_evict", dev.handle, c.ptr, to.ptr, 4, 1, x.ptr + 2048, 20, x.ptr + 2048 + 160, 4, x.ptr + 4096)
    _lib.call("wgpt_paged_evict", dev.handle, c.ptr, to.ptr, 4, 1, x.ptr + 2048, 20, x.ptr + 2048 - 32, 4, x.ptr + 4096)
    dev.synchronize()


class Described:
    """A test cache as a pass takes it."""

    def __init__(self, cache):
        self.ptr, self.n_seq, self.max_length = cache.ptr, cache.d.n_seq, cache.d.max_length


class Part:
    """A buffer from an offset on, as a pass takes it."""

    def __init__(self, buffer, offset):
        self.buffer, self.ptr = buffer, buffer.ptr + offset
