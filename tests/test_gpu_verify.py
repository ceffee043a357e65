"""wgpt_verify_drafts through the C ABI: ids and counts have to equal those of a plain 64-bit implementation."""
import ctypes as C

import numpy as np
import pytest

import serving_reference as ref
from webgpt_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from webgpt_b200 import Device
    d = Device(0)
    yield d
    d.destroy()


def verify(dev, target, draft, ids, counts, top_k, temperature, u, pad=0, V=None):
    n_seq, n1, V = target.shape[0], target.shape[1], V or target.shape[2]

    def rows(x):
        out = np.full((x.shape[0] * x.shape[1], V + pad), 1e30, np.float32)  # what lies behind a row is not part of it
        out[:, :V] = x.reshape(-1, V)
        return dev.tensor(out)

    t, d = rows(target), rows(draft) if draft is not None and n1 > 1 else None
    i = dev.tensor(np.ascontiguousarray(ids, np.uint32)) if n1 > 1 else None
    c = dev.tensor(np.array(counts, np.int32)) if counts is not None else None
    ub, out, acc = dev.tensor(np.ascontiguousarray(u, np.float64)), dev.buffer(n_seq * n1 * 4), dev.buffer(n_seq * 4)
    _lib.call("wgpt_verify_drafts", dev.handle, n_seq, n1 - 1, V, t.ptr, V + pad, d.ptr if d else None, V + pad, i.ptr if i else None,
              c.ptr if c else None, top_k, float(temperature), ub.ptr, out.ptr, acc.ptr)
    return out.read(np.uint32).reshape(n_seq, n1), acc.read(np.int32)


def check(dev, target, draft, ids, counts, top_k, temperature, u, **kw):
    got, acc = verify(dev, target, draft, ids, counts, top_k, temperature, u, **kw)
    n_draft = target.shape[1] - 1
    for s in range(len(target)):
        a, drawn = ref.verify(target[s], draft[s] if draft is not None else None, ids[s], counts[s] if counts is not None else n_draft,
                              top_k, temperature, u[s])
        assert acc[s] == a, (s, acc[s], a)
        assert list(got[s]) == list(ids[s][:a]) + [drawn] + [0xFFFFFFFF] * (n_draft - a), s
    return got, acc


def inputs(rng, n_seq, n_draft, V, temperature=1.0, top_k=0, spread=2.5, noise=0.7):
    """Logits of a target and of a draft that resembles it, tokens drawn from the draft, numbers."""
    target = (rng.standard_normal((n_seq, n_draft + 1, V)) * spread - 20).astype(np.float32)
    draft = (target[:, :n_draft] + rng.standard_normal((n_seq, n_draft, V)) * noise).astype(np.float32)
    ids = np.zeros((n_seq, n_draft), np.uint32)
    for s in range(n_seq):
        for i in range(n_draft):
            of, p = ref.distribution(draft[s, i], top_k, temperature)
            ids[s, i] = of[min(int((np.cumsum(p) <= rng.random()).sum()), len(of) - 1)]
    return target, draft, ids, rng.random((n_seq, n_draft + 1))


@pytest.mark.parametrize("V", [1, 2, 31, 65, 1000, 4097, 8193, 50257, 131073])
@pytest.mark.parametrize("top_k", [0, 1, 3, 40, 128])
def test_verify(dev, V, top_k):
    rng = np.random.default_rng(V + top_k)
    n_seq = 6 if V > 20000 else 20
    for n_draft, temperature, pad in ((4, 1.0, 0), (1, 0.5, 3), (7, 1.7, 1)):
        t, d, ids, u = inputs(rng, n_seq, n_draft, V, temperature, min(top_k, V))
        counts = rng.integers(0, n_draft + 1, n_seq)
        accepted = check(dev, t, d, ids, None, min(top_k, V), temperature, u, pad=pad)[1]
        if V > 60 and n_draft == 4:
            assert 0 < accepted.sum() < n_seq * n_draft
        check(dev, t, d, ids, counts, min(top_k, V), temperature, u)
        check(dev, t, None, ids, counts, min(top_k, V), temperature, u)  # looked up, not drawn


@pytest.mark.parametrize("top_k", [0, 5])
def test_many_drafts_and_sequences(dev, top_k):
    rng = np.random.default_rng(7)
    t, d, ids, u = inputs(rng, 3, 64, 300, 1.0, top_k, noise=0.1)
    check(dev, t, d, ids, [64, 33, 0], top_k, 1.0, u)
    t, d, ids, u = inputs(rng, 300, 2, 130, 1.0, top_k)
    check(dev, t, d, ids, None, top_k, 1.0, u)


@pytest.mark.parametrize("V", [130, 50257])
def test_no_drafts_is_sampling(dev, V):
    """Without drafts a top_k gives wgpt_sample_topk's pick from the same numbers."""
    rng = np.random.default_rng(V)
    t = (rng.standard_normal((9, 1, V)) * 3).astype(np.float32)
    t[4] = np.round(t[4])
    u = rng.random((9, 1))
    ids = np.zeros((9, 0), np.uint32)
    check(dev, t, None, ids, None, 0, 0.9, u)
    for top_k in (1, 2, 40, 128):
        got, _ = check(dev, t, None, ids, None, top_k, 0.9, u)
        lg, ub, out = dev.tensor(t), dev.tensor(u), dev.buffer(36)
        _lib.call("wgpt_sample_topk", dev.handle, lg.ptr, 9, V, top_k, 0.9, ub.ptr, out.ptr)
        assert np.array_equal(out.read(np.uint32), got[:, 0])


@pytest.mark.parametrize("V", [64, 5000, 50257])
def test_equal_logits_and_edges_of_the_numbers(dev, V):
    """Flat and two-valued rows, the draft equal to the target, numbers 0 and just below 1."""
    rng = np.random.default_rng(3)
    t = np.zeros((8, 2, V), np.float32)
    t[1:3, :, ::2] = -0.0
    t[3:5, :, ::3] = 4.0
    t[5, :, -1] = 60.0
    d = t[:, :1].copy()
    d[4] = 0.0
    ids = np.full((8, 1), V - 1, np.uint32)
    ids[6:] = 0
    last = np.nextafter(1.0, 0.0)
    for top_k in (0, 2, 33):
        for a in (0.0, 0.5, last):
            for b in (0.0, last):
                u = np.tile([a, b], (8, 1))
                check(dev, t, d, ids, None, top_k, 1.0, u)
                check(dev, t, None, ids, None, top_k, 1.0, u)


@pytest.mark.parametrize("top_k", [0, 7])
def test_logits_that_are_not_finite(dev, top_k):
    """-infinity and NaN are tokens that cannot come; a row of nothing else, or with +infinity, has no distribution."""
    rng = np.random.default_rng(9)
    V = 9000
    t, d, ids, u = inputs(rng, 10, 3, V, 1.0, top_k)
    t[0, :, ::2], t[1, 1, 100:] = -np.inf, np.nan
    d[2, :, 5:] = -np.inf
    ids[2] = 3
    check(dev, t, d, ids, None, top_k, 1.0, u)
    _lib.call("wgpt_device_check", dev.handle)
    u[:, 0] = 0.0
    for change in ((t, np.nan), (t, -np.inf), (d, np.nan), (d, -np.inf)):
        x, value = change
        old = x.copy()
        x[3, 0], x[4, 1], x[5, 2] = value, value, value
        check(dev, t, d, ids, None, top_k, 1.0, u)
        check(dev, t, None, ids, None, top_k, 1.0, u)
        x[...] = old
    for x in (t, d):
        old = x.copy()
        x[3, 0, 17], x[4, 1, 8999] = np.inf, np.inf
        check(dev, t, d, ids, None, top_k, 1.0, u)
        with pytest.raises(_lib.WgptError) as e:
            _lib.call("wgpt_device_check", dev.handle)
        assert e.value.code == _lib.ERR_ARG and "row of logits" in e.value.message
        x[...] = old
    t[6, 3] = -np.inf
    d[6], ids[6], u[6, :3] = t[6, :3], 0, 0.0  # all three are accepted: the row behind them decides
    assert check(dev, t, d, ids, None, top_k, 1.0, u)[1][6] == (3 if top_k == 0 else 0)
    try:
        _lib.call("wgpt_device_check", dev.handle)
        assert top_k
    except _lib.WgptError as e:
        assert top_k == 0 and "row of logits" in e.message


def test_extreme_temperatures(dev):
    rng = np.random.default_rng(10)
    t, d, ids, u = inputs(rng, 8, 2, 3000)
    for temperature in (1e-3, 1e-6, 50.0, 1e6):
        check(dev, t, d, ids, None, 0, temperature, u)
        check(dev, t, d, ids, None, 16, temperature, u)


@pytest.mark.parametrize("top_k", [0, 4])
def test_bad_ids_and_counts_are_reported(dev, top_k):
    rng = np.random.default_rng(11)
    t, d, ids, u = inputs(rng, 3, 2, 100, 1.0, top_k)
    ids[1, 0] = 100
    u[:, 0] = 0.0
    check(dev, t, d, ids, None, top_k, 1.0, u)
    with pytest.raises(_lib.WgptError) as e:
        _lib.call("wgpt_device_check", dev.handle)
    assert e.value.code == _lib.ERR_ARG and "token id" in e.value.message
    check(dev, t, None, ids, None, top_k, 1.0, u)
    with pytest.raises(_lib.WgptError):
        _lib.call("wgpt_device_check", dev.handle)
    ids[1, 0] = 5
    got, acc = verify(dev, t, d, ids, [5, -1, 2], top_k, 1.0, u)
    assert acc[1] == 0 and acc.max() <= 2
    with pytest.raises(_lib.WgptError) as e:
        _lib.call("wgpt_device_check", dev.handle)
    assert e.value.code == _lib.ERR_ARG and "number of drafts" in e.value.message


def test_replayed(dev):
    rng = np.random.default_rng(12)
    t, d, ids, u = inputs(rng, 4, 3, 50257)
    bufs = [dev.tensor(x) for x in (t, d, ids, u)]
    out, acc = dev.buffer(64), dev.buffer(16)
    for top_k in (0, 9):
        args = (4, 3, 50257, bufs[0].ptr, 50257, bufs[1].ptr, 50257, bufs[2].ptr, None, top_k, 1.0, bufs[3].ptr, out.ptr, acc.ptr)
        _lib.call("wgpt_verify_drafts", dev.handle, *args)
        g = C.c_void_p()
        _lib.call("wgpt_graph_begin", dev.handle)
        _lib.call("wgpt_verify_drafts", dev.handle, *args)
        _lib.call("wgpt_graph_end", dev.handle, C.byref(g))
        for _ in range(3):
            u = rng.random(u.shape)
            bufs[3].write(u)
            _lib.call("wgpt_graph_launch", dev.handle, g)
            got = acc.read(np.int32)
            assert [int(a) for a in got] == [ref.verify(t[s], d[s], ids[s], 3, top_k, 1.0, u[s])[0] for s in range(4)]
        _lib.call("wgpt_graph_destroy", dev.handle, g)


def test_refusals(dev):
    x = dev.buffer(1 << 16)
    p = x.ptr
    good = [2, 3, 100, p, 100, p, 100, p, None, 0, 1.0, p, p, p]
    S, G = _lib.ERR_SHAPE, _lib.ERR_ARG
    for at, value, code in ((0, 0, S), (0, 65536, S), (1, -1, S), (1, 65, S), (2, 0, S), (3, None, G), (4, 99, S), (6, 99, S), (7, None, G),
                            (9, -1, S), (9, 101, S), (9, 129, S), (10, 0.0, G), (10, float("nan"), G), (11, None, G), (12, None, G), (13, None, G)):
        args = good[:at] + [value] + good[at + 1:]
        with pytest.raises(_lib.WgptError) as e:
            _lib.call("wgpt_verify_drafts", dev.handle, *args)
        assert e.value.code == code, (at, value)
    assert _lib.load().wgpt_verify_drafts(None, *good) == G
