"""wgpt_verify_drafts next to the borders of its decisions: numbers a little below and above the one at which the answer changes. The
borders come from 64-bit sums, whose own error is far below the distances used: a sum of 50257 terms in any order is off by less
than V * 2^-53 = 5.6e-12 of itself, and by a hundredth of that in numpy's pairwise order."""
import numpy as np
import pytest

import serving_reference as ref
from test_gpu_verify import check, dev  # noqa: F401 (a fixture)
from webgpt_b200 import _lib

NEAR = 1e-10

pytestmark = pytest.mark.gpu


def pair(rng, V, spread=2.5, noise=0.7):
    t = (rng.standard_normal((2, V)) * spread).astype(np.float32)
    d = (t[:1] + rng.standard_normal((1, V)) * noise).astype(np.float32)
    return t, d


def turned_down(p, q):
    """An id that the draft likes better than the target, so that a number near 1 turns it down."""
    return int(np.argmax(q - p))


@pytest.mark.parametrize("V,n_seq,temperature,noise", [
    (50257, 8, 1.0, 0.7), (50257, 8, 0.9, 0.7), (50257, 64, 0.6, 0.7), (50257, 64, 1.44, 0.02), (1000, 300, 0.9, 0.7), (131073, 8, 1.2, 0.7)])
@pytest.mark.parametrize("drawn", [True, False])
def test_what_a_turned_down_draft_leaves(dev, V, n_seq, temperature, noise, drawn):  # noqa: F811
    """The id is the first whose running sum of max(p - q, 0) passes number * total: just below and above the border between two ids."""
    rng = np.random.default_rng(V + n_seq)
    t, d = pair(rng, V, noise=noise)
    p = ref.distribution(t[0], 0, temperature)[1]
    q = ref.distribution(d[0], 0, temperature)[1] if drawn else np.zeros(V)
    x = turned_down(p, q) if drawn else int(np.argmax(p))
    if not drawn:
        q[x] = 1.0
    rest = np.maximum(p - q, 0)
    sums = np.cumsum(rest) / rest.sum()
    # ids far enough from their neighbours' borders, likely and unlikely ones
    wide = np.flatnonzero(rest / rest.sum() > 50 * NEAR)
    wide = wide[np.linspace(0, len(wide) - 1, n_seq).astype(int)]
    last = np.nextafter(1.0, 0.0)
    for by in (-NEAR, NEAR):
        u = np.stack([np.full(n_seq, last), np.clip(sums[wide] + by, 0, last)], 1)
        check(dev, np.repeat(t[None], n_seq, 0), np.repeat(d[None], n_seq, 0) if drawn else None, np.full((n_seq, 1), x, np.uint32), None, 0,
              temperature, u)


@pytest.mark.parametrize("V,n_seq,temperature", [(50257, 8, 1.0), (50257, 40, 0.9), (1000, 200, 0.6), (2, 20, 1.3), (131073, 8, 1.44)])
@pytest.mark.parametrize("drawn", [True, False])
def test_numbers_next_to_acceptance(dev, V, n_seq, temperature, drawn):  # noqa: F811
    """A draft is accepted while number * q < p: numbers just below and above p / q, of several drafts behind one another too."""
    rng = np.random.default_rng(V + n_seq)
    n_draft = 3
    t = (rng.standard_normal((n_seq, n_draft + 1, V)) * 2.5).astype(np.float32)
    d = (t[:, :n_draft] + rng.standard_normal((n_seq, n_draft, V)) * 0.7).astype(np.float32)
    ids, u = np.zeros((n_seq, n_draft), np.uint32), rng.random((n_seq, n_draft + 1))
    for s in range(n_seq):
        for i in range(n_draft):
            p = ref.distribution(t[s, i], 0, temperature)[1]
            q = ref.distribution(d[s, i], 0, temperature)[1] if drawn else np.ones(V)
            likely = np.argsort(-p)[:20]
            likely = likely[p[likely] < q[likely]]
            if len(likely) == 0:
                likely = [turned_down(p, q)]
            ids[s, i] = x = likely[rng.integers(len(likely))]
            near = rng.choice([-NEAR, NEAR]) if i == n_draft - 1 else -NEAR
            u[s, i] = min(p[x] / q[x] * (1 + near), np.nextafter(1.0, 0.0))
    accepted = check(dev, t, d if drawn else None, ids, None, 0, temperature, u)[1]
    assert (accepted >= n_draft - 1).all() and (n_seq < 20 or len(set(accepted)) == 2)


@pytest.mark.parametrize("top_k", [0, 6])
@pytest.mark.parametrize("temperature", [5e-324, 1e-300, 1e-39, 3e-39, 1e-20, 1e30, 1e39, 1e300, np.inf])
def test_temperatures_at_the_ends(dev, temperature, top_k):  # noqa: F811
    """Every positive temperature is one: a tiny one leaves the largest logits alone, a huge one makes all finite ones alike."""
    rng = np.random.default_rng(3)
    V = 3000
    t = np.round(rng.standard_normal((6, 3, V)) * 4).astype(np.float32)  # several largest ones
    d = np.round(rng.standard_normal((6, 2, V)) * 4).astype(np.float32)
    if temperature < np.inf:
        t[1, :, ::3], d[2, :, 5:] = -np.inf, -np.inf
    ids = np.stack([np.argmax(t[:, i], axis=1) for i in range(2)], 1).astype(np.uint32)
    ids[4:, 1] = 17
    with np.errstate(over="ignore"):
        check(dev, t, d, ids, None, top_k, temperature, rng.random((6, 3)))
        check(dev, t, None, ids, None, top_k, temperature, rng.random((6, 3)))


@pytest.mark.parametrize("top_k", [0, 7])
@pytest.mark.parametrize("value", [np.nan, -np.inf, np.inf])
@pytest.mark.parametrize("of_draft", [False, True])
def test_rows_without_a_distribution_are_reported(dev, top_k, value, of_draft):  # noqa: F811
    """Each such row by itself, where it decides something: rows of nothing but NaN or -infinity, rows with one +infinity."""
    rng = np.random.default_rng(9)
    V, n_draft = 3000, 2
    for row in range(n_draft if of_draft else n_draft + 1):
        t, d = (rng.standard_normal((3, n, V)).astype(np.float32) for n in (n_draft + 1, n_draft))
        d[...] = t[:, :n_draft]  # accepted wherever the number is below one
        ids, u = np.argmax(t[:, :n_draft], 2).astype(np.uint32), np.full((3, n_draft + 1), 0.5)
        check(dev, t, d, ids, None, top_k, 1.0, u)
        _lib.call("wgpt_device_check", dev.handle)
        x = d if of_draft else t
        if value == np.inf:
            x[1, row, 17] = value
        else:
            x[1, row] = value
        accepted = check(dev, t, d, ids, None, top_k, 1.0, u)[1]
        assert list(accepted) == [n_draft, row, n_draft]
        with pytest.raises(_lib.WgptError) as e:
            _lib.call("wgpt_device_check", dev.handle)
        assert e.value.code == _lib.ERR_ARG and "row of logits" in e.value.message
        if row < n_draft:  # turned down before it: the row decides nothing
            ids[1, 0], u[1, 0] = np.argmin(t[1, 0] if row > 0 or of_draft else d[1, 0]), 1.0
            if row > 0:
                check(dev, t, d, ids, None, top_k, 1.0, u)
                _lib.call("wgpt_device_check", dev.handle)
