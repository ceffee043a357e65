"""Plain 64-bit implementations of the serving operators (numpy, one sequence and row at a time), for the tests."""
import math

import numpy as np

U32 = 2.0 ** -24  # half a step of f32, relative


class Pages:
    """Pools, table and lengths of a cache on the host. Values are held in f32 and are exact in the cache's type; what no
    sequence holds is NaN."""

    def __init__(self, rng, lengths, page_size, n_kv, hs, layout="positions", spare=2, max_length=None, fill=np.nan):
        self.lengths, self.page_size, self.n_kv, self.hs, self.layout = list(lengths), page_size, n_kv, hs, layout
        used = [-(-L // page_size) for L in lengths]
        self.n_pages = max(1, sum(used) + spare)
        order = list(rng.permutation(self.n_pages)[:sum(used)])
        self.max_length = max_length or max(1, max(lengths))
        self.width = max(1, -(-self.max_length // page_size))
        self.table = np.full((len(lengths), self.width), 0xFFFFFFFF, np.uint32)
        for s, n in enumerate(used):
            for i in range(n):
                self.table[s, i] = order.pop()
        self.k = np.full((self.n_pages, page_size, n_kv, hs), fill, np.float32)
        self.v = self.k.copy()

    def place(self, s, j):
        return self.table[s, j // self.page_size], j % self.page_size

    def rows(self, which, s, L=None):
        pool = getattr(self, which)
        n = self.lengths[s] if L is None else L
        return np.stack([pool[self.place(s, j)] for j in range(n)]) if n else np.zeros((0, self.n_kv, self.hs), np.float32)

    def fill(self, rng, cast, scale=1.0):
        for s, L in enumerate(self.lengths):
            for j in range(L):
                for pool in (self.k, self.v):
                    pool[self.place(s, j)] = cast(rng.standard_normal((self.n_kv, self.hs)).astype(np.float32) * scale)


def attend(pages, starts, n_head, scale, window, q, kv=None):
    """Rows [n_rows, n_head, hs] and weights [n_seq, max_length] in 64 bits, and what bounds a row's error: for each
    (row, head) the largest scale * sum |q k| and the vector sum p |v|. Rows of no sequence are NaN."""
    group, hs = n_head // pages.n_kv, pages.hs
    out = np.full((len(q), n_head, hs), np.nan)
    size, top = np.zeros((len(q), n_head, hs)), np.zeros((len(q), n_head))
    weights = np.zeros((len(pages.lengths), pages.max_length))
    for s, L in enumerate(pages.lengths):
        k, v = (pages.rows(w, s).astype(np.float64) for w in ("k", "v"))
        n = starts[s + 1] - starts[s]
        for i in range(n):
            row = starts[s] + i
            end = L - n + i + 1
            begin = max(0, end - window) if window else 0
            for h in range(n_head):
                if end <= begin:
                    out[row, h] = 0
                    continue
                x, kk, vv = q[row, h].astype(np.float64), k[begin:end, h // group], v[begin:end, h // group]
                sc = scale * (kk @ x)
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[row, h] = p @ vv
                size[row, h] = p @ np.abs(vv)
                top[row, h] = scale * (np.abs(kk) @ np.abs(x)).max()
                weights[s, begin:end] += p
    return out, weights, size, top


def attend_tolerance(pages, size, top):
    """What f32 arithmetic may be off by. A score: hs + 2 roundings of products and sums, and q as a sum of half-precision
    values, good to 2^-22 of the row's largest: below (hs + 10) U32 sum|q k|, and as much again for the tensor cores' sums,
    which cut off instead of rounding. A probability: e^(2 * that), sixteen roundings for the exponential of a product and
    its sum. The values' sum: one rounding for every position and rescaling, at most 2 L."""
    L = max(pages.lengths)
    ds = 2 * (pages.hs + 10) * U32 * top
    return size * (2 * ds[..., None] + (2 * L + 16) * U32) + 1e-30


def keep(weights, L, n_keep, recent):
    """The positions that stay."""
    if L <= n_keep:
        return list(range(L))
    old = range(L - recent)
    key = lambda j: (-math.inf if math.isnan(weights[j]) else -float(weights[j]), j)  # noqa: E731
    nan = [j for j in old if math.isnan(weights[j])]
    rest = sorted((j for j in old if not math.isnan(weights[j])), key=key)
    return sorted((nan + rest)[:n_keep - recent]) + list(range(L - recent, L))


def distribution(logits, top_k, temperature):
    """(ids, probabilities) in the order of the running sum, or None: there is none."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    ids = np.arange(len(x))
    if top_k:
        ids = np.argsort(-x, kind="stable")[:top_k]
    if not np.isfinite(x.max()):
        return None
    e = np.exp((x[ids] - x.max()) / temperature)
    return ids, e / e.sum()


def verify(target, draft, draft_ids, n, top_k, temperature, u):
    """(accepted, drawn id) of one sequence: target [n_draft + 1, V], draft [n_draft, V] or None, u [n_draft + 1]."""
    V = target.shape[1]
    for i in range(n + 1):
        d = distribution(target[i], top_k, temperature)
        if i == n:
            if d is None:
                return i, 0
            ids, p = d
            break
        x = int(draft_ids[i])
        dq = distribution(draft[i], top_k, temperature) if draft is not None else (np.array([x]), np.ones(1))
        if x < V and d is not None and dq is not None:
            p_x, q_x = (float(pr[idx == x].sum()) for idx, pr in (d, dq))
            if u[i] * q_x < p_x:
                continue
        if d is None:
            return i, 0
        ids, p = d
        if dq is not None:
            q = np.zeros(V)
            if dq[0][0] < V:
                q[dq[0]] = dq[1]
            rest = np.maximum(p - q[ids], 0)
            p = rest if rest.sum() > 0 else p
        break
    sums = np.cumsum(p)
    return i, int(ids[min(int((sums <= u[-1] * sums[-1]).sum()), len(ids) - 1)])
