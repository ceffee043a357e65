"""Operators of serving over a paged key-value cache, as cases that can be timed.

Four operators that a serving step runs one after the other: the new tokens' key and value rows go into the pages
(append), the new tokens attend over the pages (attend), positions that got little attention leave a full cache
(evict), and drafted tokens are accepted or replaced (verify). With `own` false a pass computes the operator from
elementary torch operations in 32 bits (64 for probabilities that decide a whole number); with `own` true it makes the
package's call on the same inputs.
"""
import ctypes as C
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one user's decode step on gpt2, 200 tokens into the context: the smallest call, latency counts
        {"name": "attend gpt2 1x200", "kind": "attend", "type": "f32", "n_seq": 1, "n_new": 1, "n_head": 12, "n_kv": 12,
         "hs": 64, "page": 16, "longest": 200, "window": 0, "weights": False, "layout": "positions"},
        # gpt2-xl serving sixteen users whose contexts differ
        {"name": "attend xl 16 users", "kind": "attend", "type": "f32", "n_seq": 16, "n_new": 1, "n_head": 25, "n_kv": 25,
         "hs": 64, "page": 16, "longest": 1024, "window": 0, "weights": False, "layout": "positions"},
        # eight users, up to five tokens each to verify, grouped heads, half-precision cache
        {"name": "attend drafts f16", "kind": "attend", "type": "f16", "n_seq": 8, "n_new": 5, "n_head": 32, "n_kv": 8,
         "hs": 128, "page": 64, "longest": 8192, "window": 0, "weights": False, "layout": "heads"},
        # one user with a whole book in the cache: a single token has to be spread over the GPU
        {"name": "attend long bf16", "kind": "attend", "type": "bf16", "n_seq": 1, "n_new": 1, "n_head": 32, "n_kv": 8,
         "hs": 128, "page": 64, "longest": 131072, "window": 0, "weights": False, "layout": "positions"},
        # a batch whose cache is going to be thinned out: the weight that each position got is added up
        {"name": "attend weights f16", "kind": "attend", "type": "f16", "n_seq": 32, "n_new": 1, "n_head": 12, "n_kv": 12,
         "hs": 64, "page": 32, "longest": 4097, "window": 0, "weights": True, "layout": "positions"},
        # one token's rows of one gpt2 layer
        {"name": "append gpt2 1 row", "kind": "append", "type": "f32", "n_seq": 1, "n_new": 1, "n_kv": 12, "hs": 64,
         "page": 16, "longest": 200, "layout": "positions"},
        # the prompts of a batch, of different lengths, into a half-precision cache
        {"name": "append prompts f16", "kind": "append", "type": "f16", "n_seq": 16, "n_new": 1021, "n_kv": 12, "hs": 64,
         "page": 16, "longest": 1024, "layout": "positions"},
        # a few users on gpt2 whose contexts are full: a quarter goes
        {"name": "evict gpt2 4 users", "kind": "evict", "type": "f32", "n_seq": 4, "n_kv": 12, "hs": 64, "page": 16,
         "longest": 1024, "keep": 768, "recent": 128, "layout": "positions"},
        # long contexts thinned out to a quarter
        {"name": "evict long f16", "kind": "evict", "type": "f16", "n_seq": 8, "n_kv": 8, "hs": 128, "page": 64,
         "longest": 32768, "keep": 8191, "recent": 1000, "layout": "heads"},
        # one user, four tokens that a smaller model drafted, gpt2's vocabulary
        {"name": "verify 1 user", "kind": "verify", "n_seq": 1, "n_draft": 4, "V": 50257, "top_k": 0, "temperature": 1.0,
         "draft": True},
        # a full batch of the same
        {"name": "verify 64 users", "kind": "verify", "n_seq": 64, "n_draft": 4, "V": 50257, "top_k": 0,
         "temperature": 0.8, "draft": True},
        # the sampler's kind of distribution: only the best 40 count
        {"name": "verify top 40", "kind": "verify", "n_seq": 16, "n_draft": 5, "V": 50257, "top_k": 40,
         "temperature": 1.0, "draft": True},
    ]


# ------------------------------------------------------------------------------------------ drawn cases
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_once(rng):
    kind = rng.choice(("attend", "attend", "attend", "attend", "append", "evict", "evict", "verify", "verify"))
    if kind == "verify":
        n_draft = rng.randint(0, 8)
        return {"kind": kind, "n_seq": _log_int(rng, 1, 64), "n_draft": n_draft,
                "V": rng.choice((50257, 65, _log_int(rng, 200, 130000))), "top_k": rng.choice((0, 0, rng.randint(1, 64))),
                "temperature": rng.choice((1.0, round(rng.uniform(0.4, 1.6), 2))), "draft": rng.random() < 0.7}
    type_ = rng.choice(("f32", "f16", "bf16"))
    n_kv, hs = rng.choice(((12, 64), (25, 64), (6, 64), (8, 128), (4, 128), (2, 128), (1, 128), (16, 80), (3, 256), (8, 32)))
    group = rng.choice((1, 1, 4, 8, rng.randint(2, 7)))
    case = {"kind": kind, "type": type_, "n_kv": n_kv, "hs": hs, "page": rng.choice((16, 16, 32, 64, 128, rng.randint(1, 100))),
            "layout": rng.choice(("positions", "heads"))}
    if kind == "attend":
        n_seq, longest = _log_int(rng, 1, 128), _log_int(rng, 1, 131072)
        case.update(n_seq=n_seq, n_new=rng.choice((1, 1, 1, rng.randint(2, 9))), n_head=n_kv * group, longest=longest,
                    window=rng.choice((0, 0, 0, _log_int(rng, 1, 4096))), weights=rng.random() < 0.25)
    elif kind == "append":
        longest = _log_int(rng, 1, 2048)
        case.update(n_seq=_log_int(rng, 1, 64), longest=longest, n_new=rng.choice((1, _log_int(rng, 1, longest))))
    else:
        longest = _log_int(rng, 64, 65536)
        keep = max(1, int(longest * rng.uniform(0.1, 0.9)))
        case.update(n_seq=_log_int(rng, 1, 32), longest=longest, keep=keep, recent=int(keep * rng.uniform(0, 0.5)))
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw_once(rng)
        if _cost(c) > most:
            continue
        # the plain forms hold padded rows of all sequences: room for them
        if c["kind"] == "attend" and (c["n_seq"] * c["longest"] * c["n_kv"] * c["hs"] > 3e8
                                      or c["n_seq"] * c["longest"] * c["n_head"] * c["n_new"] > 1e8):
            continue
        if c["kind"] == "append" and c["n_seq"] * c["longest"] * c["n_kv"] * c["hs"] > 1e8:
            continue
        if c["kind"] == "evict" and c["n_seq"] * c["longest"] * c["n_kv"] * c["hs"] > 6e8:
            continue
        return c


def _lengths(case):
    """The sequences' lengths: the first is the longest, the others differ from a quarter of it on."""
    r = random.Random(case["longest"] * 131 + case["n_seq"])
    return [case["longest"]] + [r.randint(max(1, case["longest"] // 4), case["longest"]) for _ in range(case["n_seq"] - 1)]


def _new(case):
    """How many new tokens each sequence has: the most for the first, one or more for the others."""
    r = random.Random(case["n_new"] * 17 + case["n_seq"])
    return [min(L, case["n_new"] if s == 0 else r.randint(max(1, case["n_new"] // 2), case["n_new"]))
            for s, L in enumerate(_lengths(case))]


def _drafted(case):
    r = random.Random(case["n_draft"] * 23 + case["n_seq"])
    return [case["n_draft"] if s == 0 else r.randint((case["n_draft"] + 1) // 2, case["n_draft"]) for s in range(case["n_seq"])]


# ------------------------------------------------------------------------------------------ what a program has in hand
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(case, lengths, g, empty=False):
    """Pools of pages, each sequence's pages scattered over them, and the table that finds them (entries behind a
    sequence's last page name no page)."""
    page, n_kv, hs = case["page"], case["n_kv"], case["hs"]
    used = [-(-L // page) for L in lengths]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda")[:sum(used)].to(torch.int32)
    width = max(used) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), torch.tensor(used, device="cuda"))
    first = torch.tensor(np.concatenate([[0], np.cumsum(used)[:-1]]), device="cuda")
    table[seq, torch.arange(sum(used), device="cuda") - first[seq]] = order
    shape = (n_pages, page, n_kv, hs) if case["layout"] == "positions" else (n_pages, n_kv, page, hs)
    pool = (lambda: torch.zeros(shape, dtype=TYPES[case["type"]], device="cuda")) if empty else \
        (lambda: torch.randn(shape, generator=g, device="cuda", dtype=TYPES[case["type"]]))
    return {"k": pool(), "v": pool(), "table": table, "lengths": _ints(lengths), "longest": max(lengths),
            "layout": case["layout"], "type": case["type"]}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "verify":
        return _prepare_verify(case, g)
    lengths = _lengths(case)
    state = {"case": dict(case), "cache": _cache(case, lengths, g)}
    if kind == "evict":
        n_seq, width = case["n_seq"], case["longest"]
        # weights as a long-running softmax leaves them: a few positions hold most, many are near zero, some equal
        w = torch.rand(n_seq, width, generator=g, device="cuda") ** 6 * 40
        state["weights"] = torch.where(w < 1e-3, torch.round(w * 1e4) / 1e4, w)
        state["to"] = _cache(case, [min(L, case["keep"]) for L in lengths], g, empty=True)
        state["weights_to"] = torch.zeros(n_seq, case["keep"], device="cuda")
        state["kept"] = torch.zeros(n_seq, case["keep"], dtype=torch.int32, device="cuda")
        return state
    new = _new(case)
    state["new"] = new
    state["starts"] = _ints([0] + list(np.cumsum(new)))
    rows = sum(new)
    if kind == "append":
        state["kv"] = torch.randn(rows, 2 * case["n_kv"] * case["hs"], generator=g, device="cuda")  # k | v, as a product leaves them
        return state
    state["q"] = torch.randn(rows, case["n_head"] * case["hs"], generator=g, device="cuda") * 1.5
    state["out"] = torch.zeros(rows, case["n_head"] * case["hs"], device="cuda")
    state["scale"] = 1 / math.sqrt(case["hs"])
    if case["weights"]:
        state["weights"] = torch.rand(case["n_seq"], case["longest"], generator=g, device="cuda")
    return state


def _prepare_verify(case, g):
    n_seq, n, V = case["n_seq"], case["n_draft"], case["V"]
    r = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    target = r(n_seq, n + 1, V) * 2.5 - 3.0
    state = {"case": dict(case), "target": target, "draft": None}
    drawn = target[:, :n] + r(n_seq, n, V) * 0.7  # the smaller model's opinion
    if case["draft"]:
        state["draft"] = drawn.contiguous()
    z = drawn.double() / case["temperature"]
    if case["top_k"] and n:
        least = torch.topk(z, min(case["top_k"], V), dim=-1).values[..., -1:]
        z = torch.where(z < least, -math.inf, z)
    if not case["draft"]:
        z = z * 4  # looked up, not drawn: mostly a likely token
    e = -torch.log(torch.rand(n_seq, n, V, generator=g, device="cuda", dtype=torch.float64).clamp_min(1e-300))
    state["draft_ids"] = torch.argmax(z - torch.log(e), dim=-1).to(torch.int32).contiguous()
    state["n_drafted"] = _ints(_drafted(case))
    state["uniforms"] = torch.rand(n_seq, n + 1, generator=g, device="cuda", dtype=torch.float64)
    state["ids"] = torch.zeros(n_seq, n + 1, dtype=torch.int32, device="cuda")
    state["accepted"] = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    return state


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        _call_now(state)
    else:
        {"attend": _attend, "append": _append, "evict": _evict, "verify": _verify}[kind](state)
    if kind == "attend":
        return {"out": state["out"], "weights": state["weights"]} if "weights" in state else {"out": state["out"]}
    if kind == "append":
        return {"k": state["cache"]["k"], "v": state["cache"]["v"]}
    if kind == "evict":
        to = state["to"]
        return {"kept": state["kept"], "lengths": to["lengths"], "k": to["k"], "v": to["v"], "weights": state["weights_to"]}
    return {"ids": state["ids"], "accepted": state["accepted"]}


# the package's calls
_devices = []


def _device():
    from webgpt_b200 import Device
    if not _devices:
        _devices.append(Device())
    return _devices[0]


def _descriptor(c):
    from webgpt_b200 import _lib
    a, b = (1, 2) if c["layout"] == "positions" else (2, 1)  # which dimension counts positions, which heads
    s = c["k"].stride()
    return _lib.PagedCache(c["k"].data_ptr(), c["v"].data_ptr(), c["table"].data_ptr(), c["lengths"].data_ptr(), s[0], s[a], s[b],
                           {"f32": _lib.TYPE_F32, "f16": _lib.TYPE_F16, "bf16": _lib.TYPE_BF16}[c["type"]], c["k"].shape[0],
                           c["k"].shape[a], c["k"].shape[b], c["k"].shape[3], len(c["lengths"]), c["table"].shape[1], c["longest"])


def _call(state):
    """The call's name and arguments, which a program builds once for its buffers."""
    case, dev = state["case"], _device()
    if case["kind"] == "verify":
        n_seq, n, V = case["n_seq"], case["n_draft"], case["V"]
        draft = state["draft"].data_ptr() if state["draft"] is not None and n else None
        return ("wgpt_verify_drafts", dev.handle, n_seq, n, V, state["target"].data_ptr(), V, draft, V,
                state["draft_ids"].data_ptr() if n else None, state["n_drafted"].data_ptr(), min(case["top_k"], V), case["temperature"],
                state["uniforms"].data_ptr(), state["ids"].data_ptr(), state["accepted"].data_ptr())
    state["descriptor"] = cache = _descriptor(state["cache"])
    if case["kind"] == "evict":
        state["descriptor_to"] = to = _descriptor(state["to"])
        return ("wgpt_paged_evict", dev.handle, C.byref(cache), C.byref(to), case["keep"], case["recent"],
                state["weights"].data_ptr(), state["weights"].shape[1], state["weights_to"].data_ptr(),
                state["weights_to"].shape[1], state["kept"].data_ptr())
    starts = state["starts"].data_ptr()
    if case["kind"] == "append":
        width = case["n_kv"] * case["hs"]
        k = state["kv"].data_ptr()
        return ("wgpt_paged_append", dev.handle, C.byref(cache), len(state["kv"]), starts, k, k + 4 * width, 2 * width)
    E = case["n_head"] * case["hs"]
    w = state.get("weights")
    return ("wgpt_paged_attention", dev.handle, C.byref(cache), len(state["q"]), starts, case["n_head"], state["scale"],
            case["window"], state["q"].data_ptr(), E, state["out"].data_ptr(), E, w.data_ptr() if w is not None else None,
            w.shape[1] if w is not None else 0)


def _call_now(state):
    from webgpt_b200 import _lib
    _lib.call(*state["call"])


# the plain forms
def _pages(c, pool):
    """The pool as [page, position, head, feature], whatever its layout."""
    return pool if c["layout"] == "positions" else pool.transpose(1, 2)


def _places(c, page, positions):
    """(page, slot) of positions [n_seq, n]; places behind a sequence's pages read page 0."""
    at = torch.gather(c["table"].long(), 1, (positions // page).clamp_max(c["table"].shape[1] - 1))
    return at.clamp_min(0), positions % page


def _attend(state):
    case, c = state["case"], state["cache"]
    n_seq, H, kv, hs, T = case["n_seq"], case["n_head"], case["n_kv"], case["hs"], max(state["new"])
    L, starts = c["lengths"].long(), state["starts"].long()
    new = starts[1:] - starts[:-1]
    j = torch.arange(c["longest"], device="cuda")
    at = _places(c, case["page"], j.expand(n_seq, -1))
    K = _pages(c, c["k"])[at].float().permute(0, 2, 1, 3)  # [sequence, head, position, feature]
    V = _pages(c, c["v"])[at].float().permute(0, 2, 1, 3)
    i = torch.arange(T, device="cuda")
    row = (starts[:-1, None] + i).clamp_max(len(state["q"]) - 1)
    q = state["q"][row].view(n_seq, T, kv, H // kv, hs).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, H // kv * T, hs)
    s = torch.matmul(q, K.transpose(2, 3)).view(n_seq, kv, H // kv, T, -1) * state["scale"]
    end = (L - new)[:, None] + i + 1
    sees = (j < end[..., None]) & (i < new[:, None])[..., None]
    if case["window"]:
        sees &= j >= (end - case["window"])[..., None]
    sees = sees[:, None, None]
    s = torch.where(sees, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(sees, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.view(n_seq, kv, H // kv * T, -1), V).view(n_seq, kv, H // kv, T, hs)
    o = o.permute(0, 3, 1, 2, 4).reshape(n_seq, T, H * hs)
    state["out"].copy_(o[i.expand(n_seq, -1) < new[:, None]])
    if "weights" in state:
        state["weights"] += p.sum((1, 2, 3))


def _append(state):
    case, c = state["case"], state["cache"]
    starts = state["starts"].long()
    new = starts[1:] - starts[:-1]
    rows = len(state["kv"])
    seq = torch.repeat_interleave(torch.arange(case["n_seq"], device="cuda"), new, output_size=rows)
    pos = (c["lengths"].long() - new)[seq] + torch.arange(rows, device="cuda") - starts[seq]
    at = c["table"].long()[seq, pos // case["page"]], pos % case["page"]
    k, v = state["kv"].view(rows, 2, case["n_kv"], case["hs"]).unbind(1)
    _pages(c, c["k"])[at] = k.to(c["k"].dtype)
    _pages(c, c["v"])[at] = v.to(c["v"].dtype)


def _evict(state):
    case, c, to = state["case"], state["cache"], state["to"]
    keep, recent, n_seq = case["keep"], case["recent"], case["n_seq"]
    L = c["lengths"].long()[:, None]
    w = state["weights"]
    j = torch.arange(w.shape[1], device="cuda")
    # the newest and, where everything fits, all positions come first, then the older by weight, then what is not there
    key = torch.where((j >= L - recent) | (L <= keep), math.inf, w)
    key = torch.where(j < L, key, -math.inf)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :keep]
    n = L.clamp_max(keep)
    i = torch.arange(order.shape[1], device="cuda")
    kept = torch.sort(torch.where(i < n, order, w.shape[1]), dim=1).values
    there = i < n
    kept = torch.where(there, kept, 0)
    state["kept"].fill_(-1)
    state["kept"][:, :len(i)] = torch.where(there, kept, -1)
    state["weights_to"].zero_()
    state["weights_to"][:, :len(i)] = torch.where(there, torch.gather(w, 1, kept), 0.0)
    to["lengths"].copy_(n[:, 0])
    page, slot = _places(c, case["page"], kept)
    page_to, slot_to = _places(to, case["page"], i.expand(n_seq, -1))
    src, dst = (page[there], slot[there]), (page_to[there], slot_to[there])
    _pages(to, to["k"])[dst] = _pages(c, c["k"])[src]
    _pages(to, to["v"])[dst] = _pages(c, c["v"])[src]


def _probabilities(logits, top_k, temperature):
    """softmax(logits / temperature) in 64 bits, over the top_k largest where that is asked for (lowest index first
    among equals): the probabilities, and the order in which they are added up."""
    z = logits.double()
    order = None
    if top_k:
        order = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :top_k]
        z = torch.full_like(z, -math.inf).scatter(-1, order, torch.gather(z, -1, order))
    e = torch.exp((z - z.amax(-1, keepdim=True)) / temperature)
    return e / e.sum(-1, keepdim=True), order


def _verify(state):
    case = state["case"]
    n_seq, n, V = case["n_seq"], case["n_draft"], case["V"]
    top_k, T = min(case["top_k"], V), case["temperature"]
    drafted, u = state["n_drafted"].long(), state["uniforms"]
    p, order = _probabilities(state["target"], top_k, T)
    s = torch.arange(n_seq, device="cuda")
    ids = state["draft_ids"].long()
    if state["draft"] is not None:
        q = _probabilities(state["draft"], top_k, T)[0]
    else:
        q = torch.zeros(n_seq, n, V, dtype=torch.float64, device="cuda").scatter_(2, ids[..., None], 1.0)
    i = torch.arange(n, device="cuda")
    px, qx = (torch.gather(x[:, :n], 2, ids[..., None])[..., 0] for x in (p, q))
    ok = (u[:, :n] * qx < px) & (i < drafted[:, None])
    accepted = torch.cumprod(ok.long(), 1).sum(1)
    p = p[s, accepted]
    q = torch.cat([q, torch.zeros(n_seq, 1, V, dtype=torch.float64, device="cuda")], 1)[s, accepted]
    rest = torch.where((accepted < drafted)[:, None], (p - q).clamp_min(0), p)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    if order is not None:
        order = order[s, accepted]
        rest = torch.gather(rest, 1, order)
    sums = torch.cumsum(rest, 1)
    pick = (sums <= u[:, n:] * sums[:, -1:]).sum(1, keepdim=True).clamp_max(rest.shape[1] - 1)
    if order is not None:
        pick = torch.gather(order, 1, pick)
    i = torch.arange(n + 1, device="cuda")
    ids = torch.cat([ids, torch.zeros_like(pick)], 1)
    state["ids"].copy_(torch.where(i < accepted[:, None], ids, torch.where(i == accepted[:, None], pick, -1)))
    state["accepted"].copy_(accepted)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "verify":
        rows = sum(n + 1 + (n if case["draft"] else 0) for n in _drafted(case))
        return {"bytes": 4.0 * rows * case["V"] + 8.0 * case["n_seq"] * (case["n_draft"] + 1), "flops": 3.0 * rows * case["V"]}
    lengths, kv, hs = _lengths(case), case["n_kv"], case["hs"]
    size = 4 if case["type"] == "f32" else 2
    if kind == "append":
        rows = sum(_new(case))
        return {"bytes": 2.0 * rows * kv * hs * (4 + size), "flops": 0.0}
    if kind == "evict":
        kept = sum(min(L, case["keep"]) for L in lengths)
        return {"bytes": 4.0 * kept * kv * hs * size + 4.0 * sum(lengths) + 8.0 * kept, "flops": 0.0}
    new = _new(case)
    window = case["window"] or case["longest"]
    seen = sum(L - max(0, L - n + 1 - window) for L, n in zip(lengths, new))  # positions that some new token sees
    pairs = sum(min(L - n + i + 1, window) for L, n in zip(lengths, new) for i in range(n))
    return {"bytes": 2.0 * seen * kv * hs * size + 8.0 * sum(new) * case["n_head"] * hs + (8.0 * seen if case["weights"] else 0.0),
            "flops": 4.0 * pairs * case["n_head"] * hs}


# ------------------------------------------------------------------------------------------ by definition, in 64 bits
def exact(case, seed):
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict, "verify": _exact_verify}[case["kind"]](
        case, prepare(case, seed))


def _one(case, c, which, s, positions):
    """Rows of one sequence at the given positions, [n, n_kv, hs]."""
    pages = c["table"][s].long()[positions // case["page"]]
    slots = positions % case["page"]
    return c[which][pages, slots] if case["layout"] == "positions" else c[which][pages, :, slots]


def _exact_attend(case, state):
    c, out, row = state["cache"], [], 0
    group = case["n_head"] // case["n_kv"]
    weights = state["weights"].double() if case["weights"] else None
    for s, (L, n) in enumerate(zip(_lengths(case), state["new"])):
        every = torch.arange(L, device="cuda")
        k, v = (_one(case, c, w, s, every).double().transpose(0, 1) for w in ("k", "v"))
        for t in range(n):
            end = L - n + t + 1
            begin = max(0, end - case["window"]) if case["window"] else 0
            q = state["q"][row].double().view(case["n_kv"], group, case["hs"])
            p = torch.softmax(torch.bmm(q, k[:, begin:end].transpose(1, 2)) / math.sqrt(case["hs"]), dim=-1)
            out.append(torch.bmm(p, v[:, begin:end]).reshape(-1))
            if weights is not None:
                weights[s, begin:end] += p.sum((0, 1))
            row += 1
    out = torch.stack(out)
    return {"out": out, "weights": weights} if case["weights"] else {"out": out}


def _exact_append(case, state):
    c, row = state["cache"], 0
    pools = {"k": c["k"].double(), "v": c["v"].double()}
    rows = state["kv"].to(c["k"].dtype).double().view(-1, 2, case["n_kv"], case["hs"])
    for s, (L, n) in enumerate(zip(_lengths(case), state["new"])):
        pos = torch.arange(L - n, L, device="cuda")
        pages, slots = c["table"][s].long()[pos // case["page"]], pos % case["page"]
        for x, which in enumerate(("k", "v")):
            if case["layout"] == "positions":
                pools[which][pages, slots] = rows[row:row + n, x]
            else:
                pools[which][pages, :, slots] = rows[row:row + n, x]
        row += n
    return pools


def _exact_evict(case, state):
    c, to = state["cache"], state["to"]
    keep, recent = case["keep"], case["recent"]
    k, v, w_to = to["k"].double(), to["v"].double(), state["weights_to"].double()
    kept_to, lengths = state["kept"].clone().fill_(-1), []
    weights = state["weights"].double().cpu().numpy()
    for s, L in enumerate(_lengths(case)):
        kept = np.arange(L)
        if L > keep:
            best = np.lexsort((np.arange(L - recent), -weights[s, :L - recent]))[:keep - recent]
            kept = np.concatenate([np.sort(best), np.arange(L - recent, L)])
        kept = torch.tensor(kept, device="cuda")
        n = len(kept)
        at = torch.arange(n, device="cuda")
        pages, slots = to["table"][s].long()[at // case["page"]], at % case["page"]
        for pool, which in ((k, "k"), (v, "v")):
            if case["layout"] == "positions":
                pool[pages, slots] = _one(case, c, which, s, kept).double()
            else:
                pool[pages, :, slots] = _one(case, c, which, s, kept).double()
        kept_to[s, :n] = kept.to(torch.int32)
        w_to[s, :n] = torch.tensor(weights[s], device="cuda")[kept]
        lengths.append(n)
    return {"kept": kept_to, "lengths": _ints(lengths), "k": k, "v": v, "weights": w_to}


def _exact_verify(case, state):
    n_seq, n, V, T = case["n_seq"], case["n_draft"], case["V"], case["temperature"]
    target = state["target"].cpu().numpy()
    draft = state["draft"].cpu().numpy() if state["draft"] is not None else None
    drafts, u, drafted = state["draft_ids"].cpu().numpy(), state["uniforms"].cpu().numpy(), _drafted(case)

    def distribution(logits):
        """(ids, probabilities) in the order of the running sum."""
        x = logits.astype(np.float64)
        ids = np.arange(V)
        if case["top_k"]:
            ids = np.argsort(-x, kind="stable")[:case["top_k"]]
        e = np.exp((x[ids] - x.max()) / T)
        return ids, e / e.sum()

    out, accepted = np.full((n_seq, n + 1), -1, np.int32), np.zeros(n_seq, np.int32)
    for s in range(n_seq):
        a = 0
        while True:
            ids, p = distribution(target[s, a])
            if a == drafted[s]:
                break
            x = drafts[s, a]
            q = np.zeros(V)
            if draft is None:
                q[x] = 1.0
            else:
                from_, by = distribution(draft[s, a])
                q[from_] = by
            if u[s, a] * q[x] < p[ids == x].sum():
                out[s, a] = x
                a += 1
                continue
            rest = np.maximum(p - q[ids], 0)
            p = rest if rest.sum() > 0 else p
            break
        sums = np.cumsum(p)
        out[s, a] = ids[min(int((sums <= u[s, n] * sums[-1]).sum()), len(ids) - 1)]
        accepted[s] = a
    return {"ids": torch.tensor(out), "accepted": torch.tensor(accepted)}
