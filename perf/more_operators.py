"""A cached history that is kept small, as cases that can be timed and compared: new tokens attend to the first keys of the cache and to a
window behind them; the attention weight that every cached key receives is added up; and the keys that received the least leave the cache, the
others move together.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, from the seed alone (ragged lengths and tree shapes come with the case)
    run(state)          one pass: the plain form, or with `own` the package's operators
    work(case)          bytes and floating-point operations the pass cannot do without
    exact(case, seed)   the same results from the definition in 64 bits

What a token sees.  Request b has lengths[b] keys in its paged cache, in places 0, 1, ...; its new tokens sit behind them, stored already.  A token
may see all cached keys, and of the new ones token j where pre[j] <= pre[i] < end[j] (spans; None: a chain, the tokens up to itself; pre = -1: padding,
which sees and is seen by nothing).  A window w and s first keys leave of these the keys whose place is behind the token's place - w, or in front of s.
A new token's place is positions[i] (in a tree: the cached keys and its depth); without positions a chain's tokens stand one behind the other, those of
other shapes all directly behind the cache."""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"


# ---- the cases --------------------------------------------------------------------------------------------------------

def _window(name, batch, tokens, cached, heads, kv_heads, dh, page, shape, *, window, sinks, cap=0.0, ragged=True, padding=0):
    return dict(name=name, kind="window", batch=batch, tokens=tokens, cached=cached, heads=heads, kv_heads=kv_heads, dh=dh, page=page, shape=shape,
                window=window, sinks=sinks, cap=cap, ragged=ragged, padding=padding, decay=1.0)


def _weights(name, batch, tokens, cached, heads, kv_heads, dh, page, shape, *, window=0, sinks=0, cap=0.0, decay=1.0, ragged=True, padding=0):
    return dict(name=name, kind="weights", batch=batch, tokens=tokens, cached=cached, heads=heads, kv_heads=kv_heads, dh=dh, page=page, shape=shape,
                window=window, sinks=sinks, cap=cap, ragged=ragged, padding=padding, decay=decay)


def _evict(name, batch, cached, budget, kv_heads, dh, page, *, sinks, recent, ragged=True):
    return dict(name=name, kind="evict", batch=batch, tokens=0, cached=cached, budget=budget, kv_heads=kv_heads, dh=dh, page=page, sinks=sinks, recent=recent,
                ragged=ragged)


def listed():
    return [
        # one new token behind a short window: launch latency is all there is
        _window("window_one_token", 1, 1, 511, 8, 8, 64, 16, "chain", window=128, sinks=4),
        # a loaded server, one new token for every user of a long history: bound by reading the windows once
        _window("window_single_tokens", 96, 1, 16384, 16, 4, 128, 64, "chain", window=2048, sinks=4),
        # long prompts enter chunk by chunk: the products of a band
        _window("window_chunk", 4, 2048, 8192, 16, 4, 128, 64, "chain", window=1024, sinks=16),
        # drafted trees of up to 32 tokens behind long histories, capped logits, small pages, some padding
        _window("window_drafts", 24, 32, 20000, 32, 8, 128, 16, "tree", window=4096, sinks=4, cap=30.0, padding=2),
        # candidates of a ranking batch over the recent part of their histories, each one seeing itself only
        _window("window_candidates", 32, 512, 4096, 8, 8, 64, 128, "isolated", window=512, sinks=1),
        # the weight that one new token gives to a short history: the smallest call
        _weights("weights_one_token", 1, 1, 127, 8, 8, 64, 16, "chain"),
        # one new token for every user, older weights fading: bound by reading the keys once
        _weights("weights_single_tokens", 96, 1, 4096, 16, 4, 128, 64, "chain", decay=0.99),
        # which posts of their histories a ranking batch's candidates look at
        _weights("weights_candidates", 32, 512, 1022, 8, 8, 64, 128, "isolated"),
        # the weights of a history that has just entered the cache, all rows seeing all: bound by products and exponentials
        _weights("weights_history", 8, 1022, 0, 16, 4, 128, 64, "whole", ragged=False),
        # one user's cache over its budget by a few keys
        _evict("evict_one", 1, 200, 128, 8, 64, 16, sinks=4, recent=32, ragged=False),
        # a server's round over many users: half of the keys leave
        _evict("evict_batch", 64, 4096, 2048, 4, 128, 64, sinks=4, recent=256),
        # two users with very long histories: the work has to be split along the cache
        _evict("evict_long", 2, 100003, 32768, 4, 128, 32, sinks=4, recent=1024),
    ]


HEADS = [(4, 4, 32), (8, 8, 64), (16, 2, 64), (16, 4, 128), (32, 8, 128), (24, 8, 128), (16, 1, 128), (10, 2, 64)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    what = rng.random()
    heads, kv_heads, dh = rng.choice(HEADS)
    page = rng.choice([16, 32, 48, 64, 128])
    if what < 0.7:
        batch = _log(rng, 1, 96)
        shape = rng.choice(["chain", "chain", "tree", "isolated"] if what < 0.4 else ["chain", "chain", "tree", "isolated", "whole"])
        tokens = _log(rng, 1, 64 if shape == "tree" else 2048)
        window, sinks = (_log(rng, 1, 8192), rng.choice([0, 1, 4, 16, 100])) if what < 0.4 or rng.random() < 0.2 else (0, 0)

        # at most about the cache bytes, the pairs and the products of the largest listed cases; `keys` per request in all, `near` of them seen
        def most():
            near = min(100000, 400_000_000 // (batch * kv_heads * dh * 4), 190_000_000 // (batch * heads * tokens), 48_000_000_000 // (4 * dh * heads * tokens * batch))
            return near, min(100000, 1_600_000_000 // (batch * kv_heads * dh * 4))
        near, keys = most()
        while near < 2 * tokens and (batch > 1 or tokens > 1):
            batch, tokens = (batch + 1) // 2, (tokens + 1) // 2 if batch == 1 else tokens
            near, keys = most()
        if what < 0.4:
            window = max(1, min(window, near - sinks - tokens))
        else:
            keys = near
        cached = _log(rng, 1, max(1, keys - tokens)) - (rng.random() < 0.1)
        more = dict(window=window, sinks=sinks, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), ragged=rng.random() < 0.7, padding=rng.choice([0, 0, 1, 3]) if shape != "chain" else 0)
        if what < 0.4:
            c = _window("", batch, tokens, cached, heads, kv_heads, dh, page, shape, **more)
        else:
            c = _weights("", batch, tokens, cached, heads, kv_heads, dh, page, shape, decay=rng.choice([1.0, 0.95]), **more)
    else:
        batch = _log(rng, 1, 128)
        cached = _log(rng, 17, max(17, min(100000, 400_000_000 // (batch * kv_heads * dh * 4))))
        budget = max(1, int(cached * rng.choice([0.1, 0.25, 0.5, 0.8, 0.97])))
        sinks = min(rng.choice([0, 1, 4, 16]), budget)
        c = _evict("", batch, cached, budget, kv_heads, dh, page, sinks=sinks, recent=rng.randrange(0, (budget - sinks) // 2 + 1), ragged=rng.random() < 0.7)
    del c["name"]
    return c


# ---- what comes with a case: ragged lengths and tree shapes -------------------------------------------------------------

def _lengths(c):
    """New tokens and cached keys of every request."""
    rng = random.Random("%d %d %d %d" % (c["batch"], c["tokens"], c["cached"], c["dh"]))
    if not c["ragged"]:
        return [c["tokens"]] * c["batch"], [c["cached"]] * c["batch"]
    tokens = [rng.randint(min(1, c["tokens"]) if c["tokens"] < 2 else c["tokens"] // 2, c["tokens"]) for _ in range(c["batch"])]
    cached = [rng.randint(c["cached"] // 4, c["cached"]) for _ in range(c["batch"])]
    at = rng.randrange(c["batch"])   # one request has the full size
    tokens[at], cached[at] = c["tokens"], c["cached"]
    return tokens, cached


def _shape(c, n, rng):
    """(pre, end, depth) of n new tokens; the last `padding` of them are padding."""
    live = max(1, n - c["padding"])
    if c["shape"] == "chain":
        made = [(i, live, i) for i in range(live)]
    elif c["shape"] == "isolated":
        made = [(i, i + 1, 0) for i in range(live)]
    elif c["shape"] == "whole":
        made = [(0, 1, 0)] * live
    else:                            # a tree in the order it grew (parents first, levels mixed)
        parent = [-1] + [rng.randint(-1 if rng.random() < 0.1 else 0, i - 1) for i in range(1, live)]
        below, depth = [1] * live, [0] * live
        for i in range(live - 1, 0, -1):
            if parent[i] >= 0:
                below[parent[i]] += below[i]
        pre, nxt, top = [0] * live, [0] * live, 0
        for i in range(live):        # a parent is placed before its children
            if parent[i] < 0:
                pre[i], top = top, top + below[i]
            else:
                pre[i], depth[i] = nxt[parent[i]], depth[parent[i]] + 1
                nxt[parent[i]] += below[i]
            nxt[i] = pre[i] + 1
        made = [(p, p + b, d) for p, b, d in zip(pre, below, depth)]
    return made + [(-1, -1, 0)] * (n - live)


def _shapes(c, tokens):
    rng = random.Random("%s %d %d" % (c["shape"], c["batch"], c["tokens"]))
    return [_shape(c, n, rng) for n in tokens]


def _seen(c, made, cached):
    """Pairs of one request's tokens and the keys that they see, and the number of different keys seen."""
    w = c["window"] or 1 << 30
    pairs = 0
    if c["shape"] == "chain":        # the window up to itself, the first keys in front of it
        pairs = sum(min(p + 1, w) + min(c["sinks"], max(0, p + 1 - w)) for p in range(cached, cached + len(made)))
    else:
        live = [m for m in made if m[0] >= 0]
        starts = [0] * (len(live) + 1)   # tokens whose place in the walk lies in front of ...
        for p, _, _ in live:
            starts[p + 1] += 1
        for i in range(len(live)):
            starts[i + 1] += starts[i]
        for p, e, d in live:         # of the cache the first keys and the window; as a new key: all tokens in its span
            first = max(0, cached + d - w + 1)
            pairs += cached - min(first, cached) + min(c["sinks"], first, cached) + starts[min(e, len(live))] - starts[p]
    first = max(0, cached - w + 1)   # of the first token behind the cache
    return pairs, len(made) + cached - min(first, cached) + min(c["sinks"], first, cached)


def work(case):
    c = case
    tokens, cached = _lengths(c)
    row = c["dh"] * 2
    if c["kind"] == "evict":
        kept = sum(min(k, c["budget"]) for k in cached)
        # every weight read, every key that stays read and written with its weight, its number written
        return {"bytes": c["kv_heads"] * (sum(cached) * 4 + kept * (2 * 2 * row + 4 + 4)), "flops": c["kv_heads"] * sum(cached)}
    seen = [_seen(c, made, k) for made, k in zip(_shapes(c, tokens), cached)]
    n, pairs, keys = sum(tokens), sum(p for p, _ in seen), sum(k for _, k in seen)
    spans = n * 8 if c["shape"] != "chain" else 0
    if c["kind"] == "weights":
        touched = keys if c["decay"] == 1.0 else sum(tokens) + sum(cached)
        return {"bytes": keys * c["kv_heads"] * row + touched * c["kv_heads"] * 8 + n * c["heads"] * (row + 4) + spans, "flops": (2 * c["dh"] + 3) * c["heads"] * pairs}
    return {"bytes": keys * c["kv_heads"] * row * 2 + n * c["heads"] * (2 * row + 4) + spans, "flops": 4 * c["dh"] * c["heads"] * pairs}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    tokens, cached = _lengths(c)
    n = sum(tokens)
    # a pool of pages that hold noise, a shuffled page table (-1 behind a request's last page)
    need = [-(-(t + k) // c["page"]) for t, k in zip(tokens, cached)]
    total = sum(need) + 3
    pages = torch.randn((total, 2, c["kv_heads"], c["page"], c["dh"]), dtype=torch.bfloat16, device=DEV, generator=gen)
    order = torch.randperm(total, device=DEV, generator=gen)
    at = torch.tensor([0] + need).cumsum(0)[:-1].to(DEV)
    col = torch.arange(max(need) + 1, device=DEV)
    table = torch.where(col[None] < torch.tensor(need, device=DEV)[:, None], order[(at[:, None] + col[None]).clamp(max=total - 1)], -1).to(torch.int32)
    s = dict(case=c, pages=pages, table=table, lengths=torch.tensor(cached, dtype=torch.int32, device=DEV), most_tokens=max(tokens),
             most_keys=max(t + k for t, k in zip(tokens, cached)))
    if c["kind"] != "window":        # what the keys received so far: a few much, most little
        s["weights"] = torch.randn((total, c["kv_heads"], c["page"]), device=DEV, generator=gen).mul_(1.5).exp_().mul_(0.05)
    if c["kind"] == "evict":
        return s
    q = torch.randn((n, c["heads"], c["dh"]), dtype=torch.bfloat16, device=DEV, generator=gen)
    made = _shapes(c, tokens)
    spans = positions = None
    if c["shape"] != "chain":
        spans = torch.tensor([(p, e) for m in made for p, e, _ in m], dtype=torch.int32).to(DEV)
    if c["shape"] == "tree" and c["window"]:
        positions = torch.tensor([k + d for m, k in zip(made, cached) for _, _, d in m], dtype=torch.int32).to(DEV)
    s.update(q=q, spans=spans, positions=positions, scale=math.sqrt(128.0) / c["dh"],
             q_start=torch.tensor([0] + tokens, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV))
    if c["kind"] == "weights":       # the rows' log of the sum of exponentials, which the attention in front gives
        x, _, _ = _logits(s, _places(s))
        request, place = _owners(s)
        s["lse"] = torch.logsumexp(x, -1).permute(0, 3, 1, 2)[request, place].reshape(n, c["heads"]).contiguous()
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    s = state
    c = s["case"]
    if own:
        from x_algorithm_b200 import decoding
        if c["kind"] == "evict":
            lengths, kept = decoding.evict(s["weights"], s["pages"], s["lengths"], s["table"], budget=c["budget"], sinks=c["sinks"], recent=c["recent"])
            return s["pages"], s["weights"], lengths, kept
        more = dict(spans=s["spans"], positions=s["positions"], window=c["window"] or None, sinks=c["sinks"], sm_scale=s["scale"], cap=c["cap"],
                    cap_method="tanh" if c["cap"] else None, max_tokens=s["most_tokens"], max_keys=s["most_keys"])
        if c["kind"] == "window":
            return decoding.window_attention(s["q"], s["pages"], s["q_start"], s["lengths"], s["table"], **more)
        return decoding.key_weights(s["q"], s["pages"], s["q_start"], s["lengths"], s["table"], s["lse"], s["weights"], decay=c["decay"], **more)
    return {"window": _plain_window, "weights": _plain_weights, "evict": _plain_evict}[c["kind"]](s)


def _owners(s):
    """The request of each new token and its place among that request's new tokens."""
    token = torch.arange(s["q"].shape[0], device=DEV)
    request = (token[:, None] >= s["q_start"][None, 1:]).sum(1)
    return request, token - s["q_start"][request]


def _places(s):
    """The places of the keys that some token of a request may see: all, or the first ones and those from the window of the first new token on."""
    c = s["case"]
    if not c["window"] or c["sinks"] + c["window"] - 1 + s["most_tokens"] >= s["most_keys"]:
        return torch.arange(s["most_keys"], device=DEV).expand(c["batch"], -1)
    col = torch.arange(c["sinks"] + c["window"] - 1 + s["most_tokens"], device=DEV)[None]
    start = (s["lengths"].long() - c["window"] + 1).clamp(min=c["sinks"])[:, None]
    return torch.where(col < c["sinks"], col, start + col - c["sinks"])


def _logits(s, place):
    """Logits [batch, key heads, group, tokens, keys], -inf where a token does not see the key; the keys and values fp32; which keys there are."""
    c = s["case"]
    n, group = s["q"].shape[0], c["heads"] // c["kv_heads"]
    count = s["q_start"][1:] - s["q_start"][:-1]
    there = place < (s["lengths"] + count)[:, None]
    page = s["table"].gather(1, (place // c["page"]).clamp(max=s["table"].shape[1] - 1)).clamp(min=0).long()
    kv = s["pages"][page, :, :, place % c["page"]]                                       # batch, keys, 2, heads, dh
    kv = torch.where(there[:, :, None, None, None], kv, 0).float()
    col = torch.arange(s["most_tokens"], device=DEV)
    token = (s["q_start"][:-1, None] + col).clamp(max=n - 1)                             # batch, tokens
    q = s["q"][token].float().reshape(c["batch"], -1, c["kv_heads"], group, c["dh"])
    x = torch.einsum("btkgd,blkd->bkgtl", q, kv[:, :, 0]) * s["scale"]
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    own_key = place - s["lengths"][:, None]                                              # < 0: cached before
    old = (own_key < 0)[:, None]
    if s["spans"] is None:
        sees = own_key[:, None] <= col[None, :, None]
        stands = s["lengths"][:, None] + col[None]
        key_place = place
        live = (col[None] < count[:, None])
    else:
        at = (s["q_start"][:-1, None] + own_key).clamp(min=0, max=n - 1)
        span, pre = s["spans"][at], s["spans"][token, 0]
        sees = old | ((span[:, None, :, 0] <= pre[:, :, None]) & (pre[:, :, None] < span[:, None, :, 1]))
        live = (pre >= 0) & (col[None] < count[:, None])
        stands = s["lengths"][:, None].expand(-1, s["most_tokens"]) if s["positions"] is None else s["positions"][token]
        new_place = s["lengths"][:, None].expand_as(place) if s["positions"] is None else s["positions"][at]
        key_place = torch.where(own_key < 0, place, new_place)
    if c["window"]:
        sees = sees & ((key_place[:, None] > stands[:, :, None] - c["window"]) | (key_place[:, None] < c["sinks"]))
    sees = (sees & there[:, None] & live[:, :, None])[:, None, None]
    return torch.where(sees, x, -math.inf), kv, there


def _plain_window(s):
    c = s["case"]
    n = s["q"].shape[0]
    x, kv, _ = _logits(s, _places(s))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bkgtl,blkd->btkgd", p, kv[:, :, 1]) / total[..., 0].clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    lse = (total.log() + top)[..., 0].permute(0, 3, 1, 2)
    request, at = _owners(s)
    return o[request, at].reshape(n, c["heads"], c["dh"]).to(torch.bfloat16), lse[request, at].reshape(n, c["heads"])


def _plain_weights(s):
    c = s["case"]
    place = _places(dict(s, case=dict(c, window=0)))                                     # older weights fade whether their key is seen or not
    x, _, there = _logits(s, place)
    token = (s["q_start"][:-1, None] + torch.arange(s["most_tokens"], device=DEV)).clamp(max=s["q"].shape[0] - 1)
    lse = s["lse"][token].reshape(c["batch"], -1, c["kv_heads"], c["heads"] // c["kv_heads"]).permute(0, 2, 3, 1)[..., None]
    got = torch.where(x == -math.inf, 0.0, torch.exp(x - lse)).sum((2, 3))               # batch, key heads, keys
    request, at = there.nonzero(as_tuple=True)
    page, slot = s["table"][request, at // c["page"]].long(), at % c["page"]
    before = torch.where((at < s["lengths"][request])[:, None], s["weights"][page, :, slot] * c["decay"], 0.0)
    s["weights"][page, :, slot] = before + got[request, :, at]
    return s["weights"]


def _plain_evict(s):
    c = s["case"]
    batch, heads = c["batch"], c["kv_heads"]
    length = s["lengths"][:, None]
    place = torch.arange(s["most_keys"], device=DEV).expand(batch, -1)
    there = place < length
    page = s["table"].gather(1, place // c["page"]).clamp(min=0).long()
    w = s["weights"][page, :, place % c["page"]].transpose(1, 2)                         # batch, heads, keys
    always = (place < c["sinks"]) | (place >= length - c["recent"])
    w = torch.where(there[:, None], torch.where(always[:, None], math.inf, w), -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :c["budget"]]    # ties: the lower place first
    lengths = s["lengths"].clamp(max=c["budget"])
    col = torch.arange(order.shape[2], device=DEV)
    kept = torch.where(col < lengths[:, None, None], torch.where(length[..., None] > c["budget"], order, col), s["most_keys"]).sort(-1)[0]
    b, h, to = (kept < s["most_keys"]).nonzero(as_tuple=True)
    at = kept[b, h, to]
    old, new = s["table"][b, at // c["page"]].long(), s["table"][b, to // c["page"]].long()
    rows, weights = s["pages"][old, :, h, at % c["page"]], s["weights"][old, h, at % c["page"]]
    s["pages"][new, :, h, to % c["page"]] = rows
    s["weights"][new, h, to % c["page"]] = weights
    out = torch.full((batch, heads, c["budget"]), -1, dtype=torch.int32, device=DEV)
    out[b, h, to] = at.to(torch.int32)
    return s["pages"], s["weights"], lengths, out


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    tokens, cached = _lengths(c)
    page, table = c["page"], s["table"].tolist()
    if c["kind"] == "evict":
        pages, weights = s["pages"].clone(), s["weights"].clone()
        for b, k in enumerate(cached):
            number = torch.tensor(table[b], device=DEV)
            for h in range(c["kv_heads"]):
                at = torch.arange(k, device=DEV)
                w = s["weights"][number[at // page], h, at % page].double()
                if k > c["budget"]:
                    middle = torch.arange(c["sinks"], max(c["sinks"], k - c["recent"]), device=DEV)
                    best = middle[torch.argsort(-w[middle], stable=True)[:c["budget"] - c["sinks"] - min(c["recent"], k)]]
                    stays = torch.zeros(k, dtype=torch.bool, device=DEV)
                    stays[:c["sinks"]] = True
                    stays[max(0, k - c["recent"]):] = True
                    stays[best] = True
                    at = torch.nonzero(stays)[:, 0]
                to = torch.arange(at.numel(), device=DEV)
                pages[number[to // page], :, h, to % page] = s["pages"][number[at // page], :, h, at % page]
                weights[number[to // page], h, to % page] = s["weights"][number[at // page], h, at % page]
        return pages.double(), weights.double(), None, None
    group, dh = c["heads"] // c["kv_heads"], c["dh"]
    out, sums, weights, n = [], [], s["weights"].double() if c["kind"] == "weights" else None, 0
    for b, (t, k) in enumerate(zip(tokens, cached)):
        number = torch.tensor(table[b][:-(-(t + k) // page)], device=DEV)
        used = s["pages"][number]
        keys, values = (used[:, i].transpose(0, 1).flatten(1, 2)[:, :t + k].double() for i in (0, 1))   # heads, keys, dh
        q = s["q"][n:n + t].double()
        row, key = torch.arange(t, device=DEV)[:, None], torch.arange(t + k, device=DEV)[None]
        if s["spans"] is None:
            hidden, stands, padding = key - k > row, k + row, torch.zeros(t, dtype=torch.bool, device=DEV)
            places = key
        else:
            pre, end = s["spans"][n:n + t].long().unbind(1)
            hidden = torch.zeros((t, t + k), dtype=torch.bool, device=DEV)
            hidden[:, k:] = (pre[None] > pre[:, None]) | (pre[:, None] >= end[None])
            padding = pre < 0
            new = s["positions"][n:n + t].long() if s["positions"] is not None else torch.full((t,), k, device=DEV)
            stands, places = new[:, None], torch.cat([key[0, :k], new])[None]
        if c["window"]:
            hidden = hidden | ((places <= stands - c["window"]) & (places >= c["sinks"]))
        hidden = hidden | padding[:, None]
        heads, logs = [], []
        for h in range(c["heads"]):
            x = q[:, h] @ keys[h // group].T * s["scale"]
            x = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
            x = x.masked_fill(hidden, -math.inf)
            if c["kind"] == "window":
                log = torch.logsumexp(x, 1)
                logs.append(log)
                heads.append((x - log.masked_fill(padding, 0)[:, None]).exp() @ values[h // group])
            else:
                p = (x - s["lse"][n:n + t, h].double().masked_fill(padding, 0)[:, None]).exp().sum(0)
                heads.append(p)
        if c["kind"] == "window":
            out.append(torch.stack(heads, 1))
            sums.append(torch.stack(logs, 1))
        else:
            got = torch.stack(heads).unflatten(0, (c["kv_heads"], group)).sum(1)         # key heads, keys
            old = weights[number].transpose(0, 1).flatten(1)[:, :t + k] * c["decay"]
            old[:, k:] = 0
            full = torch.zeros((c["kv_heads"], number.numel() * page), dtype=torch.float64, device=DEV)
            full[:, :t + k] = got + old
            rest = weights[number].transpose(0, 1).flatten(1)
            full[:, t + k:] = rest[:, t + k:]
            weights[number] = full.unflatten(1, (-1, page)).transpose(0, 1)
        n += t
    return weights if c["kind"] == "weights" else (torch.cat(out), torch.cat(sums))
