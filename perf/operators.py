"""Serving over a cached history, as cases that can be timed and compared: rows of projected queries, keys and values are
normed, rotated and appended to a paged cache; a tree of new tokens attends to that cache and to its own branch; the logits
that come out are turned into log probabilities of given ids, the entropy and the best alternatives.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, from the seed alone (ragged lengths and tree shapes come with the case)
    run(state)          one pass: the plain form, or with `own` the package's operators
    work(case)          bytes and floating-point operations the pass cannot do without
    exact(case, seed)   the same results from the definition in 64 bits

What a token sees.  Request b has lengths[b] keys in the cache that each of its new tokens sees; the new tokens sit behind
them, and token i sees token j of its request where pre[j] <= pre[i] < end[j] (spans[j] = (pre[j], end[j])).  With pre the
place in a depth-first walk and end the place behind a token's last descendant, that is "j is i or an ancestor of i"; (0, 1)
for all is a history that sees itself whole, (i, i + 1) candidates that see only themselves, (i, n) a causal chain, and pre =
-1 a padding token, which sees nothing, is seen by none and comes out as zeros."""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
ROPE_BASE = 10000.0


# ---- the cases --------------------------------------------------------------------------------------------------------

def _append(name, batch, tokens, heads, kv_heads, dh, page, *, norm, shared=False, ragged=False, cached=1000):
    return dict(name=name, kind="append", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dh=dh, page=page, norm=norm,
                shared=shared, ragged=ragged, cached=cached)


def _tree(name, batch, tokens, cached, heads, kv_heads, dh, page, shape, *, cap=0.0, ragged=True, padding=0):
    return dict(name=name, kind="tree", batch=batch, tokens=tokens, cached=cached, heads=heads, kv_heads=kv_heads, dh=dh, page=page,
                shape=shape, cap=cap, ragged=ragged, padding=padding)


def _logprobs(name, rows, vocab, top, dtype, *, given=1, cap=0.0, temperature=1.0, banned=0.0):
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, top=top, dtype=dtype, given=given, cap=cap, temperature=temperature,
                banned=banned)


def listed():
    return [
        # one user's newest action joins the cached history of the ranking model: launch latency is all there is
        _append("append_one", 1, 1, 8, 8, 64, 16, norm=False, cached=126),
        # a batch's candidates behind their histories, all of a request at the one position the model gives them
        _append("append_candidates", 32, 512, 8, 8, 64, 128, norm=False, shared=True, cached=128),
        # long histories enter an empty cache, grouped heads of 128 with their norms: the largest append, bound by memory
        _append("append_history", 16, 2500, 32, 8, 128, 64, norm=True, ragged=True, cached=0),
        # one new token over a short history: the smallest attention call
        _tree("tree_one_token", 1, 1, 127, 8, 8, 64, 16, "chain"),
        # a loaded server, one new token for every user over uneven histories: bound by reading the cache once
        _tree("tree_single_tokens", 96, 1, 4096, 16, 4, 128, 64, "chain"),
        # drafted trees of up to 32 tokens, capped logits, small pages, some padding
        _tree("tree_drafts", 24, 32, 8192, 32, 8, 128, 16, "tree", cap=30.0, padding=2),
        # candidates of a ranking batch over cached histories of a thousand posts, each one seeing itself only
        _tree("tree_candidates", 32, 512, 1022, 8, 8, 64, 128, "isolated"),
        # a history attends to itself while it enters the cache (nothing cached yet)
        _tree("tree_history", 8, 1022, 0, 16, 4, 128, 64, "whole", ragged=False),
        # two users with very long histories and a few drafted tokens: the work has to be split along the cache
        _tree("tree_long_cache", 2, 7, 100003, 16, 4, 128, 32, "tree"),
        # one row over a large table of ids: latency, one row spread over the device
        _logprobs("logprobs_one", 1, 131072, 20, "float32"),
        # a beam's rows over a codebook of odd size, some ids banned, logits capped
        _logprobs("logprobs_beam", 256, 8193, 16, "bfloat16", given=4, cap=30.0, banned=0.3),
        # scoring a batch of sequences over a large table, odd row length: bound by reading the logits once
        _logprobs("logprobs_batch", 2048, 100003, 8, "bfloat16", temperature=0.8),
    ]


HEADS = [(4, 4, 32), (8, 8, 64), (16, 2, 64), (16, 4, 128), (32, 8, 128), (24, 8, 128), (16, 1, 128), (10, 2, 64)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    what = rng.random()
    heads, kv_heads, dh = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    if what < 0.25:
        batch = _log(rng, 1, 128)
        most = 40000 * 6144 // ((heads + 2 * kv_heads) * dh)
        tokens = _log(rng, 1, max(1, min(4096, most // batch)))
        c = _append("", batch, tokens, heads, kv_heads, dh, page, norm=rng.random() < 0.6, shared=rng.random() < 0.3, ragged=rng.random() < 0.5,
                    cached=rng.randrange(0, 2000))
    elif what < 0.7:
        batch = _log(rng, 1, 96)
        shape = rng.choice(["chain", "tree", "tree", "isolated", "whole", "documents"])
        tokens = _log(rng, 1, 64 if shape == "tree" else 1024)
        # at most about the cache bytes, the pairs and the products of the largest listed cases
        keys = min(100000, 400_000_000 // (batch * kv_heads * dh * 4), 190_000_000 // (batch * heads * tokens), 48_000_000_000 // (4 * dh * heads * tokens * batch))
        while keys < 2 * tokens and batch > 1:
            batch = (batch + 1) // 2
            keys = min(100000, 400_000_000 // (batch * kv_heads * dh * 4), 190_000_000 // (batch * heads * tokens), 48_000_000_000 // (4 * dh * heads * tokens * batch))
        cached = _log(rng, 1, max(1, keys - tokens)) - (rng.random() < 0.1)
        c = _tree("", batch, tokens, cached, heads, kv_heads, dh, page, shape, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), ragged=rng.random() < 0.7,
                  padding=rng.choice([0, 0, 1, 3]))
    else:
        dtype = rng.choice(["float32", "bfloat16"])
        vocab = _log(rng, 19, 262144)
        rows = _log(rng, 1, max(1, min(8192, 400_000_000 // (vocab * (4 if dtype == "float32" else 2)))))
        c = _logprobs("", rows, vocab, min(rng.choice([0, 1, 5, 8, 20, 32, 50]), vocab), dtype, given=rng.choice([0, 1, 1, 3]), cap=rng.choice([0.0, 0.0, 30.0]),
                      temperature=rng.choice([1.0, 0.7, 1.3]), banned=rng.choice([0.0, 0.0, 0.5]))
    del c["name"]
    return c


# ---- what comes with a case: ragged lengths and tree shapes -------------------------------------------------------------

def _lengths(c):
    """Tokens and cached keys of every request."""
    rng = random.Random("%d %d %d %d" % (c["batch"], c["tokens"], c["cached"], c["dh"]))
    if not c["ragged"]:
        return [c["tokens"]] * c["batch"], [c["cached"]] * c["batch"]
    tokens = [rng.randint(max(1, c["tokens"] // 2), c["tokens"]) for _ in range(c["batch"])]
    cached = [rng.randint(0, c["cached"]) for _ in range(c["batch"])]
    at = rng.randrange(c["batch"])   # one request has the full size
    tokens[at], cached[at] = c["tokens"], c["cached"]
    return tokens, cached


def _spans(shape, n, padding, rng):
    """(pre, end) of n tokens, and how many pairs of them see each other; the last `padding` tokens are padding."""
    live = max(1, n - padding)
    if shape == "chain":
        pre, end = list(range(live)), [live] * live
    elif shape == "isolated":
        pre, end = list(range(live)), list(range(1, live + 1))
    elif shape == "whole":
        pre, end = [0] * live, [1] * live
    elif shape == "documents":   # causal runs that do not see each other
        pre, end, at = list(range(live)), [0] * live, 0
        while at < live:
            to = min(live, at + rng.randint(1, max(1, live // 3)))
            end[at:to] = [to] * (to - at)
            at = to
    else:                        # a tree in the order it grew (parents first, levels mixed)
        parent = [-1] + [rng.randint(-1 if rng.random() < 0.1 else 0, i - 1) for i in range(1, live)]
        below = [1] * live
        for i in range(live - 1, 0, -1):
            if parent[i] >= 0:
                below[parent[i]] += below[i]
        pre, nxt, top = [0] * live, [0] * live, 0
        for i in range(live):    # a parent is placed before its children
            if parent[i] < 0:
                pre[i], top = top, top + below[i]
            else:
                pre[i] = nxt[parent[i]]
                nxt[parent[i]] += below[i]
            nxt[i] = pre[i] + 1
        end = [p + b for p, b in zip(pre, below)]
    starts = [0] * (live + 1)    # pairs: for each key, the tokens whose place is in [pre, end)
    for p in pre:
        starts[p + 1] += 1
    for i in range(live):
        starts[i + 1] += starts[i]
    pairs = sum(starts[min(e, live)] - starts[p] for p, e in zip(pre, end))
    return [(p, e) for p, e in zip(pre, end)] + [(-1, -1)] * (n - live), pairs


def _trees(c, tokens):
    rng = random.Random("%s %d %d" % (c["shape"], c["batch"], c["tokens"]))
    made = [_spans(c["shape"], n, c["padding"], rng) for n in tokens]
    return [s for spans, _ in made for s in spans], [p for _, p in made]


def work(case):
    c = case
    if c["kind"] == "logprobs":
        size = 4 if c["dtype"] == "float32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * size + c["given"] * 12 + 4 + c["top"] * 12), "flops": 5 * c["rows"] * c["vocab"]}
    tokens, cached = _lengths(c)
    n, row = sum(tokens), c["dh"] * 2
    if c["kind"] == "append":
        width = c["heads"] + 2 * c["kv_heads"]
        return {"bytes": n * (2 * width * row + 4) + min(n, c["cached"] + c["tokens"]) * c["dh"] * 4, "flops": n * (c["heads"] + c["kv_heads"]) * c["dh"] * (6 if c["norm"] else 3)}
    _, pairs = _trees(c, tokens)
    seen = sum(max(1, t - c["padding"]) * k + p for t, k, p in zip(tokens, cached, pairs))
    return {"bytes": (sum(tokens) + sum(cached)) * c["kv_heads"] * row * 2 + 2 * n * c["heads"] * row + n * 8, "flops": 4 * c["dh"] * c["heads"] * seen}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _cache(c, tokens, cached, gen):
    """A pool of pages that hold noise, a shuffled page table (-1 behind a request's last page) and the ragged offsets."""
    need = [-(-(t + k) // c["page"]) for t, k in zip(tokens, cached)]
    total = sum(need) + 3
    pages = torch.randn((total, 2, c["kv_heads"], c["page"], c["dh"]), dtype=torch.bfloat16, device=DEV, generator=gen)
    order = torch.randperm(total, device=DEV, generator=gen)
    widest, at = max(need) + 1, torch.tensor([0] + need).cumsum(0)
    col = torch.arange(widest, device=DEV)
    need_t, at_t = torch.tensor(need, device=DEV), at[:-1].to(DEV)
    table = torch.where(col[None] < need_t[:, None], order[(at_t[:, None] + col[None]).clamp(max=total - 1)], -1).to(torch.int32)
    q_start = torch.tensor([0] + tokens, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
    return pages, table, q_start, torch.tensor(cached, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if c["kind"] == "logprobs":
        dtype = getattr(torch, c["dtype"])
        logits = torch.randn((c["rows"], c["vocab"]), device=DEV, generator=gen, dtype=dtype).mul_(4.0)
        if c["banned"]:
            logits.masked_fill_(torch.rand((c["rows"], c["vocab"]), device=DEV, generator=gen, dtype=torch.bfloat16) < c["banned"], -math.inf)
        given = torch.randint(0, c["vocab"], (c["rows"], c["given"]), device=DEV, generator=gen)
        return dict(case=c, logits=logits, given=given)
    tokens, cached = _lengths(c)
    n = sum(tokens)
    pages, table, q_start, lengths = _cache(c, tokens, cached, gen)
    s = dict(case=c, pages=pages, table=table, q_start=q_start, lengths=lengths, most_tokens=max(tokens), most_keys=max(t + k for t, k in zip(tokens, cached)))
    if c["kind"] == "append":
        qkv = torch.randn((n, (c["heads"] + 2 * c["kv_heads"]) * c["dh"]), dtype=torch.bfloat16, device=DEV, generator=gen)
        at = torch.cat([torch.full((t,), k) if c["shared"] else torch.arange(k, k + t) for t, k in zip(tokens, cached)])
        gain = lambda: (1 + 0.2 * torch.randn((c["dh"],), device=DEV, generator=gen)) if c["norm"] else None  # noqa: E731
        half = torch.arange(c["dh"] // 2, dtype=torch.float64, device=DEV)
        angle = torch.arange(c["cached"] + c["tokens"], dtype=torch.float64, device=DEV)[:, None] * ROPE_BASE ** (-2 * half / c["dh"])
        s.update(qkv=qkv, positions=at.to(torch.int32).to(DEV), q_gain=gain(), k_gain=gain(), cos=angle.cos().float(), sin=angle.sin().float())
    else:
        q = torch.randn((n, c["heads"], c["dh"]), dtype=torch.bfloat16, device=DEV, generator=gen)
        s.update(q=q, spans=torch.tensor(_trees(c, tokens)[0], dtype=torch.int32).to(DEV), scale=math.sqrt(128.0) / c["dh"])
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    s = state
    c = s["case"]
    if own:
        from x_algorithm_b200 import decoding
        if c["kind"] == "append":
            q = decoding.history_append(s["qkv"], s["pages"], s["q_start"], s["lengths"], s["table"], s["positions"], s["cos"], s["sin"],
                                        num_q_heads=c["heads"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS)
            return q, s["pages"]
        if c["kind"] == "tree":
            return decoding.tree_attention(s["q"], s["pages"], s["q_start"], s["lengths"], s["table"], s["spans"], sm_scale=s["scale"], cap=c["cap"],
                                           cap_method="tanh" if c["cap"] else None, max_tokens=s["most_tokens"], max_keys=s["most_keys"])
        return tuple(decoding.token_logprobs(s["logits"], s["given"], top_k=c["top"], cap=c["cap"], temperature=c["temperature"]))
    return {"append": _plain_append, "tree": _plain_tree, "logprobs": _plain_logprobs}[c["kind"]](s)


def _owners(s):
    """The request of each new token and its place among that request's new tokens."""
    n = s["q"].shape[0] if "q" in s else s["qkv"].shape[0]
    token = torch.arange(n, device=DEV)
    request = (token[:, None] >= s["q_start"][None, 1:]).sum(1)
    return request, token - s["q_start"][request]


def _plain_append(s):
    c = s["case"]
    group, dh = c["heads"] // c["kv_heads"], c["dh"]
    x = s["qkv"].float().reshape(-1, c["kv_heads"], group + 2, dh)
    qk, v = x[:, :, :group + 1], x[:, :, group + 1]
    if s["q_gain"] is not None:
        gain = torch.cat([s["q_gain"].expand(group, dh), s["k_gain"][None]])
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS) * gain
    cos, sin = (t[s["positions"]][:, None, None] for t in (s["cos"], s["sin"]))
    a, b = qk[..., :dh // 2], qk[..., dh // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)
    request, place = _owners(s)
    at = s["lengths"][request] + place
    page, slot = s["table"][request, at // c["page"]].long(), at % c["page"]
    s["pages"][page, 0, :, slot] = qk[:, :, group]
    s["pages"][page, 1, :, slot] = v.to(torch.bfloat16)
    return qk[:, :, :group].reshape(-1, c["heads"], dh), s["pages"]


def _plain_tree(s):
    c = s["case"]
    n, batch, group = s["q"].shape[0], c["batch"], c["heads"] // c["kv_heads"]
    place = torch.arange(s["most_keys"], device=DEV)
    count = s["q_start"][1:] - s["q_start"][:-1]
    page = s["table"][:, place // c["page"]].clamp(min=0).long()
    kv = s["pages"][page, :, :, place % c["page"]]                                       # batch, keys, 2, heads, dh
    there = place[None] < (s["lengths"] + count)[:, None]
    kv = torch.where(there[:, :, None, None, None], kv, 0).float()
    token = s["q_start"][:-1, None] + torch.arange(s["most_tokens"], device=DEV)         # batch, tokens
    q = s["q"][token.clamp(max=n - 1)].float().reshape(batch, -1, c["kv_heads"], group, c["dh"])
    x = torch.einsum("btkgd,blkd->bkgtl", q, kv[:, :, 0]) * s["scale"]
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    own_key = place[None] - s["lengths"][:, None]                                        # < 0: cached before
    span = s["spans"][(s["q_start"][:-1, None] + own_key).clamp(min=0, max=n - 1)]
    pre = s["spans"][token.clamp(max=n - 1), 0]
    sees = (own_key < 0)[:, None] | ((span[:, None, :, 0] <= pre[:, :, None]) & (pre[:, :, None] < span[:, None, :, 1]))
    sees = (sees & there[:, None] & (pre >= 0)[:, :, None])[:, None, None]
    x = torch.where(sees, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    o = torch.einsum("bkgtl,blkd->btkgd", p, kv[:, :, 1]) / p.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    request, at = _owners(s)
    return o[request, at].reshape(n, c["heads"], c["dh"]).to(torch.bfloat16)


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]         # ties: the lowest id first
    y = torch.where(x == -math.inf, x, c["cap"] * torch.tanh(x / c["cap"])) if c["cap"] else x
    y = y / c["temperature"]
    top = y.amax(-1, keepdim=True)
    y = y - torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(y)
    total = e.sum(-1, keepdim=True)
    entropy = total.log() - torch.where(e > 0, e * y, 0.0).sum(-1, keepdim=True) / total
    entropy = torch.where(total > 0, entropy, 0.0)[:, 0]
    logp = torch.where(y == -math.inf, y, y - total.log())
    return logp.gather(1, s["given"]), entropy, logp.gather(1, order), order


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "logprobs":
        given, entropy, best = [], [], []
        for at in range(0, c["rows"], 256):
            x = s["logits"][at:at + 256].double()
            banned = torch.isneginf(x)
            keys = torch.sort(x, dim=1, descending=True)[0][:, :c["top"]]
            if c["cap"]:
                x, keys = (torch.tanh(t / c["cap"]) * c["cap"] for t in (x, keys))
                x = x.masked_fill(banned, -math.inf)
                keys = keys.masked_fill(torch.arange(c["top"], device=DEV)[None] >= (~banned).sum(1)[:, None], -math.inf)
            logz = torch.logsumexp(x / c["temperature"], 1, keepdim=True)
            lp = x / c["temperature"] - logz
            entropy.append(-(lp.exp() * lp.masked_fill(banned, 0)).sum(1))
            given.append(torch.take_along_dim(lp, s["given"][at:at + 256], 1))
            best.append(keys / c["temperature"] - logz)
        return torch.cat(given), torch.cat(entropy), torch.cat(best), None
    tokens, cached = _lengths(c)
    page, dh, group = c["page"], c["dh"], c["heads"] // c["kv_heads"]
    table = s["table"].tolist()
    if c["kind"] == "append":
        pages = s["pages"].double()
        q_all, n = [], 0
        for b, (t, k) in enumerate(zip(tokens, cached)):
            x = s["qkv"][n:n + t].double().unflatten(1, (c["kv_heads"], group + 2, dh))
            q, key, value = x[:, :, :group].flatten(1, 2), x[:, :, group], x[:, :, group + 1]
            if c["norm"]:
                q = q * (q.square().mean(2, True) + EPS).rsqrt() * s["q_gain"].double()
                key = key * (key.square().mean(2, True) + EPS).rsqrt() * s["k_gain"].double()
            at = s["positions"][n:n + t].double()
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), at[:, None] * torch.pow(torch.tensor(ROPE_BASE, dtype=torch.float64, device=DEV), -torch.arange(0, dh, 2, dtype=torch.float64, device=DEV) / dh))
            rotated = []
            for h in (q, key):
                z = torch.complex(h[..., :dh // 2], h[..., dh // 2:]) * turn[:, None]
                rotated.append(torch.cat([z.real, z.imag], -1))
            q_all.append(rotated[0])
            at = torch.arange(k, k + t, device=DEV)
            number = torch.tensor(table[b], device=DEV)[at // page]
            pages[number, 0, :, at % page] = rotated[1]
            pages[number, 1, :, at % page] = value
            n += t
        return torch.cat(q_all), pages
    out, n = [], 0
    for b, (t, k) in enumerate(zip(tokens, cached)):
        used = s["pages"][torch.tensor(table[b][:-(-(t + k) // page)], device=DEV)]
        keys, values = (used[:, i].transpose(0, 1).flatten(1, 2)[:, :t + k].double() for i in (0, 1))   # heads, keys, dh
        q = s["q"][n:n + t].double()
        pre, end = s["spans"][n:n + t].long().unbind(1)
        hidden = torch.zeros((t, t + k), dtype=torch.bool, device=DEV)
        hidden[:, k:] = (pre[None] > pre[:, None]) | (pre[:, None] >= end[None])
        heads = []
        for h in range(c["heads"]):
            x = q[:, h] @ keys[h // group].T * s["scale"]
            x = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
            heads.append(torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ values[h // group])
        o = torch.stack(heads, 1)
        o[pre < 0] = 0
        out.append(o)
        n += t
    return torch.cat(out)
