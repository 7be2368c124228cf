"""Window attention, key weights and eviction on a paged cache against plain forms in 64 bits.

Tolerances.  A logit is off by at most (head dim + 2) roundings of 2^-24 of sum |q k| scale, capped ones by 4e-7 of the cap more (the two forms of tanh).  An exponential is off by that
and 2^-21 (ex2.approx: 2 units in the last place, and its argument's rounding, up to 2^-24 of 32); a sum of n by n 2^-24 more.  Outputs: probabilities are rounded to bf16, 2^-8 of each,
and the result once more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def make_case(batch, tokens, cached, heads, kv_heads, dh, page, shape, seed=0, ragged=True, padding=0, extra_cols=2, stride=0, positions=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = torch.Generator().manual_seed(seed + 1)
    ints = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=r).tolist()  # noqa: E731
    n_new = ints(0, tokens, batch) if ragged else [tokens] * batch
    n_old = ints(0, cached, batch) if ragged else [cached] * batch
    n_new[-1], n_old[-1] = tokens, cached
    n = sum(n_new)
    need = [-(-(a + b) // page) for a, b in zip(n_new, n_old)]
    total = sum(need) + 3
    pages = torch.randn((total, 2, kv_heads, page, dh), device=DEV, generator=g).to(torch.bfloat16)
    order = torch.randperm(total, generator=r).tolist()
    cols = max(need) + extra_cols
    table = torch.full((batch, cols), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
        at += k
    wide = torch.randn((n, heads * dh + stride), device=DEV, generator=g).to(torch.bfloat16)
    q = wide[:, :heads * dh].unflatten(1, (heads, dh))
    spans = pos = None
    if shape != "chain":
        rows, depth = [], []
        for t in n_new:
            live = max(0, t - padding)
            if shape == "isolated":
                s, d = [(i, i + 1) for i in range(live)], [0] * live
            elif shape == "whole":
                s, d = [(0, 1)] * live, [0] * live
            else:
                from x_algorithm_b200.decoding import tree_spans
                parents = [-1 if i == 0 or torch.rand(1, generator=r).item() < 0.2 else ints(0, i - 1, 1)[0] for i in range(live)]
                d = []
                for i, p in enumerate(parents):
                    d.append(0 if p < 0 else d[p] + 1)
                s = tree_spans(parents).tolist()
            rows += [tuple(x) for x in s] + [(-1, -1)] * (t - live)
            depth.append(d + [0] * (t - live))
        spans = torch.tensor(rows, dtype=torch.int32).reshape(-1, 2).to(DEV)
        if positions == "depth":
            pos = torch.tensor([k + x for k, d in zip(n_old, depth) for x in d], dtype=torch.int32).to(DEV)
    if positions == "spread":                                   # any places, some in front of the cache's end
        pos = torch.cat([torch.randint(-5, k + 50, (t,), generator=r) for t, k in zip(n_new, n_old)]).to(torch.int32).to(DEV)
    return dict(q=q, pages=pages, table=table.to(DEV), q_start=torch.tensor([0] + n_new).cumsum(0).to(torch.int32).to(DEV),
                lengths=torch.tensor(n_old, dtype=torch.int32, device=DEV), spans=spans, positions=pos, n_new=n_new, n_old=n_old, page=page,
                group=heads // kv_heads, scale=math.sqrt(128.0) / dh,
                weights=torch.rand((total, kv_heads, page), device=DEV, generator=g))


def visible(c, b, window, sinks):
    """bool [tokens, keys] of request b, from the definition."""
    t, k = c["n_new"][b], c["n_old"][b]
    row0 = int(sum(c["n_new"][:b]))
    key = torch.arange(t + k, device=DEV)
    i = torch.arange(t, device=DEV)
    if c["spans"] is None:
        see = key[None] <= (k + i)[:, None]
    else:
        pre, end = c["spans"][row0:row0 + t].long().unbind(1)
        see = torch.ones((t, t + k), dtype=torch.bool, device=DEV)
        see[:, k:] = (pre[None] <= pre[:, None]) & (pre[:, None] < end[None])
        see &= (pre >= 0)[:, None]
    if c["positions"] is not None:
        place = c["positions"][row0:row0 + t].long().clamp(min=k)
    else:
        place = k + i if c["spans"] is None else torch.full((t,), k, device=DEV)
    if window is not None:
        at = torch.cat([key[:k], place])
        see &= (at[None] > place[:, None] - window) | (at[None] < sinks)
    return see


def rows_of(c, b, which):
    t, k, page = c["n_new"][b], c["n_old"][b], c["page"]
    at = torch.arange(t + k, device=DEV)
    return c["pages"][c["table"][b, at // page].long(), which, :, at % page].double()       # keys, kv heads, dh


def plain(c, window, sinks, cap=0.0, method=None, keep=None):
    """out, lse, bounds of their errors; per request the logits' exponentials by key head."""
    outs, lses, tol_o, tol_l = [], [], [], []
    for b in range(len(c["n_new"])):
        t = c["n_new"][b]
        row0 = int(sum(c["n_new"][:b]))
        q = c["q"][row0:row0 + t].double()
        k, v = rows_of(c, b, 0), rows_of(c, b, 1)
        see = visible(c, b, window, sinks)
        if keep is not None:
            see = see & keep[b][None]
        dh = q.shape[-1]
        kk, vv = k.repeat_interleave(c["group"], 1), v.repeat_interleave(c["group"], 1)
        x = torch.einsum("thd,khd->thk", q, kk) * c["scale"]
        size = (torch.einsum("thd,khd->thk", q.abs(), kk.abs()) * abs(c["scale"])).masked_fill(~see[:, None], 0)
        if cap:
            x = cap * torch.tanh(x / cap) if method == "tanh" else x / (1 + x.abs() / cap)
        x = x.masked_fill(~see[:, None], -math.inf)
        lse = torch.logsumexp(x, -1) if x.shape[-1] else torch.full(x.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        p = torch.where(see[:, None], torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
        vm = torch.where(torch.isfinite(vv), vv, 0.0)
        o, oa = torch.einsum("thk,khd->thd", p, vm), torch.einsum("thk,khd->thd", p, vm.abs())
        off = (size.amax(-1) if size.shape[-1] else lse * 0) * (dh + 2) * 2.0 ** -24 + 4e-7 * cap + 2.0 ** -21 + see.shape[1] * 2.0 ** -24
        outs.append(o); lses.append(lse)
        tol_o.append(oa * (2.0 ** -8 + 2 * off[..., None]) + o.abs() * 2.0 ** -8 + 1e-30)
        tol_l.append(off + lse.abs().masked_fill(lse == -math.inf, 0) * 2.0 ** -23)
    return torch.cat(outs), torch.cat(lses), torch.cat(tol_o), torch.cat(tol_l)


def plain_weights(c, lse, window, sinks, cap=0.0, method=None, decay=1.0):
    """weights and the bound of their errors."""
    w, tol = c["weights"].double().clone(), torch.zeros_like(c["weights"], dtype=torch.float64)
    for b in range(len(c["n_new"])):
        t, k, page = c["n_new"][b], c["n_old"][b], c["page"]
        if t + k == 0:
            continue
        row0 = int(sum(c["n_new"][:b]))
        q, kk = c["q"][row0:row0 + t].double(), rows_of(c, b, 0).repeat_interleave(c["group"], 1)
        see = visible(c, b, window, sinks)[:, None]
        x = torch.einsum("thd,khd->thk", q, kk) * c["scale"]
        size = torch.einsum("thd,khd->thk", q.abs(), kk.abs()) * abs(c["scale"])
        if cap:
            x = cap * torch.tanh(x / cap) if method == "tanh" else x / (1 + x.abs() / cap)
        ls = lse[row0:row0 + t].double()[..., None]
        p = torch.where(see & torch.isfinite(ls), torch.exp(x - ls), 0.0)
        off = size * (q.shape[-1] + 2) * 2.0 ** -24 + 4e-7 * cap + 2.0 ** -21 + torch.where(torch.isfinite(ls), ls.abs(), 0.0) * 2.0 ** -22 + t * c["group"] * 2.0 ** -24
        fold = lambda y: y.unflatten(1, (-1, c["group"])).sum((0, 2)).T  # noqa: E731          keys, kv heads
        at = torch.arange(t + k, device=DEV)
        page_of, slot = c["table"][b, at // page].long(), at % page
        old = torch.where((at < k)[:, None], w[page_of, :, slot] * decay, 0.0)
        w[page_of, :, slot] = old + fold(p)
        tol[page_of, :, slot] = fold(torch.where(p > 0, p * off, 0.0)) + (old + fold(p)) * 2.0 ** -22 + 1e-35
    return w, tol


def close(got, want, tol, what):
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()}, allowed {tol[bad][0].item()}"


SHAPES = [
    # batch, tokens, cached, heads, kv heads, head dim, page, shape, positions
    (1, 1, 0, 8, 8, 64, 16, "chain", None),
    (1, 1, 127, 8, 8, 64, 16, "chain", None),
    (5, 1, 700, 16, 4, 128, 64, "chain", None),
    (3, 3, 300, 10, 2, 64, 48, "chain", None),
    (3, 5, 300, 4, 4, 32, 16, "tree", "depth"),
    (2, 40, 90, 4, 4, 32, 32, "chain", None),
    (3, 40, 1000, 16, 2, 64, 64, "chain", None),
    (2, 300, 500, 16, 4, 128, 48, "chain", None),
    (2, 129, 0, 16, 1, 128, 128, "chain", None),
    (3, 32, 900, 32, 8, 128, 16, "tree", "depth"),
    (3, 20, 200, 8, 8, 64, 32, "tree", None),
    (2, 200, 300, 8, 8, 64, 128, "isolated", None),
    (2, 150, 260, 24, 8, 128, 64, "whole", None),
    (2, 60, 260, 16, 4, 128, 64, "chain", "spread"),
    (3, 3, 260, 8, 8, 64, 16, "tree", "spread"),
]
WINDOWS = [(None, 0), (1, 0), (1, 3), (17, 0), (64, 4), (100, 100), (511, 1), (5000, 16)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_window_attention_and_key_weights(shape, window, sinks):
    from x_algorithm_b200 import decoding
    c = make_case(*shape[:-1], seed=3, positions=shape[-1], padding=2 if shape[-2] in ("tree", "isolated") else 0, stride=8)
    most = dict(max_tokens=max(c["n_new"]), max_keys=max(a + b for a, b in zip(c["n_new"], c["n_old"])))
    want, want_lse, tol, tol_lse = plain(c, window, sinks)
    args = (c["q"], c["pages"], c["q_start"], c["lengths"], c["table"])
    out, lse = decoding.window_attention(*args, c["spans"], c["positions"], window=window, sinks=sinks, **most)
    close(lse, want_lse, tol_lse, "lse")
    close(out, want, tol, "out")
    again, lse_again = decoding.window_attention(*args, c["spans"], c["positions"], window=window, sinks=sinks)       # without the hints: other splits
    close(lse_again, want_lse, tol_lse, "lse without hints")
    close(again, want, tol, "out without hints")
    for decay in (1.0, 0.9):
        w = c["weights"].clone()
        got = decoding.key_weights(*args, lse, w, c["spans"], c["positions"], window=window, sinks=sinks, decay=decay, **most)
        assert got is w
        ww, tw = plain_weights(c, lse, window, sinks, decay=decay)
        close(got, ww, tw, "weights, decay %g" % decay)
    decoding.check_status()


@pytest.mark.parametrize("shape", [SHAPES[2], SHAPES[3], SHAPES[6], SHAPES[9], SHAPES[12]], ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("cap,method", [(30.0, "tanh"), (2.0, "tanh"), (5000.0, "tanh"), (4.0, "soft_sign")])
@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 4)])
def test_caps(shape, cap, method, window, sinks):
    from x_algorithm_b200 import decoding
    c = make_case(*shape[:-1], seed=5, positions=shape[-1])
    if cap == 5000.0:
        cap = 1500.0
    want, want_lse, tol, tol_lse = plain(c, window, sinks, cap, method)
    args = (c["q"], c["pages"], c["q_start"], c["lengths"], c["table"])
    more = dict(window=window, sinks=sinks, cap=cap, cap_method=method)
    out, lse = decoding.window_attention(*args, c["spans"], c["positions"], **more)
    close(lse, want_lse, tol_lse, "lse")
    close(out, want, tol, "out")
    got = decoding.key_weights(*args, lse, c["weights"].clone(), c["spans"], c["positions"], **more)
    close(got, *plain_weights(c, lse, window, sinks, cap, method), "weights")


def evict_plain(c, lengths, budget, sinks, recent):
    pages, weights = c["pages"].clone(), c["weights"].clone()
    kept = torch.full((len(lengths), pages.shape[2], budget), -1, dtype=torch.int32, device=DEV)
    page, table = c["page"], c["table"]
    for b, n in enumerate(lengths):
        for h in range(pages.shape[2]):
            at = torch.arange(n, device=DEV)
            num, slot = table[b, at // page].long(), at % page
            if n > budget:
                w = c["weights"][num, h, slot].double()
                w = torch.where(torch.isnan(w), math.inf, w)
                rank = w.clone()
                rank[:sinks] = math.inf
                if recent:
                    rank[n - recent:] = math.inf
                first = torch.zeros(n, dtype=torch.long, device=DEV)     # NaN above infinity, the protected above all
                first[torch.isnan(c["weights"][num, h, slot])] = 1
                first[:sinks] = 2
                if recent:
                    first[n - recent:] = 2
                order = sorted(range(n), key=lambda i: (-first_l[i], -rank_l[i], i)) if (first_l := first.tolist()) and (rank_l := rank.tolist()) else []
                at = torch.tensor(sorted(order[:budget]), device=DEV)
            to = torch.arange(at.numel(), device=DEV)
            kept[b, h, :at.numel()] = at.to(torch.int32)
            src, dst = table[b, at // page].long(), table[b, to // page].long()
            pages[dst, :, h, to % page] = c["pages"][src, :, h, at % page]
            weights[dst, h, to % page] = c["weights"][src, h, at % page]
    return pages, weights, torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32, device=DEV), kept


EVICT = [
    # batch, cached, kv heads, head dim, page, budget, sinks, recent
    (1, 1, 8, 64, 16, 1, 0, 0),
    (1, 2, 8, 64, 16, 1, 0, 0),
    (1, 2, 2, 64, 16, 1, 1, 0),
    (1, 2, 2, 64, 16, 1, 0, 1),
    (1, 200, 8, 64, 16, 128, 4, 32),
    (4, 333, 2, 32, 48, 100, 0, 0),
    (4, 333, 2, 128, 48, 100, 50, 50),
    (3, 1000, 4, 128, 64, 999, 4, 17),
    (3, 5000, 1, 128, 16, 777, 16, 100),
    (2, 20011, 2, 64, 128, 10000, 0, 1000),
    (1, 70001, 1, 64, 128, 30000, 4, 64),
    (40, 500, 8, 64, 32, 250, 4, 64),
    (3, 30000, 2, 64, 16, 200, 4, 64),
    (2, 900, 2, 32, 128, 256, 0, 0),
    (2, 900, 2, 128, 16, 128, 4, 100),
    (2, 900, 2, 128, 16, 129, 4, 100),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("values", ["spread", "few", "same", "odd"])
def test_evict(case, values):
    from x_algorithm_b200 import decoding
    batch, cached, kv, dh, page, budget, sinks, recent = case
    c = make_case(batch, 0, cached, kv, kv, dh, page, "chain", seed=9)
    g = torch.Generator(device=DEV).manual_seed(4)
    w = torch.randn(c["weights"].shape, device=DEV, generator=g)
    if values == "spread":
        w = (w * 3).exp()
    elif values == "few":                                     # many ties
        w = (w * 2).round() / 4
    elif values == "same":
        w = torch.zeros_like(w)
    else:
        pick = torch.randint(0, 12, w.shape, device=DEV, generator=g)
        for i, x in enumerate([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38]):
            w = torch.where(pick == i, x, w)
    c["weights"] = w
    want = evict_plain(c, c["n_old"], budget, sinks, recent)
    copies = [c[k].clone() for k in ("weights", "pages", "lengths")]
    lengths, kept = decoding.evict(c["weights"], c["pages"], c["lengths"], c["table"], budget=budget, sinks=sinks, recent=recent)
    in_place, again = decoding.evict(*copies, c["table"], budget=budget, sinks=sinks, recent=recent, lengths_out=copies[2], max_keys=1)   # lengths written over, a hint too small
    assert in_place is copies[2] and torch.equal(in_place, lengths) and torch.equal(again, kept)
    assert torch.equal(copies[1].view(torch.int16), c["pages"].view(torch.int16)) and torch.equal(copies[0].view(torch.int32), c["weights"].view(torch.int32))
    decoding.check_status()
    assert torch.equal(lengths, want[2]) and torch.equal(kept, want[3])
    assert torch.equal(c["pages"].view(torch.int16), want[0].view(torch.int16))
    assert torch.equal(c["weights"].view(torch.int32), want[1].view(torch.int32))


MANY_ROWS = [
    (1, 17, 40, 4, 4, 64, 16, "chain", None),
    (2, 700, 900, 24, 8, 128, 48, "chain", None),
    (2, 333, 0, 10, 2, 64, 16, "whole", None),
    (1, 2048, 60, 16, 2, 64, 64, "isolated", None),
    (1, 1500, 100, 16, 4, 128, 128, "whole", None),
    (1, 900, 3000, 32, 1, 64, 32, "chain", None),
    (1, 4, 300, 128, 1, 128, 32, "chain", None),
    (4, 64, 700, 8, 8, 64, 48, "tree", "spread"),
]


@pytest.mark.parametrize("shape", MANY_ROWS, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("window,sinks", [(None, 0), (130, 4), (1, 200)])
def test_key_weights_of_many_rows(shape, window, sinks):
    """The tensor cores' kernel: groups that do not divide a tile, rows in chunks that are joined, hints that say too little."""
    from x_algorithm_b200 import decoding
    from x_algorithm_b200.engine import dispatch_counts
    c = make_case(*shape[:-1], seed=11, positions=shape[-1], padding=3 if shape[-2] != "chain" else 0, stride=24)
    args = (c["q"], c["pages"], c["q_start"], c["lengths"], c["table"])
    lse = plain(c, window, sinks)[1].float()
    lse[::7, 0] = math.inf                                    # rows that the caller leaves out
    lse[3 % len(lse), -1] = -math.inf
    before = dispatch_counts()["key_weights.tcgen05"]
    for decay in (1.0, 0.5):
        want, tol = plain_weights(c, lse, window, sinks, decay=decay)
        first = None
        for hints in ({}, dict(max_tokens=max(c["n_new"]), max_keys=max(a + b for a, b in zip(c["n_new"], c["n_old"]))), dict(max_tokens=17 * 4, max_keys=1)):
            got = decoding.key_weights(*args, lse, c["weights"].clone(), c["spans"], c["positions"], window=window, sinks=sinks, decay=decay, **hints)
            close(got, want, tol, f"weights, decay {decay}, {hints}")
            if hints == {}:
                first = got
        again = decoding.key_weights(*args, lse, c["weights"].clone(), c["spans"], c["positions"], window=window, sinks=sinks, decay=decay)
        assert torch.equal(again, first)                      # the order of every sum follows from the sizes
    assert dispatch_counts()["key_weights.tcgen05"] > before
    decoding.check_status()


def test_key_weights_of_more_requests_than_a_block_plans():
    from x_algorithm_b200 import decoding
    c = make_case(1500, 20, 40, 4, 2, 64, 16, "chain", seed=2)
    args = (c["q"], c["pages"], c["q_start"], c["lengths"], c["table"])
    lse = plain(c, None, 0)[1].float()
    got = decoding.key_weights(*args, lse, c["weights"].clone())
    close(got, *plain_weights(c, lse, None, 0), "weights")
    out, got_lse = decoding.window_attention(*args, window=13, sinks=2)
    want, want_lse, tol, tol_lse = plain(c, 13, 2)
    close(out, want, tol, "out")
    close(got_lse, want_lse, tol_lse, "lse")
