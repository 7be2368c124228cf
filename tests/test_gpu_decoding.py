"""Appending to a paged cache, attention of a tree of new tokens over it, and log probabilities from logits, each against
its definition in 64 bits.

Tolerances, from the arithmetic the header promises (bf16 in and out, fp32 sums), u = 2^-8 the unit roundoff of bf16:
 * appended rows: fp32 throughout, one rounding: u |y|, and a few fp32 roundings of the two products that make y
 * attention: probabilities are rounded to bf16 for the second product, u sum p |v|, then the output, u |o|; fp32 for the rest
 * log probabilities: fp32 of numbers up to 100: 2^-24 * 100 for each of a handful of operations, and the sum's own error
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
DEV = "cuda"


def _torch():
    import torch
    return torch


# ---- a cache with something in it --------------------------------------------------------------------------------------

class Cache:
    """Pages of noise, a shuffled table with -1 behind the last page, ragged requests."""

    def __init__(self, tokens, cached, kv_heads, dh, page, seed=0, spare=2):
        torch = _torch()
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.tokens, self.cached, self.page, self.kv_heads, self.dh = list(tokens), list(cached), page, kv_heads, dh
        need = [-(-(t + k) // page) for t, k in zip(tokens, cached)]
        total = sum(need) + spare
        self.pages = torch.randn((total, 2, kv_heads, page, dh), device=DEV, generator=self.g).to(torch.bfloat16)
        order = torch.randperm(total, device=DEV, generator=self.g).tolist()
        self.table_host, at = [], 0
        for k in need:
            self.table_host.append(order[at:at + k] + [-1] * (max(need) + 1 - k))
            at += k
        self.table = torch.tensor(self.table_host, dtype=torch.int32, device=DEV)
        self.q_start = torch.tensor([0] + list(np.cumsum(tokens)), dtype=torch.int32, device=DEV)
        self.lengths = torch.tensor(cached, dtype=torch.int32, device=DEV)

    @property
    def n(self):
        return sum(self.tokens)

    def args(self):
        return self.pages, self.q_start, self.lengths, self.table

    def keys(self, b, which):
        """float64 [kv heads, cached + new, dh] of request b"""
        torch = _torch()
        count = self.tokens[b] + self.cached[b]
        used = self.pages[torch.tensor(self.table_host[b][:-(-count // self.page)], dtype=torch.long, device=DEV), which]
        return used.transpose(0, 1).flatten(1, 2)[:, :count].double()


def _spans(shape, n, padding=0, seed=0):
    from x_algorithm_b200.decoding import tree_spans
    rng, live = np.random.default_rng(seed), max(n - padding, 0)
    if shape == "chain":
        s = [(i, live) for i in range(live)]
    elif shape == "isolated":
        s = [(i, i + 1) for i in range(live)]
    elif shape == "whole":
        s = [(0, 1)] * live
    else:
        parents = [-1 if i == 0 or rng.random() < 0.2 else int(rng.integers(0, i)) for i in range(live)]
        at = rng.permutation(live)                      # any order of the tokens
        mixed = np.full(live, -1, np.int64)
        for i, p in enumerate(parents):
            mixed[at[i]] = -1 if p < 0 else at[p]
        s = [tuple(x) for x in tree_spans(mixed)]
    return s + [(-1, -1)] * (n - live)


def _attend(c, q, spans, scale, cap=0.0, method=None, hide=None):
    """(o, sum p |v|) in float64; hide: (request, first key, last key) that do not exist"""
    torch = _torch()
    outs, mags, at = [], [], 0
    group = q.shape[1] // c.kv_heads
    for b, (t, k) in enumerate(zip(c.tokens, c.cached)):
        key, val = c.keys(b, 0), c.keys(b, 1)
        pre, end = spans[at:at + t].long().unbind(1)
        sees = torch.ones((t, t + k), dtype=torch.bool, device=DEV)
        sees[:, k:] = (pre[None] <= pre[:, None]) & (pre[:, None] < end[None])
        sees &= (pre >= 0)[:, None]
        if hide and hide[0] == b:
            sees[:, hide[1]:hide[2]] = False
        qh = q[at:at + t].double().transpose(0, 1)                                             # heads, t, dh
        x = qh @ key.repeat_interleave(group, 0).transpose(1, 2) * scale
        if method == "tanh":
            x = cap * torch.tanh(x / cap)
        elif method == "soft_sign":
            x = x / (1 + x.abs() / cap)
        x = x.masked_fill(~sees, -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True).nan_to_num(neginf=0.0)) if x.shape[-1] else x
        p = p.masked_fill(~sees, 0.0)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        val = val.repeat_interleave(group, 0)
        clean = val.nan_to_num(0.0, 0.0, 0.0)
        o = (p @ clean).transpose(0, 1)
        odd = torch.where(torch.isfinite(val), 0.0, val)
        if bool((odd != 0).any()):                                                             # seen infinities and NaN
            for key_at in torch.nonzero((odd != 0).any(-1).any(0))[:, 0].tolist():
                o = o + torch.where(sees[:, key_at, None, None], odd[None, :, key_at], 0.0)
        outs.append(o)
        mags.append((p @ clean.abs()).transpose(0, 1))
        at += t
    return torch.cat(outs), torch.cat(mags)


def _check(got, want, mag):
    torch = _torch()
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    bound = 1.02 * U * (want.abs() + mag) + 2e-5
    off = (got - want).abs()
    assert bool((off <= bound)[fine].all()), f"off by {float((off / bound)[fine].max()):.2f} of the bound"


def _tree_case(tokens, cached, heads, kv_heads, dh, page, shape="tree", padding=0, cap=0.0, method=None, seed=0, scale=None, **kw):
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache(tokens, cached, kv_heads, dh, page, seed)
    q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
    spans = torch.tensor([s for b, t in enumerate(tokens) for s in _spans(shape, t, min(padding, t), seed + b)], dtype=torch.int32, device=DEV).reshape(-1, 2)
    scale = math.sqrt(128.0) / dh if scale is None else scale
    out = decoding.tree_attention(q, *c.args(), spans, sm_scale=scale, cap=cap, cap_method=method, **kw)
    decoding.check_status()
    _check(out, *_attend(c, q, spans, scale, cap, method))
    return c, q, spans, out


HEADS = [(4, 4, 32), (8, 2, 32), (8, 8, 64), (16, 2, 64), (16, 4, 128), (6, 2, 128), (20, 4, 64), (16, 1, 128)]


@pytest.mark.parametrize("heads,kv_heads,dh", HEADS)
@pytest.mark.parametrize("tokens,cached,page,shape", [
    ([1], [0], 16, "chain"), ([1], [1], 16, "chain"), ([1, 1, 1], [15, 16, 17], 16, "chain"), ([5, 0, 9], [33, 7, 0], 16, "tree"),
    ([31, 32, 33], [127, 128, 129], 32, "tree"), ([70], [1], 64, "isolated"), ([3, 130], [500, 257], 128, "tree"), ([65, 1], [0, 0], 48, "whole"),
    ([7], [5001], 64, "tree"), ([200], [77], 16, "chain")])
def test_tree_attention(heads, kv_heads, dh, tokens, cached, page, shape):
    _tree_case(tokens, cached, heads, kv_heads, dh, page, shape, seed=heads + dh + sum(tokens))


@pytest.mark.parametrize("method", ["tanh", "soft_sign"])
@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 4, 32), (8, 8, 64), (16, 4, 128)])
@pytest.mark.parametrize("tokens,cached", [([2, 1], [300, 0]), ([33, 150], [90, 600])])
def test_tree_attention_capped(method, heads, kv_heads, dh, tokens, cached):
    _tree_case(tokens, cached, heads, kv_heads, dh, 32, "tree", cap=5.0, method=method, seed=3)
    _tree_case(tokens, cached, heads, kv_heads, dh, 32, "tree", cap=30.0, method=method, seed=4)


@pytest.mark.parametrize("heads,kv_heads,dh", [(4, 4, 32), (8, 8, 64), (16, 4, 128)])
@pytest.mark.parametrize("tokens,padding", [([4], 2), ([3], 3), ([40, 2, 140], 5)])
def test_padding_tokens_come_out_as_zeros(heads, kv_heads, dh, tokens, padding):
    c, q, spans, out = _tree_case(tokens, [50] * len(tokens), heads, kv_heads, dh, 16, "tree", padding=padding)
    assert bool((out[spans[:, 0] < 0] == 0).all())


@pytest.mark.parametrize("heads,kv_heads,dh,tokens", [(4, 4, 32, 9), (8, 8, 64, 9), (16, 4, 128, 4), (16, 4, 128, 60), (8, 8, 64, 150), (32, 8, 128, 17)])
def test_what_is_not_seen_leaves_no_trace(heads, kv_heads, dh, tokens):
    """NaN and infinities behind the last key, in pages of nobody, in keys and values of padding tokens and of other branches."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([tokens, tokens], [70, 3], kv_heads, dh, 32, seed=5)
    q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
    spans = torch.tensor(_spans("tree", tokens, 2, 1) + _spans("isolated", tokens, 0), dtype=torch.int32, device=DEV)
    clean = decoding.tree_attention(q, *c.args(), spans)
    live = {p for r in c.table_host for p in r if p >= 0}
    for p in range(c.pages.shape[0]):
        if p not in live:
            c.pages[p] = math.nan
    for b, (t, k) in enumerate(zip(c.tokens, c.cached)):       # the slots behind the last key
        last = c.table_host[b][(t + k - 1) // 32]
        c.pages[last, :, :, (t + k - 1) % 32 + 1:] = math.inf
    for j in (tokens - 2, tokens - 1):                         # the padding tokens of request 0
        at = 70 + j
        c.pages[c.table_host[0][at // 32], 0, :, at % 32] = math.nan
        c.pages[c.table_host[0][at // 32], 1, :, at % 32] = -math.inf
    assert torch.equal(decoding.tree_attention(q, *c.args(), spans), clean)
    # candidates that see themselves only: the odd values of one reach its own row and no other
    mid = tokens // 2
    at = 3 + mid
    c.pages[c.table_host[1][at // 32], 1, :, at % 32, 3] = math.nan
    c.pages[c.table_host[1][at // 32], 1, :, at % 32, 4] = math.inf
    out = decoding.tree_attention(q, *c.args(), spans)
    rest = [i for i in range(c.n) if i != tokens + mid]
    assert torch.equal(out[rest], clean[rest])
    own = out[tokens + mid]
    assert bool(torch.isnan(own[:, 3]).all()) and bool((own[:, 4] == math.inf).all())
    assert torch.equal(own[:, 5:], clean[tokens + mid][:, 5:])
    _check(out, *_attend(c, q, spans, math.sqrt(128.0) / dh))


@pytest.mark.parametrize("heads,kv_heads,dh,tokens", [(8, 8, 64, 3), (16, 4, 128, 50)])
def test_odd_values_that_are_seen_come_through(heads, kv_heads, dh, tokens):
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([tokens], [200], kv_heads, dh, 16, seed=8)
    c.pages[c.table_host[0][1], 1, 0, 3, 7] = math.inf          # cached: every token sees it
    q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
    spans = torch.tensor(_spans("tree", tokens, 0, 1), dtype=torch.int32, device=DEV)
    out = decoding.tree_attention(q, *c.args(), spans)
    assert bool((out[:, :heads // kv_heads, 7] == math.inf).all()) and bool(torch.isfinite(out[:, heads // kv_heads:]).all())
    c.pages[c.table_host[0][1], 0, 0, 3, 7] = math.nan          # a key: the rows are NaN, as softmax makes them
    out = decoding.tree_attention(q, *c.args(), spans)
    assert bool(torch.isnan(out[:, :heads // kv_heads]).all()) and bool(torch.isfinite(out[:, heads // kv_heads:]).all())


@pytest.mark.parametrize("heads,kv_heads,dh", [(8, 8, 64), (16, 4, 128)])
def test_extreme_logits(heads, kv_heads, dh):
    """Scores in the thousands: one key takes all; and scores that are all equal."""
    for tokens in ([2], [64]):
        _tree_case(tokens, [333], heads, kv_heads, dh, 16, "chain", scale=40.0, seed=2)
        _tree_case(tokens, [333], heads, kv_heads, dh, 16, "chain", scale=0.0, seed=2)


@pytest.mark.parametrize("heads,kv_heads,dh,tokens", [(4, 4, 32, 3), (8, 8, 64, 3), (16, 4, 128, 3), (16, 4, 128, 50), (8, 8, 64, 140)])
def test_pages_out_of_range_are_left_out_and_reported(heads, kv_heads, dh, tokens):
    from x_algorithm_b200 import PhoenixError, decoding
    torch = _torch()
    c = Cache([tokens, tokens], [300, 40], kv_heads, dh, 16, seed=4)
    q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
    spans = torch.tensor(_spans("tree", tokens, 0, 1) * 2, dtype=torch.int32, device=DEV)
    scale = math.sqrt(128.0) / dh
    for wrong in (-1, c.pages.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = c.table.clone()
        table[0, 2] = wrong
        out = decoding.tree_attention(q, c.pages, c.q_start, c.lengths, table, spans)
        _check(out, *_attend(c, q, spans, scale, hide=(0, 32, 48)))
        with pytest.raises(PhoenixError) as e:
            decoding.check_status()
        assert e.value.status == 1 and "page" in e.value.message
        decoding.check_status()
    # a table with too few columns: the keys behind it do not exist
    cut = c.table[:, :18].contiguous()
    out = decoding.tree_attention(q, c.pages, c.q_start, c.lengths, cut, spans)
    _check(out, *_attend(c, q, spans, scale, hide=(0, 288, 10 ** 6)))
    with pytest.raises(PhoenixError):
        decoding.check_status()
    # offsets that leave the rows: that request is left out, the other is right
    q_start = c.q_start.clone()
    q_start[2] = 10 ** 6
    out.fill_(7.0)
    decoding.tree_attention(q, c.pages, q_start, c.lengths, c.table, spans, out=out)
    want, mag = _attend(c, q, spans, scale)
    _check(out[:tokens], want[:tokens], mag[:tokens])
    assert bool((out[tokens:] == 7.0).all())
    with pytest.raises(PhoenixError) as e:
        decoding.check_status()
    assert "offsets" in e.value.message


def test_tree_attention_strides_streams_and_hints():
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([20, 33], [700, 90], 2, 64, 16, seed=6)
    wide = torch.randn((c.n, 24, 64), device=DEV, generator=c.g).to(torch.bfloat16)
    q, spans = wide[:, 8:16], torch.tensor(_spans("tree", 20) + _spans("tree", 33), dtype=torch.int32, device=DEV)
    table = torch.full((2, 100), -1, dtype=torch.int32, device=DEV)
    table[:, 7:7 + c.table.shape[1]] = c.table
    rows = table[:, 7:7 + c.table.shape[1]]
    out = decoding.tree_attention(q, c.pages, c.q_start, c.lengths, rows, spans)
    _check(out, *_attend(c, q, spans, math.sqrt(128.0) / 64))
    assert torch.equal(out, decoding.tree_attention(q.contiguous(), *c.args(), spans))            # equal calls, equal bits
    # hints that are too small choose other kernels, not other answers
    for kw in (dict(max_tokens=1), dict(max_keys=1), dict(max_tokens=1, max_keys=1), dict(max_tokens=1000, max_keys=100000)):
        _check(decoding.tree_attention(q, *c.args(), spans, **kw), *_attend(c, q, spans, math.sqrt(128.0) / 64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = decoding.tree_attention(q, *c.args(), spans)
    side.synchronize()
    assert torch.equal(out, again)
    decoding.check_status(stream=side.cuda_stream)


def test_tree_attention_in_a_graph():
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([3] * 4, [900, 10, 0, 333], 4, 128, 16, seed=6)
    q = torch.randn((c.n, 16, 128), device=DEV, generator=c.g).to(torch.bfloat16)
    spans = torch.tensor(_spans("tree", 3) * 4, dtype=torch.int32, device=DEV)
    side, out = torch.cuda.Stream(), torch.empty_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decoding.tree_attention(q, *c.args(), spans, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            decoding.tree_attention(q, *c.args(), spans, out=out)
    q.copy_(torch.randn(q.shape, device=DEV, generator=c.g))
    c.lengths.copy_(torch.tensor([800, 11, 0, 300]))
    c.cached = [800, 11, 0, 300]
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    _check(out, *_attend(c, q, spans, math.sqrt(128.0) / 128))


def test_candidates_over_a_cached_history_equal_the_ranker_attention():
    """The layer's own attention (history whole, candidates isolated) in two appends and two calls."""
    from x_algorithm_b200 import decoding
    from x_algorithm_b200.engine import ranker_attention
    torch = _torch()
    g = torch.Generator(device=DEV).manual_seed(9)
    B, S, Cn, heads, kv, dh = 3, 100, 50, 16, 4, 128
    qkv = torch.randn((B, S + Cn, (heads + 2 * kv) * dh), device=DEV, generator=g).to(torch.bfloat16)
    split = qkv.view(B, S + Cn, kv, heads // kv + 2, dh)
    q, k, v = split[:, :, :, :-2].flatten(2, 3).contiguous(), split[:, :, :, -2].contiguous(), split[:, :, :, -1].contiguous()
    seg = torch.ones((B, S + Cn), dtype=torch.int32, device=DEV)
    seg[:, S:] = -1
    want, _ = ranker_attention(q, k, v, seg, S, math.sqrt(128.0) / dh)
    pages = torch.full((B * 10, 2, kv, 16, dh), math.nan, dtype=torch.bfloat16, device=DEV)
    table = torch.arange(B * 10, dtype=torch.int32, device=DEV).view(B, 10)
    got = torch.empty_like(want)
    for at, count, length, span in ((0, S, 0, (0, 1)), (S, Cn, S, None)):
        rows = qkv[:, at:at + count].reshape(B * count, -1)
        q_start = torch.arange(0, B * count + 1, count, dtype=torch.int32, device=DEV)
        lengths = torch.full((B,), length, dtype=torch.int32, device=DEV)
        i = torch.arange(count, dtype=torch.int32, device=DEV)
        spans = torch.tensor([span], dtype=torch.int32, device=DEV).repeat(B * count, 1) if span else torch.stack([i, i + 1], 1).repeat(B, 1).contiguous()
        qn = decoding.history_append(rows, pages, q_start, lengths, table, None, num_q_heads=heads)
        got[:, at:at + count] = decoding.tree_attention(qn, pages, q_start, lengths, table, spans).view(B, count, heads, dh)
    decoding.check_status()
    # both round their probabilities and their output to bf16 once, in different tilings
    mag = v.abs().amax(1).repeat_interleave(heads // kv, 1)[:, None].float()
    assert bool(((got.float() - want.float()).abs() <= 2 * U * (want.float().abs() + mag)).all())


# ---- append ------------------------------------------------------------------------------------------------------------

def _append_want(c, qkv, heads, positions, base, q_gain, k_gain, eps):
    torch = _torch()
    g = heads // c.kv_heads
    x = qkv.double().view(-1, c.kv_heads, g + 2, c.dh)
    qk = x[:, :, :g + 1].clone()
    mag = qk.abs()
    if q_gain is not None:
        gain = torch.cat([q_gain.double().expand(g, c.dh), k_gain.double()[None]])
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + eps) * gain
    if base:
        half = c.dh // 2
        i = torch.arange(half, dtype=torch.float64, device=DEV)
        ang = positions.double()[:, None] * base ** (-2 * i / c.dh)
        cos, sin = ang.cos()[:, None, None], ang.sin()[:, None, None]
        a, b = qk[..., :half], qk[..., half:]
        mag = torch.cat([a.abs() + b.abs()] * 2, -1)
        qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        mag = qk.abs()
    return qk[:, :, :g].flatten(1, 2), qk[:, :, g], x[:, :, g + 1], mag[:, :, :g].flatten(1, 2), mag[:, :, g]


@pytest.mark.parametrize("heads,kv_heads,dh", HEADS)
@pytest.mark.parametrize("tokens,cached,page", [([1], [0], 16), ([3, 0, 1, 18], [15, 4, 16, 31], 16), ([100], [1], 48), ([1] * 40, list(range(40)), 32),
                                                ([2, 0, 0, 5] * 300, [7] * 1200, 16)])
@pytest.mark.parametrize("norm,base", [(True, 10000.0), (False, 500.0), (True, 0.0), (False, 0.0)])
def test_history_append(heads, kv_heads, dh, tokens, cached, page, norm, base):
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache(tokens, cached, kv_heads, dh, page, seed=len(tokens))
    width = (heads + 2 * kv_heads) * dh
    wide = torch.randn((c.n, width + 24), device=DEV, generator=c.g).to(torch.bfloat16)
    qkv = wide[:, 8:8 + width]
    positions = torch.randint(0, 300, (c.n,), device=DEV, generator=c.g, dtype=torch.int32)
    cos, sin = decoding.rope_tables(300, dh, base) if base else (None, None)
    gains = [1 + 0.3 * torch.randn(dh, device=DEV, generator=c.g) for _ in range(2)] if norm else [None, None]
    before = c.pages.clone()
    q = decoding.history_append(qkv, *c.args(), positions, cos, sin, num_q_heads=heads, q_gain=gains[0], k_gain=gains[1], eps=1e-5)
    decoding.check_status()
    wq, wk, wv, mq, mk = _append_want(c, qkv, heads, positions, base, *gains, 1e-5)
    near = lambda got, want, mag: bool(((got.double() - want).abs() <= 1.001 * U * want.abs() + 2.0 ** -20 * mag).all())  # noqa: E731
    assert near(q, wq, mq)
    at, touched = 0, torch.zeros_like(before, dtype=torch.bool)
    for b, (t, k) in enumerate(zip(tokens, cached)):
        if t == 0:
            continue
        where = torch.arange(k, k + t, device=DEV)
        number = torch.tensor(c.table_host[b], device=DEV)[where // page]
        assert near(c.pages[number, 0, :, where % page], wk[at:at + t], mk[at:at + t])
        assert torch.equal(c.pages[number, 1, :, where % page].double(), wv[at:at + t])
        touched[number, :, :, where % page] = True
        at += t
    assert torch.equal(c.pages[~touched], before[~touched])     # nothing else was written


def test_history_append_reports_what_it_left_out():
    from x_algorithm_b200 import PhoenixError, decoding
    torch = _torch()
    c = Cache([4, 4, 4], [14, 0, 30], 2, 64, 16, seed=1)
    qkv = torch.randn((c.n, (8 + 4) * 64), device=DEV, generator=c.g).to(torch.bfloat16)
    positions = torch.zeros(c.n, dtype=torch.int32, device=DEV)
    cos, sin = decoding.rope_tables(8, 64)
    good = decoding.history_append(qkv, *c.args(), positions, cos, sin, num_q_heads=8)
    stored = c.pages.clone()
    for wrong in (-1, c.pages.shape[0], 2 ** 31 - 1):
        c.pages.zero_()
        table = c.table.clone()
        table[0, 1] = wrong                                     # tokens 2 and 3 of request 0
        assert torch.equal(decoding.history_append(qkv, c.pages, c.q_start, c.lengths, table, positions, cos, sin, num_q_heads=8), good)
        with pytest.raises(PhoenixError) as e:
            decoding.check_status()
        assert e.value.status == 1 and "page" in e.value.message
        page = c.table_host[0][1]
        assert bool((c.pages[page] == 0).all())
        assert torch.equal(c.pages[c.table_host[0][0], :, :, 14:], stored[c.table_host[0][0], :, :, 14:])
    positions[5] = 8
    positions[6] = -3
    got = decoding.history_append(qkv, *c.args(), positions, cos, sin, num_q_heads=8)
    with pytest.raises(PhoenixError) as e:
        decoding.check_status()
    assert "position" in e.value.message
    near = positions.clamp(0, 7)
    assert torch.equal(got, decoding.history_append(qkv, *c.args(), near, cos, sin, num_q_heads=8))
    decoding.check_status()
    c.pages.zero_()
    q_start = torch.tensor([0, 4, 2, 12], dtype=torch.int32, device=DEV)     # does not ascend: what nobody owns is not stored
    decoding.history_append(qkv, c.pages, q_start, c.lengths, c.table, positions.zero_(), cos, sin, num_q_heads=8)
    with pytest.raises(PhoenixError) as e:
        decoding.check_status()
    assert "offsets" in e.value.message


# ---- log probabilities ---------------------------------------------------------------------------------------------------

def _logprobs_want(x, cap, temperature):
    torch = _torch()
    x = x.double()
    banned = x == -math.inf
    y = (cap * torch.tanh(x / cap) if cap else x) / temperature
    y = y.masked_fill(banned, -math.inf)
    y = y - y.amax(1, keepdim=True).nan_to_num(nan=math.nan, posinf=math.inf, neginf=0.0)   # first: 64 bits do not hold 1e30 + ln 2 either
    lp = y - torch.logsumexp(y, 1, keepdim=True)
    lp = lp.masked_fill(banned, -math.inf)
    ent = -(lp.exp() * lp.masked_fill(banned, 0.0)).sum(1)
    return lp, ent.masked_fill(banned.all(1), 0.0)


def _logprobs_check(x, given, top_k, cap=0.0, temperature=1.0):
    from x_algorithm_b200 import decoding
    torch = _torch()
    lp, entropy, top, ids = decoding.token_logprobs(x, given, top_k=top_k, cap=cap, temperature=temperature)
    want, want_h = _logprobs_want(x, cap, temperature)
    tol = lambda w: 1e-5 + 2.0 ** -21 * w.abs().nan_to_num(0.0, 0.0, 0.0)  # noqa: E731

    def near(got, w):
        got, w = got.double(), w.float().double()           # what fp32 does not hold is infinite there
        same = (got == w) | (torch.isnan(got) & torch.isnan(w))
        assert bool((same | ((got - w).abs() <= tol(w))).all()), float(((got - w).abs() - tol(w)).nan_to_num(-1.0, -1.0, -1.0).max())

    if given is not None:
        inside = (given >= 0) & (given < x.shape[1])
        g = given if given.dim() == 2 else given[:, None]
        w = want.gather(1, g.clamp(0, x.shape[1] - 1)).view(given.shape)
        near(lp, torch.where(inside, w, 0.0))
    near(entropy, want_h)
    v = torch.where(torch.isnan(x), math.inf, x.float()) + torch.where(torch.isnan(x), 1.0, 0.0)
    rank = torch.sort(torch.where(torch.isnan(x.float()), torch.full_like(v, math.nan), x.float() + 0.0), dim=1, descending=True, stable=True)[1][:, :top_k]
    assert torch.equal(ids, rank)
    near(top, want.gather(1, rank))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 19, 255, 256, 257, 1000, 2047, 4099, 8193, 40001, 131072])
@pytest.mark.parametrize("rows,top_k,given", [(1, 1, 1), (5, 20, 0), (37, 128, 3), (300, 0, 2)])
def test_token_logprobs(dtype, vocab, rows, top_k, given):
    torch = _torch()
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    x = (4 * torch.randn((rows, vocab), device=DEV, generator=g)).to(getattr(torch, dtype))
    ids = torch.randint(0, vocab, (rows, given), device=DEV, generator=g) if given else None
    _logprobs_check(x, ids, min(top_k, vocab))
    if vocab in (19, 4099):
        _logprobs_check(x, ids, min(top_k, vocab), cap=6.0, temperature=0.7)
        _logprobs_check(x, ids, min(top_k, vocab), cap=30.0, temperature=1.5)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [33, 5000, 70001])
def test_token_logprobs_orders_that_defeat_a_sampled_bound(dtype, vocab):
    """Equal logits, sorted rows, all the best in one stretch or at one distance from each other, steps, big values."""
    torch = _torch()
    t = getattr(torch, dtype)
    i = torch.arange(vocab, device=DEV, dtype=torch.float32)
    rows = [torch.zeros(vocab, device=DEV), i / vocab * 20, -i / vocab * 20, torch.where(i % 256 == 3, 9 + i / vocab, i / vocab),
            torch.where(i % 2048 < 8, 9 + i / vocab, i / vocab), torch.where(i < 3000, 9 - i / vocab, i / vocab), torch.where(i > vocab - 3000, 9.0, 0.0),
            torch.where(i == vocab // 2, 80.0, -80.0), (i % 7).floor(), torch.where(i % 2 == 0, 0.0, -0.0), 1e30 * torch.cos(i), torch.where(i < 8 * 300, 5.0, i * 0)]
    x = torch.stack(rows).to(t)
    for top_k in (1, 7, 33 if vocab == 33 else 128):
        _logprobs_check(x, torch.zeros((x.shape[0], 1), dtype=torch.int64, device=DEV), top_k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [5, 300, 9001, 66000])
def test_token_logprobs_of_banned_ids_infinities_and_nan(dtype, vocab):
    torch = _torch()
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn((8, vocab), device=DEV, generator=g)
    x[0] = -math.inf                                        # nothing allowed
    x[1] = -math.inf
    x[1, vocab - 1] = 0.25                                  # one id allowed
    x[2, torch.rand(vocab, device=DEV, generator=g) < 0.9] = -math.inf
    x[3, vocab // 2] = math.nan
    x[4, vocab // 3] = math.inf
    x[5] = torch.finfo(torch.bfloat16).min                  # a type's lowest value is a number
    x[6, :vocab // 2] = torch.finfo(torch.bfloat16).min
    x[7] = math.nan
    x = x.to(getattr(torch, dtype))
    given = torch.tensor([[0, vocab - 1, -1, vocab, 2 ** 40, -2 ** 40]] * 8, device=DEV)
    for kw in (dict(), dict(cap=20.0), dict(temperature=0.5)):
        _logprobs_check(x, given, min(vocab, 50), **kw)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_token_logprobs_strides_alignment_and_streams(dtype):
    from x_algorithm_b200 import decoding
    torch = _torch()
    g = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn((9, 5003), device=DEV, generator=g).to(getattr(torch, dtype))
    for lo, hi in ((0, 5003), (1, 4000), (3, 20), (7, 5000), (8, 4104)):
        x = wide[:, lo:hi]
        _logprobs_check(x, torch.full((9,), hi - lo - 1, dtype=torch.int64, device=DEV), 10)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = decoding.token_logprobs(x, top_k=10)
        side.synchronize()
        plain = decoding.token_logprobs(x.contiguous(), top_k=10)
        assert again[0] is None and torch.equal(again[3], plain[3])


# ---- refusals ------------------------------------------------------------------------------------------------------------

def test_refusals():
    from x_algorithm_b200 import PhoenixError, decoding
    torch = _torch()
    c = Cache([2], [5], 2, 64, 16)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)
    x = torch.zeros((2, 30), device=DEV)
    spans = torch.zeros((2, 2), dtype=torch.int32, device=DEV)
    cos, sin = decoding.rope_tables(10, 64)
    bad = [
        lambda: decoding.tree_attention(q.float(), *c.args()), lambda: decoding.tree_attention(q.cpu(), *c.args()),
        lambda: decoding.tree_attention(q[:, :, :32], *c.args()), lambda: decoding.tree_attention(q[:, ::2], *c.args()),
        lambda: decoding.tree_attention(q[:, :3].contiguous(), *c.args()), lambda: decoding.tree_attention(q, *c.args(), spans[:1]),
        lambda: decoding.tree_attention(q, *c.args(), spans.long()), lambda: decoding.tree_attention(q, *c.args(), cap=3.0, cap_method="relu"),
        lambda: decoding.tree_attention(q, c.pages[:, :1], *c.args()[1:]), lambda: decoding.tree_attention(q, c.pages, c.q_start[:1], c.lengths, c.table),
        lambda: decoding.tree_attention(q, *c.args(), sm_scale=math.nan), lambda: decoding.tree_attention(q, *c.args(), out=q[:1]),
        lambda: decoding.tree_attention(q, *c.args(), max_tokens=-1), lambda: decoding.tree_attention(q, c.pages[:, :, :, :8].contiguous(), *c.args()[1:]),
        lambda: decoding.history_append(qkv[:, :-8], *c.args(), pos, num_q_heads=4), lambda: decoding.history_append(qkv, *c.args(), pos, cos, None, num_q_heads=4),
        lambda: decoding.history_append(qkv, *c.args(), pos.long(), cos, sin, num_q_heads=4), lambda: decoding.history_append(qkv, *c.args(), pos, cos, sin, num_q_heads=3),
        lambda: decoding.history_append(qkv, *c.args(), pos, q_gain=torch.ones(64, device=DEV), num_q_heads=4),
        lambda: decoding.history_append(qkv, *c.args(), pos, q_gain=torch.ones(32, device=DEV), k_gain=torch.ones(64, device=DEV), num_q_heads=4),
        lambda: decoding.token_logprobs(x.half()), lambda: decoding.token_logprobs(x, top_k=31), lambda: decoding.token_logprobs(x, top_k=-1),
        lambda: decoding.token_logprobs(x, temperature=0.0), lambda: decoding.token_logprobs(x, temperature=math.nan), lambda: decoding.token_logprobs(x, cap=math.inf),
        lambda: decoding.token_logprobs(x, torch.zeros((1, 1), dtype=torch.int64, device=DEV)), lambda: decoding.token_logprobs(x, pos),
        lambda: decoding.token_logprobs(x.T), lambda: decoding.token_logprobs(torch.zeros((2, 200), device=DEV), top_k=129),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, PhoenixError)):
            f()
            pytest.fail(f"call {i} was not refused")
    # nothing to do is no error
    none = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert decoding.tree_attention(none, c.pages, zero, c.lengths, c.table).shape == (0, 4, 64)
    assert decoding.history_append(qkv[:0], c.pages, zero, c.lengths, c.table, pos[:0], num_q_heads=4).shape == (0, 4, 64)
    assert decoding.token_logprobs(x[:0], top_k=3)[3].shape == (0, 3)
    decoding.check_status()


# ---- which kernels run, and the ends of the ranges -------------------------------------------------------------------------

def _ran(f):
    from x_algorithm_b200.engine import dispatch_counts
    before = dispatch_counts()
    f()
    return {k for k, v in dispatch_counts().items() if v != before[k]}


def test_kernels_by_rows_of_a_key_head():
    """Up to 16 query rows of a key head, heads of 32 and groups of more than 128 are the mma.sync kernel's, the rest the tensor cores'."""
    assert _ran(lambda: _tree_case([1, 3], [100, 5], 16, 4, 128, 16)) == {"tree.mma"}
    assert _ran(lambda: _tree_case([2, 5], [100, 5], 16, 4, 128, 16, max_tokens=5)) == {"tree.tcgen05"}
    assert _ran(lambda: _tree_case([40], [100], 4, 4, 32, 16)) == {"tree.mma"}
    assert _ran(lambda: _tree_case([2], [90], 144, 1, 64, 16)) == {"tree.mma"}


@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dh", [(50, 140, 8, 8, 64), (90, 40, 16, 4, 128), (1100, 1, 16, 4, 128), (1100, 20, 4, 2, 64), (700, 2, 8, 8, 64)])
def test_many_requests(batch, tokens, heads, kv_heads, dh):
    """More units than blocks (a block takes several), more requests than the shared plan holds; empty requests among them."""
    rng = np.random.default_rng(batch)
    t = [int(x) for x in rng.integers(0, tokens + 1, batch)]
    t[3] = tokens
    _tree_case(t, [int(x) for x in rng.integers(0, 200, batch)], heads, kv_heads, dh, 16, "tree", seed=batch)


@pytest.mark.parametrize("tokens,cached,heads,kv_heads,dh,page", [([1], [40001], 8, 8, 64, 128), ([9], [30003], 16, 1, 128, 48), ([2, 30], [20000, 17], 10, 2, 64, 16),
                                                                   ([33], [12345], 24, 8, 128, 32), ([1100], [3], 4, 1, 64, 64), ([300, 2], [2500, 4001], 16, 4, 128, 112)])
@pytest.mark.parametrize("shape", ["chain", "whole", "tree"])
def test_long_caches_are_cut_and_joined(tokens, cached, heads, kv_heads, dh, page, shape):
    _tree_case(tokens, cached, heads, kv_heads, dh, page, shape, padding=1, seed=len(tokens))


def test_odd_values_in_parts():
    """Infinities and NaN of new tokens where the keys are cut into parts."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    for tokens, heads, kv_heads, dh in ((3, 16, 4, 128), (60, 16, 4, 128), (40, 8, 8, 64)):
        c = Cache([tokens], [9000], kv_heads, dh, 16, seed=2)
        q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
        spans = torch.tensor(_spans("tree", tokens, 1, 4), dtype=torch.int32, device=DEV)
        for j, value in ((0, math.inf), (tokens - 1, math.nan), (1, -math.inf)):
            at = 9000 + j
            c.pages[c.table_host[0][at // 16], 1, 0, at % 16, j + 2] = value
        out = decoding.tree_attention(q, *c.args(), spans)
        _check(out, *_attend(c, q, spans, math.sqrt(128.0) / dh))


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, its last pages in use; logits and rows further apart than 2^31 elements."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    total, kv, page, dh, heads = 18000, 8, 128, 128, 16
    pages = torch.empty((total, 2, kv, page, dh), dtype=torch.bfloat16, device=DEV)
    assert pages.numel() > 2 ** 32
    for tokens in (1, 70):
        small = Cache([tokens], [300], kv, dh, page, seed=tokens)
        numbers = [total - 1 - i for i in range(len(small.table_host[0]) - 1)]
        for i, p in enumerate(numbers):
            pages[p] = small.pages[small.table_host[0][i]]
        table = torch.tensor([numbers + [-1]], dtype=torch.int32, device=DEV)
        q = torch.randn((tokens, heads, dh), device=DEV, generator=small.g).to(torch.bfloat16)
        want = decoding.tree_attention(q, *small.args())
        assert torch.equal(decoding.tree_attention(q, pages, small.q_start, small.lengths, table), want)
        qkv = torch.randn((tokens, (heads + 2 * kv) * dh), device=DEV, generator=small.g).to(torch.bfloat16)
        a = decoding.history_append(qkv, *small.args(), None, num_q_heads=heads)
        b = decoding.history_append(qkv, pages, small.q_start, small.lengths, table, None, num_q_heads=heads)
        assert torch.equal(a, b)
        for i, p in enumerate(numbers):
            assert torch.equal(pages[p], small.pages[small.table_host[0][i]])
        decoding.check_status()
    del pages
    wide = torch.empty(2 ** 31 + 5000, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((2, 4001), device=DEV, generator=g).to(torch.bfloat16)
    far = wide.as_strided((2, 4001), (2 ** 31 + 8, 1), 3)
    far.copy_(x)
    _logprobs_check(far, torch.tensor([[0, 4000]] * 2, device=DEV), 9)    # (its words begin elsewhere than x's: the sums' last bits may differ)


def test_a_wait_that_ran_out_is_reported_once():
    """The flag that a bounded wait raises, raised by the host."""
    from x_algorithm_b200 import PhoenixError, decoding
    torch = _torch()
    _tree_case([40], [100], 8, 8, 64, 16)
    kept = decoding._kept[(0, torch._C._cuda_getCurrentRawStream(0))]
    kept.status[0] = 1
    with pytest.raises(PhoenixError) as e:
        decoding.check_status()
    assert e.value.status == 4
    decoding.check_status()
    _tree_case([40], [100], 8, 8, 64, 16)
