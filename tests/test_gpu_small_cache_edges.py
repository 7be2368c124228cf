"""Window attention, key weights and eviction where they can go wrong: hidden keys of any value, pages out of range or of others, streams, graphs, far offsets, and a run of
them together.  Tolerances are those of test_gpu_small_cache."""
import math

import pytest
import torch

from test_gpu_small_cache import DEV, close, evict_plain, make_case, plain, plain_weights, rows_of, visible

pytestmark = pytest.mark.gpu

SHAPES = [
    # batch, tokens, cached, heads, kv heads, head dim, page, shape, positions, window, sinks
    (2, 1, 500, 16, 4, 128, 64, "chain", None, 100, 3),
    (2, 3, 333, 4, 4, 32, 16, "chain", None, 70, 2),
    (2, 4, 300, 10, 2, 64, 48, "tree", "depth", 65, 1),
    (2, 70, 500, 16, 4, 128, 16, "chain", None, 100, 3),
    (2, 200, 400, 8, 8, 64, 128, "isolated", None, 130, 1),
    (2, 40, 700, 32, 8, 128, 32, "tree", "depth", 200, 20),
]
IDS = lambda s: "-".join(map(str, s))  # noqa: E731


def args_of(c):
    return c["q"], c["pages"], c["q_start"], c["lengths"], c["table"]


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_what_is_not_seen_leaves_no_trace(shape, cap):
    """Infinities, NaN and the type's largest values in keys and values that no row sees, behind the last key, and in pages of nobody."""
    from x_algorithm_b200 import decoding
    *head, positions, window, sinks = shape
    c = make_case(*head, seed=21, positions=positions, ragged=False, padding=2 if head[7] in ("tree", "isolated") else 0)
    more = dict(spans=c["spans"], positions=c["positions"], window=window, sinks=sinks, cap=cap, cap_method="tanh" if cap else None)
    out, lse = decoding.window_attention(*args_of(c), **more)
    weights = decoding.key_weights(*args_of(c), lse, c["weights"].clone(), decay=0.5, **more)
    odd = torch.tensor([math.inf, -math.inf, math.nan, 3e38, -3e38], device=DEV).to(torch.bfloat16)
    pages, page = c["pages"].clone(), c["page"]
    used = torch.zeros(pages.shape[0], page, dtype=torch.bool, device=DEV)
    for b in range(len(c["n_new"])):
        seen = visible(c, b, window, sinks).any(0)
        at = seen.nonzero()[:, 0]
        used[c["table"][b, at // page].long(), at % page] = True
    hidden = (~used)[:, None, None, :, None].expand_as(pages)
    pages[hidden] = odd[torch.arange(int(hidden.sum()), device=DEV) % 5]
    again, lse_again = decoding.window_attention(c["q"], pages, *args_of(c)[2:], **more)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)
    got = decoding.key_weights(c["q"], pages, *args_of(c)[2:], lse, c["weights"].clone(), decay=0.5, **more)
    assert torch.equal(got, weights)
    decoding.check_status()


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_odd_values_that_some_rows_see_reach_those_alone(shape):
    from x_algorithm_b200 import decoding
    *head, positions, window, sinks = shape
    c = make_case(*head, seed=22, positions=positions, ragged=False)
    k, t = c["n_old"][1], c["n_new"][1]
    at = [k - window + 2 if head[7] == "chain" else k, k + t - 1, 0]           # at a window's edge (or a new key), the last key, a first key
    for i, key in enumerate(at):
        c["pages"][c["table"][1, key // c["page"]].long(), 1, :, key % c["page"], 3 * i] = [math.inf, math.nan, -math.inf][i]
    out, _ = decoding.window_attention(*args_of(c), c["spans"], c["positions"], window=window, sinks=sinks)
    want, _, tol, _ = plain(c, window, sinks)
    row0 = c["n_new"][0]
    see = visible(c, 1, window, sinks)
    for i, key in enumerate(at):
        assert torch.equal(~torch.isfinite(out[row0:, :, 3 * i]), see[:, key, None].expand(-1, out.shape[1])), (i, key)
    fine = torch.isfinite(out.double())
    close(out[fine], want[fine], tol[fine], "out")


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_pages_in_front_of_the_window_may_be_handed_out(shape):
    from x_algorithm_b200 import decoding
    *head, positions, window, sinks = shape
    c = make_case(*head, seed=23, positions=positions, ragged=False)
    more = dict(spans=c["spans"], positions=c["positions"], window=window, sinks=sinks)
    out, lse = decoding.window_attention(*args_of(c), **more)
    weights = decoding.key_weights(*args_of(c), lse, c["weights"].clone(), **more)
    table, freed = c["table"].clone(), 0
    for b, k in enumerate(c["n_old"]):
        first, behind = -(-sinks // c["page"]), (k - window + 1) // c["page"]   # pages with a first key, the first page that the window reaches
        table[b, first:behind] = -1 if b else 2 ** 31 - 1
        freed += max(0, behind - first)
    assert freed > 0
    again, lse_again = decoding.window_attention(*args_of(c)[:4], table, **more)
    got = decoding.key_weights(*args_of(c)[:4], table, lse, c["weights"].clone(), **more)
    decoding.check_status()                                   # nothing to report
    assert torch.equal(out, again) and torch.equal(lse, lse_again) and torch.equal(got, weights)


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_bad_pages_are_left_out_and_reported(shape):
    from x_algorithm_b200 import PhoenixError, decoding
    *head, positions, window, sinks = shape
    c = make_case(*head, seed=24, positions=positions, ragged=False)
    page = c["page"]
    keep = [torch.ones(a + b, dtype=torch.bool, device=DEV) for a, b in zip(c["n_new"], c["n_old"])]
    col = c["n_old"][1] // page - 1
    bad = c["table"].clone()
    bad[1, col] = c["pages"].shape[0]
    keep[1][col * page:(col + 1) * page] = False
    want, want_lse, tol, tol_lse = plain(c, window, sinks, keep=keep)
    more = dict(spans=c["spans"], positions=c["positions"], window=window, sinks=sinks)
    out, lse = decoding.window_attention(*args_of(c)[:4], bad, **more)
    with pytest.raises(PhoenixError):
        decoding.check_status()
    close(lse, want_lse, tol_lse, "lse")
    close(out, want, tol, "out")
    full, full_tol = plain_weights(c, lse, window, sinks)
    got = decoding.key_weights(*args_of(c)[:4], bad, lse, c["weights"].clone(), **more)
    with pytest.raises(PhoenixError):
        decoding.check_status()
    full[c["table"][1, col].long()] = c["weights"][c["table"][1, col].long()].double()   # as it was
    close(got, full, full_tol, "weights")


def test_offsets_that_leave_the_rows_and_rows_of_nobody():
    from x_algorithm_b200 import PhoenixError, decoding
    for tokens in (2, 60):
        c = make_case(3, tokens, 200, 16, 4, 64, 32, "chain", seed=25, ragged=False)
        n = 3 * tokens + 4
        q = torch.cat([c["q"], c["q"][:4]])
        starts = torch.tensor([0, tokens, 2 * tokens, 3 * tokens], dtype=torch.int32, device=DEV)
        out, lse, weights = torch.full((n, 16, 64), 7.0, device=DEV, dtype=torch.bfloat16), torch.full((n, 16), 9.0, device=DEV), c["weights"].clone()
        decoding.window_attention(q, c["pages"], starts, c["lengths"], c["table"], window=50, sinks=2, out=out, lse=lse)
        assert torch.all(out[3 * tokens:] == 7) and torch.all(lse[3 * tokens:] == 9)
        want, want_lse, tol, tol_lse = plain(c, 50, 2)
        close(out[:3 * tokens], want, tol, "out")
        close(lse[:3 * tokens], want_lse, tol_lse, "lse")
        starts[2] = n + 1                                     # leaves the rows: two requests are left out
        decoding.key_weights(q, c["pages"], starts, c["lengths"], c["table"], lse, weights, window=50, sinks=2)
        with pytest.raises(PhoenixError):
            decoding.check_status()
        first, tol = plain_weights(dict(c, n_new=c["n_new"][:1], n_old=c["n_old"][:1]), lse, 50, 2)
        close(weights, first, tol, "weights")


def test_nothing_to_do():
    from x_algorithm_b200 import decoding
    c = make_case(2, 0, 100, 8, 8, 64, 16, "chain", seed=26, ragged=False)
    out, lse = decoding.window_attention(*args_of(c), window=10)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    before = c["weights"].clone()
    decoding.key_weights(*args_of(c), lse, c["weights"])
    assert torch.equal(before, c["weights"])
    empty = torch.zeros((0, c["table"].shape[1]), dtype=torch.int32, device=DEV)
    lengths, kept = decoding.evict(c["weights"], c["pages"], torch.zeros(0, dtype=torch.int32, device=DEV), empty, budget=5)
    assert lengths.shape == (0,) and kept.shape == (0, 8, 5)
    lengths, kept = decoding.evict(c["weights"], c["pages"], torch.zeros(2, dtype=torch.int32, device=DEV), c["table"], budget=5)
    assert lengths.tolist() == [0, 0] and torch.all(kept == -1)
    decoding.check_status()


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
@pytest.mark.parametrize("tokens", [1, 50])
def test_scales(scale, tokens):
    """No, turned-round and extreme logits (one key takes all weight)."""
    from x_algorithm_b200 import decoding
    c = make_case(2, tokens, 300, 16, 4, 128, 64, "chain", seed=27, ragged=False)
    c["scale"] = scale
    want, want_lse, tol, tol_lse = plain(c, 90, 2)
    out, lse = decoding.window_attention(*args_of(c), window=90, sinks=2, sm_scale=scale)
    close(lse, want_lse, tol_lse, "lse")
    close(out, want, tol, "out")
    got = decoding.key_weights(*args_of(c), lse, c["weights"].clone(), window=90, sinks=2, sm_scale=scale)
    close(got, *plain_weights(c, lse, 90, 2), "weights")


def test_bad_pages_of_an_eviction_are_reported_and_do_no_harm():
    from x_algorithm_b200 import PhoenixError, decoding
    for budget in (300, 150):                                 # chunks, and the select's own blocks
        c = make_case(2, 0, 600, 4, 4, 64, 16, "chain", seed=28, ragged=False)
        page, table = c["page"], c["table"].clone()
        table[0, 35] = -7                                     # keys 560 .. 575 have no weights: they go first
        order = c["weights"].clone()
        c["weights"][c["table"][0, 35].long()] = -1.0
        want = evict_plain(c, c["n_old"], budget, 3, 0)
        c["weights"] = order
        lengths, kept = decoding.evict(c["weights"], c["pages"], c["lengths"], table, budget=budget, sinks=3)
        with pytest.raises(PhoenixError):
            decoding.check_status()
        assert torch.equal(kept, want[3]) and torch.equal(lengths, want[2])
        assert torch.equal(c["pages"], want[0])
        lost = c["table"][0, 35].long()
        want[1][lost] = order[lost]
        assert torch.equal(c["weights"], want[1])
        c["lengths"][1] = -5                                  # a length that is none
        lengths, _ = decoding.evict(c["weights"], c["pages"], c["lengths"], c["table"], budget=100)
        with pytest.raises(PhoenixError):
            decoding.check_status()
        assert lengths.tolist() == [100, 0]


def test_a_captured_run_of_them_is_what_it_is_without():
    """Append, attention, weights and eviction in one graph, replayed on other contents of the same buffers; and on a stream of their own."""
    from x_algorithm_b200 import decoding
    H, K, D, page, budget = 16, 4, 64, 16, 96
    B, T, cached = 3, 40, [100, 300, 57]
    g = torch.Generator(device=DEV).manual_seed(1)
    cols = -(-(300 + T) // page)
    new = lambda *s: torch.randn(s, device=DEV, generator=g).to(torch.bfloat16)  # noqa: E731
    pages, weights = new(B * cols, 2, K, page, D), torch.zeros((B * cols, K, page), device=DEV)
    table = torch.randperm(B * cols, device=DEV, generator=g).view(B, cols).to(torch.int32)
    qkv, lengths = new(B * T, (H + 2 * K) * D), torch.tensor(cached, dtype=torch.int32, device=DEV)
    q_start = torch.tensor([0, T, 2 * T, 3 * T], dtype=torch.int32, device=DEV)
    positions = torch.cat([torch.arange(k, k + T) for k in cached]).to(torch.int32).to(DEV)
    cos, sin = decoding.rope_tables(400, D)

    def step(qkv, pages, weights):
        q = decoding.history_append(qkv, pages, q_start, lengths, table, positions, cos, sin, num_q_heads=H)
        out, lse = decoding.window_attention(q, pages, q_start, lengths, table, window=64, sinks=4)
        decoding.key_weights(q, pages, q_start, lengths, table, lse, weights, window=64, sinks=4, decay=0.9)
        full = lengths + T
        short, kept = decoding.evict(weights, pages, full, table, budget=budget, sinks=4, recent=20)
        last, _ = decoding.window_attention(q, pages, q_start, short - T, table, window=64, sinks=4)   # what is left serves on: the rows are its last ones
        return out, lse, short, kept, last

    state = [(qkv, pages, weights)] + [(new(*qkv.shape), new(*pages.shape), torch.rand(weights.shape, device=DEV, generator=g))]
    want = [step(*[x.clone() for x in s]) for s in state]
    after = []
    for s in state:
        s = [x.clone() for x in s]
        step(*s)
        after.append(s)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        mine = [x.clone() for x in state[0]]
        got = step(*mine)
    stream.synchronize()
    for a, b in zip(got, want[0]):
        assert torch.equal(a, b)
    graph, bufs = torch.cuda.CUDAGraph(), [x.clone() for x in state[0]]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = step(*bufs)
    for i in (0, 1, 0):
        for x, y in zip(bufs, state[i]):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b), i
        for a, b in zip(bufs, after[i]):
            assert torch.equal(a, b), i
    decoding.check_status()
    decoding.check_status(stream=stream.cuda_stream)


def test_calls_on_two_streams_at_once():
    from x_algorithm_b200 import decoding
    cases = [make_case(4, 200, 700, 16, 4, 128, 64, "whole", seed=31 + i) for i in range(2)]
    weigh = lambda c, lse: decoding.key_weights(*args_of(c), lse, c["weights"].clone(), c["spans"])  # noqa: E731
    want = []
    for c in cases:
        out, lse = decoding.window_attention(*args_of(c), c["spans"], window=None)
        want.append((out, lse, weigh(c, lse), *decoding.evict(c["weights"].clone(), c["pages"].clone(), c["lengths"], c["table"], budget=400)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [None, None]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                out, lse = decoding.window_attention(*args_of(c), c["spans"], window=None)
                got[i] = (out, lse, weigh(c, lse), *decoding.evict(c["weights"].clone(), c["pages"].clone(), c["lengths"], c["table"], budget=400))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)
    named = decoding.window_attention(*args_of(cases[0]), cases[0]["spans"], window=None, stream=streams[0].cuda_stream)
    streams[0].synchronize()
    assert torch.equal(named[0], want[0][0])


def test_offsets_past_32_bits():
    """A pool of 9 GB of which the last pages are used."""
    from x_algorithm_b200 import decoding
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 40 GB")
    small = make_case(2, 50, 400, 16, 4, 128, 64, "chain", seed=41, ragged=False)
    total, used = 70000, small["pages"].shape[0]
    pages = torch.zeros((total, 2, 4, 64, 128), dtype=torch.bfloat16, device=DEV)
    pages[total - used:] = small["pages"]
    weights = torch.zeros((total, 4, 64), device=DEV)
    weights[total - used:] = small["weights"]
    table = torch.where(small["table"] >= 0, small["table"] + (total - used), -1).to(torch.int32)
    for q, q_start in ((small["q"], small["q_start"]), (small["q"][::50].contiguous(), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV))):
        want = decoding.window_attention(q, small["pages"], q_start, small["lengths"], small["table"], window=200, sinks=4)
        got = decoding.window_attention(q, pages, q_start, small["lengths"], table, window=200, sinks=4)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a = decoding.key_weights(q, small["pages"], q_start, small["lengths"], small["table"], want[1], small["weights"].clone(), window=200, sinks=4)
        b = decoding.key_weights(q, pages, q_start, small["lengths"], table, want[1], weights.clone(), window=200, sinks=4)
        assert torch.equal(a, b[total - used:])
    for budget in (300, 100):
        p, w = small["pages"].clone(), small["weights"].clone()
        big, heavy = pages.clone(), weights.clone()
        a, b = decoding.evict(w, p, small["lengths"], small["table"], budget=budget), decoding.evict(heavy, big, small["lengths"], table, budget=budget)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(p, big[total - used:]) and torch.equal(w, heavy[total - used:])
        del big
    decoding.check_status()


def test_attention_over_a_cache_that_was_shrunk_is_attention_over_the_kept_keys():
    from x_algorithm_b200 import decoding
    c = make_case(3, 0, 900, 8, 4, 64, 32, "chain", seed=51)
    keys = [rows_of(c, b, 0) for b in range(3)], [rows_of(c, b, 1) for b in range(3)]
    lengths, kept = decoding.evict(c["weights"], c["pages"], c["lengths"], c["table"], budget=256, sinks=4, recent=32)
    n = lengths.tolist()
    q = torch.randn((3, 8, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(torch.bfloat16)
    spans = torch.tensor([[0, 1]] * 3, dtype=torch.int32, device=DEV)
    q_start = torch.arange(4, dtype=torch.int32, device=DEV)
    out = decoding.tree_attention(q, c["pages"], q_start, lengths - 1, c["table"], spans, sm_scale=0.125)   # the last kept key stands for the token's own
    for b in range(3):
        for h in range(8):
            at = kept[b, h // 2, :n[b]].long()
            k, v = keys[0][b][at, h // 2], keys[1][b][at, h // 2]
            p = torch.softmax(k @ q[b, h].double() * 0.125, 0)
            want, tol = p @ v, (p @ v.abs()) * 2.0 ** -7 + 1e-3
            assert torch.all((out[b, h].double() - want).abs() <= tol)


def test_a_wait_that_ran_out_is_reported_once():
    """The status word as a kernel's wait leaves it, behind a call of these operators."""
    from x_algorithm_b200 import PhoenixError, decoding
    c = make_case(1, 30, 300, 8, 8, 64, 16, "chain", seed=61, ragged=False)
    decoding.window_attention(*args_of(c), window=20)
    kept = decoding._kept[(0, decoding._stream(0, None))]
    kept.status[0] = 1                                        # as a wait that ran out leaves it
    with pytest.raises(PhoenixError) as e:
        decoding.check_status()
    assert e.value.status == 4
    decoding.window_attention(*args_of(c), window=20)
    decoding.check_status()


def test_refusals():
    from x_algorithm_b200 import decoding
    c = make_case(2, 3, 50, 8, 4, 64, 16, "chain", seed=71, ragged=False)
    a, n = args_of(c), c["q"].shape[0]
    lse, w = torch.zeros((n, 8), device=DEV), c["weights"]
    for bad in (dict(window=0), dict(window=4, sinks=-1), dict(window=4, cap=3.0), dict(window=4, cap_method="relu"), dict(window=4, positions=torch.zeros(n, device=DEV)),
                dict(window=4, positions=torch.zeros(n + 1, dtype=torch.int32, device=DEV)), dict(window=4, spans=torch.zeros((n, 2), device=DEV)),
                dict(window=4, lse=torch.zeros((n, 7), device=DEV)), dict(window=4, out=torch.zeros((n, 8, 64), device=DEV))):
        with pytest.raises(ValueError):
            decoding.window_attention(*a, **bad)
    for bad in (dict(lse=lse.double()), dict(lse=lse[:, :4]), dict(weights=w.half()), dict(weights=w[:-1]), dict(weights=w.transpose(1, 2)), dict(window=0), dict(cap=2.0)):
        with pytest.raises(ValueError):
            decoding.key_weights(*a, **{**dict(lse=lse, weights=w), **bad})
    with pytest.raises(Exception):
        decoding.key_weights(*a, lse, w, decay=math.nan)
    e = dict(weights=w, pages=c["pages"], lengths=c["lengths"], block_table=c["table"], budget=10)
    for bad in (dict(budget=0), dict(budget=5, sinks=3, recent=3), dict(sinks=-1), dict(recent=-1), dict(weights=w.double()), dict(weights=w[:, :2]),
                dict(lengths=c["lengths"].long()), dict(lengths=c["lengths"][:1]), dict(kept=torch.zeros((2, 4, 9), dtype=torch.int32, device=DEV)),
                dict(lengths_out=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(pages=c["pages"].float()), dict(workspace=torch.zeros(4, device=DEV))):
        with pytest.raises(ValueError):
            decoding.evict(**{**e, **bad})
    decoding.check_status()
