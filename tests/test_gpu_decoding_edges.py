"""Calls at the edges of the operators on a cached history.  Oracles and tolerances are test_gpu_decoding's unless a test says its own."""
import math

import pytest

from test_gpu_decoding import DEV, Cache, _attend, _check, _logprobs_check, _logprobs_want, _spans, _torch, _tree_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dh,page", [(16, 128, 64), (4, 64, 128), (8, 32, 16)])
@pytest.mark.parametrize("tokens,keys", [(1, k) for k in (192, 193, 256, 320, 321, 384, 385)] + [(5, k) for k in (448, 449, 512, 576, 577)] + [(30, 449), (30, 576)])
@pytest.mark.parametrize("hints", [True, False])
def test_one_request_with_one_key_head(heads, dh, page, tokens, keys, hints):
    """One unit of work and a few tiles of keys: fewer places than two blocks are worth.  The call and the next one succeed."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    kw = dict(max_tokens=tokens, max_keys=keys) if hints else {}
    c, q, _, _ = _tree_case([tokens], [keys - tokens], heads, 1, dh, page, "tree", seed=keys, **kw)
    qkv = torch.randn((tokens, (heads + 2) * dh), device=DEV, generator=c.g).to(torch.bfloat16)
    again = decoding.history_append(qkv, *c.args(), None, num_q_heads=heads)
    assert torch.equal(again, qkv.view(tokens, heads + 2, dh)[:, :heads])
    decoding.check_status()


def test_an_error_of_the_runtime_is_not_left_for_the_next_call():
    """A device that is not there is refused by the runtime; the next call, on one that is, succeeds."""
    import ctypes as C
    from x_algorithm_b200 import _lib, decoding
    torch = _torch()
    c = Cache([2], [30], 2, 64, 16, seed=1)
    qkv = torch.randn((2, 8 * 64), device=DEV, generator=c.g).to(torch.bfloat16)
    x = torch.randn((2, 100), device=DEV, generator=c.g)
    q = decoding.history_append(qkv, *c.args(), None, num_q_heads=4)
    out, probs = decoding.tree_attention(q, *c.args()), decoding.token_logprobs(x, top_k=3)
    mine, stream, bits = decoding._structs, torch.cuda.current_stream().cuda_stream, C.c_int32()
    status = decoding._kept[(0, stream)].status.data_ptr()
    none = 10 ** 6
    for f, a in ((_lib.lib.phx_history_append_device, (mine.batch_ref, mine.append_ref)), (_lib.lib.phx_tree_attention_device, (mine.batch_ref, mine.tree_ref)),
                 (_lib.lib.phx_token_logprobs_device, (mine.logprobs_ref,)), (_lib.lib.phx_decode_status, (status, stream, C.byref(bits)))):
        assert f(none, *a, *(() if f is _lib.lib.phx_decode_status else (stream,))) == 2   # PHX_E_CUDA
        assert torch.equal(decoding.history_append(qkv, *c.args(), None, num_q_heads=4), q)
    assert _lib.lib.phx_tree_workspace_bytes(none, C.byref(C.c_int64())) == 2
    assert torch.equal(decoding.tree_attention(q, *c.args()), out)
    assert all(torch.equal(a, b) for a, b in zip(decoding.token_logprobs(x, top_k=3)[1:], probs[1:]))
    decoding.check_status()


def test_a_table_that_is_broadcast_over_requests_is_refused():
    from x_algorithm_b200 import PhoenixError, decoding
    torch = _torch()
    c = Cache([1, 1, 1], [20, 20, 20], 2, 64, 16)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros((3, 8 * 64), dtype=torch.bfloat16, device=DEV)
    flat = torch.arange(16, dtype=torch.int32, device=DEV)
    for table in (c.table[:1].expand(3, -1), flat.as_strided((3, 3), (1, 1))):
        for f in (lambda: decoding.tree_attention(q, c.pages, c.q_start, c.lengths, table), lambda: decoding.history_append(qkv, c.pages, c.q_start, c.lengths, table, None, num_q_heads=4)):
            with pytest.raises((ValueError, PhoenixError)):
                f()
    one = Cache([1], [20], 2, 64, 16)                            # one row has no distance to a next
    want = decoding.tree_attention(q[:1], *one.args())
    assert torch.equal(decoding.tree_attention(q[:1], one.pages, one.q_start, one.lengths, one.table.as_strided(one.table.shape, (1, 1))), want)
    decoding.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(6, 300), (6, 1001), (6, 5000), (600, 9001), (1, 66000), (6, 131072)])
def test_token_logprobs_of_a_types_highest_value(dtype, rows, vocab):
    """An id that is forced by the largest number of the type, among ordinary, banned and lowest ones: all finite but what fp32 does not hold."""
    torch = _torch()
    t = getattr(torch, dtype)
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn((rows, vocab), device=DEV, generator=g).to(t)
    high = torch.finfo(t).max
    x[0, vocab // 2] = high
    if rows > 1:
        x[1, torch.rand(vocab, device=DEV, generator=g) < 0.5] = -math.inf
        x[1, vocab - 1] = high
        x[2, :] = high                                          # all of them
        x[3, :] = -math.inf
        x[3, 1] = high
        x[4, 0] = 2.5e38
        x[5, 0], x[5, vocab - 1], x[5, 3] = 1.2e38, -1.2e38, -math.inf
    given = torch.tensor([[0, vocab // 2, vocab - 1]] * rows, device=DEV)
    for temperature in (1.0, 0.5, 2.0):
        _logprobs_check(x, given, min(vocab, 9), temperature=temperature)


@pytest.mark.parametrize("vocab", [300, 5000, 66000])
def test_banned_ids_weigh_nothing_at_any_temperature(vocab):
    torch = _torch()
    x = torch.zeros((2, vocab), device=DEV)
    x[:, ::2] = -math.inf
    x[1, 1] = 3.0
    for temperature in (1e-6, 1e30, 1e37, 3e38):
        _logprobs_check(x, torch.tensor([[0, 1, 3]] * 2, device=DEV), 5, temperature=float(torch.tensor(temperature, dtype=torch.float32)))


@pytest.mark.parametrize("dtype,vocab", [("float32", 100003), ("bfloat16", 100003), ("float32", 1024), ("bfloat16", 1000), ("float32", 300000)])
@pytest.mark.parametrize("late", [False, True])
def test_token_logprobs_of_peaked_rows(dtype, vocab, late):
    """The best id 8.5 above all others, early and late in the row.  With the row's maximum as the reference its own exponential is 1, and log p = -ln Z, Z = 1 + r
    with r at most about 0.5.  Roundings after the 1 has been added, taken as independent, of a half ulp (2^-24) at most and so 2^-24 / sqrt(3) in the mean square: 16 within a
    batch, 74 batches at most (300000 in a cluster of blocks: fewer), 10 in the joins, 2 behind the logarithm: sqrt(102) 2^-24 / sqrt(3) = 3.5e-7, but a 1 that has equal chances to stand
    anywhere sees half of them, 2.5e-7; the exponentials' own 2^-22 on r adds 1e-7 if all were off the same way.  Root mean square at most 3.2e-7."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    rows = 64 if vocab > 2000 else 512
    t = getattr(torch, dtype)
    g = torch.Generator(device=DEV).manual_seed(vocab + late)
    x = torch.randn((rows, vocab), device=DEV, generator=g).to(t)
    at = torch.randint(0, vocab // 4, (rows,), device=DEV, generator=g)
    at = vocab - 1 - at if late else at % 32
    best = (x.float().amax(1) + 8.5).to(t)
    x[torch.arange(rows, device=DEV), at] = best
    lp, _, top, ids = decoding.token_logprobs(x, at, top_k=1)
    assert torch.equal(ids[:, 0], at) and torch.equal(lp, top[:, 0])
    want = _logprobs_want(x, 0.0, 1.0)[0].gather(1, at[:, None])[:, 0]
    off = (lp.double() - want).square().mean().sqrt().item()
    assert off <= 3.2e-7, off


@pytest.mark.parametrize("cap", [1e-3, 1e-5, 1e-20, 1e-38, 1e-41])
@pytest.mark.parametrize("vocab", [300, 5000, 66000])
def test_token_logprobs_of_very_small_caps(cap, vocab):
    torch = _torch()
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn((5, vocab), device=DEV, generator=g)
    x[1] = 0.0
    x[2] *= cap
    x[3, ::3] = 0.0
    x[4, ::2] = -math.inf
    given = torch.tensor([[0, 1, vocab - 1]] * 5, device=DEV)
    cap32 = float(torch.tensor(cap, dtype=torch.float32))
    for k in (0, 5):
        _logprobs_check(x, given, k, cap=cap32)


@pytest.mark.parametrize("method", ["tanh", "soft_sign"])
@pytest.mark.parametrize("cap", [1e-3, 1e-7, 1e-20, 1e-38, 1e-41])
@pytest.mark.parametrize("heads,kv_heads,dh,tokens", [(4, 4, 32, 3), (16, 4, 128, 3), (16, 4, 128, 50), (8, 8, 64, 40)])
def test_tree_attention_with_very_small_caps(method, cap, heads, kv_heads, dh, tokens):
    """Logits that are zero, and others, under a cap that makes them all nearly equal."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([tokens], [200], kv_heads, dh, 16, seed=5)
    q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
    q[0] = 0
    spans = torch.tensor(_spans("tree", tokens, 1, 1), dtype=torch.int32, device=DEV)
    cap = float(torch.tensor(cap, dtype=torch.float32))
    out = decoding.tree_attention(q, *c.args(), spans, cap=cap, cap_method=method)
    decoding.check_status()
    _check(out, *_attend(c, q, spans, math.sqrt(128.0) / dh, cap, method))


@pytest.mark.parametrize("method,cap", [("tanh", 5.0), ("tanh", 30.0), ("tanh", 2000.0), ("soft_sign", 5.0)])
@pytest.mark.parametrize("heads,kv_heads,dh,tokens,cached", [(4, 4, 32, 9, 70), (8, 8, 64, 9, 70), (16, 4, 128, 4, 70), (16, 4, 128, 60, 70), (8, 8, 64, 150, 70), (32, 8, 128, 17, 3000)])
def test_keys_that_are_not_seen_leave_no_trace_under_a_cap(method, cap, heads, kv_heads, dh, tokens, cached):
    """Large keys, NaN and infinities of padding tokens, of another branch and behind the last key: the same bits as without them."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([tokens, tokens], [cached, 3], kv_heads, dh, 32, seed=5)
    q = torch.randn((c.n, heads, dh), device=DEV, generator=c.g).to(torch.bfloat16)
    spans = torch.tensor(_spans("tree", tokens, 2, 1) + _spans("isolated", tokens, 0), dtype=torch.int32, device=DEV)
    run = lambda: decoding.tree_attention(q, *c.args(), spans, cap=cap, cap_method=method)  # noqa: E731
    clean = run()
    _check(clean, *_attend(c, q, spans, math.sqrt(128.0) / dh, cap, method))
    for value in (50.0, 1000.0, math.inf, math.nan):
        for b, (t, k) in enumerate(zip(c.tokens, c.cached)):       # behind the last key
            c.pages[c.table_host[b][(t + k - 1) // 32], :, :, (t + k - 1) % 32 + 1:] = value
        for j in (tokens - 2, tokens - 1):                         # the padding tokens of request 0
            c.pages[c.table_host[0][(cached + j) // 32], :, :, (cached + j) % 32] = value
        assert torch.equal(run(), clean), value
    # candidates that see themselves only: what the key of one holds is its own row's
    at = 3 + tokens // 2
    c.pages[c.table_host[1][at // 32], 0, :, at % 32] *= 40.0
    out = run()
    rest = [i for i in range(c.n) if i != tokens + tokens // 2]
    assert torch.equal(out[rest], clean[rest]) and not torch.equal(out, clean)


@pytest.mark.parametrize("method", ["tanh", "soft_sign"])
@pytest.mark.parametrize("heads,kv_heads,dh,tokens", [(4, 4, 32, 5), (8, 8, 64, 1), (16, 4, 128, 4), (16, 4, 128, 60), (8, 8, 64, 150)])
@pytest.mark.parametrize("scale", [0.3, -0.3, 3.0])
def test_logits_that_reach_their_cap(method, heads, kv_heads, dh, tokens, scale):
    """Logits of up to several times the cap beside small ones, both signs of the scale."""
    _tree_case([tokens, 2], [900, 40], heads, kv_heads, dh, 32, "tree", cap=4.0, method=method, seed=7, scale=scale)


@pytest.mark.parametrize("method", ["tanh", "soft_sign"])
@pytest.mark.parametrize("cap", [1e3, 1e5, 1e7, 1e30, 3e38])
@pytest.mark.parametrize("heads,kv_heads,dh,tokens", [(4, 4, 32, 5), (8, 8, 64, 3), (16, 4, 128, 4), (16, 4, 128, 60), (8, 8, 64, 150)])
def test_caps_far_above_the_logits(method, cap, heads, kv_heads, dh, tokens):
    """As good as no cap: the error does not grow with the cap."""
    _tree_case([tokens, 2], [900, 40], heads, kv_heads, dh, 32, "tree", cap=cap, method=method, seed=11)


def test_a_cap_without_its_method_is_refused():
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([2], [20], 2, 64, 16)
    q = torch.randn((2, 4, 64), device=DEV, generator=c.g).to(torch.bfloat16)
    with pytest.raises(ValueError, match="cap_method"):
        decoding.tree_attention(q, *c.args(), cap=30.0)
    assert torch.equal(decoding.tree_attention(q, *c.args(), cap=0.0, cap_method="tanh"), decoding.tree_attention(q, *c.args()))


def _dropped(torch, shape, dtype):
    """The address of a block that the current stream's pool will hand out next for this size."""
    t = torch.empty(shape, dtype=dtype, device=DEV)
    return t.data_ptr()


def test_results_of_a_named_stream_are_that_streams():
    """stream=: what a call allocates comes from that stream's pool, so neither a block that queued work of the current stream still uses is written, nor a
    result that is dropped early is handed to the current stream."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([300], [500], 2, 64, 16, seed=3)
    qkv = torch.randn((300, 12 * 64), device=DEV, generator=c.g).to(torch.bfloat16)
    x = torch.randn((700, 5000), device=DEV, generator=c.g)
    given = torch.randint(0, 5000, (700, 900), device=DEV, generator=c.g)
    want_q = decoding.history_append(qkv, *c.args(), None, num_q_heads=8)
    want = decoding.tree_attention(want_q, *c.args())
    want_p = decoding.token_logprobs(x, given, top_k=100)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls = [(lambda: [decoding.history_append(qkv, *c.args(), None, num_q_heads=8, stream=side.cuda_stream)], [want_q]),
             (lambda: [decoding.tree_attention(want_q, *c.args(), stream=side.cuda_stream)], [want]),
             (lambda: list(decoding.token_logprobs(x, given, top_k=100, stream=side.cuda_stream)), list(want_p))]
    for f, wants in calls:
        free = [_dropped(torch, w.shape, w.dtype) for w in wants]
        got = f()
        assert not set(free) & {g.data_ptr() for g in got}
        side.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, wants))
        addresses = {g.data_ptr() for g in got}
        del got
        assert not addresses & {torch.empty(w.shape, dtype=w.dtype, device=DEV).data_ptr() for w in wants}
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    decoding.check_status(stream=side.cuda_stream)
    same = decoding.tree_attention(want_q, *c.args(), stream=0)      # the default stream by its number
    assert torch.equal(same, want)


def _all_three(c, qkv, x):
    from x_algorithm_b200 import decoding
    q = decoding.history_append(qkv, *c.args(), None, num_q_heads=16)
    return decoding.tree_attention(q, *c.args()), decoding.token_logprobs(x, top_k=4)[2]


def test_a_capture_on_a_stream_of_its_own():
    """Warmed up on one stream, captured on the graph's own, on which nothing has run before; what a replay reports is found under the stream of the capture."""
    from x_algorithm_b200 import PhoenixError, decoding
    torch = _torch()
    c = Cache([3, 40], [9000, 700], 4, 128, 16, seed=1)
    qkv = torch.randn((c.n, 24 * 128), device=DEV, generator=c.g).to(torch.bfloat16)
    x = torch.randn((3, 9000), device=DEV, generator=c.g)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _all_three(c, qkv, x)
    warm.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.cuda.current_stream().cuda_stream
        out = _all_three(c, qkv, x)
    qkv.copy_(torch.randn(qkv.shape, device=DEV, generator=c.g))
    graph.replay()
    got = [t.clone() for t in out]
    for a, b in zip(got, _all_three(c, qkv, x)):
        assert torch.equal(a, b)
    decoding.check_status()
    decoding.check_status(stream=captured)
    c.table[0, 2] = -1
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(PhoenixError, match="page"):
        decoding.check_status(stream=captured)


def test_the_first_call_on_a_stream_does_not_wait_for_it():
    """Work that is queued on a new stream is still running when the first call returns."""
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([3], [50], 2, 64, 16, seed=1)
    q = torch.randn((3, 4, 64), device=DEV, generator=c.g).to(torch.bfloat16)
    decoding.tree_attention(q, *c.args())
    torch.cuda.synchronize()
    for _ in range(40):                                            # one that has no call behind it
        side = torch.cuda.Stream()
        if (0, side.cuda_stream) not in decoding._kept:
            break
    else:
        pytest.skip("every stream of the pool has been used")
    done = torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                             # about 0.1 s
        done.record()
        decoding.tree_attention(q, *c.args())
        assert not done.query()
    side.synchronize()


def test_graphs_that_are_replayed_beside_each_other_share_no_workspace():
    from x_algorithm_b200 import decoding
    torch = _torch()
    caches = [Cache([3, 40], [9000, 7000], 4, 128, 16, seed=s) for s in (1, 2, 3)]
    q = [torch.randn((c.n, 16, 128), device=DEV, generator=c.g).to(torch.bfloat16) for c in caches]
    want = [decoding.tree_attention(r, *c.args()) for c, r in zip(caches, q)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs, used = [], [], []
    with torch.cuda.stream(side):
        decoding.tree_attention(q[0], *caches[0].args())     # the stream has a workspace of its own
        for c, r in zip(caches, q):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append([decoding.tree_attention(r, *c.args()) for _ in range(4)])
                used.append(decoding._structs.tree.workspace)
            graphs.append(graph)
        used.append(decoding._kept[(0, side.cuda_stream)].workspace.data_ptr())
    assert len(set(used)) == 4
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):
            last = decoding.tree_attention(q[0], *caches[0].args())
    torch.cuda.synchronize()
    assert torch.equal(last, want[0])
    for o, w in zip(outs, want):
        assert all(torch.equal(t, w) for t in o)
    decoding.check_status()


def test_appending_keeps_no_workspace_and_it_can_be_given_back():
    from x_algorithm_b200 import decoding
    torch = _torch()
    c = Cache([3], [50], 2, 64, 16, seed=1)
    qkv = torch.randn((3, 8 * 64), device=DEV, generator=c.g).to(torch.bfloat16)
    side = torch.cuda.Stream()
    decoding.release(stream=side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        before = torch.cuda.memory_allocated()
        q = decoding.history_append(qkv, *c.args(), None, num_q_heads=4)
        assert torch.cuda.memory_allocated() - before < 1 << 20
        out = decoding.tree_attention(q, *c.args())
        assert torch.cuda.memory_allocated() - before > 1 << 20
        decoding.release()
        assert torch.cuda.memory_allocated() - before < 1 << 20
        assert torch.equal(decoding.tree_attention(q, *c.args()), out)
        decoding.check_status()
