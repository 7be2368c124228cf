"""Key weights, window attention and eviction in calls that are seldom made: no new token in the whole call, a table that is too short for a request's keys, threads that share a stream.
Checks and tolerances are those of test_gpu_small_cache."""
import pytest
import torch

from test_gpu_small_cache import DEV, close, make_case, plain, plain_weights

pytestmark = pytest.mark.gpu
IDS = lambda s: "-".join(map(str, s))  # noqa: E731


def args_of(c):
    return c["q"], c["pages"], c["q_start"], c["lengths"], c["table"]


@pytest.mark.parametrize("shape", [
    # batch, cached, heads, kv heads, head dim, page
    (3, 300, 16, 4, 64, 32),
    (1, 1, 8, 8, 64, 16),
    (4, 700, 32, 1, 128, 48),
    (2, 90, 4, 4, 32, 16),
], ids=IDS)
@pytest.mark.parametrize("decay", [0.5, 0.0, 1.0])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
def test_weights_fade_without_new_tokens(shape, decay, window, sinks):
    from x_algorithm_b200 import decoding
    batch, cached, heads, kv_heads, dh, page = shape
    c = make_case(batch, 0, cached, heads, kv_heads, dh, page, "chain", seed=81)
    lse = torch.zeros((0, heads), device=DEV)
    want, tol = plain_weights(c, lse, window, sinks, decay=decay)
    for hints in ({}, dict(max_tokens=100, max_keys=1)):
        got = decoding.key_weights(*args_of(c), lse, c["weights"].clone(), window=window, sinks=sinks, decay=decay, **hints)
        close(got, want, tol, f"weights, {hints}")
    decoding.check_status()


@pytest.mark.parametrize("tokens", [2, 60])
def test_weights_fade_alike_beside_a_request_with_tokens(tokens):
    """The weights of a request without tokens are the same in a call of its own."""
    from x_algorithm_b200 import decoding
    c = make_case(2, tokens, 400, 16, 4, 64, 32, "chain", seed=82, ragged=False)
    c["q"], c["n_new"] = c["q"][tokens:], [0, tokens]
    c["q_start"] = torch.tensor([0, 0, tokens], dtype=torch.int32, device=DEV)
    lse = plain(c, None, 0)[1].float()
    want, tol = plain_weights(c, lse, None, 0, decay=0.75)
    both = decoding.key_weights(*args_of(c), lse, c["weights"].clone(), decay=0.75)
    close(both, want, tol, "weights of both")
    alone = decoding.key_weights(c["q"][:0], c["pages"], c["q_start"][:2], c["lengths"][:1], c["table"][:1], lse[:0], c["weights"].clone(), decay=0.75)
    mine = c["table"][0, :-(-400 // c["page"])].long()
    assert torch.equal(alone[mine], both[mine])
    decoding.check_status()


def test_bad_pages_and_lengths_are_reported_without_new_tokens():
    from x_algorithm_b200 import PhoenixError, decoding
    c = make_case(2, 0, 200, 8, 4, 64, 16, "chain", seed=83, ragged=False)
    lse = torch.zeros((0, 8), device=DEV)
    full, tol = plain_weights(c, lse, None, 0, decay=0.5)
    bad = c["table"].clone()
    bad[1, 3] = c["pages"].shape[0]
    got = decoding.key_weights(c["q"], c["pages"], c["q_start"], c["lengths"], bad, lse, c["weights"].clone(), decay=0.5)
    with pytest.raises(PhoenixError):
        decoding.check_status()
    lost = c["table"][1, 3].long()
    full[lost] = c["weights"][lost].double()
    close(got, full, tol, "weights")
    c["lengths"][0] = -1
    decoding.key_weights(*args_of(c), lse, c["weights"].clone(), decay=0.5)
    with pytest.raises(PhoenixError):
        decoding.check_status()


@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("window,sinks", [(100, 0), (100, 4), (None, 0)])
@pytest.mark.parametrize("decay", [1.0, 0.5])
def test_keys_behind_the_table_are_reported_by_the_weights(tokens, window, sinks, decay):
    """A table without columns for a request's last keys: they get no weight, and the call says so, whichever kernel takes it."""
    from x_algorithm_b200 import PhoenixError, decoding
    from x_algorithm_b200.engine import dispatch_counts
    c = make_case(2, tokens, 512, 16, 4, 128, 16, "chain", seed=84, ragged=False, extra_cols=0)
    lse = plain(c, window, sinks)[1].float()
    want, tol = plain_weights(c, lse, window, sinks, decay=decay)
    cols = 512 // 16
    for b in range(2):                                        # pages behind the last column: as they were
        lost = c["table"][b, cols:].long()
        want[lost] = c["weights"][lost].double()
    before = dispatch_counts()["key_weights.tcgen05"]
    got = decoding.key_weights(*args_of(c)[:4], c["table"][:, :cols], lse, c["weights"].clone(), window=window, sinks=sinks, decay=decay, max_tokens=tokens)
    assert (dispatch_counts()["key_weights.tcgen05"] > before) == (tokens == 70)
    with pytest.raises(PhoenixError):
        decoding.check_status()
    close(got, want, tol, "weights")


@pytest.mark.parametrize("tokens", [3, 70])
def test_a_table_without_columns_is_reported_by_the_weights(tokens):
    from x_algorithm_b200 import PhoenixError, decoding
    c = make_case(2, tokens, 0, 16, 4, 64, 16, "chain", seed=85, ragged=False)
    lse, before = torch.zeros((2 * tokens, 16), device=DEV), c["weights"].clone()
    decoding.key_weights(*args_of(c)[:4], c["table"][:, :0], lse, c["weights"], decay=0.5)
    with pytest.raises(PhoenixError):
        decoding.check_status()
    assert torch.equal(c["weights"], before)


@pytest.mark.parametrize("name", ["window_attention", "tree_attention", "key_weights", "evict"])
@pytest.mark.parametrize("tokens", [2, 60])
def test_a_threads_first_call(name, tokens):
    """A thread that has made no CUDA call before has no context; its outputs are there, so that torch makes none for it either."""
    import threading
    from x_algorithm_b200 import decoding
    c = make_case(2, tokens, 300, 16, 4, 64, 32, "chain", seed=95, ragged=False)
    n = 2 * tokens
    out, lse = torch.zeros((n, 16, 64), dtype=torch.bfloat16, device=DEV), torch.zeros((n, 16), device=DEV)
    decoding.window_attention(*args_of(c), window=90, out=out, lse=lse)
    lengths, kept = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros((2, 4, 280), dtype=torch.int32, device=DEV)
    call = dict(window_attention=lambda: decoding.window_attention(*args_of(c), window=90, out=out, lse=lse), tree_attention=lambda: decoding.tree_attention(*args_of(c), out=out),
                key_weights=lambda: decoding.key_weights(*args_of(c), lse, c["weights"], window=90),
                evict=lambda: decoding.evict(c["weights"], c["pages"], c["lengths"], c["table"], budget=280, lengths_out=lengths, kept=kept))[name]
    torch.cuda.synchronize()
    raised = []

    def body():
        try:
            call()
        except Exception as e:  # noqa: BLE001
            raised.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not raised, raised
    decoding.check_status()


@pytest.mark.parametrize("own_stream", [False, True])
def test_threads_that_share_a_stream(own_stream):
    """Calls of several kernels (parts and their join; plan, product and join; select and move) from threads at once, on the default stream and on one of their own, are what they are
    one after the other."""
    import threading
    from x_algorithm_b200 import decoding
    cases = [make_case(*shape, seed=91 + i, ragged=False) for i, shape in enumerate([
        (2, 40, 3000, 16, 2, 64, 64, "chain"), (4, 200, 700, 16, 4, 128, 64, "whole"), (1, 900, 1500, 32, 1, 64, 32, "chain"), (6, 30, 2000, 8, 4, 128, 16, "chain")])]

    def step(c):
        out, lse = decoding.window_attention(*args_of(c), c["spans"], window=1200, sinks=4)
        tree = decoding.tree_attention(*args_of(c), c["spans"])
        weights = decoding.key_weights(*args_of(c), lse, c["weights"].clone(), c["spans"], window=1200, sinks=4, decay=0.9)
        heavy, pages = weights.clone(), c["pages"].clone()
        return out, lse, tree, weights, heavy, pages, *decoding.evict(heavy, pages, c["lengths"], c["table"], budget=600, sinks=4, recent=50)

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    stream, wrong = torch.cuda.Stream() if own_stream else torch.cuda.current_stream(), []

    def body(c, expected):
        try:
            with torch.cuda.stream(stream):
                for _ in range(15):
                    wrong.extend(i for i, (x, y) in enumerate(zip(step(c), expected)) if not torch.equal(x, y))
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=body, args=pair) for pair in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong[:5]
    decoding.check_status(stream=stream.cuda_stream)
