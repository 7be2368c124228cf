"""Window attention, key weights and eviction: what is decided on the host - argument blocks, refusals, and the beam search's caches that shrink."""
import contextlib
import ctypes as C

import pytest
import torch

from x_algorithm_b200 import PhoenixError, _lib, beam, decoding


def _cache(**kw):
    c = _lib.CacheBatch(16, 10, 16, 16, 16, 4, 16, 4, 16, 2, 64, 1, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


WINDOW = dict(positions=16, lse_out=16, window=8, sinks=1)
TREE = dict(q=16, q_stride=256, out=16, workspace=256, workspace_bytes=1 << 40, max_keys=64, max_tokens=1, num_q_heads=4, sm_scale=0.1)
WEIGHTS = dict(q=16, q_stride=256, lse=16, weights=16, workspace=256, workspace_bytes=1 << 40, max_keys=64, max_tokens=1, num_q_heads=4, sm_scale=0.1, decay=1.0)
EVICT = dict(weights=16, lengths_out=16, kept_out=16, workspace=256, workspace_bytes=1 << 40, max_keys=64, budget=8, sinks=1, recent=2)


def _window(tree=None, **kw):
    return _lib.lib.phx_window_attention_device, _lib.WindowArgs(attention=_lib.TreeArgs(**{**TREE, **(tree or {})}), **{**WINDOW, **kw})


def _weights(**kw):
    return _lib.lib.phx_key_weights_device, _lib.KeyWeightsArgs(**{**WEIGHTS, **kw})


def _evict(**kw):
    return _lib.lib.phx_evict_device, _lib.EvictArgs(**{**EVICT, **kw})


def test_struct_layouts():
    assert C.sizeof(_lib.WindowArgs) == C.sizeof(_lib.TreeArgs) + 2 * 8 + 2 * 4
    assert C.sizeof(_lib.KeyWeightsArgs) == 9 * 8 + 8 * 4
    assert C.sizeof(_lib.EvictArgs) == 6 * 8 + 4 * 4


def test_argument_blocks_are_filled_field_by_field():
    mine = decoding._Structs()
    decoding._WINDOW(mine.window, 0, *range(1, 18))
    tree = [getattr(mine.window.attention, n) for n, _ in _lib.TreeArgs._fields_]
    assert tree + [getattr(mine.window, n) for n, _ in _lib.WindowArgs._fields_[1:]] == list(range(1, 18))
    decoding._WEIGHTS(mine.weights, 0, *range(1, 18))
    assert [getattr(mine.weights, n) for n, _ in _lib.KeyWeightsArgs._fields_] == list(range(1, 18))
    decoding._EVICT(mine.evict, 0, *range(1, 11))
    assert [getattr(mine.evict, n) for n, _ in _lib.EvictArgs._fields_] == list(range(1, 11))


@pytest.mark.parametrize("wrong", [dict(key_size=48), dict(page_size=8), dict(page_size=40), dict(num_kv_heads=0), dict(batch=-1), dict(status_dev=None),
                                   dict(lengths=None), dict(block_table=None), dict(table_stride=3), dict(pages=8), dict(pages=None), dict(table_cols=2 ** 30),
                                   dict(num_pages=2 ** 40), dict(num_pages=0), dict(batch=70000)])
@pytest.mark.parametrize("call", [_window, _weights, _evict])
def test_a_wrong_cache_is_refused(call, wrong):
    """Before any CUDA call: the addresses are made up."""
    f, a = call()
    assert f(0, C.byref(_cache(**wrong)), C.byref(a), None) == 1
    assert f.__name__.encode() in _lib.lib.phx_global_error()


@pytest.mark.parametrize("call,wrong", [(_window, w) for w in (
    dict(lse_out=None), dict(window=-1), dict(sinks=-1), dict(tree=dict(q=None)), dict(tree=dict(q=2)), dict(tree=dict(out=None)), dict(tree=dict(q_stride=248)),
    dict(tree=dict(num_q_heads=5)), dict(tree=dict(cap_method=3)), dict(tree=dict(sm_scale=float("nan"))), dict(tree=dict(workspace=None)), dict(tree=dict(spans=4)),
    dict(tree=dict(max_tokens=-1)), dict(tree=dict(max_keys=-1)))] + [(_weights, w) for w in (
        dict(q=None), dict(q=2), dict(q_stride=248), dict(q_stride=260), dict(lse=None), dict(weights=None), dict(num_q_heads=5), dict(num_q_heads=0), dict(cap_method=-1),
        dict(sm_scale=float("inf")), dict(cap=float("nan")), dict(decay=float("nan")), dict(decay=float("inf")), dict(window=-1), dict(sinks=-1), dict(spans=4),
        dict(max_tokens=-1), dict(max_keys=-1), dict(workspace=8), dict(workspace=None), dict(workspace_bytes=-1))] + [(_evict, w) for w in (
            dict(weights=None), dict(lengths_out=None), dict(kept_out=None), dict(budget=0), dict(budget=-3), dict(budget=2), dict(sinks=-1), dict(recent=-1), dict(sinks=7),
            dict(max_keys=-1), dict(workspace=None), dict(workspace=8), dict(workspace_bytes=16))])
def test_wrong_arguments_are_refused(call, wrong):
    f, a = call(**wrong)
    assert f(0, C.byref(_cache()), C.byref(a), None) == 1, wrong
    assert f.__name__.encode() in _lib.lib.phx_global_error()


def test_missing_blocks_are_refused_and_empty_batches_are_not():
    for call in (_window, _weights, _evict):
        f, a = call()
        assert f(0, None, None, None) == 1 and f(0, C.byref(_cache()), None, None) == 1 and f(0, None, C.byref(a), None) == 1
        assert f(0, C.byref(_cache(batch=0)), C.byref(a), None) == 0
        if call is not _evict:
            assert f(0, C.byref(_cache(num_tokens=0)), C.byref(a), None) == 0


def test_the_python_calls_refuse_what_is_no_cuda_tensor():
    q, pages, i = torch.zeros((1, 4, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 2, 16, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    w, table = torch.zeros((2, 2, 16)), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: decoding.window_attention(q, pages, i, i[:1], table, window=4), lambda: decoding.key_weights(q, pages, i, i[:1], table, w[0], w),
                 lambda: decoding.evict(w, pages, i[:1], table, budget=4)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for window, sinks in ((0, 0), (-1, 0), (2 ** 31, 0), (4, -1), (4, 2 ** 31)):
        with pytest.raises(ValueError):
            decoding._seen(None, None, window, sinks, 1, 0)
    assert decoding._seen(None, None, None, 0, 1, 0) == (0, 0, 0, 0) and decoding._seen(None, None, 7, 3, 1, 0) == (0, 0, 7, 3)


# ---- the beam search's caches ----------------------------------------------------------------------------------------------------


@pytest.fixture
def host(monkeypatch):
    seen = dict(window=[], weights=[], evict=[], tree=0, positions=[])

    def gemm(a, wt, residual=None, epilogue=0, impl=0, device=0):
        c = a.float() @ wt.float().T
        c = torch.nn.functional.gelu(c) if epilogue == 2 else c + residual.float() if epilogue == 1 else c
        return c.to(torch.bfloat16), 0.0

    def history_append(qkv, pages, q_start, lengths, table, positions, cos, sin, *, num_q_heads, q_gain, k_gain, eps):
        seen["positions"].append(positions.tolist())
        return qkv[:, :num_q_heads * pages.shape[-1]].reshape(qkv.shape[0], num_q_heads, -1)

    def token_logprobs(logits, given=None, *, top_k=0, cap=0.0, temperature=1.0):
        best, ids = torch.log_softmax(logits.float(), -1).topk(top_k, dim=1)
        return None, None, best, ids

    def window_attention(q, pages, q_start, lengths, table, **kw):
        seen["window"].append(kw)
        return q, torch.zeros(q.shape[:2])

    def tree_attention(q, *a, **k):
        seen["tree"] += 1
        return q

    def evict(weights, pages, lengths, table, **kw):
        seen["evict"].append((lengths.tolist(), table.tolist(), kw))

    monkeypatch.setattr(beam, "gemm", gemm)
    for name, f in dict(history_append=history_append, tree_attention=tree_attention, window_attention=window_attention, token_logprobs=token_logprobs, evict=evict,
                        key_weights=lambda *a, **k: seen["weights"].append(k), check_status=lambda *a, **k: None).items():
        monkeypatch.setattr(decoding, name, f)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return seen


def _decoder(**kw):
    cfg = beam.BeamConfig(emb_size=64, num_layers=2, ffn_size=64, vocab=32, page_size=16, num_pages=12, **kw)
    return beam.SemanticIdBeam(cfg, beam.make_weights(cfg, device="cpu"), max_users=4, device="cpu")


def _rows(n):
    return torch.randn(n, 64).to(torch.bfloat16)


def test_a_shrunk_history_keeps_its_positions_and_gives_its_pages_back(host):
    d = _decoder(sinks=2, keep_weights=True)
    d.remember([0, 1], [_rows(70), _rows(20)])
    assert len(host["weights"]) == 2 and host["tree"] == 0 and all(k["window"] is None for k in host["window"])
    free, first = len(d.free), d.owned[0][:3]
    d.shrink([0, 1], budget=40, recent=5)
    assert [e[0] for e in host["evict"]] == [[70], [70]] and host["evict"][0][2] == dict(budget=40, sinks=2, recent=5, max_keys=70)   # user 1 is within the budget
    assert d.length == [40, 20, 0, 0] and d.place == [70, 20, 0, 0] and d.owned[0] == first and len(d.free) == free + 2
    host["positions"].clear()
    d.search([0, 1], [3, 4], steps=2, beam=2)
    assert host["positions"][0] == [70, 20] and host["positions"][2] == [70, 71, 71, 20, 21, 21] and host["tree"] == 4
    d.forget(0)
    assert d.place[0] == 0 and d.length[0] == 0


def test_a_window_takes_places_behind_the_cache(host):
    d = _decoder(window=8, sinks=1)
    d.remember([0], [_rows(30)])
    assert host["window"][0]["positions"] is None and host["window"][0]["window"] == 8 and not host["weights"]
    host["window"].clear()
    d.search([0], [3], steps=2, beam=2)
    assert host["tree"] == 0 and [k["positions"].tolist() for k in host["window"][::2]] == [[30], [30, 31, 31]]


def test_shrinking_needs_weights(host):
    d = _decoder()
    with pytest.raises(ValueError):
        d.shrink([0], budget=4)
    e = _decoder(keep_weights=True)
    with pytest.raises(ValueError):
        e.shrink([1, 1], budget=4)
    e.shrink([0, 1], budget=4)                               # nothing cached
    assert not host["evict"]


@pytest.mark.parametrize("budget", [2 ** 30 + 1, 2 ** 31 - 1])
def test_a_budget_that_a_grid_would_count_past_is_refused(budget):
    f, a = _evict(budget=budget)
    assert f(0, C.byref(_cache()), C.byref(a), None) == 1 and b"2^30" in _lib.lib.phx_global_error()


def test_fading_weights_are_asked_for_without_new_tokens_too():
    """With a decay cached weights change in a call without tokens: what such a call reads has to be there, and its queries need not."""
    f, a = _weights(decay=0.5, q=None, lse=None)
    for wrong in (dict(lengths=None), dict(q_start=None), dict(block_table=None), dict(table_stride=3), dict(pages=8), dict(table_cols=2 ** 30), dict(num_pages=2 ** 40)):
        assert f(0, C.byref(_cache(num_tokens=0, **wrong)), C.byref(a), None) == 1, wrong
        assert b"phx_key_weights_device" in _lib.lib.phx_global_error()
    for kw in (dict(weights=None), dict(decay=float("nan")), dict(max_keys=-1)):
        f, a = _weights(**{"decay": 0.5, **kw})
        assert f(0, C.byref(_cache(num_tokens=0)), C.byref(a), None) == 1, kw
    f, a = _weights(decay=0.5)
    for empty in (dict(batch=0), dict(num_pages=0), dict(table_cols=0)):
        assert f(0, C.byref(_cache(num_tokens=0, **empty)), C.byref(a), None) == 0, empty


# ---- threads ---------------------------------------------------------------------------------------------------------------------


class _OnDevice:
    """A host tensor that says it is on device 0."""
    is_cuda = True

    def __init__(self, t):
        self._t = t

    def __getattr__(self, name):
        return getattr(self._t, name)

    def get_device(self):
        return 0


def _calls_of(kept_args):
    z = lambda *s, dtype=torch.int32: _OnDevice(torch.zeros(s, dtype=dtype))  # noqa: E731
    q, pages, w = z(1, 4, 64, dtype=torch.bfloat16), z(2, 2, 2, 16, 64, dtype=torch.bfloat16), z(2, 2, 16, dtype=torch.float32)
    q_start, lengths, table, lse = z(2), z(1), z(1, 2), z(1, 4, dtype=torch.float32)
    return [lambda: decoding.tree_attention(q, pages, q_start, lengths, table, **kept_args), lambda: decoding.window_attention(q, pages, q_start, lengths, table, window=4, **kept_args),
            lambda: decoding.key_weights(q, pages, q_start, lengths, table, lse, w, **kept_args), lambda: decoding.evict(w, pages, lengths, table, budget=4, **kept_args)]


@pytest.fixture
def launches(monkeypatch):
    """The entry points as functions that take a while: [stream, calls in them, the most at once, workspaces seen] of each stream; `current` is a thread's stream."""
    import threading
    import time
    import types
    seen, guard, current = {}, threading.Lock(), threading.local()

    def entry(device, batch, args, stream):
        with guard:
            s = seen.setdefault(stream, dict(now=0, most=0, calls=0, freed=False))
            s["now"] += 1
            s["calls"] += 1
            s["most"] = max(s["most"], s["now"])
            kept = decoding._kept[(0, stream)]
            had = kept.space
        time.sleep(0.002)
        with guard:
            s["now"] -= 1
            s["freed"] |= kept.space is not had
        return 0

    names = ("phx_tree_attention_device", "phx_window_attention_device", "phx_key_weights_device", "phx_evict_device")
    monkeypatch.setattr(decoding, "lib", types.SimpleNamespace(phx_global_error=lambda: b"", **{n: entry for n in names}))
    monkeypatch.setattr(decoding, "_kept", {})
    monkeypatch.setattr(decoding, "_status_block", lambda device: torch.zeros(4, dtype=torch.int32))
    monkeypatch.setattr(decoding, "_workspace", lambda device: torch.zeros(64, dtype=torch.uint8))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: getattr(current, "stream", 0), raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    return seen, current


def _at_once(current, streams, work):
    import threading
    errors = []

    def body(stream):
        current.stream = stream
        try:
            for _ in range(3):
                for f in work:
                    f()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=body, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("workspace", [False, True])
def test_calls_of_threads_on_one_stream_do_not_interleave(launches, workspace):
    """A call's kernels talk through its workspace, so no other call's launches may come between them, whoever owns it; other streams' may."""
    seen, current = launches
    work = _calls_of(dict(workspace=_OnDevice(torch.zeros(64, dtype=torch.uint8))) if workspace else {})
    _at_once(current, [0, 0, 0, 7], work)
    assert seen[0]["most"] == 1 and seen[7]["most"] == 1 and seen[0]["calls"] == 36 and seen[7]["calls"] == 12


def test_a_workspace_is_not_given_back_under_a_call(launches):
    seen, current = launches
    _at_once(current, [0, 0], _calls_of({}) + [lambda: decoding.release(0, 0)])
    assert not seen[0]["freed"]


def test_a_refused_call_lets_the_next_one_in(launches, monkeypatch):
    monkeypatch.setattr(decoding.lib, "phx_evict_device", lambda *a: 1)
    tree, _, _, evict = _calls_of({})
    with pytest.raises(PhoenixError):
        evict()
    tree()


def test_an_error_is_the_calling_threads():
    """The message of a refused call is still there, and the caller's, after another thread's call was refused."""
    import threading
    first, second, seen = threading.Event(), threading.Event(), {}

    def body(call, mine, other, name):
        f, a = call(**({"budget": 0} if call is _evict else {"window": -1}))
        if other is first:
            first.wait(10)
        f(0, C.byref(_cache()), C.byref(a), None)
        mine.set()
        other.wait(10)
        seen[name] = _lib.lib.phx_global_error()

    threads = [threading.Thread(target=body, args=(_evict, first, second, "evict")), threading.Thread(target=body, args=(_window, second, first, "window"))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert b"phx_evict_device" in seen["evict"] and b"phx_window_attention_device" in seen["window"]
