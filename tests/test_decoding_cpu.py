"""What the operators on a paged cache decide on the host: spans of a tree, refusals of the C entry points."""
import ctypes as C

import numpy as np
import pytest

from x_algorithm_b200 import PhoenixError, _lib


def _ancestors(parents):
    n = len(parents)
    see = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0 and parents[i] != -2:
            see[i, j] = True
            j = parents[j]
    return see


@pytest.mark.parametrize("n", [0, 1, 2, 7, 40, 300])
@pytest.mark.parametrize("roots", [0.0, 0.3, 1.0])
def test_tree_spans_are_the_ancestors(n, roots):
    from x_algorithm_b200.decoding import tree_spans
    rng = np.random.default_rng(n)
    for _ in range(5):
        grown = [-1 if i == 0 or rng.random() < roots else int(rng.integers(0, i)) for i in range(n)]
        at = rng.permutation(n)
        parents = np.full(n, -1, np.int64)
        for i, p in enumerate(grown):
            parents[at[i]] = -1 if p < 0 else at[p]
        for i in range(n):                                   # leaves may be padding
            if i not in parents and rng.random() < 0.1:
                parents[i] = -2
        s = tree_spans(parents)
        see = (s[None, :, 0] <= s[:, None, 0]) & (s[:, None, 0] < s[None, :, 1])
        np.testing.assert_array_equal(see, _ancestors(parents))


def test_tree_spans_refuse_what_is_no_forest():
    from x_algorithm_b200.decoding import tree_spans
    for parents in ([0], [1, 0], [3, -1], [-3], [1, 2, 0], [-1, 5], [-2, 0]):
        with pytest.raises(PhoenixError) as e:
            tree_spans(parents)
        assert e.value.status == 1
    with pytest.raises(ValueError):
        tree_spans([[0]])


def _cache(**kw):
    c = _lib.CacheBatch(16, 10, 16, 16, 16, 4, 16, 4, 16, 2, 64, 1, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_struct_layouts():
    assert C.sizeof(_lib.CacheBatch) == 7 * 8 + 6 * 4
    assert C.sizeof(_lib.AppendArgs) == 8 * 8 + 4 * 4
    assert C.sizeof(_lib.TreeArgs) == 7 * 8 + 6 * 4
    assert C.sizeof(_lib.LogprobsArgs) == 7 * 8 + 8 * 4


def test_argument_blocks_are_filled_field_by_field():
    from x_algorithm_b200 import decoding
    mine = decoding._Structs()
    decoding._BATCH(mine.batch, 0, *range(1, 14))
    assert [getattr(mine.batch, n) for n, _ in _lib.CacheBatch._fields_] == list(range(1, 14))
    decoding._APPEND(mine.append, 0, *range(1, 13))
    assert [getattr(mine.append, n) for n, _ in _lib.AppendArgs._fields_] == list(range(1, 13))
    decoding._TREE(mine.tree, 0, *range(1, 14))
    assert [getattr(mine.tree, n) for n, _ in _lib.TreeArgs._fields_] == list(range(1, 14))
    decoding._LOGPROBS(mine.logprobs, 0, *range(1, 16))
    assert [getattr(mine.logprobs, n) for n, _ in _lib.LogprobsArgs._fields_] == list(range(1, 16))


@pytest.mark.parametrize("wrong", [dict(key_size=48), dict(page_size=8), dict(page_size=40), dict(num_kv_heads=0), dict(batch=-1), dict(status_dev=None),
                                   dict(q_start=None), dict(lengths=None), dict(block_table=None), dict(table_stride=3), dict(pages=8), dict(pages=None),
                                   dict(table_cols=2 ** 30), dict(num_pages=2 ** 40), dict(num_tokens=-1)])
def test_entry_points_refuse_a_wrong_cache(wrong):
    """Refused before any CUDA call: the addresses are made up."""
    c = _cache(**wrong)
    a = _lib.AppendArgs(16, 512, 16, None, None, None, None, 16, 4, 0, 1e-6, 0)
    t = _lib.TreeArgs(16, 256, None, 16, 16, 1 << 30, 64, 1, 4, 0.1, 0.0, 0, 0)
    assert _lib.lib.phx_history_append_device(0, C.byref(c), C.byref(a), None) == 1
    assert b"phx_history_append_device" in _lib.lib.phx_global_error()
    assert _lib.lib.phx_tree_attention_device(0, C.byref(c), C.byref(t), None) == 1
    assert b"phx_tree_attention_device" in _lib.lib.phx_global_error()


def test_entry_points_refuse_wrong_arguments():
    c = _cache()
    append = dict(qkv=16, qkv_stride=512, positions=16, num_q_heads=4, q_out=16, eps=1e-6)
    for wrong in (dict(qkv=None), dict(qkv=24), dict(qkv_stride=504), dict(qkv_stride=516), dict(num_q_heads=3), dict(num_q_heads=0), dict(q_out=None),
                  dict(cos_tab=16), dict(cos_tab=16, sin_tab=16, num_positions=0), dict(cos_tab=16, sin_tab=20, num_positions=4),
                  dict(cos_tab=16, sin_tab=16, num_positions=4, positions=None), dict(q_gain=16), dict(q_gain=16, k_gain=8), dict(q_gain=16, k_gain=16, eps=-1.0)):
        a = _lib.AppendArgs(**{**append, **wrong})
        assert _lib.lib.phx_history_append_device(0, C.byref(c), C.byref(a), None) == 1, wrong
    tree = dict(q=16, q_stride=256, out=16, workspace=256, workspace_bytes=1 << 40, max_keys=64, max_tokens=1, num_q_heads=4, sm_scale=0.1)
    for wrong in (dict(q=None), dict(q=2), dict(out=None), dict(out=8), dict(q_stride=248), dict(q_stride=260), dict(num_q_heads=5), dict(cap_method=3),
                  dict(sm_scale=float("nan")), dict(cap=float("nan")), dict(workspace=None), dict(workspace=8), dict(spans=4), dict(max_tokens=-1), dict(max_keys=-1)):
        a = _lib.TreeArgs(**{**tree, **wrong})
        assert _lib.lib.phx_tree_attention_device(0, C.byref(c), C.byref(a), None) == 1, wrong
    logp = dict(logits=16, stride=100, given=16, given_out=16, entropy_out=16, top_out=16, top_ids_out=16, rows=1, vocab=100, num_given=1, top_k=5, temperature=1.0)
    for wrong in (dict(logits=None), dict(logits=2), dict(stride=99), dict(given=None), dict(rows=-1), dict(vocab=0), dict(num_given=-1), dict(top_k=129),
                  dict(top_k=101), dict(top_k=-1), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
                  dict(cap=float("nan")), dict(is_bf16=2)):
        a = _lib.LogprobsArgs(**{**logp, **wrong})
        assert _lib.lib.phx_token_logprobs_device(0, C.byref(a), None) == 1, wrong
    for f in (_lib.lib.phx_history_append_device, _lib.lib.phx_tree_attention_device):
        assert f(0, None, None, None) == 1 and f(0, C.byref(c), None, None) == 1
    assert _lib.lib.phx_token_logprobs_device(0, None, None) == 1
    assert _lib.lib.phx_decode_status(0, None, None, None) == 1 and _lib.lib.phx_tree_workspace_bytes(0, None) == 1


def test_the_rows_of_a_block_table_keep_their_distance():
    """A table that is broadcast over requests reaches the entry point with its stride of 0, which refuses it; one row has no distance to a next."""
    import torch
    from types import SimpleNamespace as Fake
    from x_algorithm_b200 import decoding

    def on_gpu(t):
        return Fake(shape=t.shape, dtype=t.dtype, stride=t.stride, is_contiguous=t.is_contiguous, get_device=lambda: 0, data_ptr=lambda: 16)

    pages = on_gpu(torch.zeros((4, 2, 2, 16, 64), dtype=torch.bfloat16))
    kept, flat = Fake(status_ptr=16), torch.zeros(40, dtype=torch.int32)
    for table, stride in ((flat.view(4, 10), 10), (flat[:10].expand(4, 10), 0), (flat.as_strided((4, 10), (3, 1)), 3), (flat.as_strided((4, 5), (10, 1)), 10), (flat.as_strided((1, 10), (1, 1)), 10)):
        n, mine = table.shape[0], decoding._Structs()
        decoding._batch(mine.batch, pages, on_gpu(torch.zeros(n + 1, dtype=torch.int32)), on_gpu(torch.zeros(n, dtype=torch.int32)), on_gpu(table), n, 0, kept)
        assert mine.batch.table_stride == stride and mine.batch.table_cols == table.shape[1]
        if stride < table.shape[1]:
            a = _lib.AppendArgs(16, 512, 16, None, None, None, None, 16, 4, 0, 1e-6, 0)
            assert _lib.lib.phx_history_append_device(0, mine.batch_ref, C.byref(a), None) == 1 and b"table_cols apart" in _lib.lib.phx_global_error()


def test_check_status_asks_the_current_device(monkeypatch):
    import torch
    from types import SimpleNamespace as Fake
    from x_algorithm_b200 import decoding
    asked = []

    def decode_status(device, status, stream, bits):
        asked.append((device, status, stream))
        return 0

    monkeypatch.setattr(decoding, "lib", Fake(phx_decode_status=decode_status))
    monkeypatch.setattr(decoding, "_kept", {(d, 70 + d): Fake(status=Fake(data_ptr=lambda d=d: 100 + d)) for d in (0, 1)})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 70 + d, raising=False)
    decoding.check_status()
    decoding.check_status(0)
    decoding.check_status(device=0, stream=70)
    assert asked == [(1, 101, 71), (0, 100, 70), (0, 100, 70)]


def test_threads_that_meet_on_a_stream_keep_one_block(monkeypatch):
    """Both make the first call on a stream at once: one status block and one workspace, not one each."""
    import threading
    import time
    from x_algorithm_b200 import decoding

    class Slow:
        made = 0

        def __init__(self, *_):
            Slow.made += 1
            time.sleep(0.05)

    monkeypatch.setattr(decoding, "_Kept", Slow)
    monkeypatch.setattr(decoding, "_kept", {})
    got, start = [], threading.Barrier(4)

    def first():
        start.wait()
        got.append(decoding._keep(0, 5))

    threads = [threading.Thread(target=first) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert Slow.made == 1 and len({id(k) for k in got}) == 1 and len(got) == 4


def test_parents_are_integers_and_keep_all_their_bits():
    from x_algorithm_b200.decoding import tree_spans
    for parents in (np.array([-1, 2 ** 32]), np.array([-1, 2 ** 32 - 2]), np.array([2 ** 64 - 1, 0], np.uint64), [-1, 2 ** 40]):
        with pytest.raises(PhoenixError) as e:
            tree_spans(parents)
        assert e.value.status == 1
    for parents in ([-1, 0.5], np.array([-1.0, 0.0])):
        with pytest.raises(ValueError):
            tree_spans(parents)
    np.testing.assert_array_equal(tree_spans(np.array([-1, 0], np.int8)), [[0, 2], [1, 2]])
    assert tree_spans([]).shape == (0, 2)
