"""Window attention, key weights and eviction at sizes where another kernel or another cut of the work takes the call: heads of 32 with many rows, more units than blocks, more
heads than SMs.  Checks and tolerances are those of test_gpu_small_cache."""
import pytest

import test_gpu_small_cache as base
import test_gpu_small_cache_edges as edges

pytestmark = pytest.mark.gpu
IDS = edges.IDS

HEADS_OF_32 = [
    # batch, tokens, cached, heads, kv heads, head dim, page, shape, positions
    (2, 17, 40, 4, 4, 32, 16, "chain", None),
    (2, 300, 500, 4, 4, 32, 48, "chain", None),
    (1, 130, 0, 32, 1, 32, 128, "chain", None),
    (3, 70, 300, 12, 4, 32, 32, "tree", "depth"),
    (3, 70, 300, 10, 2, 32, 16, "tree", "spread"),
    (2, 200, 300, 4, 4, 32, 64, "isolated", None),
    (2, 260, 64, 4, 2, 32, 112, "whole", None),
]


@pytest.mark.parametrize("shape", HEADS_OF_32, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (64, 4), (511, 70)])
def test_heads_of_32(shape, window, sinks):
    from x_algorithm_b200.engine import dispatch_counts
    before = dispatch_counts()
    base.test_window_attention_and_key_weights(shape, window, sinks)
    assert dispatch_counts()["key_weights.tcgen05"] > before["key_weights.tcgen05"]


@pytest.mark.parametrize("shape", HEADS_OF_32[1:4], ids=IDS)
@pytest.mark.parametrize("cap,method", [(30.0, "tanh"), (2.0, "tanh"), (4.0, "soft_sign")])
def test_capped_heads_of_32(shape, cap, method):
    base.test_caps(shape, cap, method, 90, 4)


@pytest.mark.parametrize("shape", [
    (2, 70, 500, 4, 4, 32, 16, "chain", None, 100, 3),
    (2, 200, 400, 4, 2, 32, 128, "isolated", None, 130, 1),
    (2, 40, 700, 8, 4, 32, 32, "tree", "depth", 200, 20),
], ids=IDS)
def test_hidden_keys_of_heads_of_32(shape):
    edges.test_what_is_not_seen_leaves_no_trace(shape, 0.0)
    edges.test_what_is_not_seen_leaves_no_trace(shape, 20.0)
    edges.test_odd_values_that_some_rows_see_reach_those_alone(shape)
    edges.test_pages_in_front_of_the_window_may_be_handed_out(shape)


@pytest.mark.parametrize("shape", [
    (60, 200, 150, 8, 8, 64, 32, "chain", None),
    (40, 260, 90, 16, 4, 128, 16, "chain", None),
    (50, 130, 260, 8, 8, 64, 128, "isolated", None),
    (90, 260, 40, 4, 4, 32, 48, "chain", None),
    (70, 60, 100, 24, 8, 128, 64, "tree", "depth"),
], ids=IDS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 3)])
def test_more_units_than_blocks(shape, window, sinks):
    base.test_window_attention_and_key_weights(shape, window, sinks)


@pytest.mark.parametrize("case", [
    # batch, cached, kv heads, head dim, page, budget, sinks, recent
    (40, 60, 8, 128, 48, 16, 0, 7),
    (40, 60, 8, 64, 16, 59, 3, 20),
    (24, 1025, 8, 32, 64, 600, 4, 64),
    (38, 4096, 4, 32, 64, 300, 4, 64),
    (19, 4113, 8, 32, 16, 4100, 0, 0),
], ids=IDS)
@pytest.mark.parametrize("values", ["few", "odd"])
def test_evict_of_more_heads_than_sms(case, values):
    base.test_evict(case, values)
