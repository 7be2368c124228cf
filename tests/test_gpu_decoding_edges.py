"""Calls at the edges of the operators on a cached history.  Oracles and tolerances are test_gpu_decoding's unless a test says its own."""
import pytest

from test_gpu_decoding import DEV, Cache, _torch, _tree_case

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
