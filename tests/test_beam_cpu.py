"""What the beam search decides on the host, with stand-ins for the operators."""
import contextlib

import pytest
import torch

from x_algorithm_b200 import beam, decoding


@pytest.fixture
def host(monkeypatch):
    """The operators in plain torch on the CPU (attention as an average of the queries); what they were called with."""
    seen = dict(gemm=[], status=[], device=[], tables=[])

    def gemm(a, wt, residual=None, epilogue=0, impl=0, device=0):
        seen["gemm"].append(device)
        c = a.float() @ wt.float().T
        c = torch.nn.functional.gelu(c) if epilogue == 2 else c + residual.float() if epilogue == 1 else c
        return c.to(torch.bfloat16), 0.0

    def history_append(qkv, pages, q_start, lengths, table, positions, cos, sin, *, num_q_heads, q_gain, k_gain, eps):
        seen["tables"].append(table.clone())
        return qkv[:, :num_q_heads * pages.shape[-1]].reshape(qkv.shape[0], num_q_heads, -1)

    def token_logprobs(logits, given=None, *, top_k=0, cap=0.0, temperature=1.0):
        lp = torch.log_softmax(logits.float(), -1)
        best, ids = lp.topk(top_k, dim=1)
        return None, None, best, ids

    @contextlib.contextmanager
    def device(index):
        seen["device"].append(index)
        yield

    monkeypatch.setattr(beam, "gemm", gemm)
    monkeypatch.setattr(decoding, "history_append", history_append)
    monkeypatch.setattr(decoding, "tree_attention", lambda q, *a, **k: q)
    monkeypatch.setattr(decoding, "token_logprobs", token_logprobs)
    monkeypatch.setattr(decoding, "check_status", lambda device=None, stream=None: seen["status"].append(device))
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    return seen


def _decoder(**kw):
    cfg = beam.BeamConfig(emb_size=64, num_layers=1, ffn_size=64, vocab=32, **kw)
    return beam.SemanticIdBeam(cfg, beam.make_weights(cfg, device="cpu"), max_users=4, device="cpu")


def test_every_call_goes_to_the_decoders_device(host):
    d = _decoder()
    assert d.index == 2                                      # "cuda" is the current device
    d.index = 3
    d.remember([0, 1], [torch.randn(5, 64).to(torch.bfloat16), torch.randn(2, 64).to(torch.bfloat16)])
    ids, scores = d.search([1, 0], [3, 4], steps=2, beam=3)
    assert ids.shape == (2, 3, 2) and scores.shape == (2, 3)
    assert set(host["gemm"]) == {3} and host["status"] == [3] and host["device"] == [3, 3]


def test_a_user_may_be_named_once_a_call(host):
    d = _decoder()
    row = torch.randn(5, 64).to(torch.bfloat16)
    with pytest.raises(ValueError, match="once"):
        d.remember([1, 1], [row, row])
    assert d.length == [0] * 4 and len(d.free) == d.cfg.num_pages
    d.remember([1], [row])
    with pytest.raises(ValueError, match="once"):
        d.search([1, 1], [3, 4], steps=1, beam=2)
    d.search([1], [3], steps=1, beam=2)


def test_a_pool_that_is_too_small_hands_out_nothing(host):
    d = _decoder(num_pages=4, page_size=16)
    row = torch.randn(40, 64).to(torch.bfloat16)                 # three pages
    with pytest.raises(MemoryError, match="6 pages"):
        d.remember([0, 1], [row, row])
    assert len(d.free) == 4 and d.owned == [[]] * 4 and d.length == [0] * 4
    d.remember([0], [row])
    d.search([0], [3], steps=2, beam=3)
    with pytest.raises(MemoryError):
        d.remember([1], [row])
    assert d.length[1] == 0 and len(d.free) + len(d.owned[0]) == 4
    d.forget(0)
    d.remember([1], [row])
    tables = host["tables"]
    assert all(len(set(t[t >= 0].tolist())) == int((t >= 0).sum()) for t in tables)


def test_what_has_no_position_or_no_candidates_is_refused(host):
    d = _decoder(max_positions=40)
    row = torch.randn(41, 64).to(torch.bfloat16)
    with pytest.raises(ValueError, match="41 positions"):
        d.remember([0], [row])
    assert d.length[0] == 0 and not d.owned[0]
    d.remember([0], [row[:38]])
    with pytest.raises(ValueError, match="41 positions"):
        d.search([0], [3], steps=3, beam=2)
    for beam_size in (0, 33, 129):
        with pytest.raises(ValueError, match="beam"):
            d.search([0], [3], steps=2, beam=beam_size)
    assert d.search([0], [3], steps=2, beam=32)[0].shape == (1, 32, 2)
