"""Beam search behind a cached history against plain torch in 64 bits without a cache: every sequence that the search returns
is sent through the same layers by itself, with its whole history, and has to get the log probability that the search gave it.

Tolerance: a layer rounds its activations to bf16 about ten times (u = 2^-8 each), two layers and the logits make log probabilities of size 5 off by a
few u times the logits' own size (about 1): 20 u."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _plain(cfg, w, history, ids):
    """log p of ids[1:] given ids[0] and the history, float64"""
    import torch
    D, dh, g = cfg.emb_size, cfg.key_size, cfg.num_q_heads // cfg.num_kv_heads
    n, t = history.shape[0], len(ids)
    x = torch.cat([history.double(), w["embed"][torch.tensor(ids, device="cuda")].double()])
    sees = torch.zeros((n + t, n + t), dtype=torch.bool, device="cuda")
    sees[:, :n] = True
    sees[n:, n:] = torch.ones((t, t), dtype=torch.bool, device="cuda").tril()
    pos = torch.arange(n + t, dtype=torch.float64, device="cuda")
    ang = pos[:, None] * 10000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64, device="cuda") / dh)
    norm = lambda y, gain, eps=cfg.rms_eps: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * gain.double()  # noqa: E731

    def turn(y):
        a, b = y[..., :dh // 2], y[..., dh // 2:]
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    for l in w["layers"]:
        qkv = (norm(x, l["pre_attn"]) @ l["qkv"].double().T).view(n + t, cfg.num_kv_heads, g + 2, dh)
        q, k, v = turn(norm(qkv[:, :, :g].flatten(1, 2), l["q_gain"])), turn(norm(qkv[:, :, g], l["k_gain"])), qkv[:, :, g + 1]
        s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * math.sqrt(128.0) / dh
        a = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~sees, -math.inf), -1), v.repeat_interleave(g, 1))
        x = x + a.flatten(1) @ l["out"].double().T
        x = x + torch.nn.functional.gelu(norm(x, l["pre_ffn"]) @ l["up"].double().T, approximate="tanh") @ l["down"].double().T
    y = norm(x[n:], w["final"]) @ w["unembed"].double().T
    lp = torch.log_softmax(cfg.logit_cap * torch.tanh(y / cfg.logit_cap), -1)
    return sum(float(lp[i, ids[i + 1]]) for i in range(t - 1))


def test_beam_search_scores_are_those_of_its_sequences():
    import torch
    from x_algorithm_b200.beam import BeamConfig, SemanticIdBeam, make_weights
    cfg = BeamConfig(vocab=512)
    w = make_weights(cfg, seed=2)
    g = torch.Generator(device="cuda").manual_seed(3)
    histories = [torch.randn((n, cfg.emb_size), device="cuda", generator=g).to(torch.bfloat16) for n in (130, 1, 47)]
    d = SemanticIdBeam(cfg, w, max_users=4)
    d.remember([2, 0, 3], histories)
    ids, scores = d.search([2, 0, 3], [5, 6, 7], steps=3, beam=6)
    assert ids.shape == (3, 6, 3) and scores.shape == (3, 6)
    for u in range(3):
        rows = [tuple(r) for r in ids[u].tolist()]
        assert len(set(rows)) == 6 and scores[u].tolist() == sorted(scores[u].tolist(), reverse=True)
        for i in (0, 3, 5):
            want = _plain(cfg, w, histories[u], [5 + u] + list(rows[i]))
            assert abs(float(scores[u, i]) - want) <= 20 / 256 * 3, (float(scores[u, i]), want)
    again, same = d.search([2, 0, 3], [5, 6, 7], steps=3, beam=6)     # the search left the histories as they were
    assert torch.equal(ids, again) and torch.equal(scores, same)
    d.forget(2)
    d.remember([2], [histories[1]])
    assert torch.equal(d.search([2], [6], steps=2, beam=3)[0], d.search([0], [6], steps=2, beam=3)[0])
