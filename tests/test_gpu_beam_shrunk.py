"""Beam search behind a history that was shrunk, and through a window, against plain torch in 64 bits over the cached keys and values themselves.

Tolerance.  From an id to its log probability a token's vector is rounded to bf16 about 18 times (two layers of two norms, merged projection, rotation, attention, out-projection, up, down; the last
norm), each time by 2^-9 / sqrt(3) of its size (root mean square), and nothing in between makes a relative error larger: norms bring every vector back to unit size.  Logits have unit size, so
they are off by sqrt(18) 1.13e-3 = 0.0048, and their own rounding, at sizes of 2 to 4, adds 2^-7 / sqrt(3) = 0.0045: 0.0066 a step, 0.0114 over three (SIGMA).  Errors of that many
independent parts are normal: a sequence may be off by 8 SIGMA, all of a search by 2.5 SIGMA (root mean square)."""
import math

import pytest
import torch

SIGMA = 0.0114


def cached(pages, owned, n):
    """Keys and values [n, kv heads, head dim] of a history's pages."""
    at = torch.arange(n, device=pages.device)
    table, page = torch.tensor(owned, device=pages.device), pages.shape[3]
    return [pages[table[at // page], i, :, at % page] for i in (0, 1)]


def score(cfg, w, caches, place, ids, window=0, sinks=0):
    """log p of ids[1:] behind cached (keys, values) of each layer, float64: the ids are rotated from position `place` on; an id in place n + i of the cache's count sees cached keys and ids in
    front of it that stand behind n + i - window, and the first `sinks`."""
    dh, g, t = cfg.key_size, cfg.num_q_heads // cfg.num_kv_heads, len(ids)
    dev = w["embed"].device
    x = w["embed"][torch.tensor(ids, device=dev)].double()
    pos = place + torch.arange(t, dtype=torch.float64, device=dev)
    ang = pos[:, None] * 10000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64, device=dev) / dh)
    norm = lambda y, gain: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + cfg.rms_eps) * gain.double()  # noqa: E731

    def turn(y):
        a, b = y[..., :dh // 2], y[..., dh // 2:]
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    n = caches[0][0].shape[0]
    i, key = torch.arange(t, device=dev)[:, None], torch.arange(n + t, device=dev)[None]
    sees = key <= n + i
    if window:
        sees = sees & ((key > n + i - window) | (key < sinks))
    for l, (old_k, old_v) in zip(w["layers"], caches):
        qkv = (norm(x, l["pre_attn"]) @ l["qkv"].double().T).view(t, cfg.num_kv_heads, g + 2, dh)
        q, k, v = turn(norm(qkv[:, :, :g].flatten(1, 2), l["q_gain"])), turn(norm(qkv[:, :, g], l["k_gain"])), qkv[:, :, g + 1]
        k, v = (torch.cat([a.double(), b]).repeat_interleave(g, 1) for a, b in ((old_k, k), (old_v, v)))
        s = torch.einsum("qhd,khd->hqk", q, k) * math.sqrt(128.0) / dh
        a = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~sees, -math.inf), -1), v)
        x = x + a.flatten(1) @ l["out"].double().T
        x = x + torch.nn.functional.gelu(norm(x, l["pre_ffn"]) @ l["up"].double().T, approximate="tanh") @ l["down"].double().T
    y = norm(x, w["final"]) @ w["unembed"].double().T
    lp = torch.log_softmax(cfg.logit_cap * torch.tanh(y / cfg.logit_cap), -1)
    return sum(float(lp[j, ids[j + 1]]) for j in range(t - 1))


def agree(scores, want):
    off = (scores.double().cpu() - torch.tensor(want, dtype=torch.float64)).abs()
    assert off.max() <= 8 * SIGMA and off.square().mean().sqrt() <= 2.5 * SIGMA, (off.max().item(), off.square().mean().sqrt().item())


def _history(n, cfg, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, cfg.emb_size), device="cuda", generator=g).to(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 3), (40, 3)])
def test_a_search_behind_a_shrunk_history_is_one_over_the_kept_keys(window, sinks):
    from x_algorithm_b200 import decoding
    from x_algorithm_b200.beam import BeamConfig, SemanticIdBeam, make_weights
    cfg = BeamConfig(vocab=512, keep_weights=True, window=window, sinks=sinks)
    w = make_weights(cfg, seed=14)
    d = SemanticIdBeam(cfg, w, max_users=2)
    d.remember([0, 1], [_history(150, cfg, 15), _history(33, cfg, 16)])
    caches = []                                               # the kept keys and values, gathered from the whole history
    for pages, weights in zip(d.pages, d.weights):
        keys, values = cached(pages, d.owned[0], 150)
        _, kept = decoding.evict(weights.clone(), pages.clone(), torch.tensor([150], dtype=torch.int32, device="cuda"),
                                 torch.tensor([d.owned[0]], dtype=torch.int32, device="cuda"), budget=64, sinks=sinks, recent=10)
        at = kept[0].long().T[..., None].expand(-1, -1, cfg.key_size)
        caches.append((keys.gather(0, at), values.gather(0, at)))
    d.shrink([0], budget=64, recent=10)
    e = SemanticIdBeam(cfg, w, max_users=1)                   # a decoder that holds them from the start
    e.free.reverse()                                          # in other pages
    e._reserve([0], [64])
    e.length[0], e.place[0] = 64, 150
    for pages, (keys, values) in zip(e.pages, caches):
        at = torch.arange(64, device="cuda")
        number = torch.tensor(e.owned[0], device="cuda")[at // cfg.page_size]
        pages[number, 0, :, at % cfg.page_size], pages[number, 1, :, at % cfg.page_size] = keys, values
    ids, scores = d.search([0], [5], steps=3, beam=8)
    same_ids, same = e.search([0], [5], steps=3, beam=8)
    assert torch.equal(ids, same_ids) and torch.equal(scores, same)
    agree(scores[0], [score(cfg, w, caches, 150, [5] + r, window, sinks) for r in ids[0].tolist()])
    both_ids, both = d.search([1, 0], [7, 5], steps=3, beam=8)   # beside a user that was not shrunk
    agree(both[1], [score(cfg, w, caches, 150, [5] + r, window, sinks) for r in both_ids[1].tolist()])
    whole = [cached(p, d.owned[1], 33) for p in d.pages]
    agree(both[0], [score(cfg, w, whole, 33, [7] + r, window, sinks) for r in both_ids[0].tolist()])


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(2, 0), (20, 2), (89, 0), (500, 1), (0, 0)])
def test_scores_through_a_window_are_those_of_its_keys(window, sinks):
    from x_algorithm_b200.beam import BeamConfig, SemanticIdBeam, make_weights
    cfg = BeamConfig(vocab=512, window=window, sinks=sinks)
    w = make_weights(cfg, seed=17)
    d = SemanticIdBeam(cfg, w, max_users=2)
    d.remember([0, 1], [_history(90, cfg, 18), _history(17, cfg, 19)])
    ids, scores = d.search([0, 1], [9, 4], steps=3, beam=8)
    for u, (n, first) in enumerate(((90, 9), (17, 4))):
        caches = [cached(p, d.owned[u], n) for p in d.pages]
        agree(scores[u], [score(cfg, w, caches, n, [first] + r, window, sinks) for r in ids[u].tolist()])
