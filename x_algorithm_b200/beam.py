"""Beam search over semantic ids behind a user's cached history: an example of the operators of `decoding` run together.

A small decoder in the trunk's arithmetic (pre-norm layers, merged QKV, rotation, GELU feed-forward; transformer.py:461-618) keeps the keys and
values of every user's history in one paged cache a layer.  `remember` sends history rows through the layers once, each
seeing the whole history; `search` grows a tree of ids behind it: every step sends the tree's tokens through the layers, appended behind the history
and seeing it and their own branch, and extends the best branches by the best alternatives of the next id.  The projections are the
engine's GEMM call, which waits for the device each time; norms and the choice of branches are plain torch.  (A new token sees all that is cached, so a tree is not
cached level by level: each step sends it whole.)"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List

import torch

from . import decoding
from .engine import gemm


@dataclass
class BeamConfig:
    emb_size: int = 256
    num_layers: int = 2
    num_q_heads: int = 4
    num_kv_heads: int = 2
    key_size: int = 64
    ffn_size: int = 512
    vocab: int = 1024            # semantic ids
    page_size: int = 16
    num_pages: int = 256
    max_positions: int = 4096
    rms_eps: float = 1e-5
    logit_cap: float = 30.0


def make_weights(cfg: BeamConfig, seed: int = 0, device="cuda"):
    """Random weights; matrices bf16 [out, in] as the GEMM reads them."""
    g = torch.Generator(device=device).manual_seed(seed)

    def mat(n, k):
        return (torch.randn((n, k), device=device, generator=g) / math.sqrt(k)).to(torch.bfloat16)

    D, width = cfg.emb_size, (cfg.num_q_heads + 2 * cfg.num_kv_heads) * cfg.key_size
    gain = lambda n: 1 + 0.1 * torch.randn(n, device=device, generator=g)  # noqa: E731
    layers = [dict(pre_attn=gain(D), qkv=mat(width, D), q_gain=gain(cfg.key_size), k_gain=gain(cfg.key_size), out=mat(D, cfg.num_q_heads * cfg.key_size),
                   pre_ffn=gain(D), up=mat(cfg.ffn_size, D), down=mat(D, cfg.ffn_size)) for _ in range(cfg.num_layers)]
    return dict(layers=layers, embed=mat(cfg.vocab, D), final=gain(D), unembed=mat(cfg.vocab, D))


class SemanticIdBeam:
    """Caches and weights of one decoder; users are slots 0 .. max_users - 1."""

    def __init__(self, cfg: BeamConfig, weights, max_users: int, device="cuda"):
        self.cfg, self.w, self.device = cfg, weights, torch.device(device)
        self.index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        shape = (cfg.num_pages, 2, cfg.num_kv_heads, cfg.page_size, cfg.key_size)
        self.pages = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(cfg.num_layers)]
        self.cos, self.sin = decoding.rope_tables(cfg.max_positions, cfg.key_size, device=device)
        self.free = list(range(cfg.num_pages))
        self.owned: List[List[int]] = [[] for _ in range(max_users)]
        self.length = [0] * max_users

    @staticmethod
    def _distinct(users: List[int]):
        """Two rows of one call for the same user would write the same places of its pages."""
        if len(set(users)) != len(users):
            raise ValueError("a user may be named once a call")

    def _placed(self, positions: int):
        if positions > self.cfg.max_positions:
            raise ValueError(f"{positions} positions are needed, the rotation has {self.cfg.max_positions}")

    def _reserve(self, users: List[int], keys: List[int]):
        """Pages for so many keys of each user: all that are missing, or none and an error."""
        more = [max(0, -(-k // self.cfg.page_size) - len(self.owned[u])) for u, k in zip(users, keys)]
        if sum(more) > len(self.free):
            raise MemoryError(f"{sum(more)} pages are needed, {len(self.free)} are free: forget a user, or make the pool larger")
        for u, n in zip(users, more):
            self.owned[u] += [self.free.pop() for _ in range(n)]

    def _gemm(self, a, wt, residual=None, epilogue=0):
        return gemm(a, wt, residual, epilogue=epilogue, device=self.index)[0]

    def _norm(self, x, gain):
        x = x.float()
        return (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.cfg.rms_eps) * gain).to(torch.bfloat16)

    def _layers(self, x, users: List[int], counts: List[int], positions, spans):
        """Token rows x bf16 [N, D] of the users, counts[i] each, behind what their caches hold; appends their keys, returns the rows."""
        cfg = self.cfg
        self._reserve(users, [self.length[u] + n for u, n in zip(users, counts)])
        cols = max(len(self.owned[u]) for u in users)
        dev = dict(dtype=torch.int32, device=self.device)
        table = torch.tensor([self.owned[u] + [-1] * (cols - len(self.owned[u])) for u in users], **dev)
        lengths = torch.tensor([self.length[u] for u in users], **dev)
        q_start = torch.tensor([0] + counts, **dev).cumsum(0).to(torch.int32)
        most = dict(max_tokens=max(counts), max_keys=max(self.length[u] + n for u, n in zip(users, counts)))
        for w, pages in zip(self.w["layers"], self.pages):
            qkv = self._gemm(self._norm(x, w["pre_attn"]), w["qkv"])
            q = decoding.history_append(qkv, pages, q_start, lengths, table, positions, self.cos, self.sin, num_q_heads=cfg.num_q_heads,
                                        q_gain=w["q_gain"], k_gain=w["k_gain"], eps=cfg.rms_eps)
            a = decoding.tree_attention(q, pages, q_start, lengths, table, spans, **most)
            x = self._gemm(a.view(a.shape[0], -1), w["out"], x, epilogue=1)
            h = self._gemm(self._norm(x, w["pre_ffn"]), w["up"], epilogue=2)
            x = self._gemm(h, w["down"], x, epilogue=1)
        return x

    def remember(self, users: List[int], rows: List[torch.Tensor]):
        """History rows bf16 [n, D] of each user join the cache (a user's first: its rows see each other, none comes later than its history)."""
        counts = [r.shape[0] for r in rows]
        self._distinct(users)
        for u in users:
            if self.length[u]:
                raise ValueError(f"user {u} has a history already: forget it first")
        self._placed(max(counts, default=0))
        positions = torch.cat([torch.arange(n, dtype=torch.int32, device=self.device) for n in counts])
        spans = torch.tensor([[0, 1]], dtype=torch.int32, device=self.device).repeat(sum(counts), 1)
        with torch.cuda.device(self.index):
            self._layers(torch.cat(rows), users, counts, positions, spans)
        for u, n in zip(users, counts):
            self.length[u] = n

    def forget(self, user: int):
        self.free += self.owned[user]
        self.owned[user], self.length[user] = [], 0

    def search(self, users: List[int], first_ids: List[int], steps: int, beam: int):
        """The `beam` best continuations of `steps` ids behind each user's history and first id: (ids int64 [users, beam, steps],
        log probabilities fp32 [users, beam])."""
        self._distinct(users)
        if not 1 <= beam <= min(self.cfg.vocab, 128):
            raise ValueError("beam must be 1 to the vocabulary, at most 128")
        self._placed(max((self.length[u] for u in users), default=0) + steps)
        with torch.cuda.device(self.index):
            return self._search(users, first_ids, steps, beam)

    def _search(self, users, first_ids, steps, beam):
        cfg, count = self.cfg, len(users)
        # a user's tree: ids, parents (-1: behind the history), depth of each token; leaves of the last level and their scores
        ids, parents, depth = [[f] for f in first_ids], [[-1] for _ in users], [[0] for _ in users]
        leaves, scores = [[0] for _ in users], torch.zeros((count, 1), device=self.device)
        for step in range(steps):
            counts = [len(t) for t in ids]
            spans = torch.cat([torch.from_numpy(decoding.tree_spans(p)) for p in parents]).to(self.device)
            positions = torch.tensor([self.length[u] + d for u, ds in zip(users, depth) for d in ds], dtype=torch.int32, device=self.device)
            x = self.w["embed"][torch.tensor([i for t in ids for i in t], device=self.device)]
            x = self._layers(x, users, counts, positions, spans)
            starts = [sum(counts[:i]) for i in range(count)]
            last = torch.tensor([s + leaf for s, ls in zip(starts, leaves) for leaf in ls], device=self.device)
            logits = self._gemm(self._norm(x[last], self.w["final"]), self.w["unembed"])
            width = len(leaves[0])
            _, _, best, best_ids = decoding.token_logprobs(logits, top_k=min(beam, cfg.vocab), cap=cfg.logit_cap)
            total = scores[:, :, None] + best.view(count, width, -1)
            scores, at = total.view(count, -1).topk(beam, dim=1)
            chosen, leaf_of = best_ids.view(count, -1).gather(1, at).tolist(), (at // total.shape[2]).tolist()
            for u in range(count):
                first_new = len(ids[u])
                for i, leaf in zip(chosen[u], leaf_of[u]):
                    parent = leaves[u][leaf]
                    ids[u].append(i); parents[u].append(parent); depth[u].append(step + 1)
                leaves[u] = list(range(first_new, first_new + beam))
        decoding.check_status(self.index)
        paths = []
        for u in range(count):
            rows = []
            for leaf in leaves[u]:
                path = []
                while parents[u][leaf] >= 0:
                    path.append(ids[u][leaf])
                    leaf = parents[u][leaf]
                rows.append(path[::-1])
            paths.append(rows)
        return torch.tensor(paths), scores


def main():
    cfg = BeamConfig()
    weights = make_weights(cfg)
    decoder = SemanticIdBeam(cfg, weights, max_users=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    histories = [torch.randn((n, cfg.emb_size), device="cuda", generator=g).to(torch.bfloat16) for n in (200, 37, 1)]
    decoder.remember([0, 1, 2], histories)
    ids, scores = decoder.search([0, 1, 2], [1, 2, 3], steps=3, beam=8)
    for u in range(3):
        print("user %d: best ids %s, log probability %.3f" % (u, ids[u, 0].tolist(), scores[u, 0].item()))


if __name__ == "__main__":
    main()
