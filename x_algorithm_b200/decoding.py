"""Serving over a cached history: rows enter a paged cache (`history_append`), a tree of new tokens attends to it
(`tree_attention`), logits become log probabilities, entropy and best alternatives (`token_logprobs`).  torch CUDA tensors in
and out, asynchronous on torch's current stream unless `stream` says otherwise; nothing here waits for the GPU but
`check_status`.

The cache is a tensor `pages` bf16 [num_pages, 2 (key, value), kv heads, page size, head dim] that the caller owns and hands out page by
page; `block_table` int32 [B, columns] names a request's pages in order, `lengths` int32 [B] counts its cached keys, and the new tokens of
request b are rows q_start[b] .. q_start[b + 1] - 1 of every token array (int32 [B + 1])."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import PhoenixError, lib

CAP_METHODS = {None: 0, "soft_sign": 1, "tanh": 2}


class _Kept:
    """What one stream of one device keeps between calls: the status block and the attention's workspace."""

    def __init__(self, device: int):
        self.status = torch.zeros(4, dtype=torch.int32, device=f"cuda:{device}")
        need = C.c_int64()
        _ok(lib.phx_tree_workspace_bytes(device, C.byref(need)))
        self.workspace = torch.empty(need.value, dtype=torch.uint8, device=f"cuda:{device}")
        # made on torch's current stream, used on others: both must be there before any of them reads
        torch.cuda.current_stream(device).synchronize()


_kept = {}


def _ok(status: int) -> None:
    if status != 0:
        raise PhoenixError(status, lib.phx_global_error().decode())


def _stream(device: int, stream: Optional[int]) -> int:
    return torch.cuda.current_stream(device).cuda_stream if stream is None else stream


def _keep(device: int, stream: int) -> _Kept:
    kept = _kept.get((device, stream))
    if kept is None:
        kept = _kept[(device, stream)] = _Kept(device)
    return kept


def _is(t, name: str, dtype, ndim: int, device: Optional[torch.device] = None):
    """`t` is a CUDA tensor of this type and rank whose last dimension is dense."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != ndim or not t.is_cuda:
        raise ValueError(f"{name} must be a {ndim}-dimensional {dtype} tensor on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be dense in its last dimension")
    return t


def _dense(t, name: str, dtype, shape, device):
    _is(t, name, dtype, len(shape), device)
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {list(shape)} tensor, got {list(t.shape)}")
    return t


def _batch(pages, q_start, lengths, block_table, tokens: int, kept: _Kept) -> _lib.CacheBatch:
    _is(pages, "pages", torch.bfloat16, 5)
    if pages.shape[1] != 2 or not pages.is_contiguous():
        raise ValueError("pages must be a contiguous [pages, 2, kv heads, page size, head dim] tensor")
    _is(block_table, "block_table", torch.int32, 2, pages.device)
    batch = block_table.shape[0]
    _dense(q_start, "q_start", torch.int32, (batch + 1,), pages.device)
    _dense(lengths, "lengths", torch.int32, (batch,), pages.device)
    return _lib.CacheBatch(pages.data_ptr(), pages.shape[0], q_start.data_ptr(), lengths.data_ptr(), block_table.data_ptr(),
                           max(block_table.stride(0), block_table.shape[1]), kept.status.data_ptr(), block_table.shape[1], pages.shape[3],
                           pages.shape[2], pages.shape[4], batch, tokens)


def rope_tables(num_positions: int, head_dim: int, base: float = 10000.0, device="cuda"):
    """cos and sin fp32 [num_positions, head_dim / 2] of position * base^(-2 i / head_dim) (layers.py:52-60), the angles in 64 bits."""
    i = torch.arange(head_dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * i / head_dim)
    return angle.cos().float(), angle.sin().float()


def tree_spans(parents) -> np.ndarray:
    """int32 [n, 2] (pre, end) of one request's tokens from their parents (host ints: the parent's place among them, -1: hangs on
    the cached history, -2: padding), any order."""
    p = np.ascontiguousarray(parents, dtype=np.int32)
    if p.ndim != 1:
        raise ValueError("parents must be one-dimensional")
    out = np.empty((p.shape[0], 2), np.int32)
    _ok(lib.phx_tree_spans(p.ctypes.data, p.shape[0], out.ctypes.data))
    return out


def history_append(qkv, pages, q_start, lengths, block_table, positions, cos=None, sin=None, *, num_q_heads: int, q_gain=None, k_gain=None,
                   eps: float = 1e-6, out=None, stream: Optional[int] = None):
    """qkv bf16 [N, (num_q_heads + 2 kv heads) * head dim] in the merged order [kv head][queries, key, value] (rows may be apart).  Query and key heads are
    normed (q_gain, k_gain fp32 [head dim]; None: not) and rotated by positions int32 [N] (cos, sin fp32 [positions, head dim / 2];
    None: not); keys and values go to the cache behind `lengths`, the queries come back as bf16 [N, num_q_heads, head dim]."""
    _is(qkv, "qkv", torch.bfloat16, 2)
    device, n = qkv.device, qkv.shape[0]
    stream = _stream(device.index, stream)
    kept = _keep(device.index, stream)
    batch = _batch(pages, q_start, lengths, block_table, n, kept)
    _is(pages, "pages", torch.bfloat16, 5, device)
    dh = batch.key_size
    if qkv.shape[1] != (num_q_heads + 2 * batch.num_kv_heads) * dh:
        raise ValueError(f"qkv rows have {qkv.shape[1]} columns, {(num_q_heads + 2 * batch.num_kv_heads) * dh} are needed")
    if cos is not None or sin is not None:
        _is(cos, "cos", torch.float32, 2, device)
        _dense(cos, "cos", torch.float32, (cos.shape[0], dh // 2), device)
        _dense(sin, "sin", torch.float32, (cos.shape[0], dh // 2), device)
        _dense(positions, "positions", torch.int32, (n,), device)
    for g, name in ((q_gain, "q_gain"), (k_gain, "k_gain")):
        if g is not None:
            _dense(g, name, torch.float32, (dh,), device)
    if out is None:
        out = torch.empty((n, num_q_heads, dh), dtype=torch.bfloat16, device=device)
    else:
        _dense(out, "out", torch.bfloat16, (n, num_q_heads, dh), device)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    args = _lib.AppendArgs(qkv.data_ptr(), qkv.stride(0) if n > 1 else qkv.shape[1], p(positions), p(cos), p(sin), p(q_gain), p(k_gain), out.data_ptr(), num_q_heads,
                           0 if cos is None else cos.shape[0], eps, 0)
    _ok(lib.phx_history_append_device(device.index, C.byref(batch), C.byref(args), stream))
    return out


def tree_attention(q, pages, q_start, lengths, block_table, spans=None, *, sm_scale: Optional[float] = None, cap: float = 0.0,
                   cap_method: Optional[str] = None, max_tokens: Optional[int] = None, max_keys: Optional[int] = None, out=None, workspace=None,
                   stream: Optional[int] = None):
    """q bf16 [N, heads, head dim] (tokens may be apart) attends to the cached keys of its request and to the new ones - appended
    already - that spans int32 [N, 2] lets it see: (pre, end) per token, i sees j where pre[j] <= pre[i] < end[j] (`tree_spans`; None: a
    chain).  sm_scale defaults to sqrt(128) / head dim (scaling.py:46-47).  max_tokens and max_keys: the most new tokens and keys
    (cached + new) of a request, if the caller knows them; they only choose kernels.  workspace: uint8, phx_tree_workspace_bytes; the stream's own if None.
    Returns bf16 [N, heads, head dim]."""
    _is(q, "q", torch.bfloat16, 3)
    n, heads, dh = q.shape
    device = q.device
    stream = _stream(device.index, stream)
    kept = _keep(device.index, stream)
    batch = _batch(pages, q_start, lengths, block_table, n, kept)
    _is(pages, "pages", torch.bfloat16, 5, device)
    if batch.key_size != dh or (heads > 1 and q.stride(1) != dh):
        raise ValueError("q must have the cache's head dim, its heads side by side")
    if cap_method not in CAP_METHODS:
        raise ValueError(f"cap_method must be one of {list(CAP_METHODS)}")
    if spans is not None:
        _dense(spans, "spans", torch.int32, (n, 2), device)
    if out is None:
        out = torch.empty((n, heads, dh), dtype=torch.bfloat16, device=device)
    else:
        _dense(out, "out", torch.bfloat16, (n, heads, dh), device)
    if workspace is None:
        workspace = kept.workspace
    else:
        _is(workspace, "workspace", torch.uint8, 1, device)
    args = _lib.TreeArgs(q.data_ptr(), q.stride(0) if n > 1 else heads * dh, None if spans is None else spans.data_ptr(), out.data_ptr(), workspace.data_ptr(), workspace.numel(),
                         batch.table_cols * batch.page_size if max_keys is None else max_keys, n if max_tokens is None else max_tokens, heads,
                         math.sqrt(128.0) / dh if sm_scale is None else sm_scale, cap, CAP_METHODS[cap_method], 0)
    _ok(lib.phx_tree_attention_device(device.index, C.byref(batch), C.byref(args), stream))
    return out


def token_logprobs(logits, given=None, *, top_k: int = 0, cap: float = 0.0, temperature: float = 1.0, stream: Optional[int] = None):
    """logits fp32 or bf16 [N, vocab] (rows may be apart; -inf: not allowed), given int64 [N, n] or [N] ids (outside the
    vocabulary: none).  Returns (log probabilities of given fp32, of its shape, None without given; entropy fp32 [N]; the top_k best ids' log probabilities fp32
    [N, top_k]; the ids int64 [N, top_k]) of softmax(cap tanh(logits / cap) / temperature), best first, ties by the lower id."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be a float32 or bfloat16 tensor")
    _is(logits, "logits", logits.dtype, 2)
    rows, vocab = logits.shape
    device = logits.device
    if not 0 <= top_k <= vocab:
        raise ValueError(f"top_k must be 0 to vocab ({vocab})")
    given_out = None
    if given is not None:
        _dense(given, "given", torch.int64, (rows,) if given.dim() == 1 else (rows, given.shape[-1]), device)
        given_out = torch.empty(given.shape, dtype=torch.float32, device=device)
    entropy = torch.empty((rows,), dtype=torch.float32, device=device)
    top = torch.empty((rows, top_k), dtype=torch.float32, device=device)
    ids = torch.empty((rows, top_k), dtype=torch.int64, device=device)
    args = _lib.LogprobsArgs(logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, None if given is None else given.data_ptr(), None if given is None else given_out.data_ptr(), entropy.data_ptr(), top.data_ptr(),
                             ids.data_ptr(), rows, vocab, 0 if given is None else given.numel() // max(rows, 1), top_k,
                             int(logits.dtype == torch.bfloat16), cap, temperature, 0)
    _ok(lib.phx_token_logprobs_device(device.index, C.byref(args), _stream(device.index, stream)))
    return given_out, entropy, top, ids


def check_status(device: int = 0, stream: Optional[int] = None) -> None:
    """Waits for the stream and raises PhoenixError if a call on it since the last check met a page, position or offset out of range
    (PHX_E_ARG: what it named was left out) or a bounded wait that ran out (PHX_E_TIMEOUT)."""
    stream = _stream(device, stream)
    kept = _kept.get((device, stream))
    if kept is not None:
        bits = C.c_int32()
        _ok(lib.phx_decode_status(device, kept.status.data_ptr(), stream, C.byref(bits)))
