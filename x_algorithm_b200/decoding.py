"""Serving over a cached history: rows enter a paged cache (`history_append`), a tree of new tokens attends to it
(`tree_attention`), logits become log probabilities, entropy and best alternatives (`token_logprobs`).  torch CUDA tensors in
and out, asynchronous on torch's current stream; nothing here waits for what is queued but `check_status`.  `stream`, a raw handle, names another
as `with torch.cuda.stream(...)` around the call would: what the call allocates is that stream's, and what it reads has to be there and stay until it
has run.

The cache is a tensor `pages` bf16 [num_pages, 2 (key, value), kv heads, page size, head dim] that the caller owns and hands out page by
page; `block_table` int32 [B, columns] names a request's pages in order, `lengths` int32 [B] counts its cached keys, and the new tokens of
request b are rows q_start[b] .. q_start[b + 1] - 1 of every token array (int32 [B + 1])."""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import PhoenixError, lib

STATUS_BLOCKS = 1024                # cleared at a time, one a stream
CAP_METHODS = {None: 0, "soft_sign": 1, "tanh": 2}


class _Kept:
    """What one stream of one device keeps between calls: the status block and, from its first attention on, that one's workspace."""

    def __init__(self, device: int):
        self.status = _status_block(device)
        self.status_ptr, self.workspace, self.space = self.status.data_ptr(), None, None


def _take_space(kept, device: int):
    with _kept_lock:
        if kept.space is None:
            kept.workspace = _workspace(device)
            kept.space = kept.workspace.data_ptr(), kept.workspace.numel()
        return kept.space


def _workspace(device: int):
    need = C.c_int64()
    _ok(lib.phx_tree_workspace_bytes(device, C.byref(need)))
    return torch.empty(need.value, dtype=torch.uint8, device=f"cuda:{device}")


_kept, _kept_lock = {}, threading.Lock()
_cleared = {}                       # device -> status blocks that no stream has yet


def _status_block(device: int):
    """A status block of zeros.  They are cleared many at a time, on a stream of its own whose work is waited for: neither the caller's queue is, nor is
    the clearing recorded where the caller is capturing a graph."""
    blocks = _cleared.setdefault(device, [])
    if not blocks:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call on a device must not be captured: make one before")
        side = torch.cuda.Stream(device, priority=-1)
        with torch.cuda.stream(side):
            blocks.extend(torch.zeros((STATUS_BLOCKS, 4), dtype=torch.int32, device=f"cuda:{device}").unbind(0))
        side.synchronize()
    return blocks.pop()


class _Structs(threading.local):
    """One set of argument blocks a thread, filled anew for every call: a call costs the host less than its launch."""

    def __init__(self):
        self.batch, self.append, self.tree, self.logprobs = _lib.CacheBatch(), _lib.AppendArgs(), _lib.TreeArgs(), _lib.LogprobsArgs()
        self.batch_ref, self.append_ref, self.tree_ref, self.logprobs_ref = (C.byref(x) for x in (self.batch, self.append, self.tree, self.logprobs))


_structs = _Structs()
_BATCH, _APPEND, _TREE, _LOGPROBS = (struct.Struct(f).pack_into for f in ("=7q6i", "=8q2ifi", "=7q2i2f2i", "=7q5i2fi"))   # the blocks' fields, in order
_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


def _ok(status: int) -> None:
    if status != 0:
        raise PhoenixError(status, lib.phx_global_error().decode())


def _stream(device: int, stream: Optional[int]) -> int:
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream


def _elsewhere(device: int, stream: Optional[int]) -> bool:
    """Whether `stream` is another than torch's current one.  A call for it runs under it: outputs from the current stream's pool could still be in
    use by work that is queued there, or be handed out again there while the call writes them."""
    return stream is not None and stream != torch._C._cuda_getCurrentRawStream(device)


def _under(device: int, stream: int):
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def _keep(device: int, stream: int) -> _Kept:
    kept = _kept.get((device, stream))
    if kept is None:
        with _kept_lock:                                     # made once: what a second one held would be lost, or freed under a kernel
            kept = _kept.get((device, stream))
            if kept is None:
                kept = _kept[(device, stream)] = _Kept(device)
    return kept


def _need(t, name: str, dtype, shape, device):
    """`t` is a contiguous tensor of this type and shape on this device."""
    try:
        if t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    raise ValueError(f"{name} must be a contiguous {list(shape)} {dtype} tensor on cuda:{device}")


def _rows(t, name: str, dtype, ndim: int):
    """The device of `t`, a CUDA tensor of this type and rank whose last dimension is dense."""
    try:
        if t.dtype is dtype and t.is_cuda:
            shape, stride = t.shape, t.stride()
            if len(shape) == ndim:
                if stride[-1] == 1 or shape[-1] < 2:
                    return t.get_device()
                raise ValueError(f"{name} must be dense in its last dimension")
    except AttributeError:
        pass
    raise ValueError(f"{name} must be a {ndim}-dimensional {dtype} tensor on a CUDA device")


def _batch(block, pages, q_start, lengths, block_table, tokens: int, device: int, kept: _Kept):
    """Fills the cache's block; (kv heads, page size, head dim, table columns)."""
    try:
        num_pages, two, kv_heads, page_size, dh = pages.shape
        batch, cols = block_table.shape
        good = (pages.dtype is _BF16 and pages.get_device() == device and pages.is_contiguous() and two == 2 and
                block_table.dtype is _I32 and block_table.get_device() == device and (cols < 2 or block_table.stride(1) == 1) and
                q_start.dtype is _I32 and q_start.get_device() == device and q_start.shape == (batch + 1,) and q_start.is_contiguous() and
                lengths.dtype is _I32 and lengths.get_device() == device and lengths.shape == (batch,) and lengths.is_contiguous())
    except (AttributeError, ValueError, TypeError):
        good = False
    if not good:                                             # say which
        if _rows(pages, "pages", _BF16, 5) != device or _rows(block_table, "block_table", _I32, 2) != device:
            raise ValueError(f"pages and block_table must be on cuda:{device}")
        _need(q_start, "q_start", _I32, (block_table.shape[0] + 1,), device)
        _need(lengths, "lengths", _I32, (block_table.shape[0],), device)
        raise ValueError("pages must be a contiguous [pages, 2, kv heads, page size, head dim] tensor")
    # one row has no distance to a next, whatever its stride says; rows that overlap (a table broadcast over requests) are refused below
    _BATCH(block, 0, pages.data_ptr(), num_pages, q_start.data_ptr(), lengths.data_ptr(), block_table.data_ptr(), block_table.stride(0) if batch > 1 else cols,
           kept.status_ptr, cols, page_size, kv_heads, dh, batch, tokens)
    return kv_heads, page_size, dh, cols


def rope_tables(num_positions: int, head_dim: int, base: float = 10000.0, device="cuda"):
    """cos and sin fp32 [num_positions, head_dim / 2] of position * base^(-2 i / head_dim) (layers.py:52-60), the angles in 64 bits."""
    i = torch.arange(head_dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * i / head_dim)
    return angle.cos().float(), angle.sin().float()


def tree_spans(parents) -> np.ndarray:
    """int32 [n, 2] (pre, end) of one request's tokens from their parents (host ints: the parent's place among them, -1: hangs on
    the cached history, -2: padding), any order."""
    p = np.asarray(parents)
    if p.ndim != 1 or (p.size and p.dtype.kind not in "iu"):
        raise ValueError("parents must be one-dimensional integers")
    if p.size and (p.min() < -2 or p.max() >= p.size):         # before they are narrowed to 32 bits
        raise PhoenixError(1, "a parent must be -1, -2 (padding) or another token that is no padding")
    p = np.ascontiguousarray(p, dtype=np.int32)
    out = np.empty((p.shape[0], 2), np.int32)
    _ok(lib.phx_tree_spans(p.ctypes.data, p.shape[0], out.ctypes.data))
    return out


def history_append(qkv, pages, q_start, lengths, block_table, positions, cos=None, sin=None, *, num_q_heads: int, q_gain=None, k_gain=None,
                   eps: float = 1e-6, out=None, stream: Optional[int] = None):
    """qkv bf16 [N, (num_q_heads + 2 kv heads) * head dim] in the merged order [kv head][queries, key, value] (rows may be apart).  Query and key heads are
    normed (q_gain, k_gain fp32 [head dim]; None: not) and rotated by positions int32 [N] (cos, sin fp32 [positions, head dim / 2];
    None: not); keys and values go to the cache behind `lengths`, the queries come back as bf16 [N, num_q_heads, head dim]."""
    device = _rows(qkv, "qkv", _BF16, 2)
    if _elsewhere(device, stream):
        with _under(device, stream):
            return history_append(qkv, pages, q_start, lengths, block_table, positions, cos, sin, num_q_heads=num_q_heads, q_gain=q_gain, k_gain=k_gain, eps=eps, out=out)
    n, width = qkv.shape
    stream = _stream(device, stream)
    mine = _structs
    kv_heads, _, dh, _ = _batch(mine.batch, pages, q_start, lengths, block_table, n, device, _keep(device, stream))
    if width != (num_q_heads + 2 * kv_heads) * dh:
        raise ValueError(f"qkv rows have {width} columns, {(num_q_heads + 2 * kv_heads) * dh} are needed")
    places = at = cos_ptr = sin_ptr = q_gain_ptr = k_gain_ptr = 0
    if cos is not None or sin is not None:
        _rows(cos, "cos", _F32, 2)
        places = cos.shape[0]
        cos_ptr, sin_ptr = _need(cos, "cos", _F32, (places, dh // 2), device), _need(sin, "sin", _F32, (places, dh // 2), device)
        at = _need(positions, "positions", _I32, (n,), device)
    if q_gain is not None:
        q_gain_ptr = _need(q_gain, "q_gain", _F32, (dh,), device)
    if k_gain is not None:
        k_gain_ptr = _need(k_gain, "k_gain", _F32, (dh,), device)
    shape = (n, num_q_heads, dh)
    if out is None:
        out = torch.empty_strided(shape, (num_q_heads * dh, dh, 1), dtype=_BF16, device=qkv.device)
    else:
        _need(out, "out", _BF16, shape, device)
    _APPEND(mine.append, 0, qkv.data_ptr(), qkv.stride(0) if n > 1 else width, at, cos_ptr, sin_ptr, q_gain_ptr, k_gain_ptr, out.data_ptr(), num_q_heads, places, eps, 0)
    _ok(lib.phx_history_append_device(device, mine.batch_ref, mine.append_ref, stream))
    return out


def tree_attention(q, pages, q_start, lengths, block_table, spans=None, *, sm_scale: Optional[float] = None, cap: float = 0.0,
                   cap_method: Optional[str] = None, max_tokens: Optional[int] = None, max_keys: Optional[int] = None, out=None, workspace=None,
                   stream: Optional[int] = None):
    """q bf16 [N, heads, head dim] (tokens may be apart) attends to the cached keys of its request and to the new ones - appended
    already - that spans int32 [N, 2] lets it see: (pre, end) per token, i sees j where pre[j] <= pre[i] < end[j] (`tree_spans`; None: a
    chain).  sm_scale defaults to sqrt(128) / head dim (scaling.py:46-47).  cap > 0 caps the logits by cap_method.  max_tokens and max_keys: the most new tokens and keys
    (cached + new) of a request, if the caller knows them; they only choose kernels.  workspace: uint8, phx_tree_workspace_bytes; the stream's own if None, in a capture the graph's own.
    Returns bf16 [N, heads, head dim]."""
    device = _rows(q, "q", _BF16, 3)
    if _elsewhere(device, stream):
        with _under(device, stream):
            return tree_attention(q, pages, q_start, lengths, block_table, spans, sm_scale=sm_scale, cap=cap, cap_method=cap_method, max_tokens=max_tokens,
                                  max_keys=max_keys, out=out, workspace=workspace)
    n, heads, dh = shape = q.shape
    stream = _stream(device, stream)
    kept, mine = _keep(device, stream), _structs
    _, page_size, cache_dh, cols = _batch(mine.batch, pages, q_start, lengths, block_table, n, device, kept)
    if cache_dh != dh or (heads > 1 and q.stride(1) != dh):
        raise ValueError("q must have the cache's head dim, its heads side by side")
    if cap_method not in CAP_METHODS:
        raise ValueError(f"cap_method must be one of {list(CAP_METHODS)}")
    if cap > 0 and cap_method is None:
        raise ValueError("a cap needs its cap_method")
    if out is None:
        out = torch.empty_strided(shape, (heads * dh, dh, 1), dtype=_BF16, device=q.device)
    else:
        _need(out, "out", _BF16, shape, device)
    if workspace is None:
        if stream != 0 and torch._C._cuda_isCurrentStreamCapturing():   # (the default stream cannot be captured)
            workspace = _workspace(device)                   # a graph may be replayed on any stream: it has a workspace of its own, from its own pool
            space, size = workspace.data_ptr(), workspace.numel()
        else:
            space, size = kept.space or _take_space(kept, device)
    else:
        size = workspace.numel()
        space = _need(workspace, "workspace", _U8, (size,), device)
    _TREE(mine.tree, 0, q.data_ptr(), q.stride(0) if n > 1 else heads * dh, 0 if spans is None else _need(spans, "spans", _I32, (n, 2), device),
          out.data_ptr(), space, size, cols * page_size if max_keys is None else max_keys, n if max_tokens is None else max_tokens, heads,
          math.sqrt(128.0) / dh if sm_scale is None else sm_scale, cap, CAP_METHODS[cap_method], 0)
    _ok(lib.phx_tree_attention_device(device, mine.batch_ref, mine.tree_ref, stream))
    return out


def token_logprobs(logits, given=None, *, top_k: int = 0, cap: float = 0.0, temperature: float = 1.0, stream: Optional[int] = None):
    """logits fp32 or bf16 [N, vocab] (rows may be apart; -inf: not allowed), given int64 [N, n] or [N] ids (outside the
    vocabulary: none), top_k at most 128.  Returns (log probabilities of given fp32, of its shape, None without given; entropy fp32 [N]; the top_k best ids' log probabilities fp32
    [N, top_k]; the ids int64 [N, top_k]) of softmax(cap tanh(logits / cap) / temperature), best first, ties by the lower id."""
    bf16 = isinstance(logits, torch.Tensor) and logits.dtype is _BF16
    device = _rows(logits, "logits", _BF16 if bf16 else _F32, 2)
    if _elsewhere(device, stream):
        with _under(device, stream):
            return token_logprobs(logits, given, top_k=top_k, cap=cap, temperature=temperature)
    rows, vocab = logits.shape
    if not 0 <= top_k <= vocab:
        raise ValueError(f"top_k must be 0 to vocab ({vocab})")
    where = logits.device
    given_out, given_ptr, given_out_ptr, num_given = None, 0, 0, 0
    if given is not None:
        shape = tuple(given.shape)
        num_given = shape[-1] if len(shape) == 2 else 1
        given_ptr = _need(given, "given", _I64, (rows,) if len(shape) == 1 else (rows, num_given), device)
        given_out = torch.empty_strided(shape, given.stride(), dtype=_F32, device=where)
        given_out_ptr = given_out.data_ptr()
    entropy = torch.empty_strided((rows,), (1,), dtype=_F32, device=where)
    top = torch.empty_strided((rows, top_k), (top_k, 1), dtype=_F32, device=where)
    ids = torch.empty_strided((rows, top_k), (top_k, 1), dtype=_I64, device=where)
    mine = _structs
    _LOGPROBS(mine.logprobs, 0, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, given_ptr, given_out_ptr, entropy.data_ptr(), top.data_ptr(), ids.data_ptr(),
              rows, vocab, num_given, top_k, bf16, cap, temperature, 0)
    _ok(lib.phx_token_logprobs_device(device, mine.logprobs_ref, _stream(device, stream)))
    return given_out, entropy, top, ids


def release(device: Optional[int] = None, stream: Optional[int] = None) -> None:
    """Gives the workspace of a stream (torch's current one if None) back to torch's allocator, 39 MB on a B200; its next attention takes one again."""
    device = torch.cuda.current_device() if device is None else device
    kept = _kept.get((device, _stream(device, stream)))
    if kept is not None:
        kept.workspace = kept.space = None


def check_status(device: Optional[int] = None, stream: Optional[int] = None) -> None:
    """Waits for the stream (torch's current one of `device`, of the current device if None) and raises PhoenixError if a call on it since the last check met a page, position or offset out of range
    (PHX_E_ARG: what it named was left out) or a bounded wait that ran out (PHX_E_TIMEOUT)."""
    device = torch.cuda.current_device() if device is None else device
    stream = _stream(device, stream)
    kept = _kept.get((device, stream))
    if kept is not None:
        bits = C.c_int32()
        _ok(lib.phx_decode_status(device, kept.status.data_ptr(), stream, C.byref(bits)))
