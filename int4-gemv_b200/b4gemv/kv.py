"""The 4-bit key/value cache: torch wrappers of the b4_kv_* entry points
(include/b4gemv.h, which defines the layout and the semantics).

    cache = KVCache.alloc(KV_INT4, n_pages, kv_heads, page_size=64, head_dim=128, device="cuda")
    step = kv_tables(cache.page_size, tables, cached, added, free_pages, free_state, max_tokens)
    kv_append(cache, k, v, step.slots)
    out = kv_attention(cache, q, tables, step.ctx_len, step.q_starts, max_q)

Every call goes to the current stream of the tensors' device and returns without
waiting.  Refused arguments raise ValueError before anything is launched; what
only the library can refuse raises B4Error.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

from ._lib import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, KV_FULL, KV_INT4, KV_NF4, KvAttn, KvCache, KvStep, check, load)

__all__ = ["KV_INT4", "KV_NF4", "KVCache", "KVStep", "kv_block_bytes", "kv_tables", "kv_append", "kv_read",
           "kv_attention", "kv_attention_workspace"]

_byref = ctypes.byref


def _torch():
    import torch
    return torch


def _raw_stream(device):
    return _torch().cuda.current_stream(device).cuda_stream


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _ints(name, t, device, least):
    torch = _torch()
    _need(t.dtype == torch.int32 and t.device == device and t.is_contiguous(), f"{name}: a contiguous int32 tensor on {device}")
    _need(t.numel() >= least, f"{name}: {least} values at least, got {t.numel()}")


def kv_block_bytes(fmt: int, page_size: int, head_dim: int) -> int:
    """Bytes of one kv head's part of a page."""
    n = ctypes.c_size_t(0)
    check("b4_kv_block_bytes", load().b4_kv_block_bytes(fmt, page_size, head_dim, _byref(n)))
    return n.value


class KVCache:
    """One layer's cache over `blocks`, a contiguous uint8 CUDA tensor
    [pages][kv_heads][kv_block_bytes(fmt, page_size, head_dim)]."""

    def __init__(self, blocks, fmt: int, page_size: int, head_dim: int):
        size = kv_block_bytes(fmt, page_size, head_dim)
        _need(blocks.is_cuda and blocks.dtype == _torch().uint8 and blocks.is_contiguous(), "blocks: a contiguous uint8 CUDA tensor")
        _need(blocks.dim() == 3 and blocks.shape[2] == size, f"blocks: [pages][kv_heads][{size}], got {tuple(blocks.shape)}")
        self.blocks, self.fmt, self.page_size, self.head_dim = blocks, fmt, page_size, head_dim
        self.n_pages, self.kv_heads = blocks.shape[0], blocks.shape[1]
        self.device = blocks.device
        self._c = KvCache(blocks.data_ptr(), fmt, self.n_pages, page_size, self.kv_heads, head_dim)
        self._ref = _byref(self._c)

    @classmethod
    def alloc(cls, fmt: int, n_pages: int, kv_heads: int, page_size: int = 64, head_dim: int = 128, device="cuda"):
        """A cache of n_pages pages (zero-filled)."""
        torch = _torch()
        return cls(torch.zeros((n_pages, kv_heads, kv_block_bytes(fmt, page_size, head_dim)), dtype=torch.uint8,
                               device=device), fmt, page_size, head_dim)


class KVStep(NamedTuple):
    """What kv_tables returns, int32 CUDA tensors (b4_kv_step's outputs)."""
    ctx_len: object
    q_starts: object
    slots: object
    positions: object
    free_state: object


def kv_tables(page_size: int, tables, cached, added, free_pages, free_state, max_tokens: int, out: KVStep | None = None,
              stream=None) -> KVStep:
    """b4_kv_tables: block tables (int32 [requests][width], updated in place),
    slots, positions, starts and lengths of one step.  free_pages is the ring
    of free pages, free_state its (place, pages left); the returned free_state is
    the next step's.  out: buffers to reuse (free_state must be another one)."""
    torch = _torch()
    dev = tables.device
    n = cached.numel()
    _need(tables.is_cuda and tables.dtype == torch.int32 and tables.dim() == 2 and tables.shape[0] >= n
          and (tables.shape[1] <= 1 or tables.stride(1) == 1), "tables: int32 CUDA [requests][width], columns contiguous")
    _ints("cached", cached, dev, 0)
    _ints("added", added, dev, n)
    _ints("free_pages", free_pages, dev, 0)
    _ints("free_state", free_state, dev, 2)
    if out is None:
        # one buffer for the five outputs, each on a 16-byte boundary
        sizes = [n, n + 1, max_tokens, max_tokens, 3]
        flat = torch.empty(sum((s + 3) // 4 * 4 for s in sizes), dtype=torch.int32, device=dev)
        parts, at = [], 0
        for s in sizes:
            parts.append(flat[at:at + s])
            at += (s + 3) // 4 * 4
        out = KVStep(*parts)
    else:
        for name, least in (("ctx_len", n), ("q_starts", n + 1), ("slots", max_tokens), ("positions", max_tokens), ("free_state", 3)):
            _ints(name, getattr(out, name), dev, least)
    c = KvStep(n, page_size, tables.shape[1], free_pages.numel(), max_tokens, max(tables.stride(0), tables.shape[1]),
               tables.data_ptr(), cached.data_ptr(), added.data_ptr(), free_pages.data_ptr(), free_state.data_ptr(),
               out.ctx_len.data_ptr(), out.q_starts.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(),
               out.free_state.data_ptr())
    check("b4_kv_tables", load().b4_kv_tables(_byref(c), stream.cuda_stream if stream is not None else _raw_stream(dev)))
    return out


def _dtype(t):
    torch = _torch()
    return {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_F32}.get(t.dtype)


def kv_append(cache: KVCache, k, v, slots, stream=None) -> None:
    """b4_kv_append: k and v [tokens][kv_heads][head_dim] (fp16, bf16 or fp32, any
    token and head strides, columns contiguous) into the cache at slots."""
    shape = (slots.numel(), cache.kv_heads, cache.head_dim)
    _ints("slots", slots, cache.device, 0)
    code = _dtype(k)
    _need(code is not None and v.dtype == k.dtype, "k and v: fp16, bf16 or fp32, both alike")
    for t in (k, v):
        _need(tuple(t.shape) == shape and t.device == cache.device and t.stride(2) == 1,
              f"k and v: {shape} on {cache.device}, columns contiguous")
    check("b4_kv_append", load().b4_kv_append(
        cache._ref, k.data_ptr(), v.data_ptr(), code, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        slots.data_ptr(), shape[0], stream.cuda_stream if stream is not None else _raw_stream(cache.device)))


def kv_read(cache: KVCache, slots, k=None, v=None, stream=None):
    """b4_kv_read: the fp32 values held at slots, as (k, v) [tokens][kv_heads][head_dim]."""
    torch = _torch()
    shape = (slots.numel(), cache.kv_heads, cache.head_dim)
    _ints("slots", slots, cache.device, 0)
    k = torch.empty(shape, device=cache.device) if k is None else k
    v = torch.empty(shape, device=cache.device) if v is None else v
    for t in (k, v):
        _need(tuple(t.shape) == shape and t.dtype == torch.float32 and t.device == cache.device and t.is_contiguous(),
              f"k and v: contiguous fp32 {shape} on {cache.device}")
    check("b4_kv_read", load().b4_kv_read(cache._ref, slots.data_ptr(), shape[0], k.data_ptr(), v.data_ptr(),
                                          stream.cuda_stream if stream is not None else _raw_stream(cache.device)))
    return k, v


_WS = {}


def _workspace(device, nbytes: int):
    """The package's workspace for attention on `device`: zero-filled, grown on demand."""
    ws = _WS.get(device.index)
    if ws is None or ws.numel() < nbytes:
        torch = _torch()
        ws = torch.zeros(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=device)
        _WS[device.index] = ws
    return ws


def _attn(cache, q, tables, ctx_len, q_starts, max_q, scale, window, causal, out, lse):
    torch = _torch()
    dev = cache.device
    code = _dtype(q)
    _need(code in (DTYPE_F16, DTYPE_BF16) and q.dim() == 3 and q.device == dev and q.shape[2] == cache.head_dim
          and q.stride(2) == 1, f"q: fp16 or bf16 [tokens][heads][{cache.head_dim}] on {dev}, columns contiguous")
    total, heads, _ = q.shape
    _need(heads % cache.kv_heads == 0, f"heads: a multiple of {cache.kv_heads}, got {heads}")
    n = ctx_len.numel()
    _need(tables.dtype == torch.int32 and tables.device == dev and tables.dim() == 2 and tables.shape[0] >= n
          and (tables.shape[1] <= 1 or tables.stride(1) == 1), "tables: int32 [requests][width], columns contiguous")
    _ints("ctx_len", ctx_len, dev, 0)
    _ints("q_starts", q_starts, dev, n + 1)
    if out is None:
        out = torch.empty((total, heads, cache.head_dim), dtype=q.dtype, device=dev)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev and out.stride(2) == 1, "out: as q, columns contiguous")
    if lse is not None:
        _need(tuple(lse.shape) == (total, heads) and lse.dtype == torch.float32 and lse.device == dev and lse.is_contiguous(),
              "lse: contiguous fp32 [tokens][heads]")
    a = KvAttn(q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None, tables.data_ptr(),
               ctx_len.data_ptr(), q_starts.data_ptr(), max(tables.stride(0), tables.shape[1]), q.stride(0), q.stride(1),
               out.stride(0), out.stride(1), tables.shape[1], n, total, max_q, heads, code, window,
               0 if causal else KV_FULL, cache.head_dim ** -0.5 if scale is None else scale)
    return a, out


def kv_attention_workspace(cache: KVCache, q, tables, ctx_len, q_starts, max_q: int) -> int:
    """Bytes of workspace that kv_attention needs for such a call (b4_kv_attention_workspace)."""
    a, _ = _attn(cache, q, tables, ctx_len, q_starts, max_q, None, 0, True, q, None)
    n = ctypes.c_size_t(0)
    check("b4_kv_attention_workspace", load().b4_kv_attention_workspace(cache._ref, _byref(a), _byref(n)))
    return n.value


def kv_attention(cache: KVCache, q, tables, ctx_len, q_starts, max_q: int, scale: float | None = None, window: int = 0,
                 causal: bool = True, out=None, lse=None, ws=None, stream=None):
    """b4_kv_attention: softmax(scale * q K^T + mask) V over the cached pages of
    each query's request; q [tokens][heads][head_dim] fp16 or bf16, packed by
    request (q_starts).  scale None = head_dim ** -0.5; window 0 = none; lse: an
    fp32 [tokens][heads] tensor that receives the log-sum-exp of the scores.
    ws: a zero-filled uint8 CUDA tensor of kv_attention_workspace() bytes, or
    None for the package's own of the device (calls that may overlap on the GPU
    need their own).  Returns out."""
    a, out = _attn(cache, q, tables, ctx_len, q_starts, max_q, scale, window, causal, out, lse)
    lib = load()
    if ws is None:
        n = ctypes.c_size_t(0)
        check("b4_kv_attention_workspace", lib.b4_kv_attention_workspace(cache._ref, _byref(a), _byref(n)))
        ws = _workspace(cache.device, n.value)
    check("b4_kv_attention", lib.b4_kv_attention(cache._ref, _byref(a), ws.data_ptr(), ws.numel(),
                                                 stream.cuda_stream if stream is not None else _raw_stream(cache.device)))
    return out
