"""The 4-bit key/value cache: torch wrappers of the b4_kv_* entry points
(include/b4gemv.h, which defines the layout and the semantics).

    cache = KVCache.alloc(KV_INT4, n_pages, kv_heads, page_size=64, head_dim=128, device="cuda")
    step = kv_tables(cache.page_size, tables, cached, added, free_pages, free_state, max_tokens)
    kv_append(cache, k, v, step.slots)
    out = kv_attention(cache, q, tables, step.ctx_len, step.q_starts, max_q)

Every call goes to the current stream of the tensors' device (or `stream`),
whichever device is current, and returns without waiting.  Refused arguments raise ValueError before anything is
launched; what only the library can refuse raises B4Error.

A decode step calls these for every layer, with kernels of a few microseconds:
the checks make no objects, and a call's structure is packed as bytes in one
go.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

from ._lib import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, KV_FULL, KV_INT4, KV_NF4, KvAttn, KvCache, KvStep, check, load)

__all__ = ["KV_INT4", "KV_NF4", "KVCache", "KVStep", "kv_block_bytes", "kv_tables", "kv_append", "kv_read",
           "kv_attention", "kv_attention_workspace"]

# b4_kv_step and b4_kv_attn as the C compiler lays them out (KvStep, KvAttn in _lib)
_STEP = struct.Struct("@5i4xq10P")
_ATTN = struct.Struct("@6P5q8if4x")
assert _STEP.size == ctypes.sizeof(KvStep) and _ATTN.size == ctypes.sizeof(KvAttn)

_torch = _int32 = _float32 = _uint8 = _raw_stream = _device = _codes = None


def _load():
    """torch's names and the library, once."""
    global _torch, _int32, _float32, _uint8, _raw_stream, _device, _codes
    import torch
    _torch, _int32, _float32, _uint8 = torch, torch.int32, torch.float32, torch.uint8
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: torch.cuda.current_stream(index).cuda_stream)
    _device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    _codes = {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_F32}
    return load()


def _lib():
    return load() if _torch is not None else _load()


def _ints(name, t, index, least):
    if t.dtype is not _int32 or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor on cuda:{index}")
    if least and t.numel() < least:
        raise ValueError(f"{name}: {least} values at least, got {t.numel()}")


def _table(tables, index, n):
    """(width, stride) of int32 [requests][width] with contiguous columns."""
    if tables.dtype is not _int32 or tables.get_device() != index or index < 0 or tables.dim() != 2:
        raise ValueError("tables: an int32 CUDA tensor [requests][width], on the device of the others")
    rows, width = tables.shape
    stride, one = tables.stride()
    if rows < n or (n > 0 and width > 1 and one != 1):    # an empty table's strides are any
        raise ValueError(f"tables: {n} rows at least, columns contiguous")
    if stride < width:
        if n > 1:                              # expanded or overlapping rows: no stride of such a table's is the library's
            raise ValueError("tables: rows must not overlap (an expanded table needs contiguous())")
        stride = width                         # of a single row, that nothing is addressed by
    return width, stride


def kv_block_bytes(fmt: int, page_size: int, head_dim: int) -> int:
    """Bytes of one kv head's part of a page."""
    n = ctypes.c_size_t(0)
    check("b4_kv_block_bytes", load().b4_kv_block_bytes(fmt, page_size, head_dim, ctypes.byref(n)))
    return n.value


class KVCache:
    """One layer's cache over `blocks`, a contiguous uint8 CUDA tensor
    [pages][kv_heads][kv_block_bytes(fmt, page_size, head_dim)]."""

    def __init__(self, blocks, fmt: int, page_size: int, head_dim: int):
        size = kv_block_bytes(fmt, page_size, head_dim)
        _load()
        if not blocks.is_cuda or blocks.dtype != _torch.uint8 or not blocks.is_contiguous():
            raise ValueError("blocks: a contiguous uint8 CUDA tensor")
        if blocks.dim() != 3 or blocks.shape[2] != size:
            raise ValueError(f"blocks: [pages][kv_heads][{size}], got {tuple(blocks.shape)}")
        self.blocks, self.fmt, self.page_size, self.head_dim = blocks, fmt, page_size, head_dim
        self.n_pages, self.kv_heads = blocks.shape[0], blocks.shape[1]
        self.device, self.index = blocks.device, blocks.get_device()
        self._c = KvCache(blocks.data_ptr(), fmt, self.n_pages, page_size, self.kv_heads, head_dim)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def alloc(cls, fmt: int, n_pages: int, kv_heads: int, page_size: int = 64, head_dim: int = 128, device="cuda"):
        """A cache of n_pages pages (zero-filled)."""
        import torch
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
    the next step's.  out: buffers to reuse; none of them may be one that the call
    reads (the last step's ctx_len as `cached`, its free_state)."""
    lib = _lib()
    index, n = tables.get_device(), cached.numel()
    width, stride = _table(tables, index, n)
    _ints("cached", cached, index, 0)
    _ints("added", added, index, n)
    _ints("free_pages", free_pages, index, 0)
    _ints("free_state", free_state, index, 2)
    if out is None:
        if max_tokens < 0:
            raise ValueError("max_tokens: 0 or more")
        out = KVStep(*_torch.empty(2 * n + 2 * max_tokens + 4, dtype=_int32, device=tables.device).split(
            (n, n + 1, max_tokens, max_tokens, 3)))
    else:
        for name, least in (("ctx_len", n), ("q_starts", n + 1), ("slots", max_tokens), ("positions", max_tokens), ("free_state", 3)):
            _ints(name, getattr(out, name), index, least)
    if _device() != index:
        with _torch.cuda.device(index):
            return kv_tables(page_size, tables, cached, added, free_pages, free_state, max_tokens, out, stream)
    args = _STEP.pack(n, page_size, width, free_pages.numel(), max_tokens, stride, tables.data_ptr(), cached.data_ptr(),
                      added.data_ptr(), free_pages.data_ptr(), free_state.data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                      out[2].data_ptr(), out[3].data_ptr(), out[4].data_ptr())
    status = lib.b4_kv_tables(args, stream.cuda_stream if stream is not None else _raw_stream(index))
    if status:
        check("b4_kv_tables", status)
    return out


def kv_append(cache: KVCache, k, v, slots, stream=None) -> None:
    """b4_kv_append: k and v [tokens][kv_heads][head_dim] (fp16, bf16 or fp32, any
    token and head strides, columns contiguous) into the cache at slots."""
    index, n = cache.index, slots.numel()
    _ints("slots", slots, index, 0)
    code = _codes.get(k.dtype)
    shape, ks, vs = (n, cache.kv_heads, cache.head_dim), k.stride(), v.stride()
    if (code is None or v.dtype is not k.dtype or k.shape != shape or v.shape != shape or k.get_device() != index
            or v.get_device() != index or ks[2] != 1 or vs[2] != 1):
        raise ValueError(f"k and v: {shape}, both fp16, bf16 or fp32, on cuda:{index}, columns contiguous")
    if _device() != index:                     # the library launches on the current device
        with _torch.cuda.device(index):
            return kv_append(cache, k, v, slots, stream)
    status = load().b4_kv_append(cache._ref, k.data_ptr(), v.data_ptr(), code, ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), n,
                                 stream.cuda_stream if stream is not None else _raw_stream(index))
    if status:
        check("b4_kv_append", status)


def kv_read(cache: KVCache, slots, k=None, v=None, stream=None):
    """b4_kv_read: the fp32 values held at slots, as (k, v) [tokens][kv_heads][head_dim]."""
    index, n = cache.index, slots.numel()
    _ints("slots", slots, index, 0)
    shape = (n, cache.kv_heads, cache.head_dim)
    k = _torch.empty(shape, device=cache.device) if k is None else k
    v = _torch.empty(shape, device=cache.device) if v is None else v
    for x in (k, v):
        if x.shape != shape or x.dtype is not _float32 or x.get_device() != index or not x.is_contiguous():
            raise ValueError(f"k and v: contiguous fp32 {shape} on cuda:{index}")
    if _device() != index:
        with _torch.cuda.device(index):
            return kv_read(cache, slots, k, v, stream)
    status = load().b4_kv_read(cache._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(),
                               stream.cuda_stream if stream is not None else _raw_stream(index))
    if status:
        check("b4_kv_read", status)
    return k, v


_WS = {}


def _workspace_most():
    """Bytes that serve every attention call on the current device: the tile kernel's, and the warp kernel's 16 columns, of 128."""
    most = 0
    for group, queries in ((1, 1 << 20), (16, 1)):
        cache = KvCache(blocks=16, fmt=KV_INT4, n_pages=1, page_size=16, kv_heads=1, head_dim=128)      # an address that nothing reads
        n = ctypes.c_size_t(0)
        check("b4_kv_attention_workspace", load().b4_kv_attention_workspace(
            ctypes.byref(cache), ctypes.byref(KvAttn(n_req=1, total_q=queries, max_q=queries, heads=group)), ctypes.byref(n)))
        most = max(most, n.value)
    return most


def _workspace(index, stream=None):
    """The package's workspace for attention on a device.  Captured graphs and kernels on any stream hold its address, so
    there is one, of the largest size, made and zeroed once, outside captures, and never replaced."""
    ws = _WS.get(index)
    if ws is None:
        with _torch.cuda.device(index):
            for s in (None, stream):                           # the caller's and the call's
                with _torch.cuda.stream(s):
                    if _torch.cuda.is_current_stream_capturing():
                        raise ValueError("ws: the first call on a device makes the package's workspace, which a capture would "
                                         "only record; call once before the capture, or pass ws")
            ws = _torch.zeros(_workspace_most(), dtype=_torch.uint8, device=f"cuda:{index}")
            _torch.cuda.current_stream().synchronize()         # zero for every stream from here on
        ws = _WS.setdefault(index, ws)
    return ws


def _attn(cache, q, tables, ctx_len, q_starts, max_q, scale, window, causal, out, lse):
    """A call's b4_kv_attn, packed, and its output."""
    index, dim, n = cache.index, cache.head_dim, ctx_len.numel()
    code = _codes.get(q.dtype)
    if (code is None or code == DTYPE_F32 or q.dim() != 3 or q.get_device() != index or q.shape[2] != dim
            or q.stride(2) != 1):
        raise ValueError(f"q: fp16 or bf16 [tokens][heads][{dim}] on cuda:{index}, columns contiguous")
    total, heads, _ = q.shape
    if heads % cache.kv_heads:
        raise ValueError(f"heads: a multiple of {cache.kv_heads}, got {heads}")
    width, stride = _table(tables, index, n)
    _ints("ctx_len", ctx_len, index, 0)
    _ints("q_starts", q_starts, index, n + 1)
    if out is None:
        out = _torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != index or out.stride(2) != 1:
        raise ValueError("out: as q, columns contiguous")
    if lse is not None and (lse.shape != (total, heads) or lse.dtype is not _float32 or lse.get_device() != index
                            or not lse.is_contiguous()):
        raise ValueError("lse: contiguous fp32 [tokens][heads]")
    qs, os = q.stride(), out.stride()
    return _ATTN.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else 0, tables.data_ptr(),
                      ctx_len.data_ptr(), q_starts.data_ptr(), stride, qs[0], qs[1], os[0], os[1], width, n, total, max_q, heads,
                      code, window, 0 if causal else KV_FULL, dim ** -0.5 if scale is None else scale), out


def kv_attention_workspace(cache: KVCache, q, tables, ctx_len, q_starts, max_q: int) -> int:
    """Bytes of workspace that kv_attention needs for such a call (b4_kv_attention_workspace)."""
    n = ctypes.c_size_t(0)
    args, _ = _attn(cache, q, tables, ctx_len, q_starts, max_q, None, 0, True, q, None)
    with _torch.cuda.device(cache.index):      # whose SMs are counted
        check("b4_kv_attention_workspace", load().b4_kv_attention_workspace(cache._ref, args, ctypes.byref(n)))
    return n.value


def kv_attention(cache: KVCache, q, tables, ctx_len, q_starts, max_q: int, scale: float | None = None, window: int = 0,
                 causal: bool = True, out=None, lse=None, ws=None, stream=None):
    """b4_kv_attention: softmax(scale * q K^T + mask) V over the cached pages of
    each query's request; q [tokens][heads][head_dim] fp16 or bf16, packed by
    request (q_starts).  scale None = head_dim ** -0.5; window 0 = none; lse: an
    fp32 [tokens][heads] tensor that receives the log-sum-exp of the scores.
    ws: a zero-filled uint8 CUDA tensor of kv_attention_workspace() bytes, or
    None for the package's own of the device (39.4 MB on a B200; the first call
    makes it and waits for its zeros, and is refused inside a graph capture).
    Calls that may overlap on the GPU need their own.  Returns out."""
    args, out = _attn(cache, q, tables, ctx_len, q_starts, max_q, scale, window, causal, out, lse)
    if ws is None:
        ws = _workspace(cache.index, stream)
    elif ws.dtype is not _uint8 or ws.get_device() != cache.index or not ws.is_contiguous():
        raise ValueError(f"ws: a contiguous uint8 tensor on cuda:{cache.index}")
    if _device() != cache.index:
        with _torch.cuda.device(cache.index):
            return kv_attention(cache, q, tables, ctx_len, q_starts, max_q, scale, window, causal, out, lse, ws, stream)
    status = load().b4_kv_attention(cache._ref, args, ws.data_ptr(), ws.numel(),
                                    stream.cuda_stream if stream is not None else _raw_stream(cache.index))
    if status:
        check("b4_kv_attention", status)
    return out
