"""What stands around the 4-bit cache in a layer whose queries read a choice of its
pages: torch wrappers of b4_kv_append_rotary, b4_kv_boxes, b4_kv_select and
b4_kv_attention_lists (include/b4gemv.h, which defines the semantics).

    rotary, boxes = Rotary(128, base=1e6), kv_new_boxes(cache)            # once; boxes beside the cache, per layer
    q = kv_append_rotary(cache, rotary, q, k, v, step.positions, step.slots)
    kv_boxes(cache, boxes, step.slots)
    lists = kv_select(cache, boxes, q, tables, step.ctx_len, step.q_starts, max_q, keep=64)
    out = kv_attention_lists(cache, q, lists)

Streams, devices and refusals are as in kv.py.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import struct
from typing import NamedTuple

from . import kv as _kv
from ._lib import DTYPE_BF16, DTYPE_F16, DTYPE_F32, ROTARY_ADJACENT, KvAttn, KvChoice, KvRows, RotaryTable, check
from .kv import _ints, _table, _workspace

__all__ = ["Rotary", "KVLists", "kv_append_rotary", "kv_box_bytes", "kv_new_boxes", "kv_boxes", "kv_select",
           "kv_attention_lists", "kv_attention_lists_workspace"]

# b4_kv_rows, b4_kv_choice and b4_kv_attn as the C compiler lays them out
_ROWS = struct.Struct("@6P9q4i")
_CHOICE = struct.Struct("@7P3q9i4x")
_ATTN = struct.Struct("@6P5q8if4x")
assert _ROWS.size == ctypes.sizeof(KvRows) and _CHOICE.size == ctypes.sizeof(KvChoice) and _ATTN.size == ctypes.sizeof(KvAttn)

# torch's names, as kv.py has them once it is loaded: a call looks each up once
_torch = _int32 = _float32 = _uint8 = _float16 = _codes = None


def _lib():
    """The library; torch's names, once."""
    global _torch, _int32, _float32, _uint8, _float16, _codes
    lib = _kv._lib()
    if _torch is None:
        _torch, _int32, _float32, _uint8, _codes = _kv._torch, _kv._int32, _kv._float32, _kv._uint8, _kv._codes
        _float16 = _torch.float16
    return lib


def _on(stream):
    """Where a call's own outputs are allocated: on the stream that writes them, whose memory no other stream still uses."""
    return _torch.cuda.stream(stream) if stream is not None else _here


_here = contextlib.nullcontext()


class Rotary:
    """The angles of b4_kv_append_rotary: the first `dim` columns of a head turn, in pairs.

    base: pair i's frequency is base ** (-2 i / dim) radians a position; inv_freq: the dim / 2 frequencies themselves, for
    scaled forms.  sections: how many pairs, in order, follow each axis of the positions (time, height, width: three
    numbers); axes: the axis of every pair, where they are mixed.  adjacent: pairs (2i, 2i + 1) instead of (i, i + dim / 2).
    scale: a factor of cosine and sine."""

    def __init__(self, dim: int, base: float = 1e6, inv_freq=None, sections=None, axes=None, adjacent: bool = False, scale: float = 1.0,
                 device="cuda"):
        lib = _lib()
        torch = _torch
        if dim < 16 or dim % 16 or dim > 128:
            raise ValueError(f"dim: a multiple of 16 up to 128, got {dim}")
        half = dim // 2
        if inv_freq is None:
            if not base > 0:
                raise ValueError("base: above 0")
            inv_freq = [base ** (-i / half) for i in range(half)]
        inv_freq = [float(f) for f in inv_freq]
        if len(inv_freq) != half or not all(map(math.isfinite, inv_freq)):
            raise ValueError(f"inv_freq: {half} finite frequencies")
        if sections is not None:
            if axes is not None or any(n < 0 for n in sections) or sum(sections) != half:
                raise ValueError(f"sections: numbers of pairs that add up to {half}, without axes")
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
            n_axes = len(sections)
        elif axes is not None:
            axes = [int(a) for a in axes]
            n_axes = max(axes, default=0) + 1
        else:
            n_axes = 1
        if axes is not None and (len(axes) != half or min(axes) < 0 or n_axes > 256):
            raise ValueError(f"axes: the axis, 0 to 255, of each of {half} pairs")
        if not math.isfinite(scale):
            raise ValueError("scale: finite")
        turns = (ctypes.c_uint64 * half)()
        check("b4_rotary_turns", lib.b4_rotary_turns((ctypes.c_double * half)(*inv_freq), half, turns))
        self.dim, self.n_axes, self.adjacent, self.scale = dim, n_axes, bool(adjacent), float(scale)
        # signed: torch's int64 holds the same bits
        self.turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=device)
        self.axes = torch.tensor(axes, dtype=torch.uint8, device=device) if n_axes > 1 else None
        self.index = self.turns.get_device()
        if self.index >= 0:
            torch.cuda.current_stream(self.index).synchronize()        # there for every stream from here on
        self._c = RotaryTable(self.turns.data_ptr(), self.axes.data_ptr() if self.axes is not None else None, dim, n_axes,
                              ROTARY_ADJACENT if adjacent else 0, scale)
        self._ref = ctypes.byref(self._c)


def kv_append_rotary(cache, rotary: Rotary, q, k, v, positions, slots, out=None, stream=None):
    """b4_kv_append_rotary: q [tokens][heads][head_dim] (or None) and k [tokens][kv_heads][head_dim] rotated by positions,
    k and v quantised into the cache at slots.  q, k, v: all fp16, bf16 or fp32, any token and head strides, columns
    contiguous.  positions: int32 [tokens], or [axes][tokens] where the rotary has several.  Returns the rotated q:
    out, which may be q itself but lies on nothing else that the call reads, or a new tensor of q's type (fp16 for fp32)."""
    lib = _lib()
    index, n, dim, dtype = cache.index, slots.numel(), cache.head_dim, k.dtype
    if slots.dtype is not _int32 or slots.get_device() != index or not slots.is_contiguous():
        raise ValueError(f"slots: a contiguous int32 tensor on cuda:{index}")
    code = _codes.get(dtype)
    shape, ks, vs = (n, cache.kv_heads, dim), k.stride(), v.stride()
    if (code is None or v.dtype is not dtype or k.shape != shape or v.shape != shape or k.get_device() != index
            or v.get_device() != index or ks[2] != 1 or vs[2] != 1):
        raise ValueError(f"k and v: {shape}, both fp16, bf16 or fp32, on cuda:{index}, columns contiguous")
    if rotary.index != index or rotary.dim > dim:
        raise ValueError(f"rotary: {dim} columns at most, on cuda:{index}")
    axes, along = rotary.n_axes, positions.stride()
    if (positions.dtype is not _int32 or positions.get_device() != index
            or positions.shape != ((n,) if axes == 1 and len(along) == 1 else (axes, n)) or (n > 1 and along[-1] != 1)):
        raise ValueError(f"positions: int32 [{axes}][{n}] on cuda:{index}, an axis contiguous")
    along = along[0] if axes > 1 else n
    if along < n:
        raise ValueError("positions: axes must not overlap (an expanded tensor needs contiguous())")
    if q is None:
        if out is not None:
            raise ValueError("out: without q nothing is rotated into it")
        heads, qs, os, out_code, q_at, out_at = 0, (0, 0), (0, 0), DTYPE_F16 if code == DTYPE_F32 else code, 0, 0
    else:
        of_q, qs = q.shape, q.stride()
        if (len(of_q) != 3 or q.dtype is not dtype or of_q[0] != n or of_q[2] != dim or q.get_device() != index or qs[2] != 1):
            raise ValueError(f"q: [{n}][heads][{dim}] of k's type on cuda:{index}, columns contiguous")
        heads = of_q[1]
        if out is None:
            with _on(stream):
                out = _torch.empty(of_q, dtype=_float16 if code == DTYPE_F32 else dtype, device=q.device)
        out_code, os = _codes.get(out.dtype), out.stride()
        if (out.shape != of_q or out_code not in (DTYPE_F16, DTYPE_BF16) or (code != DTYPE_F32 and out_code != code)
                or out.get_device() != index or os[2] != 1):
            raise ValueError("out: as q, of its type (fp16 or bf16 for fp32), columns contiguous")
        q_at, out_at = q.data_ptr(), out.data_ptr()
    if _kv._device() != index:                 # the library launches on the current device
        with _torch.cuda.device(index):
            return kv_append_rotary(cache, rotary, q, k, v, positions, slots, out, stream)
    args = _ROWS.pack(q_at, k.data_ptr(), v.data_ptr(), out_at, positions.data_ptr(), slots.data_ptr(), along, qs[0], qs[1], ks[0], ks[1],
                      vs[0], vs[1], os[0], os[1], n, heads, code, out_code)
    status = lib.b4_kv_append_rotary(cache._ref, rotary._ref, args,
                                     stream.cuda_stream if stream is not None else _kv._raw_stream(index))
    if status:
        check("b4_kv_append_rotary", status)
    return out


def kv_box_bytes(head_dim: int) -> int:
    """Bytes of one kv head's box of a page."""
    n = ctypes.c_size_t(0)
    check("b4_kv_box_bytes", _kv.load().b4_kv_box_bytes(head_dim, ctypes.byref(n)))
    return n.value


def kv_new_boxes(cache):
    """Room for the boxes of a cache's pages: zeros, uint8 [pages][kv_heads][kv_box_bytes]."""
    _lib()
    return _torch.zeros((cache.n_pages, cache.kv_heads, kv_box_bytes(cache.head_dim)), dtype=_torch.uint8, device=cache.device)


def _boxes(cache, boxes):
    if (boxes.dtype is not _uint8 or boxes.shape != (cache.n_pages, cache.kv_heads, 2 * cache.head_dim + 16)
            or boxes.get_device() != cache.index or not boxes.is_contiguous()):
        raise ValueError(f"boxes: as kv_new_boxes makes them, on cuda:{cache.index}")


def kv_boxes(cache, boxes, slots, stream=None) -> None:
    """b4_kv_boxes: the boxes of the pages whose last token is among slots, into boxes (kv_new_boxes)."""
    lib = _lib()
    index = cache.index
    if slots.dtype is not _int32 or slots.get_device() != index or not slots.is_contiguous():
        raise ValueError(f"slots: a contiguous int32 tensor on cuda:{index}")
    _boxes(cache, boxes)
    if _kv._device() != index:
        with _torch.cuda.device(index):
            return kv_boxes(cache, boxes, slots, stream)
    status = lib.b4_kv_boxes(cache._ref, slots.data_ptr(), slots.numel(), boxes.data_ptr(),
                             stream.cuda_stream if stream is not None else _kv._raw_stream(index))
    if status:
        check("b4_kv_boxes", status)


class KVLists(NamedTuple):
    """Each query's pages of each kv head, int32 [tokens][kv_heads][keep], and the tokens that it sees of them, int32 [tokens]."""
    pages: object
    seen: object


_new_lists = tuple.__new__


def kv_select(cache, boxes, q, tables, ctx_len, q_starts, max_q: int, keep: int, first: int = 1, last: int = 1, out: KVLists | None = None,
              stream=None) -> KVLists:
    """b4_kv_select: for every query and kv head the `keep` pages that it reads: the first `first` and the last `last` of its
    request's up to its own place, and of the others those whose boxes bound its scores highest.  q, tables, ctx_len,
    q_starts and max_q as kv_attention takes them; out: buffers to reuse, none that the call reads.  Its time follows the
    tables' width: pass tables[:, :pages] where that is far beyond the longest context."""
    lib = _lib()
    index, dim, kv_heads, n = cache.index, cache.head_dim, cache.kv_heads, ctx_len.numel()
    code, shape, qs = _codes.get(q.dtype), q.shape, q.stride()
    if code is None or code == DTYPE_F32 or len(shape) != 3 or q.get_device() != index or shape[2] != dim or qs[2] != 1:
        raise ValueError(f"q: fp16 or bf16 [tokens][heads][{dim}] on cuda:{index}, columns contiguous")
    total, heads, _ = shape
    if heads % kv_heads:
        raise ValueError(f"heads: a multiple of {kv_heads}, got {heads}")
    if keep < 1 or first < 0 or last < 1 or first + last > keep:
        raise ValueError(f"keep {keep}: at least first {first} (0 or more) and last {last} (1 or more)")
    width, stride = _table(tables, index, n)
    if (ctx_len.dtype is not _int32 or ctx_len.get_device() != index or not ctx_len.is_contiguous() or q_starts.dtype is not _int32
            or q_starts.get_device() != index or not q_starts.is_contiguous() or q_starts.numel() <= n):
        raise ValueError(f"ctx_len and q_starts: contiguous int32 tensors on cuda:{index}, q_starts of {n + 1} values at least")
    _boxes(cache, boxes)
    if out is None:
        # (empty_like is the quickest: single tokens have as many rows as requests)
        with _on(stream):
            out = _new_lists(KVLists, (ctx_len.new_empty((total, kv_heads, keep)), _torch.empty_like(ctx_len) if total == n else ctx_len.new_empty(total)))
    else:
        _ints("out.pages", out.pages, index, 0)
        _ints("out.seen", out.seen, index, total)
        if out.pages.shape != (total, kv_heads, keep):
            raise ValueError(f"out.pages: [{total}][{kv_heads}][{keep}]")
    if _kv._device() != index:
        with _torch.cuda.device(index):
            return kv_select(cache, boxes, q, tables, ctx_len, q_starts, max_q, keep, first, last, out, stream)
    args = _CHOICE.pack(q.data_ptr(), boxes.data_ptr(), tables.data_ptr(), ctx_len.data_ptr(), q_starts.data_ptr(), out[0].data_ptr(),
                        out[1].data_ptr(), stride, qs[0], qs[1], width, n, total, max_q, heads, code, keep, first, last)
    status = lib.b4_kv_select(cache._ref, args, stream.cuda_stream if stream is not None else _kv._raw_stream(index))
    if status:
        check("b4_kv_select", status)
    return out


def _list_attn(cache, q, lists, scale, out, lse, stream=None):
    """A call's b4_kv_attn, packed, the lists' head stride, and its output."""
    index, dim, kv_heads = cache.index, cache.head_dim, cache.kv_heads
    code, shape, qs = _codes.get(q.dtype), q.shape, q.stride()
    if code is None or code == DTYPE_F32 or len(shape) != 3 or q.get_device() != index or shape[2] != dim or qs[2] != 1:
        raise ValueError(f"q: fp16 or bf16 [tokens][heads][{dim}] on cuda:{index}, columns contiguous")
    total, heads, _ = shape
    if heads % kv_heads:
        raise ValueError(f"heads: a multiple of {kv_heads}, got {heads}")
    pages, seen = lists
    of_lists = pages.shape
    if pages.dtype is not _int32 or pages.get_device() != index or len(of_lists) != 3 or of_lists[0] != total or of_lists[1] != kv_heads:
        raise ValueError(f"lists.pages: int32 [{total}][{kv_heads}][pages] on cuda:{index}")
    width = of_lists[2]
    along, across, one = pages.stride()
    if (width > 1 and one != 1) or (kv_heads > 1 and across < width) or (total > 1 and along < width):
        raise ValueError("lists.pages: entries contiguous, rows that do not overlap")
    if seen.dtype is not _int32 or seen.get_device() != index or not seen.is_contiguous() or seen.numel() < total:
        raise ValueError(f"lists.seen: a contiguous int32 tensor on cuda:{index}, {total} values at least")
    if out is None:
        with _on(stream):
            out = _torch.empty_like(q) if q.is_contiguous() else _torch.empty(shape, dtype=q.dtype, device=q.device)
    elif out.shape != shape or out.dtype is not q.dtype or out.get_device() != index or out.stride(2) != 1:
        raise ValueError("out: as q, columns contiguous")
    if lse is not None and (lse.shape != (total, heads) or lse.dtype is not _float32 or lse.get_device() != index
                            or not lse.is_contiguous()):
        raise ValueError("lse: contiguous fp32 [tokens][heads]")
    os = out.stride()
    args = _ATTN.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else 0, pages.data_ptr(), seen.data_ptr(), 0,
                      max(along, width), qs[0], qs[1], os[0], os[1], width, total, total, 1, heads, code, 0, 0,
                      dim ** -0.5 if scale is None else scale)
    return args, max(across, width), out


def kv_attention_lists_workspace(cache, q, lists: KVLists) -> int:
    """Bytes of workspace that kv_attention_lists needs for such a call (b4_kv_attention_lists_workspace)."""
    lib = _lib()
    n = ctypes.c_size_t(0)
    args, _, _ = _list_attn(cache, q, lists, None, q, None)
    with _torch.cuda.device(cache.index):  # whose SMs are counted
        check("b4_kv_attention_lists_workspace", lib.b4_kv_attention_lists_workspace(cache._ref, args, ctypes.byref(n)))
    return n.value


def kv_attention_lists(cache, q, lists: KVLists, scale: float | None = None, out=None, lse=None, ws=None, stream=None):
    """b4_kv_attention_lists: every query's attention over its own lists of pages, one for each kv head (kv_select's, or any
    others: page ids of the cache in the order of the tokens, of which the first lists.seen are seen).  The rest is as
    kv_attention: q and out [tokens][heads][head_dim] fp16 or bf16, scale None = head_dim ** -0.5, lse, ws and the package's
    workspace of the device.  Rows whose lists.seen is below 0 are left as they are.  Returns out, which may be q itself but
    lies on nothing else that the call reads."""
    lib = _lib()
    args, across, out = _list_attn(cache, q, lists, scale, out, lse, stream)
    if ws is None:
        ws = _workspace(cache.index, stream)
    elif ws.dtype is not _uint8 or ws.get_device() != cache.index or not ws.is_contiguous():
        raise ValueError(f"ws: a contiguous uint8 tensor on cuda:{cache.index}")
    if _kv._device() != cache.index:
        with _torch.cuda.device(cache.index):
            return kv_attention_lists(cache, q, lists, scale, out, lse, ws, stream)
    status = lib.b4_kv_attention_lists(cache._ref, args, across, ws.data_ptr(), ws.numel(),
                                       stream.cuda_stream if stream is not None else _kv._raw_stream(cache.index))
    if status:
        check("b4_kv_attention_lists", status)
    return out
