"""The rotated append, the boxes, the choice of pages and attention over lists, restated in numpy / 64-bit torch from their
definitions for their tests."""
from __future__ import annotations

import numpy as np
import torch

import kv_ref as ref

U32 = np.float32


def turns(inv_freq):
    """A position's part of a turn as whole numbers of 2^-64, by Python's integers from the fp64 quotient."""
    out = []
    for f in inv_freq:
        num, den = (float(f) / 6.283185307179586).as_integer_ratio()
        t, rest = divmod(abs(num) << 64, den)
        t += 2 * rest > den or (2 * rest == den and t & 1)
        out.append((t if num >= 0 else -t) % (1 << 64))
    return out


def angles(positions, axes, inv_freq):
    """fp64 radians [tokens][pairs]: positions int [axes][tokens]."""
    out = np.empty((positions.shape[1], len(inv_freq)))
    for i, (t, a) in enumerate(zip(turns(inv_freq), axes)):
        for j, p in enumerate(positions[a].tolist()):
            whole = p * t % (1 << 64)
            out[j, i] = (whole - (1 << 64) if whole >> 63 else whole) / float(1 << 63) * np.pi
    return out


def rotate(x, angle, adjacent, scale=1.0):
    """float64 [tokens][heads][D] with the first 2 * pairs columns turned."""
    x = np.asarray(x, np.float64).copy()
    half = angle.shape[1]
    c, s = np.cos(angle)[:, None] * scale, np.sin(angle)[:, None] * scale
    at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if adjacent else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., at[0]].copy(), x[..., at[1]].copy()
    with np.errstate(all="ignore"):
        x[..., at[0]], x[..., at[1]] = a * c - b * s, b * c + a * s
    return x


def boxes(fmt, page, d, blocks):
    """uint8 [n][heads][2 d + 16] of pages [n][heads][block bytes]."""
    codes, s = ref.unpack_blocks(fmt, page, d, blocks)
    k = ref.values(fmt, codes[0], s[0])
    out = np.zeros(k.shape[:2] + (2 * d + 16,), np.uint8)
    with np.errstate(all="ignore"):
        hi = np.where(np.isnan(k), -np.inf, k).max(-2).astype(U32)
        lo = np.where(np.isnan(k), np.inf, k).min(-2).astype(U32)
        none = hi < lo
        hi, lo = np.where(none, U32(0), hi), np.where(none, U32(0), lo)
        box = np.concatenate([hi, lo], -1)
        top = np.abs(box).max(-1, keepdims=True)
        unit = np.where(top > 0, top * (U32(1) / U32(127)), U32(1)).astype(U32)
        codes = int8(box, unit)
    out[..., : 2 * d] = codes.view(np.uint8)
    out[..., 2 * d: 2 * d + 4] = np.ascontiguousarray(unit).view(np.uint8)
    return out


def int8(x, unit):
    q = (x / unit).astype(U32)
    return np.clip(np.rint(np.where(np.isnan(q), U32(0), q)), -127, 127).astype(np.int8)


def scores(d, box, q):
    """fp32 [tokens][pages] of q [tokens][group][D] (fp32) over boxes [pages][2 d + 16]."""
    x = q.astype(np.float64)
    with np.errstate(all="ignore"):
        s = np.concatenate([np.where(x > 0, x, 0).sum(1), np.where(x > 0, 0, x).sum(1)], -1).astype(U32)
        finite = np.isfinite(s).all(-1)
        s[~finite] = 0
        top = np.abs(s).max(-1, keepdims=True)
        codes = int8(s, np.where(top > 0, top * (U32(1) / U32(127)), U32(1)).astype(U32))
        unit = np.ascontiguousarray(box[:, 2 * d: 2 * d + 4]).view(U32)[:, 0]
        dot = codes.astype(np.int64) @ np.ascontiguousarray(box[:, : 2 * d]).view(np.int8).astype(np.int64).T
        return np.where(np.isfinite(unit), dot.astype(U32) * np.where(np.isfinite(unit), unit, 0).astype(U32), U32(np.inf))


def select(page, d, box, q, tab, ctx_len, q_starts, keep, first, last, n_pages, seen=None):
    """(lists [tokens][kv heads][keep], seen [tokens]); rows of no request keep what they hold: -7, -1 in seen."""
    total, heads = q.shape[:2]
    kvh, group, width = box.shape[1], heads // box.shape[1], tab.shape[1]
    lists, seen = np.full((total, kvh, keep), -7, np.int32), np.full(total, -1, np.int32)
    x = q.float().cpu().numpy()
    for r in range(len(ctx_len)):
        a, b, ctx = int(q_starts[r]), int(q_starts[r + 1]), max(int(ctx_len[r]), 0)
        there = (tab[r] >= 0) & (tab[r] < n_pages)
        ids = np.where(there, tab[r], -1)
        for h in range(kvh):
            s = scores(d, box[np.where(there, ids, 0), h], x[a:b, h * group:(h + 1) * group]) if b > a and width else None
            for t in range(a, b):
                visible = min(ctx - (b - a) + t - a + 1, width * page)
                row = np.full(keep, -1, np.int32)
                seen[t] = 0
                if visible > 0:
                    c = -(-visible // page)
                    take = np.arange(c)
                    if c > keep:
                        middle = np.arange(first, c - last)
                        value = s[t - a][middle].astype(np.float64)
                        value[value == 0] = 0                                    # no -0
                        value = np.where(there[middle], value, -np.inf)
                        # a missing page is behind every other, those at -infinity too
                        order = np.lexsort((middle, -value, ~there[middle]))
                        take = np.concatenate([np.arange(first), np.sort(middle[order[: keep - first - last]]), np.arange(c - last, c)])
                    row[: len(take)] = ids[take]
                    seen[t] = (len(take) - 1) * page + visible - (c - 1) * page
                lists[t, h] = row
    return lists, seen


def attention(fmt, page, d, blocks, q, lists, seen, scale):
    """(out, lse, bound) as kv_ref.attention: every query and kv head a request over its own list."""
    total, heads = q.shape[:2]
    kvh = blocks.shape[1]
    group = heads // kvh
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -np.inf, dtype=torch.float64, device=q.device)
    weight, size = torch.zeros_like(out), torch.zeros_like(lse)
    ones = np.arange(total + 1)
    for h in range(kvh):
        at = slice(h * group, (h + 1) * group)
        o, l, (w, s) = ref.attention(fmt, page, d, blocks[:, h:h + 1].contiguous(), q[:, at], torch.as_tensor(lists[:, h]), np.maximum(seen, 0), ones, scale)
        out[:, at], lse[:, at], weight[:, at], size[:, at] = o, l, w, s
    return out, lse, (weight, size)
