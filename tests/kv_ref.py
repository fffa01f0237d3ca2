"""The 4-bit key/value cache restated in numpy / 64-bit torch for its tests: the
block layout, the quantisers, the step's bookkeeping and attention, each from
its definition."""
from __future__ import annotations

import numpy as np
import torch

NF4 = np.array([-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
                -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
                0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941,
                0.7229568362236023, 1.0], np.float32)
INT4, NF = 0, 1


def scale_bytes(fmt):
    return 2 if fmt == INT4 else 4


def quantise(fmt, x):
    """fp32 [..., D] -> (codes uint8 [..., D], scales [...] as fp16 / fp32), the weight quantisers' steps in fp32."""
    with np.errstate(all="ignore"):
        a = np.abs(x)
        amax = np.where(np.isnan(a), np.float32(0), a).max(-1).astype(np.float32)
        if fmt == INT4:
            s = np.where(amax > 0, amax * (np.float32(1) / np.float32(7)), np.float32(1)).astype(np.float16)
            q = (x / s.astype(np.float32)[..., None]).astype(np.float32)
            ok = np.abs(q) < np.float32(2.0 ** 63)
            d = np.where(ok, q, 0).astype(np.float64)
            codes = np.where(ok, np.clip(np.sign(d) * np.floor(np.abs(d) + 0.5) + 8, 0, 15), 8)
            return codes.astype(np.uint8), s
        s = np.where(amax > 0, amax, np.float32(1)).astype(np.float32)
        q = (x / s[..., None]).astype(np.float32)
        best = np.zeros(q.shape, np.uint8)
        bd = np.abs(q - NF4[0])
        for c in range(1, 16):
            d = np.abs(q - NF4[c])
            take = d < bd
            best[take] = c
            bd = np.where(take, d, bd)
        return best, s


def values(fmt, codes, s):
    with np.errstate(all="ignore"):
        lev = (np.arange(16) - 8).astype(np.float32) if fmt == INT4 else NF4
        return lev[codes] * s.astype(np.float32)[..., None]


def unpack_blocks(fmt, page, d, blocks):
    """uint8 [pages][heads][block] -> codes uint8 [2][pages][heads][page][d], scales [2][pages][heads][page]."""
    b = np.asarray(blocks)
    n, h, size = b.shape
    sb = scale_bytes(fmt)
    assert size == 2 * page * (d // 2 + sb)
    c = b[..., : page * d].reshape(n, h, 2, page, d // 2).transpose(2, 0, 1, 3, 4)
    codes = np.stack([c & 15, c >> 4], -1).reshape(2, n, h, page, d)
    s = np.ascontiguousarray(b[..., page * d:]).view(np.float16 if fmt == INT4 else np.float32).reshape(n, h, 2, page)
    return codes, s.transpose(2, 0, 1, 3)


def pack_blocks(fmt, codes, s):
    """The inverse of unpack_blocks."""
    _, n, h, page, d = codes.shape
    c = (codes[..., 0::2] | codes[..., 1::2] << 4).transpose(1, 2, 0, 3, 4).reshape(n, h, page * d)
    t = np.ascontiguousarray(s.transpose(1, 2, 0, 3).astype(np.float16 if fmt == INT4 else np.float32))
    return np.concatenate([c, t.view(np.uint8).reshape(n, h, -1)], -1)


def tables(page, tab, cached, added, ring, state, max_tokens):
    tab = tab.copy()
    width = tab.shape[1]
    ctx, starts, slots, pos = [], [0], [], []
    head = state[0] % len(ring) if len(ring) else 0
    left, taken, missing = min(max(state[1], 0), len(ring)), 0, 0
    for r, (c, a) in enumerate(zip(cached, added)):
        c, a = max(int(c), 0), max(int(a), 0)
        held, need = min(-(-c // page), width), min(-(-(c + a) // page), width)
        for p in range(held, need):
            if taken < left:
                tab[r, p] = ring[(head + taken) % len(ring)]
                taken += 1
            else:
                tab[r, p] = -1
                missing += 1
        for i in range(a):
            p = (c + i) // page
            ok = p < width and tab[r, p] >= 0
            slots.append(tab[r, p] * page + (c + i) % page if ok else -1)
            pos.append(c + i)
        ctx.append(c + a)
        starts.append(starts[-1] + a)
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    pos = (pos + [0] * max_tokens)[:max_tokens]
    out = [(head + taken) % len(ring) if len(ring) else 0, left - taken, missing]
    return (tab, *(np.array(v, np.int32) for v in (ctx, starts, slots, pos, out)))


def attention(fmt, page, d, blocks, q, tab, ctx_len, q_starts, scale, window=0, full=False):
    """(out, lse, bound) in 64 bits; bound: how far an output may be, per unit of the weights' and the scores' relative errors:
    the sum of p |v|, and the largest sum of |scale q k| of a row."""
    dev = q.device
    codes, s = unpack_blocks(fmt, page, d, blocks.cpu().numpy())
    lev = torch.tensor((np.arange(16) - 8).astype(np.float64) if fmt == INT4 else NF4.astype(np.float64), device=dev)
    codes, s = torch.from_numpy(np.ascontiguousarray(codes)).to(dev), torch.from_numpy(np.ascontiguousarray(s)).to(dev).double()
    heads, kvh, n_pages = q.shape[1], codes.shape[2], codes.shape[1]
    group = heads // kvh
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:2], -np.inf, dtype=torch.float64, device=dev)
    weight = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    size = torch.zeros(q.shape[:2], dtype=torch.float64, device=dev)
    for r in range(len(ctx_len)):
        a, b, ctx = int(q_starts[r]), int(q_starts[r + 1]), min(max(int(ctx_len[r]), 0), tab.shape[1] * page)
        n = b - a
        if n <= 0 or ctx == 0:
            continue
        ids = tab[r, : -(-ctx // page)].long().to(dev)
        there = ((ids >= 0) & (ids < n_pages)).repeat_interleave(page)[:ctx]
        ids = ids.clamp(0, n_pages - 1)
        for h in range(kvh):
            k, v = (lev[codes[o, ids, h].reshape(-1, d)[:ctx].long()] * s[o, ids, h].reshape(-1)[:ctx, None] for o in (0, 1))
            place = torch.arange(ctx, device=dev)
            end = torch.arange(n, device=dev) + (ctx - n + 1) if not full else torch.full((n,), ctx, device=dev)
            seen = (place[None] < end[:, None]) & there[None]
            if window:
                seen &= place[None] >= end[:, None] - window
            k, v = (torch.where(seen.any(0)[:, None], t, torch.zeros((), dtype=t.dtype, device=dev)) for t in (k, v))
            x = q[a:b, h * group:(h + 1) * group].double()
            sc = torch.einsum("ngd,kd->ngk", x, k) * scale
            sc = sc.masked_fill(~seen[:, None], -np.inf)
            m = sc.amax(-1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(sc - m)
            total = p.sum(-1, keepdim=True)
            p = p / total.clamp(min=1e-300)
            at = (slice(a, b), slice(h * group, (h + 1) * group))
            out[at] = torch.einsum("ngk,kd->ngd", p, v)
            weight[at] = torch.einsum("ngk,kd->ngd", p, v.abs())
            lse[at] = torch.where(total[..., 0] > 0, m[..., 0] + torch.log(total[..., 0]), -np.inf)
            size[at] = (torch.einsum("ngd,kd->ngk", x.abs(), k.abs()) * abs(scale)).masked_fill(~seen[:, None], 0).amax(-1)
    return out, lse, (weight, size)
