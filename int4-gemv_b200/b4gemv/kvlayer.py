"""The attention half of a decode layer in 4 bits throughout: q/k/v projections
(the 4-bit GEMVs), rotary embedding at the step's positions, the quantising
append, attention over the 4-bit pages, the o projection.

    layer = CachedAttention(FMT_NF4_B64, hidden=3584, heads=28, kv_heads=4, n_pages=1024, max_requests=16)
    y = layer.step(x, [17])          # x fp16 [17][hidden]: a prompt of 17 tokens
    y = layer.step(x, [1])           # its next token

Requests are the first len(added) rows of the layer's block tables; a step's
tokens are packed by request.  The host keeps nothing but max_tokens: lengths,
tables and the ring of free pages stay on the device.
"""
from __future__ import annotations

from . import FMT_INT4_G128, FMT_NF4_B64, gemv_ws, quantise_device, quantise_nf4_device
from .kv import KV_INT4, KV_NF4, KVCache, kv_append, kv_attention, kv_tables

ROWS = 16                # of a GEMV call at most


def rotate(x, positions, base: float = 1e6):
    """Rotary embedding of fp32 x [tokens][heads][dim], halves paired."""
    import torch
    half = x.shape[2] // 2
    angle = positions[:, None].double() * base ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


class CachedAttention:
    def __init__(self, fmt: int, hidden: int, heads: int, kv_heads: int, n_pages: int, max_requests: int, head_dim: int = 128,
                 page_size: int = 64, max_context: int = 4096, seed: int = 0, device="cuda"):
        import torch
        if fmt not in (FMT_INT4_G128, FMT_NF4_B64):
            raise ValueError("fmt: FMT_INT4_G128 or FMT_NF4_B64")
        self.fmt, self.heads, self.kv_heads, self.dim = fmt, heads, kv_heads, head_dim
        g = torch.Generator(device=device).manual_seed(seed)
        quant = quantise_nf4_device if fmt == FMT_NF4_B64 else quantise_device
        self.weights = {}
        for name, out_f, in_f in (("q", heads * head_dim, hidden), ("k", kv_heads * head_dim, hidden),
                                  ("v", kv_heads * head_dim, hidden), ("o", hidden, heads * head_dim)):
            w = torch.randn((out_f, in_f), generator=g, device=device) * in_f ** -0.5
            self.weights[name] = quant(w)[:2]
        self.cache = KVCache.alloc(KV_NF4 if fmt == FMT_NF4_B64 else KV_INT4, n_pages, kv_heads, page_size, head_dim, device)
        ints = dict(dtype=torch.int32, device=device)
        self.tables = torch.full((max_requests, -(-max_context // page_size)), -1, **ints)
        self.cached = torch.zeros(max_requests, **ints)
        self.free = torch.arange(n_pages, **ints)
        self.free_state = torch.tensor([0, n_pages, 0], **ints)

    def _project(self, name, x):
        import torch
        qw, scale = self.weights[name]
        y = torch.empty((x.shape[0], qw.shape[0]), dtype=torch.float32, device=x.device)
        for at in range(0, x.shape[0], ROWS):
            gemv_ws(self.fmt, qw, scale, x[at:at + ROWS], y[at:at + ROWS])
        return y

    def step(self, x, added):
        """x fp16 [sum(added)][hidden], added: new tokens of each request (0 or more); returns fp32 [sum(added)][hidden]."""
        import torch
        n, total = len(added), x.shape[0]
        if total != sum(added) or n > self.cached.numel() or min(added, default=0) < 0:
            raise ValueError(f"x: {sum(added)} rows, {self.cached.numel()} requests at most, of 0 tokens or more")
        more = torch.tensor(list(added), dtype=torch.int32, device=x.device)
        step = kv_tables(self.cache.page_size, self.tables[:n], self.cached[:n], more, self.free, self.free_state, total)
        q, k, v = (self._project(name, x).view(total, h, self.dim) for name, h in
                   (("q", self.heads), ("k", self.kv_heads), ("v", self.kv_heads)))
        kv_append(self.cache, rotate(k, step.positions), v, step.slots)
        out = kv_attention(self.cache, rotate(q, step.positions).half(), self.tables[:n], step.ctx_len, step.q_starts,
                           max(added, default=0))
        self.cached[:n] = step.ctx_len
        self.free_state = step.free_state
        return self._project("o", out.view(total, self.heads * self.dim))
