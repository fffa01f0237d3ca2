"""Cached values at the ends of what a scale can be."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_ref as ref
from test_kv_gpu import F16, INT4, NF4, bounds, make

pytestmark = pytest.mark.gpu


def set_scales(cache, fmt, page, d, change):
    """change(key scales, value scales), fp32 [pages][heads][page] each, written back."""
    codes, s = ref.unpack_blocks(fmt, page, d, cache.blocks.cpu().numpy())
    s = s.astype(np.float32)
    change(s[0], s[1])
    cache.blocks.copy_(torch.from_numpy(ref.pack_blocks(fmt, codes.copy(), s)))


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [2, 4, 90])
@pytest.mark.parametrize("size", [1e-3, 1.0, 100.0])
def test_infinite_values_stay_with_the_queries_that_see_them(cuda, fmt, new, size):
    """The last token's values are infinite: only the last query sees them, whatever the other values' size."""
    ctx = [40, 200, 91] if new < 40 else [190, 200, 91]
    state = make(cuda, fmt, F16, 8, 2, 128, 16, ctx, [new] * 3)
    cache, q, tab, lens, starts, most = state

    def scaled(k, v):
        v *= size

    set_scales(cache, fmt, 16, 128, scaled)
    want, wl, aux = ref.attention(fmt, 16, 128, cache.blocks, q, tab, ctx, starts.tolist(), 128 ** -0.5)
    tl = tab.cpu().numpy()

    def infinite(k, v):
        for r, c in enumerate(ctx):
            v[tl[r, (c - 1) // 16], :, (c - 1) % 16] = np.inf

    set_scales(cache, fmt, 16, 128, infinite)
    got = b4gemv.kv_attention(*state)
    last = torch.zeros(q.shape[0], dtype=torch.bool, device=cuda)
    last[(starts[1:] - 1).long()] = True
    tol, _ = bounds(fmt, F16, want, wl, aux, max(ctx))
    assert bool(((got.double() - want).abs() <= tol)[~last].all())
    assert not bool(torch.isfinite(got[last]).any())


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [2, 4, 90])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_unusable_keys_stay_with_the_queries_that_see_them(cuda, fmt, new, bad):
    ctx = [40, 200, 91] if new < 40 else [190, 200, 91]
    state = make(cuda, fmt, F16, 8, 2, 128, 16, ctx, [new] * 3)
    cache, q, tab, lens, starts, most = state
    want, wl, aux = ref.attention(fmt, 16, 128, cache.blocks, q, tab, ctx, starts.tolist(), 128 ** -0.5)
    tl = tab.cpu().numpy()

    def spoilt(k, v):
        for r, c in enumerate(ctx):
            k[tl[r, (c - 1) // 16], :, (c - 1) % 16] = bad

    set_scales(cache, fmt, 16, 128, spoilt)
    got = b4gemv.kv_attention(*state)
    rows = torch.ones(q.shape[0], dtype=torch.bool, device=cuda)
    rows[(starts[1:] - 1).long()] = False
    tol, _ = bounds(fmt, F16, want, wl, aux, max(ctx))
    assert bool(((got.double() - want).abs() <= tol)[rows].all())
