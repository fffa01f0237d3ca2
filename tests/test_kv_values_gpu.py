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


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 4, 90])
@pytest.mark.parametrize("late", [False, True])
def test_a_token_that_counts_beside_larger_values_that_do_not(cuda, fmt, new, late):
    """One token takes the whole weight; its value scale is 2^18 below the others'."""
    ctx, heads, kvh, d = 200, 8, 2, 128
    state = make(cuda, fmt, F16, heads, kvh, d, 16, [ctx], [new])
    cache, q, tab, lens, starts, most = state
    at = ctx - new - 1 if late else 0                            # seen by every query
    tl = tab.cpu().numpy()[0]
    page, row = tl[at // 16], at % 16
    key = b4gemv.kv_read(cache, torch.tensor([page * 16 + row], dtype=torch.int32, device=cuda))[0][0]
    key = key / key.norm(dim=-1, keepdim=True) * 45 * d ** 0.5
    q.copy_(key.repeat_interleave(heads // kvh, 0).half().expand_as(q))

    def change(k, v):
        norm = k[page, :, row].copy()
        k[:] = 0                               # scores of 0
        k[page, :, row] = norm
        v[:] = 2.0 ** 10
        v[page, :, row] = 1.3701171875 * 2.0 ** -8

    set_scales(cache, fmt, 16, d, change)
    want, _, (weight, size) = ref.attention(fmt, 16, d, cache.blocks, q, tab, [ctx], starts.tolist(), d ** -0.5)
    assert float(size.amin()) > 40             # so the others weigh e^-40, 2^-57, each: 2^-47 of their value scale
    got = b4gemv.kv_attention(*state)
    # a rounding of the weight to fp16 and of the output; of NF4's levels (1e-4); 2^-32 of 2^11 for a product below fp16's
    # normal numbers, times the level
    level = 8 if fmt == INT4 else 1
    tol = weight * (2.0 ** -11 + 2.0 ** -16 + (1e-4 if fmt == NF4 else 0)) + want.abs() * 2.0 ** -11 + level * 2.0 ** -21
    if fmt == NF4:
        tol = tol + 2.0 ** -8 * 1e-4           # a level's rounding is relative to the scale
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
