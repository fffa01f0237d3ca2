"""Attention over the 4-bit cache for batches drawn at random: how the work is split over CTAs and warps depends on every
length of the batch, so many small different ones, and the largest group, against 64 bits."""
import numpy as np
import pytest
import torch

import b4gemv
from test_kv_gpu import BF16, F16, INT4, NF4, check_attention, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(24))
def test_drawn_batches(cuda, seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 30))
    d, page = int(rng.choice([64, 128])), int(rng.choice([16, 32, 64]))
    kvh, group = int(rng.integers(1, 5)), int(rng.choice([1, 2, 3, 5, 7, 8, 9, 16, 20]))
    kind = seed % 4                                              # single tokens, drafts, prompts, all of them
    new = {0: np.ones(n), 1: rng.integers(0, 9, n), 2: rng.integers(1, 400, n),
           3: np.where(rng.random(n) < 0.5, 1, rng.integers(0, 300, n))}[kind].astype(int)
    ctx = np.where(rng.random(n) < 0.3, new, new + rng.integers(0, 900, n))
    ctx = np.where(rng.random(n) < 0.1, rng.integers(0, 40, n), ctx)               # some shorter than their queries
    window = int(rng.integers(1, 500)) if seed % 5 == 4 else 0
    check_attention(cuda, int(rng.integers(0, 2)), F16 if seed & 1 else BF16, kvh * group, kvh, d, page, ctx.tolist(), new.tolist(),
                    window=window, causal=bool(window or seed % 7 != 6), seed=seed)
    assert b4gemv.load().b4_device_error(0) == 0


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("group,new", [(64, 1), (64, 5), (3, 43), (11, 12)])
def test_large_groups_and_odd_rows(cuda, fmt, group, new):
    """64 heads over one; row tiles of 129 and 132 rows, whose second half is nearly empty."""
    check_attention(cuda, fmt, F16, group, 1, 128, 16, [700, 64, 131], [new, min(new, 64), new])


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("ctx,new", [([9000, 4000], [1, 1]), ([3000, 2000, 700], [5, 70, 300]), ([400] * 20, [9] * 20)])
def test_same_bits_every_time(cuda, fmt, ctx, new):
    """Segments that cross warps and CTAs are added up in their order, whichever arrives last."""
    cache, q, tab, lens, starts, most = make(cuda, fmt, BF16, 16, 2, 128, 32, ctx, new)
    first = b4gemv.kv_attention(cache, q, tab, lens, starts, most)
    for _ in range(20):
        assert torch.equal(first, b4gemv.kv_attention(cache, q, tab, lens, starts, most))


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("new", [1, 4, 150])
def test_scales_of_no_and_other_sign(cuda, scale, new):
    for fmt, dtype in ((INT4, F16), (NF4, BF16)):
        check_attention(cuda, fmt, dtype, 8, 2, 128, 32, [200, 333], [new, min(new, 200)], scale=scale)
