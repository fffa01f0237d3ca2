"""NF4 with fp16 queries: both fp16 parts of a level count, in keys and in values, for few queries and for many."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_ref as ref
from test_kv_gpu import F16, NF4, check_attention, make

pytestmark = pytest.mark.gpu
N = 64                                         # tokens, alike in weight


def cancelling(rng, columns):
    """Codes [N][columns] of three levels a column that sum to nearly nothing, in an order of chance: the output is so small
    that its own rounding hides nothing, while the levels' roundings, were they those of fp16 alone, leave 1.5e-5."""
    lev = ref.NF4.astype(np.float64)
    ups = [1.67766535282135, 1.6775788]        # factors that the levels may be rounded with
    eps = [(np.float32(u) * ref.NF4).astype(np.float16).astype(np.float64) / np.float32(u) - lev for u in ups]
    found = []
    i, j = np.meshgrid(np.arange(1, N), np.arange(1, N), indexing="ij")
    ok = i + j < N
    counts = np.stack([i[ok], j[ok], N - i[ok] - j[ok]], 1)
    for a in range(16):
        for b in range(a + 1, 16):
            for c in range(b + 1, 16):
                mean = counts @ lev[[a, b, c]] / N
                lost = np.minimum(*(np.abs(counts @ e[[a, b, c]]) / N for e in eps))
                for n in counts[(np.abs(mean) < 1e-3) & (lost > 1.5e-5)]:
                    found.append(np.repeat([a, b, c], n))
    assert len(found) > 100
    return np.stack([rng.permutation(found[k]) for k in rng.integers(len(found), size=columns)], 1).astype(np.uint8)


@pytest.mark.parametrize("group,new", [(1, 1), (8, 1), (16, 1), (8, 20), (4, 100)])
@pytest.mark.parametrize("d,page", [(128, 64), (128, 16), (64, 32)])
def test_levels_of_values(cuda, group, new, d, page):
    rng = np.random.default_rng(d + page + group)
    kvh, pages = 3, N // page
    codes = rng.integers(0, 16, (2, pages, kvh, page, d)).astype(np.uint8)
    v = np.stack([cancelling(rng, d) for _ in range(kvh)])                                  # [head][token][column]
    codes[1] = v.reshape(kvh, pages, page, d).transpose(1, 0, 2, 3)
    scales = np.ones((2, pages, kvh, page), np.float32)
    cache = b4gemv.KVCache(torch.from_numpy(ref.pack_blocks(NF4, codes, scales)).to(cuda), NF4, page, d)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.zeros((new, kvh * group, d), dtype=torch.float16, device=cuda)
    got = b4gemv.kv_attention(cache, q, t([list(range(pages))]), t([N]), t([0, new]), new, causal=False).cpu().numpy().astype(np.float64)
    want = np.repeat(ref.NF4.astype(np.float64)[v].mean(1), group, 0)
    # a level in two parts is off by 2^-22; a product of 16 tokens adds to a sum of fewer than 32 levels, off by 2^-22 of it,
    # and N / 8 of them make the sum of N: 2^-20; the output is rounded once
    assert bool((np.abs(got - want) <= 2.0 ** -22 + 2.0 ** -20 + np.abs(want) * 2.0 ** -11).all())


@pytest.mark.parametrize("group,new", [(1, 1), (8, 1), (16, 1), (8, 20), (4, 100)])
@pytest.mark.parametrize("d,page", [(128, 64), (128, 16), (64, 32)])
def test_levels_of_keys(cuda, group, new, d, page):
    """Requests of one key: the log-sum-exp is its score, queries of ones make it the sum of its levels."""
    rng = np.random.default_rng(d + page + group + new)
    kvh, n = 2, 9
    codes = rng.integers(0, 16, (2, n, kvh, page, d)).astype(np.uint8)
    k = np.concatenate([cancelling(rng, n * kvh) for _ in range(d // N)]).T.reshape(n, kvh, d)
    codes[0, :, :, 0] = k
    cache = b4gemv.KVCache(torch.from_numpy(ref.pack_blocks(NF4, codes, np.ones((2, n, kvh, page), np.float32))).to(cuda), NF4, page, d)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.ones((n * new, kvh * group, d), dtype=torch.float16, device=cuda)
    lse = torch.empty(q.shape[:2], device=cuda)
    b4gemv.kv_attention(cache, q, t(range(n)).view(n, 1), t([1] * n), t(range(0, n * new + 1, new)), new, scale=1.0, causal=False, lse=lse)
    want = np.repeat(np.repeat(ref.NF4.astype(np.float64)[k].sum(-1), group, 1), new, 0)
    # as above, summed: a level 2^-22, D / 8 products 2^-22 of 32 levels each; fp16 alone would leave 1e-3 for 64 columns
    assert bool((np.abs(lse.cpu().numpy() - want) <= d * 2.0 ** -22 + d / 8 * 32 * 2.0 ** -22 + 2.0 ** -20).all())


@pytest.mark.parametrize("d,heads,kvh", [(128, 16, 2), (64, 28, 4)])
@pytest.mark.parametrize("ctx,new", [([9000, 4000], [1, 1]), ([3000, 2000, 700], [5, 70, 300]), ([400] * 20, [9] * 20), ([1500, 90], [1500, 90])])
def test_same_bits_every_time(cuda, d, heads, kvh, ctx, new):
    """Levels in two parts have their own order of barriers: the same bits whatever it comes to."""
    state = make(cuda, NF4, F16, heads, kvh, d, 32, ctx, new)
    first = check_attention(cuda, NF4, F16, heads, kvh, d, 32, ctx, new, state=state).clone()
    for _ in range(20):
        assert torch.equal(first, b4gemv.kv_attention(*state))
