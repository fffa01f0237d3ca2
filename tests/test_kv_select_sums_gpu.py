"""The sums of a choice's queries where bf16's range decides a code: columns whose sum in 64 bits, rounded to fp32, lies one
step above a border between codes, for a term that 48 bits do not hold beside the largest."""
import numpy as np
import pytest
import torch

from test_kv_select_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [3, 8, 11, 64])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 5, 20])
def test_terms_of_unlike_size(cuda, group, d, new):
    """A column's heads hold m + 1/2 with m even, half of its fp32 step and 2^-48, in any order: 50 bits, so the sum in 64 bits is exact
    whatever its order, and rounds to fp32 away from the tie.  A head of 127 in column 0 makes the unit 1."""
    assert np.float32(127) * (np.float32(1) / np.float32(127)) == 1
    rng = np.random.default_rng(group + d + new)
    s = make(cuda, torch.bfloat16, group, 1, d, 16, [16 * 200 + new], [new])
    q = np.zeros((new, group, d))
    for t in range(new):
        for c in range(1, d):
            m = 2 * int(rng.integers(1, 32))
            half = 2.0 ** (int(np.log2(m + 0.5)) - 24)
            heads = rng.permutation(group)[:3]
            q[t, heads, c] = np.array([m + 0.5, half, 2.0 ** -48]) * (1 if rng.random() < 0.5 else -1)
        q[t, rng.integers(group), 0] = 127
    s["q"].copy_(torch.from_numpy(q))
    assert np.array_equal(s["q"].double().cpu().numpy(), q)                # bf16 holds every term
    check(cuda, s, 20, 0, 1)
