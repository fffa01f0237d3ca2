"""Requests that have outgrown their row of the block table: keys past it are masked like missing pages, the queries stay at
their places among all of the request's tokens."""
import pytest
import torch

import b4gemv
import kv_ref as ref
from test_kv_gpu import BF16, F16, INT4, NF4, bounds, make

pytestmark = pytest.mark.gpu


def check(cuda, fmt, dtype, heads, kvh, d, page, width, ctx, new, window=0, causal=True):
    cache, q, tab, lens, starts, most = make(cuda, fmt, dtype, heads, kvh, d, page, ctx, new)
    lse = torch.empty(q.shape[:2], device=cuda)
    got = b4gemv.kv_attention(cache, q, tab[:, :width], lens, starts, most, window=window, causal=causal, lse=lse)
    full = tab.clone()
    full[:, width:] = -1                       # the same keys, as pages that are missing
    want, wl, aux = ref.attention(fmt, page, d, cache.blocks, q, full, ctx, starts.tolist(), d ** -0.5, window, not causal)
    tol, ltol = bounds(fmt, dtype, want, wl, aux, width * page)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert torch.equal(torch.isinf(lse), torch.isinf(wl))
    seen = ~torch.isinf(wl)
    assert bool(((lse.double() - wl)[seen].abs() <= ltol[seen]).all())


@pytest.mark.parametrize("fmt,dtype", [(INT4, F16), (NF4, BF16)])
@pytest.mark.parametrize("new", [[10, 1, 3, 8, 64], [1] * 5, [70, 64, 65, 200, 30]])
@pytest.mark.parametrize("window", [0, 7, 100])
def test_past_the_table(cuda, fmt, dtype, new, window):
    check(cuda, fmt, dtype, 8, 2, 128, 16, 4, [70, 64, 65, 300, 64], new, window)
    check(cuda, fmt, dtype, 12, 1, 64, 64, 3, [400, 192, 193, 1000, 191], new, window)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 6, 150])
def test_every_key_that_the_table_holds(cuda, fmt, new):
    check(cuda, fmt, F16, 8, 2, 128, 32, 5, [161, 700, 160, 33], [new, new, new, min(new, 33)], causal=False)


def test_a_step_past_the_table(cuda):
    """cached + added beyond the table's pages, as kv_tables leaves it: the first of ten new tokens sees all before it."""
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    cache = b4gemv.KVCache.alloc(INT4, 4, 1, 16, 64, cuda)
    tab, ring = t([[-1] * 4]), t([2, 0, 3, 1])
    k, v = (torch.randn((70, 1, 64), device=cuda) for _ in range(2))
    a = b4gemv.kv_tables(16, tab, t([0]), t([60]), ring, t([0, 4, 0]), 60)
    b4gemv.kv_append(cache, k[:60], v[:60], a.slots)
    b = b4gemv.kv_tables(16, tab, a.ctx_len, t([10]), ring, a.free_state, 10)
    assert b.slots.tolist()[:4] == [tab[0, 3].item() * 16 + 12 + i for i in range(4)] and b.slots.tolist()[4:] == [-1] * 6
    b4gemv.kv_append(cache, k[60:], v[60:], b.slots)
    kc, vc = b4gemv.kv_read(cache, torch.cat([a.slots, b.slots[:4]]))
    q = torch.randn((10, 1, 64), device=cuda).half()
    out = b4gemv.kv_attention(cache, q, tab, b.ctx_len, b.q_starts, 10)
    for i in range(10):
        n = min(61 + i, 64)
        p = torch.softmax((kc[:n, 0].double() @ q[i, 0].double()) / 8, 0)
        want = p @ vc[:n, 0].double()
        assert bool(((out[i, 0].double() - want).abs() <= 2 ** -9 * (p @ vc[:n, 0].double().abs())).all())
