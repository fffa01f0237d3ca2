"""The 4-bit cache's operators together with the GEMVs: a layer's attention half over several steps against the same in 64
bits, from the weights' and the cache's own dequantised values."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_ref as ref
from b4gemv.kvlayer import CachedAttention, rotate

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,kv_fmt", [(b4gemv.FMT_INT4_G128, b4gemv.KV_INT4), (b4gemv.FMT_NF4_B64, b4gemv.KV_NF4)])
@pytest.mark.parametrize("heads,kvh,dim,page", [(4, 2, 128, 16), (8, 1, 64, 32)])
def test_steps(cuda, fmt, kv_fmt, heads, kvh, dim, page):
    hidden = 512
    layer = CachedAttention(fmt, hidden, heads, kvh, n_pages=40, max_requests=4, head_dim=dim, page_size=page, max_context=10 * page, seed=3)
    dequant = b4gemv.dequant_nf4 if fmt == b4gemv.FMT_NF4_B64 else b4gemv.dequant_int4
    w = {n: dequant(*layer.weights[n]).double().view(-1, hidden if n != "o" else heads * dim) for n in "qkvo"}
    g = torch.Generator(device="cuda").manual_seed(1)
    done = [0, 0, 0]
    for added in ([37, 1, 60], [1, 1, 1], [0, 5, 2], [1, 1, 1]):
        x = torch.randn((sum(added), hidden), generator=g, device="cuda").half()
        y = layer.step(x, added)
        done = [a + b for a, b in zip(done, added)]
        assert layer.cached.tolist()[:3] == done
        place = torch.cat([torch.arange(d - a, d) for d, a in zip(done, added)]).int().cuda()
        q = rotate((x.double() @ w["q"].T).float().view(-1, heads, dim), place)
        starts = np.concatenate([[0], np.cumsum(added)])
        out, _, (weight, size) = ref.attention(kv_fmt, page, dim, layer.cache.blocks, q.half(), layer.tables[:3], done, starts, dim ** -0.5)
        # q's rounding to fp16 may fall to either side (2^-10 of q, so of the largest score, then twice in a weight), the NF4
        # code book in fp16 3e-4 of a level; weights and outputs are rounded to fp16 once each
        book = 3e-4 if kv_fmt == b4gemv.KV_NF4 else 0.0
        tol = weight * (2 ** -11 + book + 2 * size[..., None] * (2.0 ** -10 + book)) + out.abs() * 2 ** -11 + 2.0 ** -20
        got, want = y.double(), out.view(x.shape[0], -1) @ w["o"].T
        assert bool(((got - want).abs() <= tol.view(x.shape[0], -1) @ w["o"].abs().T + 1e-4 * want.abs().max()).all())
        # what was appended: the new tokens' keys, from the layer's own projections, within a step of their codes
        k = rotate((x.double() @ w["k"].T).float().view(-1, kvh, dim), place)
        v = (x.double() @ w["v"].T).view(-1, kvh, dim)
        table = layer.tables.cpu().numpy()
        row = np.repeat(np.arange(3), added)
        slots = torch.from_numpy(table[row, place.cpu().numpy() // page] * page + place.cpu().numpy() % page).int().cuda()
        for a, b in zip(b4gemv.kv_read(layer.cache, slots), (k, v)):
            # half the widest step (INT4: 1 / 14 of the largest column; NF4: 0.152 of it), and what is rounded before
            step = (1 / 14 if kv_fmt == b4gemv.KV_INT4 else 0.152) * b.abs().amax(-1, keepdim=True)
            assert bool(((a - b).abs() <= step * 1.01 + 1e-3).all())
    assert layer.free_state.tolist()[2] == 0
    assert b4gemv.load().b4_device_error(0) == 0


def test_step_refusals(cuda):
    layer = CachedAttention(b4gemv.FMT_INT4_G128, 256, 2, 1, n_pages=4, max_requests=2, page_size=16, max_context=32)
    x = torch.zeros((3, 256), dtype=torch.float16, device="cuda")
    for added in ([1, 1], [1, 1, 1]):
        with pytest.raises(ValueError):
            layer.step(x, added)
    with pytest.raises(ValueError):
        CachedAttention(7, 256, 2, 1, n_pages=4, max_requests=2)
