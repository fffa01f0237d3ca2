"""A layer's attention half with the rotation in the append and a choice of pages, over several steps: what its operators made
of the layer's own queries against the same in 64 bits, and the layer without them."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_lists_ref as lists_ref
from b4gemv import kvlayer
from b4gemv.kvlayer import CachedAttention
from test_kv_gpu import bounds

pytestmark = pytest.mark.gpu
FORMATS = [(b4gemv.FMT_INT4_G128, b4gemv.KV_INT4), (b4gemv.FMT_NF4_B64, b4gemv.KV_NF4)]
STEPS = ([137, 1, 60], [1, 1, 1], [0, 50, 2], [1, 1, 1])


@pytest.mark.parametrize("fmt,kv_fmt", FORMATS)
@pytest.mark.parametrize("heads,kvh,dim,page", [(4, 2, 128, 16), (8, 1, 64, 32)])
def test_steps_with_a_choice(cuda, monkeypatch, fmt, kv_fmt, heads, kvh, dim, page):
    made = {}

    def noted(name):
        f = getattr(kvlayer, name)

        def call(*args, **more):
            made[name] = f(*args, **more)
            return made[name]
        monkeypatch.setattr(kvlayer, name, call)
    for name in ("kv_append_rotary", "kv_select", "kv_attention_lists"):
        noted(name)
    hidden, keep, first, last = 512, 4, 1, 2
    layer = CachedAttention(fmt, hidden, heads, kvh, n_pages=60, max_requests=4, head_dim=dim, page_size=page, max_context=16 * page, seed=3,
                            rotary=b4gemv.Rotary(dim, device=cuda), keep=keep, first=first, last=last)
    g = torch.Generator(device="cuda").manual_seed(1)
    done = [0, 0, 0]
    for added in STEPS:
        x = torch.randn((sum(added), hidden), generator=g, device="cuda").half()
        y = layer.step(x, added)
        done = [a + b for a, b in zip(done, added)]
        q, out = made["kv_append_rotary"], made["kv_attention_lists"]
        starts = np.concatenate([[0], np.cumsum(added)])
        lists, seen = lists_ref.select(page, dim, layer.boxes.cpu().numpy(), q, layer.tables[:3].cpu().numpy(), done, starts, keep, first, last, 60)
        assert np.array_equal(made["kv_select"].pages.cpu().numpy(), lists) and np.array_equal(made["kv_select"].seen.cpu().numpy(), seen)
        want, wl, aux = lists_ref.attention(kv_fmt, page, dim, layer.cache.blocks, q, lists, seen, dim ** -0.5)
        tol, _ = bounds(kv_fmt, torch.float16, want, wl, aux, keep * page)
        assert bool(((out.double() - want).abs() <= tol).all())
        assert torch.equal(y, layer._project("o", out.view(sum(added), -1)))
    assert layer.cached.tolist()[:3] == done and layer.free_state.tolist()[2] == 0
    assert b4gemv.load().b4_device_error(0) == 0


@pytest.mark.parametrize("fmt,kv_fmt", FORMATS)
def test_rotary_turns_as_before(cuda, fmt, kv_fmt):
    """With rotate()'s base and pairs keys differ by their roundings alone: 3 * 2^-24 of |a| + |b|, some 2^-21 of a column's
    range.  A code differs where a border lies between the two, by one step: for 15 borders in a range some 15 * 2^-20 of the
    values, 2e-5.  An INT4 scale may be the next fp16 number: 2^-10 of a value, 0.007 of a step."""
    a, b = (CachedAttention(fmt, 512, 4, 2, n_pages=40, max_requests=3, page_size=16, max_context=256, seed=3, rotary=r)
            for r in (None, b4gemv.Rotary(128, base=1e6, device=cuda)))
    g = torch.Generator(device="cuda").manual_seed(2)
    slots = None
    for added in STEPS:
        x = torch.randn((sum(added), 512), generator=g, device="cuda").half()
        assert a.step(x, added).shape == b.step(x, added).shape
        assert torch.equal(a.tables, b.tables)
    slots = torch.arange(40 * 16, dtype=torch.int32, device=cuda)
    for p, q in zip(b4gemv.kv_read(a.cache, slots), b4gemv.kv_read(b.cache, slots)):
        step = (1 / 7 if kv_fmt == b4gemv.KV_INT4 else 0.304) * p.abs().amax(-1, keepdim=True)
        assert bool(((p - q).abs() <= step * 1.01 + 1e-6).all())
        assert float(((p - q).abs() > 0.01 * step).float().mean()) < 1e-3


def test_positions_of_several_axes(cuda):
    rotary = b4gemv.Rotary(128, sections=(16, 24, 24), device=cuda)
    layer = CachedAttention(b4gemv.FMT_INT4_G128, 256, 4, 2, n_pages=20, max_requests=2, page_size=16, max_context=128, rotary=rotary, keep=3)
    x = torch.randn((70, 256), device=cuda).half()
    place = torch.arange(35, dtype=torch.int32, device=cuda).repeat(2)
    same = layer.step(x, [35, 35], positions=place.expand(3, 70).contiguous())
    plain = CachedAttention(b4gemv.FMT_INT4_G128, 256, 4, 2, n_pages=20, max_requests=2, page_size=16, max_context=128,
                            rotary=b4gemv.Rotary(128, device=cuda), keep=3)
    assert torch.equal(same, plain.step(x, [35, 35]))                # the same place on every axis is one axis
    y = layer.step(x[:2], [1, 1], positions=torch.randint(0, 90, (3, 2), dtype=torch.int32, device=cuda))
    assert y.shape == (2, 256) and bool(torch.isfinite(y).all())


def test_steps_without_tokens_and_refusals(cuda):
    layer = CachedAttention(b4gemv.FMT_INT4_G128, 256, 2, 1, n_pages=4, max_requests=2, page_size=16, max_context=32, rotary=b4gemv.Rotary(128, device=cuda), keep=2)
    x = torch.zeros((3, 256), dtype=torch.float16, device="cuda")
    for added in ([0, 0], [0], []):
        assert layer.step(x[:0], added).shape == (0, 256)
    with pytest.raises(ValueError):
        layer.step(x, [1, 1])
    for bad in (dict(keep=-1), dict(keep=1), dict(keep=3, first=2, last=2), dict(keep=3, last=0)):
        with pytest.raises(ValueError):
            CachedAttention(b4gemv.FMT_INT4_G128, 256, 2, 1, n_pages=4, max_requests=2, **bad)
    with pytest.raises(ValueError):
        CachedAttention(b4gemv.FMT_INT4_G128, 256, 2, 1, n_pages=4, max_requests=2).step(x, [3], positions=torch.zeros(3, dtype=torch.int32, device=cuda))


def test_command(cuda, capsys):
    from b4gemv import diag
    diag.main(["kv", "--fmt", "int4", "--requests", "3", "--prompt", "300", "--tokens", "5", "--rotary", "--keep", "4"])
    assert "us a" in capsys.readouterr().out
