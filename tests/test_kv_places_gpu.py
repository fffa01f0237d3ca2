"""Where outputs may lie: the rotated append in place among fused rows of queries, keys and values, whatever their order; attention
over its own queries."""
import pytest
import torch

import b4gemv
from test_kv_rotary_gpu import check, rows

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t", [1, 40, 700])
@pytest.mark.parametrize("layout", ["columns", "head by head", "heads first"])
def test_in_place_among_fused_rows(cuda, dtype, t, layout):
    """check compares the pages and the queries; keys and values stay as they were."""
    heads, d = 4, 128
    if layout == "columns":
        fused = rows(t, heads + 4, d, dtype, 7, cuda)
        q, k, v = fused[:, :heads], fused[:, heads:heads + 2], fused[:, heads + 2:]
    elif layout == "head by head":
        fused = rows(t, 3 * heads, d, dtype, 7, cuda)
        q, k, v = (fused[:, i::3] for i in range(3))
    else:
        fused = rows(heads + 4, t, d, dtype, 7, cuda)
        q, k, v = (x.transpose(0, 1) for x in (fused[:heads], fused[heads:heads + 2], fused[heads + 2:]))
    before, plain = fused.clone(), check(cuda, NF4, dtype, t, heads, k.shape[1], d, 16, d, q=q.clone(), k=k, v=v)
    got = check(cuda, NF4, dtype, t, heads, k.shape[1], d, 16, d, q=q, k=k, v=v, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, plain)
    q.zero_()
    after = fused.clone()
    fused.copy_(before)
    q.zero_()
    assert torch.equal(after, fused)


def test_outputs_on_inputs_are_refused(cuda):
    t, d = 20, 64
    fused = rows(t, 12, d, F16, 1, cuda)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:8]
    cache = b4gemv.KVCache.alloc(INT4, 4, 2, 16, d, cuda)
    at = torch.arange(t, dtype=torch.int32, device=cuda)
    rotary, before = b4gemv.Rotary(d, device=cuda), fused.clone()
    for out in (fused[:, 2:6], fused[:, 4:8], fused[:, 6:10], fused[:, 1:5], fused[:, 3:4].expand(t, 4, d), fused[:1, 8:].expand(t, 4, d),
                fused.view(-1)[:t * 4 * d].view(t, 4, d)):
        with pytest.raises(b4gemv.B4Error):
            b4gemv.kv_append_rotary(cache, rotary, q, k, v, at, at, out=out)
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_append_rotary(cache, rotary, *(x[:16].float() for x in (q, k, v)), at[:16], at[:16],
                                out=cache.blocks.view(-1)[:16 * 4 * d * 2].view(F16).view(16, 4, d))
    assert torch.equal(fused, before) and not bool(cache.blocks.any())
    b4gemv.kv_append_rotary(cache, rotary, q, k, v, at, at, out=fused[:, 8:])
    assert torch.equal(fused[:, :8], before[:, :8]) and not torch.equal(fused[:, 8:], before[:, 8:])


def test_attention_in_place(cuda):
    """Over its own queries; a few heads off is refused."""
    for total, keep in ((3, 40), (200, 6)):                        # lists shared by teams, and not
        g = torch.Generator(device=cuda).manual_seed(total)
        cache = b4gemv.KVCache.alloc(INT4, 60, 2, 16, 128, cuda)
        at = torch.arange(60 * 16, dtype=torch.int32, device=cuda)
        b4gemv.kv_append(cache, *(torch.randn((60 * 16, 2, 128), generator=g, device=cuda) for _ in range(2)), at)
        room = torch.randn((total, 24, 128), generator=g, device=cuda).half()
        q = room[:, 2:22]
        lists = b4gemv.KVLists(torch.randint(0, 60, (total, 2, keep), generator=g, device=cuda).int(), torch.randint(0, 16 * keep + 1, (total,), generator=g, device=cuda).int())
        want, before = b4gemv.kv_attention_lists(cache, q.clone(), lists), room.clone()
        for out in (room[:, 1:21], room[:, 4:], room[:, 2:3].expand(total, 20, 128)):
            with pytest.raises(b4gemv.B4Error):
                b4gemv.kv_attention_lists(cache, q, lists, out=out)
        assert torch.equal(room, before)
        b4gemv.kv_attention_lists(cache, q, lists, out=q)
        assert torch.equal(q, want) and torch.equal(room[:, :2], before[:, :2]) and torch.equal(room[:, 22:], before[:, 22:])
