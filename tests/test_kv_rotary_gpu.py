"""The rotated append against its restatement in 64 bits: pages equal byte for byte, queries within their own rounding."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_lists_ref as lists_ref
import kv_ref as ref

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rows(t, heads, d, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((t, heads, d), generator=g) * torch.exp(torch.randn((t, heads, 1), generator=g))
    return x.to(dtype).to(device)


def check(cuda, fmt, dtype, t, heads, kvh, d, page, rot, adjacent=False, n_axes=1, far=100000, out_dtype=None, scale=1.0, seed=0, q=None, k=None, v=None,
          positions=None, slots=None, out=None, **more):
    """Pages, and queries, of one call.  A page's bytes are those of the 64-bit rotation rounded to fp32 once: they could differ
    only where it lies within some 2^-50 of a border between fp32 numbers, which no value of these does."""
    rng = np.random.default_rng(seed)
    inv = [1e6 ** (-i / (rot // 2)) for i in range(rot // 2)]
    axes = rng.integers(0, n_axes, rot // 2).tolist()
    axes[0] = n_axes - 1
    if positions is None:
        positions = rng.integers(0, far, (n_axes, t)).astype(np.int32)
    pages = t // page + 2
    if slots is None:
        slots = rng.permutation(pages * page)[:t].astype(np.int32)
        if t > 3:
            slots[0], slots[2] = -1, pages * page                # skipped
    rotary = b4gemv.Rotary(rot, inv_freq=inv, axes=axes, adjacent=adjacent, scale=scale, device=cuda)
    q = rows(t, heads, d, dtype, 1, cuda) if q is None else q
    k = rows(t, kvh, d, dtype, 2, cuda) if k is None else k
    v = rows(t, kvh, d, dtype, 3, cuda) if v is None else v
    blocks = torch.randint(0, 256, (pages, kvh, b4gemv.kv_block_bytes(fmt, page, d)), dtype=torch.uint8, device=cuda)
    before = blocks.cpu().numpy()
    cache = b4gemv.KVCache(blocks, fmt, page, d)
    x = q.float().cpu().numpy()
    if out_dtype is not None:
        out = torch.empty(q.shape, dtype=out_dtype, device=cuda)
    where = torch.from_numpy(positions).to(cuda)
    got = b4gemv.kv_append_rotary(cache, rotary, q, k, v, where[0] if n_axes == 1 else where, torch.from_numpy(slots).to(cuda), out=out, **more)
    torch.cuda.synchronize()
    angle = lists_ref.angles(positions, axes, inv)
    ok = (slots >= 0) & (slots < pages * page)
    codes, scales = ref.unpack_blocks(fmt, page, d, before)
    codes, scales = codes.copy(), scales.copy()
    turned = lists_ref.rotate(k.float().cpu().numpy(), angle, adjacent, float(np.float32(scale))).astype(np.float32)
    for o, y in enumerate((turned, v.float().cpu().numpy())):
        c, s = ref.quantise(fmt, y)
        codes[o, slots[ok] // page, :, slots[ok] % page], scales[o, slots[ok] // page, :, slots[ok] % page] = c[ok], s[ok]
    assert blocks.cpu().numpy().tobytes() == ref.pack_blocks(fmt, codes, scales).tobytes()
    want = lists_ref.rotate(x, angle, adjacent, float(np.float32(scale)))
    # cosine and sine rounded to fp32 (2^-24 of each), two products and a sum (2^-24 each): 3 * 2^-24 of |a| + |b| times the
    # scale at most; then the type's own half step, fp16's least step among them
    size = lists_ref.rotate(np.abs(x), np.zeros_like(angle), adjacent)
    other = np.zeros_like(size)
    h = rot // 2
    if adjacent:
        other[..., 0:rot:2], other[..., 1:rot:2] = size[..., 1:rot:2], size[..., 0:rot:2]
    else:
        other[..., :h], other[..., h:rot] = size[..., h:rot], size[..., :h]
    far_off = np.where(np.arange(d) < rot, (size + other) * abs(scale) * 4 * 2.0 ** -24, 0)
    half_step = torch.finfo(got.dtype).eps / 2
    tol = far_off * (1 + half_step) + np.abs(want) * half_step + (2.0 ** -25 if got.dtype == F16 else 0)
    assert bool((np.abs(got.float().cpu().numpy() - want) <= tol).all())
    return got


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("dtype,out_dtype", [(F16, None), (BF16, None), (F32, None), (F32, BF16)])
@pytest.mark.parametrize("t,heads,kvh,d,page,rot,adjacent,n_axes", [
    (1, 1, 1, 64, 16, 64, False, 1), (17, 28, 4, 128, 16, 128, False, 1), (700, 8, 8, 128, 64, 128, True, 3), (77, 15, 5, 64, 32, 32, True, 1),
    (64, 64, 8, 128, 16, 96, False, 2), (1203, 6, 3, 64, 16, 48, False, 3), (601, 3, 1, 128, 32, 16, True, 2)])
def test_rotated_append(cuda, fmt, dtype, out_dtype, t, heads, kvh, d, page, rot, adjacent, n_axes):
    got = check(cuda, fmt, dtype, t, heads, kvh, d, page, rot, adjacent, n_axes, out_dtype=out_dtype)
    assert got.dtype == (out_dtype or (F16 if dtype == F32 else dtype))


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("adjacent", [False, True])
def test_far_positions_and_scale(cuda, fmt, adjacent):
    """To the ends of 32 bits, below 0 too: the whole turns leave exactly."""
    p = np.array([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9, -123456789, 131071]], np.int32)
    check(cuda, fmt, F32, 8, 4, 2, 128, 16, 128, adjacent, positions=p, scale=1.1877)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_and_alignment(cuda, fmt, dtype):
    """Column slices of a fused projection's rows, at addresses that 16-byte loads do not take too; out with strides of its own."""
    t, heads, kvh, d = 37, 6, 2, 128
    for shift in (0, 1, 3):
        wide = rows(t, 1, (heads + 2 * kvh) * d + 40, dtype, 5, cuda)[:, 0, shift:]
        q, k, v = (wide[:, a * d:(a + n) * d].unflatten(1, (n, d)) for a, n in ((0, heads), (heads, kvh), (heads + kvh, kvh)))
        room = torch.full((t, heads + 1, d + 8), 3.0, dtype=F16, device=cuda)
        check(cuda, fmt, dtype, t, heads, kvh, d, 32, 128, q=q, k=k, v=v, out=room[:, 1:, :d])
        assert bool((room[:, :, d:] == 3).all()) and bool((room[:, 0] == 3).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t", [5, 800])
def test_in_place_and_without_queries(cuda, dtype, t):
    q = rows(t, 12, 128, dtype, 9, cuda)
    first = check(cuda, INT4, dtype, t, 12, 2, 128, 16, 128, q=q.clone())
    mine = q.clone()
    assert check(cuda, INT4, dtype, t, 12, 2, 128, 16, 128, q=mine, out=mine).data_ptr() == mine.data_ptr()
    assert torch.equal(mine, first)
    a, b = (b4gemv.KVCache.alloc(INT4, t // 16 + 1, 2, 16, 128, cuda) for _ in range(2))
    rotary = b4gemv.Rotary(128, device=cuda)
    k, v, at = rows(t, 2, 128, dtype, 2, cuda), rows(t, 2, 128, dtype, 3, cuda), torch.arange(t, dtype=torch.int32, device=cuda)
    assert b4gemv.kv_append_rotary(a, rotary, None, k, v, at, at) is None
    b4gemv.kv_append_rotary(b, rotary, q, k, v, at, at)
    assert torch.equal(a.blocks, b.blocks) and bool(a.blocks.any())


@pytest.mark.parametrize("fmt", [INT4, NF4])
def test_turn_of_nothing_is_the_plain_append(cuda, fmt):
    """At position 0 keys are written as kv_append writes them, whatever they hold, and queries stay."""
    from test_kv_gpu import data
    for dtype in (F16, BF16, F32):
        t, kvh, d, page = 40, 3, 128, 16
        k, v = (data((t, kvh, d), dtype, s, special=True).to(cuda) for s in (1, 2))
        # inf and NaN columns would make NaN of their pairs' others, which take no part in a scale: kept to columns that do not turn
        k = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
        a, b = (b4gemv.KVCache.alloc(fmt, 4, kvh, page, d, cuda) for _ in range(2))
        slots = torch.arange(t, dtype=torch.int32, device=cuda)
        q = torch.randn((t, 7, d), device=cuda).to(dtype)
        out = b4gemv.kv_append_rotary(a, b4gemv.Rotary(64, device=cuda), q, k, v, torch.zeros_like(slots), slots)
        b4gemv.kv_append(b, k, v, slots)
        assert torch.equal(a.blocks, b.blocks)
        assert torch.equal(out, q.to(out.dtype))


def test_columns_without_a_number_stay_with_their_pairs(cuda):
    """An infinite or missing number in a query reaches its pair's two columns alone; in a key its code is NaN's."""
    t, d = 3, 128
    q, k, v = (torch.randn((t, 2, d), device=cuda) for _ in range(3))
    q[0, 0, 5], q[1, 1, 70], k[0, 0, 3] = float("inf"), float("nan"), float("nan")
    cache = b4gemv.KVCache.alloc(INT4, 1, 2, 16, d, cuda)
    slots = torch.arange(t, dtype=torch.int32, device=cuda)
    out = b4gemv.kv_append_rotary(cache, b4gemv.Rotary(d, device=cuda), q, k, v, slots + 3, slots)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 0, 5] = bad[0, 0, 69] = bad[1, 1, 70] = bad[1, 1, 6] = True
    assert torch.equal(~torch.isfinite(out), bad)
    got, _ = b4gemv.kv_read(cache, slots)
    assert got[0, 0, 3] == 0 and got[0, 0, 67] == 0 and bool(torch.isfinite(got).all())


def test_graph_stream_and_repeats(cuda):
    t, heads, kvh, d, page = 50, 8, 2, 128, 16
    cache = b4gemv.KVCache.alloc(NF4, 8, kvh, page, d, cuda)
    rotary = b4gemv.Rotary(d, sections=(16, 24, 24), device=cuda)
    q, k, v = (rows(t, n, d, BF16, n, cuda) for n in (heads, kvh, kvh))
    positions = torch.randint(0, 5000, (3, 64), dtype=torch.int32, device=cuda)[:, :t]     # axes wider apart than their tokens
    slots = torch.randperm(100, device=cuda)[:t].int()
    first = b4gemv.kv_append_rotary(cache, rotary, q, k, v, positions, slots)
    blocks = cache.blocks.clone()
    out, side = torch.empty_like(q), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b4gemv.kv_append_rotary(cache, rotary, q, k, v, positions, slots, out=out, stream=side)
    side.synchronize()
    assert torch.equal(out, first) and torch.equal(cache.blocks, blocks)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b4gemv.kv_append_rotary(cache, rotary, q, k, v, positions, slots, out=out)
    positions += 17
    q.copy_(q.flip(0))
    graph.replay()
    want = b4gemv.kv_append_rotary(cache, rotary, q, k, v, positions, slots)
    assert torch.equal(out, want) and not torch.equal(out, first)
    del graph


def test_nothing_to_append(cuda):
    cache = b4gemv.KVCache.alloc(INT4, 2, 2, 16, 64, cuda)
    none = torch.empty((0, 2, 64), dtype=F16, device=cuda)
    ints = torch.empty(0, dtype=torch.int32, device=cuda)
    assert b4gemv.kv_append_rotary(cache, b4gemv.Rotary(64, device=cuda), none, none, none, ints, ints).shape == (0, 2, 64)
    assert not bool(cache.blocks.any())
