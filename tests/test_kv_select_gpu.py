"""Boxes and the choice of pages against their restatements in numpy: every byte and every page equal, since scores are whole
numbers times one scale."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_lists_ref as lists_ref
import kv_ref as ref

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16 = torch.float16, torch.bfloat16


def ints(x, cuda):
    return torch.tensor(np.asarray(x, np.int32), device=cuda)


# ---- boxes ----------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("d,page,kvh", [(64, 16, 1), (128, 16, 3), (64, 32, 5), (128, 32, 8), (64, 64, 2), (128, 64, 12)])
@pytest.mark.parametrize("few", [True, False])
def test_boxes(cuda, fmt, d, page, kvh, few):
    """Of the pages whose last token is in the slots, no others, in any order of the slots."""
    rng = np.random.default_rng(d + page + kvh)
    pages = 9 if few else 700
    cache = b4gemv.KVCache.alloc(fmt, pages, kvh, page, d, cuda)
    every = torch.arange(pages * page, dtype=torch.int32, device=cuda)
    x = torch.randn((pages * page, kvh, d), device=cuda) * torch.exp(torch.randn((pages * page, kvh, 1), device=cuda))
    x[: 2 * page] = x[: 2 * page].abs()                                    # minima above 0
    x[2 * page: 3 * page] = 0.0
    x[3 * page: 4 * page] *= 1e-30                                         # INT4: scales of 0
    b4gemv.kv_append(cache, x, x, every)
    slots = rng.permutation(pages * page)[: max(1, pages * page * 2 // 3)].astype(np.int32)
    slots[rng.integers(0, len(slots), 5)] = -1
    slots = np.concatenate([slots, [-5, pages * page + page - 1, 2 ** 31 - 1]]).astype(np.int32)
    boxes = torch.full((pages, kvh, b4gemv.kv_box_bytes(d)), 201, dtype=torch.uint8, device=cuda)
    b4gemv.kv_boxes(cache, boxes, ints(slots, cuda))
    ok = (slots >= 0) & (slots < pages * page) & (slots % page == page - 1)
    want = np.full(boxes.shape, 201, np.uint8)
    done = np.unique(slots[ok] // page)
    assert len(done)
    want[done] = lists_ref.boxes(fmt, page, d, cache.blocks.cpu().numpy()[done])
    assert np.array_equal(boxes.cpu().numpy(), want)


@pytest.mark.parametrize("fmt", [INT4, NF4])
def test_boxes_of_keys_that_are_no_numbers(cuda, fmt):
    """Scales of infinity and NaN in the pages, a page whose scales are all of them."""
    page, d, kvh = 16, 64, 2
    cache = b4gemv.KVCache.alloc(fmt, 4, kvh, page, d, cuda)
    x = torch.randn((4 * page, kvh, d), device=cuda)
    every = torch.arange(4 * page, dtype=torch.int32, device=cuda)
    b4gemv.kv_append(cache, x, x, every)
    codes, s = ref.unpack_blocks(fmt, page, d, cache.blocks.cpu().numpy())
    s = s.copy()
    s[0, 0, 0, 3], s[0, 1, 1, 5], s[0, 2] = np.nan, np.inf, np.nan
    cache.blocks.copy_(torch.from_numpy(ref.pack_blocks(fmt, codes, s)))
    boxes = b4gemv.kv_new_boxes(cache)
    b4gemv.kv_boxes(cache, boxes, every)
    assert np.array_equal(boxes.cpu().numpy(), lists_ref.boxes(fmt, page, d, cache.blocks.cpu().numpy()))


def test_a_box_bounds_its_keys(cuda):
    """To the roundings of its two corners: half a unit a column each."""
    cache = b4gemv.KVCache.alloc(INT4, 6, 2, 64, 128, cuda)
    every = torch.arange(6 * 64, dtype=torch.int32, device=cuda)
    x = torch.randn((6 * 64, 2, 128), device=cuda)
    b4gemv.kv_append(cache, x, x, every)
    boxes = b4gemv.kv_new_boxes(cache)
    b4gemv.kv_boxes(cache, boxes, every)
    k = b4gemv.kv_read(cache, every)[0].view(6, 64, 2, 128).transpose(1, 2)
    unit = boxes[..., 256:260].contiguous().view(torch.float32)
    hi, lo = (boxes[..., a:a + 128].view(torch.int8).float() * unit for a in (0, 128))
    assert bool((k <= hi[:, :, None] + 0.5001 * unit[:, :, None]).all()) and bool((k >= lo[:, :, None] - 0.5001 * unit[:, :, None]).all())


# ---- the choice -----------------------------------------------------------------------

def make(cuda, dtype, heads, kvh, d, page, ctx, new, seed=0, extra=0, spare=2):
    """Boxes of every page at random (a choice reads nothing else of a page), tables in a random order, packed queries."""
    rng = np.random.default_rng(seed)
    need = [-(-max(c, 0) // page) for c in ctx]
    pages, width = sum(need) + spare, max(need + [1])
    order = rng.permutation(pages)
    tab = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        tab[r, :n] = order[at:at + n]
        at += n
    box = rng.integers(0, 256, (pages, kvh, 2 * d + 16)).astype(np.uint8)
    box[..., : 2 * d][box[..., : 2 * d] == 128] = 0
    box[..., 2 * d: 2 * d + 4] = np.exp(rng.standard_normal((pages, kvh, 1))).astype(np.float32).view(np.uint8)
    cache = b4gemv.KVCache.alloc(INT4, pages, kvh, page, d, cuda)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    g = torch.Generator(device=cuda).manual_seed(seed)
    q = torch.randn((int(starts[-1]) + extra, heads, d), generator=g, device=cuda).to(dtype)
    return dict(cache=cache, box=box, q=q, tab=tab, ctx=list(ctx), starts=starts, most=max(list(new) + [0]))


def check(cuda, s, keep, first=1, last=1, most=None, **more):
    total, kvh = s["q"].shape[0], s["cache"].kv_heads
    out = b4gemv.KVLists(torch.full((total, kvh, keep), -7, dtype=torch.int32, device=cuda), torch.full((total,), -7, dtype=torch.int32, device=cuda))
    boxes = torch.from_numpy(s["box"]).to(cuda)
    table = s["tab"] if torch.is_tensor(s["tab"]) else ints(s["tab"], cuda)
    b4gemv.kv_select(s["cache"], boxes, s["q"], table, ints(s["ctx"], cuda), ints(s["starts"], cuda), s["most"] if most is None else most,
                     keep, first=first, last=last, out=out, **more)
    torch.cuda.synchronize()
    lists, seen = lists_ref.select(s["cache"].page_size, s["cache"].head_dim, s["box"], s["q"], table.cpu().numpy(), s["ctx"], s["starts"],
                                   keep, first, last, s["cache"].n_pages)
    assert np.array_equal(out.seen.cpu().numpy(), seen)
    assert np.array_equal(out.pages.cpu().numpy(), lists)
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kvh,d,page", [(28, 4, 128, 16), (64, 8, 128, 64), (4, 4, 64, 32), (32, 2, 64, 16), (64, 1, 128, 32)])
@pytest.mark.parametrize("keep,first,last", [(1, 0, 1), (4, 1, 2), (9, 0, 1), (16, 8, 8), (40, 1, 3)])
def test_single_tokens(cuda, dtype, heads, kvh, d, page, keep, first, last):
    s = make(cuda, dtype, heads, kvh, d, page, [1, 2, page - 1, page, page + 1, 7 * page, 9 * page + 1, 300, 2111, 40 * page, 41 * page, 41 * page + 1], [1] * 12)
    check(cuda, s, keep, first, last)


@pytest.mark.parametrize("new", [[3, 1, 8, 0, 5], [8] * 5, [9, 40, 0, 1, 17], [100, 3, 31, 8, 60], [1, 0, 0, 0, 700]])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 64)])
def test_several_tokens(cuda, new, d, page):
    ctx = [n + c for n, c in zip(new, (900, 0, 3000, 50, 1700))]
    check(cuda, make(cuda, F16, 12, 4, d, page, ctx, new, extra=5), 12, 2, 3)
    check(cuda, make(cuda, BF16, 6, 3, d, page, ctx, new), 5, 0, 1)


@pytest.mark.parametrize("pages", [130, 257, 511, 1025, 2500, 8192])
@pytest.mark.parametrize("new", [1, 4, 20])
def test_long_contexts(cuda, pages, new):
    """One request and few heads: a cluster of CTAs for a tile."""
    s = make(cuda, F16, 4, 2, 64, 16, [pages * 16 - 5], [new])
    check(cuda, s, 64, 1, 2)
    check(cuda, s, 129, 5, 40)


def test_the_widest_tables(cuda):
    width = 49152
    for new in (1, 3, 30):
        s = make(cuda, F16, 2, 1, 64, 16, [width * 16 - 3], [new])
        check(cuda, s, 100, 1, 2)
    assert s["tab"].shape[1] == width
    with pytest.raises(b4gemv.B4Error):
        check(cuda, make(cuda, F16, 2, 1, 64, 16, [width * 16 + 1], [1]), 100, 1, 2)


def test_many_requests(cuda):
    rng = np.random.default_rng(3)
    for n, hi in ((300, 1), (1100, 3), (90, 30)):
        new = rng.integers(0, hi + 1, n).tolist()
        ctx = [a + int(c) for a, c in zip(new, rng.integers(0, 900, n))]
        check(cuda, make(cuda, F16, 4, 2, 64, 16, ctx, new, extra=3), 6, 1, 1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_more_than_fit_at_once(cuda, dtype, d):
    """More CTAs than the GPU holds: of a token each, of several, of 16."""
    rng = np.random.default_rng(d)
    for n, new in ((150, 1), (130, 4), (2, 300)):
        s = make(cuda, dtype, 8, 4 if n > 2 else 8, d, 16, (new + rng.integers(0, 2500, n)).tolist(), [new] * n)
        check(cuda, s, 24, 1, 2)
        if n > 2:
            s["box"][::11, :, 2 * d: 2 * d + 4] = np.float32([np.nan]).view(np.uint8)
            s["tab"][::3, ::5] = -1
            check(cuda, s, 24, 1, 2)


@pytest.mark.parametrize("new", [1, 5, 12])
def test_ties_go_to_the_earlier(cuda, new):
    """Boxes that are all alike, or of three kinds, and queries of zeros."""
    s = make(cuda, F16, 4, 2, 64, 16, [2000 + new, 900, 333], [new, 1, new])
    s["box"][:] = s["box"][0]
    check(cuda, s, 20, 1, 2)
    s["box"][1::3], s["box"][2::3] = s["box"][1], s["box"][2] ^ 3
    check(cuda, s, 20, 1, 2)
    s["box"][..., 128:132] = np.float32([1.0]).view(np.uint8)
    s["q"].zero_()
    check(cuda, s, 20, 0, 1)


@pytest.mark.parametrize("new", [1, 10])
def test_boxes_and_queries_without_numbers(cuda, new):
    s = make(cuda, F16, 4, 2, 64, 16, [1500, 1500], [new, new])
    s["box"][::5, :, 128:132] = np.float32([np.inf]).view(np.uint8)
    s["box"][::7, :, 128:132] = np.float32([np.nan]).view(np.uint8)
    s["box"][1, :, 128:132] = np.float32([3e38]).view(np.uint8)                      # scores that overflow to either side
    s["box"][2, :, 128:132] = np.float32([1e-44]).view(np.uint8)
    check(cuda, s, 30, 1, 1)
    s["q"][0, 1, 3], s["q"][new, 2, 60] = float("nan"), float("inf")
    check(cuda, s, 30, 1, 1)


@pytest.mark.parametrize("new", [1, 9])
def test_missing_pages_come_last(cuda, new):
    s = make(cuda, F16, 4, 2, 64, 16, [1500, 700, 100], [new, new, new])
    s["tab"][:, 3::4] = -1
    s["tab"][0, 8::9] = s["cache"].n_pages
    s["tab"][1] = -1
    check(cuda, s, 30, 1, 2)
    check(cuda, s, 80, 1, 2)                                                         # more than are there


def test_requests_at_their_edges(cuda):
    """No tokens, more queries than tokens, rows of no request, no request at all, tables narrower than a context, more to keep
    than a table holds."""
    s = make(cuda, F16, 4, 2, 64, 16, [0, 3, -4, 40, 700], [2, 5, 1, 0, 3], extra=9)
    check(cuda, s, 4, 1, 1)
    s = make(cuda, F16, 4, 2, 64, 16, [300, 900, 10], [12, 2, 20], extra=100)
    check(cuda, s, 6, 1, 2)
    s["tab"] = np.ascontiguousarray(s["tab"][:, :9])
    check(cuda, s, 6, 1, 2)
    check(cuda, s, 70, 1, 2)
    s["tab"] = np.ascontiguousarray(s["tab"][:, :0])
    check(cuda, s, 6, 1, 2)
    s.update(tab=np.zeros((0, 3), np.int32), ctx=[], starts=np.zeros(1, np.int32))
    check(cuda, s, 6, 1, 2)
    s = make(cuda, F16, 4, 2, 64, 16, [300], [0])
    assert check(cuda, s, 6).pages.shape == (0, 2, 6)


def test_max_q_is_a_hint(cuda):
    s = make(cuda, F16, 4, 2, 64, 16, [900, 400, 2000], [11, 1, 30])
    for most in (0, 1, 4, 8, 9, 31, 5000):
        check(cuda, s, 10, 1, 2, most=most)


def test_strides_and_streams(cuda):
    s = make(cuda, F16, 8, 2, 128, 32, [900, 4000, 64], [1, 1, 1])
    first = check(cuda, s, 10, 1, 2)
    wide = torch.zeros((3, 11, 160), dtype=F16, device=cuda)
    wide[:, 2:10, 16:144] = s["q"]
    table = torch.full((3, s["tab"].shape[1] + 13), -1, dtype=torch.int32, device=cuda)[:, : s["tab"].shape[1]]
    table.copy_(ints(s["tab"], cuda))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again = check(cuda, {**s, "q": wide[:, 2:10, 16:144], "tab": table}, 10, 1, 2, stream=side)
    assert torch.equal(first.pages, again.pages)


def test_box_past_4_gib(cuda):
    """Boxes whose bytes lie past 32 bits."""
    kvh, d = 1024, 128
    pages = (1 << 32) // (kvh * 272) + 40
    cache = object.__new__(b4gemv.KVCache)                                            # the choice reads no page
    small = b4gemv.KVCache.alloc(INT4, 1, kvh, 16, d, cuda)
    cache.__dict__.update(small.__dict__)
    cache.n_pages = pages
    cache._c = type(small._c)(small.blocks.data_ptr(), INT4, pages, 16, kvh, d)
    import ctypes
    cache._ref = ctypes.byref(cache._c)
    boxes = torch.empty((pages, kvh, 272), dtype=torch.uint8, device=cuda)
    ids = list(range(pages - 20, pages)) + [0, 1, 2]
    few = torch.randint(0, 127, (23, kvh, 272), dtype=torch.uint8, device=cuda)
    few[..., 256:260] = torch.rand((23, kvh, 1), device=cuda).view(torch.uint8).view(23, kvh, 4)
    boxes[ids] = few
    q = torch.randn((1, kvh, d), device=cuda).half()
    a = b4gemv.kv_select(cache, boxes, q, ints([ids], cuda), ints([23 * 16], cuda), ints([0, 1], cuda), 1, 7)
    other = b4gemv.KVCache.alloc(INT4, 23, kvh, 16, d, cuda)
    b = b4gemv.kv_select(other, few, q, ints([range(23)], cuda), ints([23 * 16], cuda), ints([0, 1], cuda), 1, 7)
    assert torch.equal(a.pages, ints(ids, cuda)[b.pages.long()].view_as(b.pages))


def test_refused_on_the_gpu(cuda):
    s = make(cuda, F16, 4, 2, 64, 16, [30], [1])
    boxes, t = torch.from_numpy(s["box"]).to(cuda), lambda x: ints(x, cuda)
    odd = torch.zeros(s["q"].numel() + 8, dtype=F16, device=cuda)[1:1 + s["q"].numel()].view_as(s["q"])
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_select(s["cache"], boxes, odd, t(s["tab"]), t(s["ctx"]), t(s["starts"]), 1, 4)
    with pytest.raises(ValueError):
        b4gemv.kv_select(s["cache"], boxes[:-1], s["q"], t(s["tab"]), t(s["ctx"]), t(s["starts"]), 1, 4)
    with pytest.raises(ValueError):
        b4gemv.kv_select(s["cache"], boxes, s["q"], t(s["tab"]), t(s["ctx"]), t(s["starts"]), 1, 2, first=1, last=2)
    assert b4gemv.load().b4_device_error(0) == 0
