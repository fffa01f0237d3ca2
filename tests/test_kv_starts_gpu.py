"""Batches whose first request does not begin at row 0: a part of a step's requests, with the whole step's rows."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_lists_ref as lists_ref
from test_kv_gpu import bounds
from test_kv_select_gpu import check, ints, make

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16 = torch.float16, torch.bfloat16


def later(s, before, after):
    """The same requests, `before` rows of none in front of them and `after` behind (make's `extra` has the room)."""
    assert s["q"].shape[0] == int(s["starts"][-1]) + before + after
    s["starts"] = s["starts"] + np.int32(before)
    return s


@pytest.mark.parametrize("before", [1, 7, 8, 16, 31, 100])
@pytest.mark.parametrize("new,heads,kvh,pages", [
    ([20], 4, 2, 40), ([9, 40, 0, 1, 17], 12, 4, 60),              # tiles of 8
    ([12], 4, 2, 900), ([9, 30], 2, 1, 2500),                      # shared by a cluster of CTAs
    ([300], 8, 8, 40), ([150, 1, 180], 8, 8, 60),                  # tiles of 16
    ([300], 8, 8, 1500),                                           # shared by a cluster
    ([5], 4, 2, 300), ([1, 8, 0, 3], 4, 2, 40)])                   # a tile's place is its request's
def test_rows_before_the_first_request(cuda, before, new, heads, kvh, pages):
    """Lists of the rows before it are left, and their `seen` is -1 (lists_ref.select and check hold both)."""
    for dtype, d in ((F16, 64), (BF16, 128)):
        s = later(make(cuda, dtype, heads, kvh, d, 16, [pages * 16 - 5 - 7 * r for r in range(len(new))], new, extra=before + 3), before, 3)
        for most in {max(new), 1, 9}:                              # a hint: each way to find a tile's request
            out = check(cuda, s, 12, 1, 2, most=most)
            assert bool((out.pages[:before] == -7).all()) and bool((out.seen[:before] == -1).all())


def test_first_requests_without_rows(cuda):
    s = later(make(cuda, F16, 4, 2, 64, 16, [300, 900, 700, 40], [0, 0, 30, 2], extra=70), 50, 20)
    check(cuda, s, 6, 1, 2)
    s = later(make(cuda, F16, 4, 2, 64, 16, [300, 900], [0, 0], extra=70), 50, 20)
    check(cuda, s, 6, 1, 2, most=20)


@pytest.mark.parametrize("fmt,dtype", [(INT4, F16), (NF4, BF16)])
def test_a_mixed_batch_in_two_calls(cuda, fmt, dtype):
    """A step's single tokens, then its prompts, each with the step's whole rows and a call of its own: the second leaves what the
    first made of its rows."""
    page, kvh, heads, d, keep = 16, 2, 8, 64, 6
    singles = 20
    ctx, new = [300, 41, 700, 16] * 5 + [1000, 64], [1] * singles + [30, 64]
    s = make(cuda, dtype, heads, kvh, d, page, ctx, new, extra=4)
    cache = b4gemv.KVCache.alloc(fmt, s["cache"].n_pages, kvh, page, d, cuda)
    g = torch.Generator(device=cuda).manual_seed(4)
    x, y = (torch.randn((cache.n_pages * page, kvh, d), generator=g, device=cuda) for _ in range(2))
    every = torch.arange(cache.n_pages * page, dtype=torch.int32, device=cuda)
    b4gemv.kv_append(cache, x, y, every)
    boxes = b4gemv.kv_new_boxes(cache)
    b4gemv.kv_boxes(cache, boxes, every)
    out = torch.full_like(s["q"], 9.0)
    tab, lens, starts = ints(s["tab"], cuda), ints(s["ctx"], cuda), ints(s["starts"], cuda)
    for part, most in ((slice(0, singles), 1), (slice(singles, singles + 2), 64)):
        lists = b4gemv.kv_select(cache, boxes, s["q"], tab[part], lens[part], starts[part.start:part.stop + 1], most, keep, 1, 2)
        b4gemv.kv_attention_lists(cache, s["q"], lists, out=out)
    lists, seen = lists_ref.select(page, d, boxes.cpu().numpy(), s["q"], s["tab"], ctx, s["starts"], keep, 1, 2, cache.n_pages)
    n = int(s["starts"][-1])
    want, wl, aux = lists_ref.attention(fmt, page, d, cache.blocks, s["q"][:n], lists[:n], seen[:n], d ** -0.5)
    tol, _ = bounds(fmt, dtype, want, wl, aux, keep * page)
    assert bool(((out[:n].double() - want).abs() <= tol).all()) and bool((out[n:] == 9.0).all())
