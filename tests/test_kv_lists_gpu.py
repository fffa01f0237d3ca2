"""Attention over lists of pages against 64 bits, and the operators of a layer with a choice of pages together: append, boxes,
choice, attention."""
import numpy as np
import pytest
import torch

import b4gemv
import kv_lists_ref as lists_ref
import kv_ref as ref
from test_kv_gpu import bounds

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16 = torch.float16, torch.bfloat16
FORMS = [(INT4, F16), (INT4, BF16), (NF4, F16), (NF4, BF16)]


def ints(x, cuda):
    return torch.tensor(np.asarray(x, np.int32), device=cuda)


def filled(cuda, fmt, pages, kvh, page, d, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    cache = b4gemv.KVCache.alloc(fmt, pages, kvh, page, d, cuda)
    k, v = (torch.randn((pages * page, kvh, d), generator=g, device=cuda) * torch.exp(0.3 * torch.randn((pages * page, kvh, 1), generator=g, device=cuda))
            for _ in range(2))
    b4gemv.kv_append(cache, k, v, torch.arange(pages * page, dtype=torch.int32, device=cuda))
    return cache


def check(cuda, cache, q, lists, seen, scale=None, **more):
    """The bounds of attention over a whole context (test_kv_gpu): a list is one."""
    heads, page, width = q.shape[1], cache.page_size, lists.shape[2]
    out, lse = torch.full_like(q, 9.0), torch.full((q.shape[0], heads), 5.0, device=cuda)
    pages = lists if torch.is_tensor(lists) else ints(lists, cuda)
    got = b4gemv.kv_attention_lists(cache, q, b4gemv.KVLists(pages, ints(seen, cuda)), scale=scale, out=out, lse=lse, **more)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    sc = cache.head_dim ** -0.5 if scale is None else scale
    seen = np.asarray(seen)
    want, wl, aux = lists_ref.attention(cache.fmt, page, cache.head_dim, cache.blocks, q, pages.cpu().numpy(), seen, sc)
    tol, ltol = bounds(cache.fmt, q.dtype, want, wl, aux, width * page)
    there = torch.from_numpy(seen >= 0).to(cuda)
    err = (out.double() - want).abs()
    assert bool((err <= tol)[there].all()), f"worst {float((err / tol)[there].max()):.2f} of its bound"
    empty = torch.isinf(wl)
    assert torch.equal((torch.isinf(lse) & (lse < 0))[there], empty[there])
    assert not bool(((lse.double() - wl).abs() > ltol)[there & ~empty.any(-1)].any())
    assert bool((out[~there] == 9.0).all()) and bool((lse[~there] == 5.0).all())
    assert b4gemv.load().b4_device_error(0) == 0
    return out


def random_lists(rng, total, kvh, keep, pages):
    return np.stack([[rng.permutation(pages)[:keep] for _ in range(kvh)] for _ in range(total)]).astype(np.int32)


@pytest.mark.parametrize("fmt,dtype", FORMS)
@pytest.mark.parametrize("heads,kvh,d,page", [(28, 4, 128, 16), (64, 8, 128, 64), (4, 4, 64, 32), (32, 2, 64, 16), (5, 1, 128, 32), (64, 1, 128, 64), (40, 1, 64, 32)])
def test_lists(cuda, fmt, dtype, heads, kvh, d, page):
    rng = np.random.default_rng(heads + page)
    cache = filled(cuda, fmt, 40, kvh, page, d)
    q = torch.randn((9, heads, d), device=cuda).to(dtype)
    keep = 7
    seen = [1, page - 1, page, page + 1, 3 * page + 5, keep * page, 0, -1, keep * page - 1]
    check(cuda, cache, q, random_lists(rng, 9, kvh, keep, 40), seen)


@pytest.mark.parametrize("fmt,dtype", FORMS)
@pytest.mark.parametrize("total,keep", [(1, 64), (1, 300), (32, 32), (200, 9), (300, 5), (1100, 2), (3, 1)])
def test_numbers_of_queries_and_pages(cuda, fmt, dtype, total, keep):
    rng = np.random.default_rng(total)
    cache = filled(cuda, fmt, 320, 2, 16, 64)
    q = torch.randn((total, 14, 64), device=cuda).to(dtype)
    seen = rng.integers(0, keep * 16 + 1, total)
    seen[rng.integers(0, total, total // 5)] = -1
    check(cuda, cache, q, random_lists(rng, total, 2, keep, 320), seen)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_missing_and_repeated_pages(cuda, fmt, page):
    """An entry outside the cache is masked, wherever it stands; a page listed twice counts twice; more seen than listed."""
    rng = np.random.default_rng(page)
    cache = filled(cuda, fmt, 12, 2, page, 128)
    q = torch.randn((8, 6, 128), device=cuda).half()
    lists = random_lists(rng, 8, 2, 6, 12)
    lists[0, :, 1:3], lists[1, 0, 5], lists[2] = -1, 12, -1
    lists[3, 1, :], lists[4, :, 0], lists[5, 0, 2] = 4, -2 ** 31, 2 ** 31 - 1
    check(cuda, cache, q, lists, [6 * page, 6 * page, 6 * page, 6 * page, 2 * page + 3, 3 * page - 1, 7 * page, 2 ** 31 - 1])


@pytest.mark.parametrize("fmt", [INT4, NF4])
def test_what_is_not_seen_holds_anything(cuda, fmt):
    """NaN and infinite scales behind the last token seen, and in pages of other lists."""
    cache = filled(cuda, fmt, 10, 1, 32, 64)
    codes, s = ref.unpack_blocks(fmt, 32, 64, cache.blocks.cpu().numpy())
    s = s.copy()
    s[:, 5, :, 20:] = np.nan
    s[:, 6, :, 1:] = np.inf
    s[:, 9] = np.nan
    cache.blocks.copy_(torch.from_numpy(ref.pack_blocks(fmt, codes, s)))
    q = torch.randn((3, 8, 64), device=cuda).half()
    lists = np.array([[[0, 3, 5]], [[6, 9, 9]], [[1, 2, 9]]], np.int32)
    out = check(cuda, cache, q, lists, [84, 1, 64])
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
def test_scales(cuda, scale):
    rng = np.random.default_rng(1)
    cache = filled(cuda, INT4, 30, 2, 16, 128)
    check(cuda, cache, torch.randn((5, 8, 128), device=cuda).half(), random_lists(rng, 5, 2, 20, 30), [320, 300, 17, 1, 0], scale=scale)


def test_strides_streams_and_repeats(cuda):
    rng = np.random.default_rng(2)
    cache = filled(cuda, INT4, 100, 4, 32, 128)
    total, keep = 40, 12
    q = torch.randn((total, 28, 128), device=cuda).half()
    lists, seen = random_lists(rng, total, 4, keep, 100), rng.integers(1, keep * 32, total)
    first = check(cuda, cache, q, lists, seen)
    room = torch.full((total, 4, keep + 5), -1, dtype=torch.int32, device=cuda)
    room[..., :keep] = ints(lists, cuda)
    wide = torch.zeros((total, 30, 136), dtype=F16, device=cuda)
    wide[:, 1:29, :128] = q
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again = check(cuda, cache, wide[:, 1:29, :128], room[..., :keep], seen, stream=side)
    assert torch.equal(first, again)
    ws = torch.zeros(b4gemv.kv_attention_lists_workspace(cache, q, b4gemv.KVLists(room[..., :keep], ints(seen, cuda))), dtype=torch.uint8, device=cuda)
    for _ in range(2):
        assert torch.equal(first, check(cuda, cache, q, lists, seen, ws=ws))
    with pytest.raises(b4gemv.B4Error):
        check(cuda, cache, q, lists, seen, ws=ws[:-16])


def test_equal_to_attention_over_the_whole_context(cuda):
    """Lists that hold a request's every page are its context.  The two kernels add in orders of their own; each is within its
    bound of the exact values, so they are within twice that of one another."""
    page, kvh, d = 16, 2, 128
    cache = filled(cuda, NF4, 60, kvh, page, d)
    ctx, order = [1, 100, 333, 480], torch.randperm(60).int()
    tab, at = torch.full((4, 30), -1, dtype=torch.int32), 0
    for r, c in enumerate(ctx):
        n = -(-c // page)
        tab[r, :n] = order[at:at + n]
        at += n
    tab = tab.to(cuda)
    q = torch.randn((4, 16, d), device=cuda).bfloat16()
    a = b4gemv.kv_attention(cache, q, tab, ints(ctx, cuda), ints(range(5), cuda), 1)
    lists = tab[:, None].expand(4, kvh, 30).contiguous()
    b = b4gemv.kv_attention_lists(cache, q, b4gemv.KVLists(lists, ints(ctx, cuda)))
    want, wl, aux = lists_ref.attention(NF4, page, d, cache.blocks, q, lists.cpu().numpy(), np.array(ctx), d ** -0.5)
    tol, _ = bounds(NF4, BF16, want, wl, aux, 480)
    assert bool(((a.double() - b.double()).abs() <= 2 * tol).all())


def test_no_queries(cuda):
    cache = filled(cuda, INT4, 2, 2, 16, 64)
    q = torch.empty((0, 4, 64), dtype=F16, device=cuda)
    lists = b4gemv.KVLists(torch.empty((0, 2, 3), dtype=torch.int32, device=cuda), torch.empty(0, dtype=torch.int32, device=cuda))
    assert b4gemv.kv_attention_lists(cache, q, lists).shape == (0, 4, 64)
    q, lists = torch.full((2, 4, 64), 2.0, dtype=F16, device=cuda), b4gemv.KVLists(torch.empty((2, 2, 0), dtype=torch.int32, device=cuda), ints([0, 5], cuda))
    assert not bool(b4gemv.kv_attention_lists(cache, q, lists).any())                    # of no pages


def test_calls_at_once_on_two_streams(cuda):
    """Choices and attention of two layers side by side, with outputs of their own streams and workspaces of their own."""
    layers, want = [], []
    for seed in range(2):
        cache = filled(cuda, INT4, 300, 2, 16, 128, seed)
        boxes = b4gemv.kv_new_boxes(cache)
        b4gemv.kv_boxes(cache, boxes, torch.arange(300 * 16, dtype=torch.int32, device=cuda))
        q = torch.randn((3, 14, 128), generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).half()
        tab = torch.randperm(300, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).int().view(3, 100)
        ctx, starts = ints([1600, 900, 1333], cuda), ints(range(4), cuda)
        lists = b4gemv.kv_select(cache, boxes, q, tab, ctx, starts, 1, 40)
        ws = torch.zeros(b4gemv.kv_attention_lists_workspace(cache, q, lists), dtype=torch.uint8, device=cuda)
        layers.append((cache, boxes, q, tab, ctx, starts, ws))
        want.append((lists.pages.clone(), b4gemv.kv_attention_lists(cache, q, lists)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for stream, (cache, boxes, q, tab, ctx, starts, ws) in zip(streams, layers):
            lists = b4gemv.kv_select(cache, boxes, q, tab, ctx, starts, 1, 40, stream=stream)
            got.append((lists.pages, b4gemv.kv_attention_lists(cache, q, lists, ws=ws, stream=stream)))
    torch.cuda.synchronize()
    for i, (pages, out) in enumerate(got):
        assert torch.equal(pages, want[i % 2][0]) and torch.equal(out, want[i % 2][1])


# ---- together -------------------------------------------------------------------------

class Layer:
    """A layer's cache, boxes and bookkeeping over steps, as a program holds them."""

    def __init__(self, cuda, fmt, dtype, heads, kvh, d, page, requests, pages, room, keep, first, last):
        self.cuda, self.keep, self.first, self.last, self.room = cuda, keep, first, last, room
        self.cache = b4gemv.KVCache.alloc(fmt, pages, kvh, page, d, cuda)
        self.boxes = b4gemv.kv_new_boxes(self.cache)
        self.rotary = b4gemv.Rotary(d, device=cuda)
        self.tab = torch.full((requests, pages), -1, dtype=torch.int32, device=cuda)
        self.ring, self.state = torch.randperm(pages, device=cuda).int(), ints([3, pages, 0], cuda)
        self.cached = torch.zeros(requests, dtype=torch.int32, device=cuda)
        self.q, self.k, self.v = (torch.zeros((room, h, d), dtype=dtype, device=cuda) for h in (heads, kvh, kvh))
        self.added = torch.zeros(requests, dtype=torch.int32, device=cuda)
        self.out = torch.full_like(self.q, 9.0)

    def step(self, most):
        s = b4gemv.kv_tables(self.cache.page_size, self.tab, self.cached, self.added, self.ring, self.state, self.room)
        self.turned = b4gemv.kv_append_rotary(self.cache, self.rotary, self.q, self.k, self.v, s.positions, s.slots)
        b4gemv.kv_boxes(self.cache, self.boxes, s.slots)
        self.lists = b4gemv.kv_select(self.cache, self.boxes, self.turned, self.tab, s.ctx_len, s.q_starts, most, self.keep, self.first, self.last)
        b4gemv.kv_attention_lists(self.cache, self.turned, self.lists, out=self.out)
        self.s = s
        self.cached.copy_(s.ctx_len)
        self.state.copy_(s.free_state)

    def check(self, done):
        c = self.cache
        box = self.boxes.cpu().numpy()
        ctx, starts, tab = self.s.ctx_len.tolist(), self.s.q_starts.tolist(), self.tab.cpu().numpy()
        assert ctx == done
        full = [int(p) for r, n in enumerate(ctx) for p in tab[r, : n // c.page_size]]
        assert np.array_equal(box[full], lists_ref.boxes(c.fmt, c.page_size, c.head_dim, c.blocks.cpu().numpy()[full]))
        lists, seen = lists_ref.select(c.page_size, c.head_dim, box, self.turned, tab, ctx, starts, self.keep, self.first, self.last, c.n_pages)
        n = starts[-1]
        assert np.array_equal(self.lists.seen.cpu().numpy(), seen) and np.array_equal(self.lists.pages.cpu().numpy()[:n], lists[:n])
        want, wl, aux = lists_ref.attention(c.fmt, c.page_size, c.head_dim, c.blocks, self.turned[:n], lists[:n], seen[:n], c.head_dim ** -0.5)
        tol, _ = bounds(c.fmt, self.q.dtype, want, wl, aux, self.keep * c.page_size)
        assert bool(((self.out[:n].double() - want).abs() <= tol).all())
        assert bool((self.out[n:] == 9.0).all())
        self.out.fill_(9.0)


@pytest.mark.parametrize("fmt,dtype", FORMS)
def test_a_layers_steps(cuda, fmt, dtype):
    """Prompts, single tokens and drafts in turn; a choice once a context is longer than it."""
    layer = Layer(cuda, fmt, dtype, 8, 2, 64, 16, 3, 80, 600, 6, 1, 2)
    done = [0, 0, 0]
    for i, added in enumerate(([300, 15, 96], [1, 1, 1], [0, 90, 3], [5, 0, 1], [1, 1, 1])):
        for x in (layer.q, layer.k, layer.v):
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device=cuda).manual_seed(i), device=cuda))
        layer.added.copy_(ints(added, cuda))
        layer.step(max(added))
        done = [a + b for a, b in zip(done, added)]
        layer.check(done)


@pytest.mark.parametrize("new", [1, 12])
def test_a_captured_step_replayed(cuda, new):
    """The whole step in a graph, replayed as the contexts grow past what is kept, page ends among the steps."""
    layer = Layer(cuda, INT4, F16, 8, 2, 128, 16, 3, 90, 3 * new + 7, 4, 1, 1)
    layer.added.fill_(new)
    for x in (layer.q, layer.k, layer.v):
        x.normal_()
    layer.step(new)                                                                      # makes the package's workspace
    torch.cuda.synchronize()
    layer.check([new] * 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(new)
    for i in range(2, 40 if new == 1 else 12):
        for x in (layer.q, layer.k, layer.v):
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        if new > 1 or i % 16 in (0, 1) or i > 80:
            layer.check([i * new] * 3)
        layer.out.fill_(9.0)
    del graph
