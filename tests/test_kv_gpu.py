"""The 4-bit key/value cache on the GPU against its restatement in kv_ref:
bookkeeping and codes equal, attention within bounds derived from the roundings
that the kernels make."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import b4gemv
import kv_ref as ref

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16 = torch.float16, torch.bfloat16


# ---- tables ---------------------------------------------------------------------

def check_tables(cuda, page, width, cached, added, ring, state, max_tokens, seed=0, stride=None):
    rng = np.random.default_rng(seed)
    n = len(cached)
    tab = rng.integers(0, 1000, (n, width)).astype(np.int32)
    want = ref.tables(page, tab, cached, added, ring, state, max_tokens)
    wide = torch.full((n, stride or width), 77, dtype=torch.int32, device=cuda)
    dev = wide[:, :width]
    dev.copy_(torch.from_numpy(tab))
    t = lambda v: torch.tensor(np.asarray(v, np.int32), device=cuda)  # noqa: E731
    step = b4gemv.kv_tables(page, dev, t(cached), t(added), t(ring), t(state), max_tokens)
    got = [dev, step.ctx_len, step.q_starts, step.slots, step.positions, step.free_state]
    for name, g, w in zip(("tables", "ctx_len", "q_starts", "slots", "positions", "free_state"), got, want):
        assert np.array_equal(g.cpu().numpy(), w), name
    assert stride is None or bool((wide[:, width:] == 77).all())


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("n,lo,hi", [(1, 1, 1), (3, 0, 2), (33, 1, 1), (257, 0, 90), (1000, 0, 40), (7000, 0, 3)])
def test_tables(cuda, page, n, lo, hi):
    rng = np.random.default_rng(n * 100 + page)
    cached, added = rng.integers(0, 300, n), rng.integers(lo, hi + 1, n)
    width = int(-(-(cached + added).max() // page)) + 1
    need = int((-(-(cached + added) // page) - -(-cached // page)).sum())
    ring = rng.permutation(need + 7)
    check_tables(cuda, page, width, cached, added, ring, [int(rng.integers(len(ring))), need + 3, 0], int(added.sum()) + 5)


def test_tables_edges(cuda):
    ring = np.arange(100, 140)
    check_tables(cuda, 16, 4, [], [], ring, [3, 20, 0], 8)                                # no request
    check_tables(cuda, 16, 4, [0, 16, 5], [0, 0, 0], ring, [3, 20, 0], 8)                 # no token
    check_tables(cuda, 16, 8, [15, 16, 17], [1, 1, 1], ring, [39, 20, 0], 3)              # page ends; the ring wraps
    check_tables(cuda, 16, 8, [10, 30, 0], [60, 40, 70], ring, [0, 4, 0], 170)            # pages run out
    check_tables(cuda, 16, 3, [40, 100, 0], [20, 5, 60], ring, [0, 30, 0], 85)            # past the table's width
    check_tables(cuda, 32, 5, [-4, 7], [9, -3], ring, [45, 60, 0], 10)                    # lengths below 0, a place past the ring
    check_tables(cuda, 16, 4, [3, 20], [20, 20], ring, [0, 30, 0], 13)                    # fewer slots than tokens
    check_tables(cuda, 16, 6, [3, 20], [20, 20], [], [0, 0, 0], 40)                       # no free page at all
    check_tables(cuda, 16, 5, [3, 20, 33], [20, 9, 1], ring, [0, 30, 0], 30, stride=9)    # rows wider than the table


def test_tables_buffers_reused_and_refusals(cuda):
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    tab, ring, state = t([[-1] * 4] * 2), t(list(range(8))), t([0, 8, 0])
    a = b4gemv.kv_tables(16, tab, t([0, 0]), t([17, 5]), ring, state, 22)
    b = b4gemv.kv_tables(16, tab, a.ctx_len, t([1, 1]), ring, a.free_state, 2)
    c = b4gemv.kv_tables(16, tab, b.ctx_len, t([1, 1]), ring, b.free_state, 2, out=a)      # a's buffers, b's state
    assert c.slots.data_ptr() == a.slots.data_ptr() and c.free_state.tolist() == [3, 5, 0]
    assert c.slots[:2].tolist() == [1 * 16 + 2, 2 * 16 + 6] and tab.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]]
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_tables(16, tab, t([0, 0]), t([1, 1]), ring, c.free_state, 2, out=c)      # the state in place
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_tables(8, tab, t([0, 0]), t([1, 1]), ring, state, 2)
    with pytest.raises(ValueError):
        b4gemv.kv_tables(16, tab, t([0, 0]), t([1]), ring, state, 2)
    with pytest.raises(ValueError):
        b4gemv.kv_tables(16, tab, torch.zeros(2, dtype=torch.int64, device=cuda), t([1, 1]), ring, state, 2)


# ---- append and read-back ----------------------------------------------------------

def data(shape, dtype, seed, special=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=g))
    if special:
        flat = x.reshape(-1, shape[-1])
        flat[0] = 0.0
        flat[1, 3] = float("nan")
        flat[2, 5] = float("inf")
        flat[3] = 1e-30                                  # INT4: the fp16 scale rounds to 0
        flat[4] *= 1e30 if dtype != F16 else 100         # INT4: the fp16 scale overflows
        flat[5] = float("nan")
        flat[6, :8] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 7.0, -7.0])   # ties of lround at scale 1
        flat[6, 8:] = 0.25
        flat[7] = 1e-41                                  # subnormal
        flat[8, :2] = torch.tensor([float("-inf"), float("nan")])
    return x.to(dtype)


def check_append(cuda, fmt, dtype, t, h, d, page, k, v, slots, pages):
    g = torch.Generator(device=cuda).manual_seed(1)
    blocks = torch.randint(0, 256, (pages, h, b4gemv.kv_block_bytes(fmt, page, d)), dtype=torch.uint8, device=cuda, generator=g)
    before = blocks.cpu().numpy()
    cache = b4gemv.KVCache(blocks, fmt, page, d)
    b4gemv.kv_append(cache, k, v, slots)
    s = slots.cpu().numpy()
    ok = (s >= 0) & (s < pages * page)
    codes, scales = ref.unpack_blocks(fmt, page, d, before)
    codes, scales = codes.copy(), scales.copy()
    at, row = s[ok] // page, s[ok] % page
    want = []
    for o, x in enumerate((k, v)):
        c, sc = ref.quantise(fmt, x.float().cpu().numpy())
        codes[o, at, :, row], scales[o, at, :, row] = c[ok], sc[ok]
        val = ref.values(fmt, c, sc)
        val[~ok] = 0
        want.append(val)
    got = blocks.cpu().numpy()
    assert got.tobytes() == ref.pack_blocks(fmt, codes, scales).tobytes()
    for g_, w in zip(b4gemv.kv_read(cache, slots), want):
        assert np.array_equal(g_.cpu().numpy(), w, equal_nan=True)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("t,h,d,page", [(1, 1, 64, 16), (17, 3, 128, 16), (301, 8, 128, 64), (77, 5, 64, 32)])
def test_append_and_read(cuda, fmt, dtype, t, h, d, page):
    pages = t // page + 2
    g = torch.Generator().manual_seed(t)
    slots = torch.randperm(pages * page, generator=g)[:t].to(torch.int32)
    if t > 3:
        slots[0], slots[2] = -1, pages * page                    # skipped
    k, v = (data((t, h, d), dtype, s, special=t > 9).to(cuda) for s in (1, 2))
    check_append(cuda, fmt, dtype, t, h, d, page, k, v, slots.to(cuda), pages)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("dtype", [F16, torch.float32])
def test_append_strides(cuda, fmt, dtype):
    """Columns of a fused row, heads outermost, a base that is no multiple of 16 bytes, one token broadcast to all."""
    t, h, d, page = 50, 4, 128, 16
    slots = torch.arange(t, dtype=torch.int32, device=cuda)
    rows = data((t, 2 * h * d + 24), dtype, 3).to(cuda)
    a = rows[:, 8:8 + h * d].view(t, h, d)
    b = data((h, t, d), dtype, 4).to(cuda).transpose(0, 1)
    c = rows[:, 1:1 + h * d].view(t, h, d)
    e = data((1, h, d), dtype, 5).to(cuda).expand(t, h, d)
    for k, v in ((a, b), (c, a), (e, c)):
        check_append(cuda, fmt, dtype, t, h, d, page, k, v, slots, 4)


def test_nf4_codes_beside_every_threshold(cuda):
    """Quotients within a few ulp of each place where the nearest level changes, with an absmax of 1, 3 and 0.7."""
    mid = (ref.NF4[1:].astype(np.float64) + ref.NF4[:-1]) / 2
    for a in (1.0, 3.0, 0.7):
        rows = []
        for m in mid:
            x = np.float32(m * a)
            near = [x]
            for _ in range(31):
                near.append(np.nextafter(near[-1], np.float32(9)))
            down = [x]
            for _ in range(31):
                down.append(np.nextafter(down[-1], np.float32(-9)))
            row = np.array(near + down, np.float32)
            row[31] = a
            rows.append(row)
        k = torch.from_numpy(np.array(rows)[:, None]).to(cuda)
        check_append(cuda, NF4, torch.float32, len(rows), 1, 64, 16, k, k.neg(), torch.arange(len(rows), dtype=torch.int32, device=cuda), 1)


def test_int4_codes_beside_every_tie(cuda):
    rows = []
    for s in (1.0, 0.3, 11.0):
        sc = np.float32(np.float16(np.float32(7 * s) * (np.float32(1) / np.float32(7))))
        row = []
        for m in np.arange(-7.5, 8):
            x = np.float32(m * sc)
            row += [x, np.nextafter(x, np.float32(99)), np.nextafter(x, np.float32(-99))]
        row = np.array(row + [0.0] * 15 + [7 * s], np.float32).clip(-7 * np.float32(s), 7 * np.float32(s))
        rows.append(row)
    k = torch.from_numpy(np.array(rows)[:, None]).to(cuda)
    check_append(cuda, INT4, torch.float32, 3, 1, 64, 16, k, k.neg(), torch.arange(3, dtype=torch.int32, device=cuda), 1)


def test_append_equals_the_weight_quantiser(cuda):
    """A cached head vector of 64 columns is a row in the weights' NF4 format."""
    x = torch.randn((48, 1, 64), device=cuda)
    slots = torch.arange(48, dtype=torch.int32, device=cuda)
    cache = b4gemv.KVCache.alloc(NF4, 3, 1, 16, 64, cuda)
    b4gemv.kv_append(cache, x, x, slots)
    assert torch.equal(b4gemv.kv_read(cache, slots)[1][:, 0], b4gemv.quantise_nf4_device(x[:, 0].contiguous(), True)[2])


# ---- attention -----------------------------------------------------------------------

def make(cuda, fmt, dtype, heads, kvh, d, page, ctx, new, seed=0, spare=3, extra=0):
    """A filled cache, its tables in a random order of pages, and packed queries (`extra` rows past the last)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    need = [-(-max(c, 0) // page) for c in ctx]
    pages, width = sum(need) + spare, max(need + [1])
    order = torch.randperm(pages, generator=g, device=cuda).int()
    tab = torch.full((len(ctx), width), -1, dtype=torch.int32, device=cuda)
    at = 0
    for r, n in enumerate(need):
        tab[r, :n] = order[at:at + n]
        at += n
    cache = b4gemv.KVCache.alloc(fmt, pages, kvh, page, d, cuda)
    every = torch.arange(pages * page, dtype=torch.int32, device=cuda)
    k, v = (torch.randn((pages * page, kvh, d), generator=g, device=cuda) * torch.exp(0.3 * torch.randn((pages * page, kvh, 1), generator=g, device=cuda))
            for _ in range(2))
    b4gemv.kv_append(cache, k, v, every)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=cuda)
    q = torch.randn((sum(new) + extra, heads, d), generator=g, device=cuda).to(dtype)
    return cache, q, tab, torch.tensor(ctx, dtype=torch.int32, device=cuda), starts, max(new + [0])


def bounds(fmt, dtype, out, lse, aux, keys, scale_rel=0.0):
    """What the kernels' roundings allow.  Weights are rounded to fp16 (2^-11 of each, and 2^-24 of the largest at least: then
    `keys` of them), the output once more to its type; scores and sums are in fp32 (2^-24 a step: 2^-16 of the sum of |q k|
    covers 128 columns and the exponential's error).  The NF4 code book in fp16 is within 3e-4 of each level, in keys
    and in values."""
    weight, size = aux
    book = 3e-4 if fmt == NF4 else 0.0
    score = size * (2.0 ** -16 + book) + 2.0 ** -18
    top = weight.amax(-1, keepdim=True)
    tol = weight * (2.0 ** -11 + 2.0 ** -16 + book + 2 * score[..., None]) + out.abs() * (2.0 ** -11 if dtype == F16 else 2.0 ** -8)
    tol = tol + keys * 2.0 ** -24 * top + (2.0 ** -24 if dtype == F16 else 0.0)
    return tol, score + 2.0 ** -20 * lse.abs().clamp(max=1e30)


def check_attention(cuda, fmt, dtype, heads, kvh, d, page, ctx, new, window=0, causal=True, scale=None, seed=0, state=None,
                    out=None, lse=True, **more):
    cache, q, tab, ctx_t, starts, most = state or make(cuda, fmt, dtype, heads, kvh, d, page, ctx, new, seed)
    total = int(starts[-1])
    ls = torch.full((q.shape[0], heads), 5.0, device=cuda) if lse else None
    if out is None:
        out = torch.full_like(q, 9.0)
    got = b4gemv.kv_attention(cache, q, tab, ctx_t, starts, most, scale=scale, window=window, causal=causal, out=out, lse=ls, **more)
    sc = d ** -0.5 if scale is None else scale
    want, wl, aux = ref.attention(fmt, page, d, cache.blocks, q, tab, ctx_t.tolist(), starts.tolist(), sc, window, not causal)
    tol, ltol = bounds(fmt, dtype, want, wl, aux, max([min(c, window + 8) if window else c for c in ctx] + [1]))
    err = (got[:total].double() - want[:total]).abs()
    assert bool(torch.isfinite(got[:total]).all())
    bad = err > tol[:total]
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / tol[:total]).max()):.2f} of its bound"
    if lse:
        empty = torch.isinf(wl[:total])
        assert torch.equal(torch.isinf(ls[:total]) & (ls[:total] < 0), empty)
        le = (ls[:total].double() - wl[:total])[~empty].abs()
        assert not bool((le > ltol[:total][~empty]).any())
        assert bool((ls[total:] == 5.0).all())
    assert bool((got[total:] == 9.0).all()) or total == q.shape[0]
    return got


FORMS = [(INT4, F16), (INT4, BF16), (NF4, F16), (NF4, BF16)]


@pytest.mark.parametrize("fmt,dtype", FORMS)
@pytest.mark.parametrize("heads,kvh,d,page", [(28, 4, 128, 16), (64, 8, 128, 64), (4, 4, 64, 32), (32, 2, 64, 16), (5, 1, 128, 32)])
def test_single_tokens(cuda, fmt, dtype, heads, kvh, d, page):
    check_attention(cuda, fmt, dtype, heads, kvh, d, page, [1, 2, 15, 16, 17, 63, 64, 65, 130, 700, 31, 33], [1] * 12)


@pytest.mark.parametrize("fmt,dtype", FORMS)
@pytest.mark.parametrize("n,ctx", [(1, 1), (1, 5000), (2, 20001), (300, 40)])
def test_single_tokens_batches(cuda, fmt, dtype, n, ctx):
    check_attention(cuda, fmt, dtype, 16, 2, 128, 64, [ctx - r % 7 if ctx > 7 else ctx for r in range(n)], [1] * n)


@pytest.mark.parametrize("fmt,dtype", FORMS)
@pytest.mark.parametrize("heads,kvh,d", [(28, 4, 128), (8, 8, 64), (32, 4, 128), (64, 1, 64)])
def test_few_tokens_ragged(cuda, fmt, dtype, heads, kvh, d):
    """Drafted tokens: 0 to 8 queries a request, the first of them beside short contexts."""
    check_attention(cuda, fmt, dtype, heads, kvh, d, 16, [8, 5, 100, 1, 64, 65, 333, 17, 0], [8, 3, 0, 1, 5, 2, 7, 4, 0])


@pytest.mark.parametrize("fmt,dtype", FORMS)
@pytest.mark.parametrize("heads,kvh,d,page", [(28, 4, 128, 64), (16, 2, 64, 16), (6, 6, 128, 32), (3, 1, 128, 64)])
def test_prompts(cuda, fmt, dtype, heads, kvh, d, page):
    """Chunks of prompts, alone and behind cached tokens, with single tokens among them."""
    check_attention(cuda, fmt, dtype, heads, kvh, d, page, [200, 301, 77, 1, 500, 129, 260], [200, 64, 77, 1, 1, 129, 33])


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 5, 70])
@pytest.mark.parametrize("window", [1, 16, 100, 4096])
def test_windows(cuda, fmt, new, window):
    check_attention(cuda, fmt, F16, 14, 2, 128, 32, [90, 300, 65, 1000], [new] * 4 if new < 65 else [70, 200, 65, 3], window=window)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_rows_that_see_nothing(cuda, fmt, new):
    """More queries than tokens: the first see no key; requests without any token; a request whose pages are all missing."""
    state = make(cuda, fmt, F16, 8, 2, 128, 16, [0, 3, 40, 16, 33], [new, new, new, 2, 1])
    state[2][3, :] = -1
    got = check_attention(cuda, fmt, F16, 8, 2, 128, 16, [0, 3, 40, 16, 33], [new, new, new, 2, 1], state=state)
    assert bool((got[:new] == 0).all()) and bool((got[3 * new:3 * new + 2] == 0).all())


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 4, 80])
def test_every_key_seen(cuda, fmt, new):
    check_attention(cuda, fmt, BF16, 8, 4, 64, 16, [50, 7, 333], [new, 2, new], causal=False)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_masked_places_hold_anything(cuda, fmt, new):
    """Slots past the last token hold NaN and infinite scales, and pages outside the cache are not read."""
    ctx = [100, 33, 129, 250]
    state = make(cuda, fmt, F16, 8, 2, 128, 32, ctx, [new] * 4)
    cache, _, tab, _, _, _ = state
    codes, s = ref.unpack_blocks(fmt, 32, 128, cache.blocks.cpu().numpy())
    s = s.copy()
    tl = tab.cpu().numpy()
    used = np.zeros(s.shape[1:2] + s.shape[3:], bool)
    for r, c in enumerate(ctx):
        for p in range(c):
            used[tl[r, p // 32], p % 32] = True
    s[0][np.broadcast_to(~used[:, None], s[0].shape)] = np.nan
    s[1][np.broadcast_to(~used[:, None], s[1].shape)] = np.inf
    cache.blocks.copy_(torch.from_numpy(ref.pack_blocks(fmt, codes.copy(), s)))
    tab[3, 2] = cache.n_pages + 5
    tab[3, 4] = -7
    check_attention(cuda, fmt, F16, 8, 2, 128, 32, ctx, [new] * 4, state=state)


@pytest.mark.parametrize("new", [1, 4, 90])
def test_scores_of_any_size(cuda, new):
    """Scales far from 1: scores in the thousands (one key takes all), scores of 0, values near fp16's ends, bf16 queries past fp16."""
    for fmt in (INT4, NF4):
        for mul_k, mul_v, mul_q, dtype in ((60.0, 1.0, 30.0, F16), (0.0, 1.0, 1.0, F16), (1.0, 1e-3, 1.0, F16), (1.0, 3000.0, 1.0, F16),
                                           (1e-3, 1.0, 1e5, BF16), (1.0, 1.0, 1e-6, BF16)):
            cache, q, tab, ctx, starts, most = make(cuda, fmt, dtype, 8, 2, 128, 16, [70, 300], [new, new])
            codes, s = ref.unpack_blocks(fmt, 16, 128, cache.blocks.cpu().numpy())
            s = s.astype(np.float32)
            s[0] *= mul_k
            s[1] *= mul_v
            cache.blocks.copy_(torch.from_numpy(ref.pack_blocks(fmt, codes.copy(), s)))
            check_attention(cuda, fmt, dtype, 8, 2, 128, 16, [70, 300], [new, new], state=(cache, (q * mul_q).contiguous(), tab, ctx, starts, most))


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 70])
def test_values_of_unlike_size(cuda, fmt, new):
    """Tokens whose value scales differ by 2^20, the large ones late and early."""
    for flip in (False, True):
        state = make(cuda, fmt, F16, 4, 1, 128, 16, [200], [new])
        cache, _, tab, _, _, _ = state
        codes, s = ref.unpack_blocks(fmt, 16, 128, cache.blocks.cpu().numpy())
        s = s.astype(np.float32)
        order = tab[0].cpu().numpy()[:13]
        ramp = np.exp2(np.linspace(-14, 6, 13))[::-1 if flip else 1]
        s[1][order] = ramp[:, None, None]
        cache.blocks.copy_(torch.from_numpy(ref.pack_blocks(fmt, codes.copy(), s)))
        check_attention(cuda, fmt, F16, 4, 1, 128, 16, [200], [new], state=state)


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 3, 66])
def test_strides_scale_stream_and_rows_past_the_last(cuda, fmt, new):
    """Queries as columns of a fused row, the output as heads outermost, tables wider than needed, rows past q_starts' last
    left alone, on a stream of the caller's."""
    heads, kvh, d, page, ctx = 6, 2, 128, 16, [40, 200, 129]
    cache, q, tab, ctx_t, starts, most = make(cuda, fmt, F16, heads, kvh, d, page, ctx, [new] * 3, extra=4)
    wide = torch.zeros((q.shape[0], heads * d + 512), dtype=F16, device=cuda)
    wide[:, 256:256 + heads * d] = q.reshape(q.shape[0], -1)
    q = wide[:, 256:256 + heads * d].view(q.shape[0], heads, d)
    big = torch.full((len(ctx), tab.shape[1] + 5), 10 ** 9, dtype=torch.int32, device=cuda)
    big[:, :tab.shape[1]] = tab
    out = torch.full((heads, q.shape[0], d), 9.0, dtype=F16, device=cuda).transpose(0, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check_attention(cuda, fmt, F16, heads, kvh, d, page, ctx, [new] * 3, scale=0.2, out=out,
                        state=(cache, q, big[:, :tab.shape[1]], ctx_t, starts, most))
    torch.cuda.current_stream().wait_stream(s)


@pytest.mark.parametrize("fmt", [INT4, NF4])
def test_one_workspace_serves_calls_of_every_shape_and_repeats_bits(cuda, fmt):
    """Calls one after another, without a wait between them, leave the workspace ready; a call's bits do not vary."""
    states = [make(cuda, fmt, F16, 8, 2, 128, 32, c, n, seed=i) for i, (c, n) in enumerate(
        (([3000], [1]), ([50] * 40, [1] * 40), ([700, 90, 2000], [4, 1, 6]), ([600, 400], [300, 1]), ([9000, 10], [1, 1])))]
    need = max(b4gemv.kv_attention_workspace(*s) for s in states)
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device=cuda)
    first = [b4gemv.kv_attention(*s, ws=ws) for s in states]
    for _ in range(3):
        for s, f in zip(states, first):
            assert torch.equal(b4gemv.kv_attention(*s, ws=ws), f)
    for s, f in zip(states, first):
        assert torch.equal(b4gemv.kv_attention(*s), f)                       # and not with the package's


def test_max_q_is_a_hint(cuda):
    """Requests with more queries than max_q says, and fewer, give the same within the bounds."""
    ctx, new = [300, 90, 40], [60, 1, 9]
    s = make(cuda, INT4, F16, 8, 2, 128, 32, ctx, new)
    for most in (1, 4, 9, 60, 4000):
        check_attention(cuda, INT4, F16, 8, 2, 128, 32, ctx, new, state=s[:5] + (most,))


def test_cache_past_4_gib(cuda):
    """Pages whose bytes lie past 32 bits."""
    pages = (1 << 32) // (8 * b4gemv.kv_block_bytes(INT4, 64, 128)) + 100
    cache = b4gemv.KVCache(torch.empty((pages, 8, b4gemv.kv_block_bytes(INT4, 64, 128)), dtype=torch.uint8, device=cuda), INT4, 64, 128)
    ids = [pages - 1, 0, pages - 40, 7, pages - 2]
    slots = torch.tensor([i * 64 + j for i in ids for j in range(64)], dtype=torch.int32, device=cuda)
    k, v = (torch.randn((320, 8, 128), device=cuda) for _ in range(2))
    b4gemv.kv_append(cache, k, v, slots)
    small = b4gemv.KVCache.alloc(INT4, 5, 8, 64, 128, cuda)
    b4gemv.kv_append(small, k, v, torch.arange(320, dtype=torch.int32, device=cuda))
    for a, b in zip(b4gemv.kv_read(cache, slots), b4gemv.kv_read(small, torch.arange(320, dtype=torch.int32, device=cuda))):
        assert torch.equal(a, b)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    for new in (1, 100):
        q = torch.randn((new, 16, 128), device=cuda).half()
        a = b4gemv.kv_attention(cache, q, t([ids]), t([310]), t([0, new]), new)
        b = b4gemv.kv_attention(small, q, t([[0, 1, 2, 3, 4]]), t([310]), t([0, new]), new)
        assert torch.equal(a, b)


@pytest.mark.parametrize("new", [1, 40])
def test_graph_replay(cuda, new):
    """A captured step (tables, append, attention) replayed with other lengths in the same buffers."""
    heads, kvh, d, page = 8, 2, 128, 16
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    cache = b4gemv.KVCache.alloc(INT4, 64, kvh, page, d, cuda)
    tab, ring, state = torch.full((3, 20), -1, dtype=torch.int32, device=cuda), torch.randperm(64, device=cuda).int(), t([5, 64, 0])
    cached, added = t([0, 0, 0]), t([new, new, new])
    k, v = (torch.randn((3 * new, kvh, d), device=cuda).half() for _ in range(2))
    q = torch.randn((3 * new, heads, d), device=cuda).half()
    out = torch.empty_like(q)

    def step():
        s = b4gemv.kv_tables(page, tab, cached, added, ring, state, 3 * new)
        b4gemv.kv_append(cache, k, v, s.slots)
        b4gemv.kv_attention(cache, q, tab, s.ctx_len, s.q_starts, new, out=out)
        cached.copy_(s.ctx_len)
        state.copy_(s.free_state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="relaxed"):
        step()
    for i in range(2, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert cached.tolist() == [i * new] * 3
        want, wl, aux = ref.attention(INT4, page, d, cache.blocks, q, tab, cached.tolist(), [0, new, 2 * new, 3 * new], d ** -0.5)
        tol, _ = bounds(INT4, F16, want, wl, aux, i * new)
        assert bool(((out.double() - want).abs() <= tol).all())
    del graph


def test_refused_on_the_gpu(cuda):
    s = make(cuda, INT4, F16, 8, 2, 128, 16, [30], [1])
    cache, q, tab, ctx, starts, most = s
    with pytest.raises(ValueError):
        b4gemv.kv_attention(cache, q.float(), tab, ctx, starts, most)
    with pytest.raises(ValueError):
        b4gemv.kv_attention(cache, q[:, :7], tab, ctx, starts, most)
    with pytest.raises(ValueError):
        b4gemv.kv_attention(cache, q, tab.long(), ctx, starts, most)
    with pytest.raises(ValueError):
        b4gemv.kv_attention(cache, q, tab, ctx, starts[:1], most)
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_attention(cache, q, tab, ctx, starts, most, window=5, causal=False)
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_attention(cache, q, tab, ctx, starts, most, scale=float("nan"))
    odd = torch.zeros(q.numel() + 8, dtype=F16, device=cuda)[1:1 + q.numel()].view_as(q)
    with pytest.raises(b4gemv.B4Error):
        b4gemv.kv_attention(cache, odd, tab, ctx, starts, most)
    with pytest.raises(ValueError):
        b4gemv.KVCache(cache.blocks[:, :, :-1], INT4, 16, 128)
    with pytest.raises(b4gemv.B4Error):
        b4gemv.KVCache.alloc(INT4, 4, 2, 16, 96, cuda)
    with pytest.raises(ValueError):
        b4gemv.kv_append(cache, q, q, torch.zeros(1, dtype=torch.int32, device=cuda))
    assert b4gemv.kv_attention(cache, q[:0], tab, ctx, starts, most).shape[0] == 0
