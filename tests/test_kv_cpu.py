"""The 4-bit key/value cache's entry points without a GPU: sizes, refusals before
any launch, and the layout's restatement."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import b4gemv
import kv_ref as ref
from b4gemv import _lib

INV = 1          # cudaErrorInvalidValue
P = 4096         # an address that nothing reads


def cache(**kw):
    a = dict(blocks=P, fmt=0, n_pages=10, page_size=16, kv_heads=2, head_dim=128)
    a.update(kw)
    return _lib.KvCache(*[a[n] for n, _ in _lib.KvCache._fields_])


BAD_CACHES = [dict(blocks=None), dict(blocks=P + 8), dict(fmt=2), dict(fmt=-1), dict(n_pages=0), dict(page_size=8),
              dict(page_size=48), dict(page_size=128), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=256),
              dict(n_pages=1 << 28)]


@pytest.mark.parametrize("fmt,scale", [(0, 2), (1, 4)])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("d", [64, 128])
def test_block_bytes(fmt, scale, page, d):
    n = b4gemv.kv_block_bytes(fmt, page, d)
    assert n == 2 * page * (d // 2 + scale) and n % 16 == 0
    rng = np.random.default_rng(0)
    b = rng.integers(0, 256, (3, 2, n)).astype(np.uint8)
    codes, s = ref.unpack_blocks(fmt, page, d, b)
    assert codes.shape == (2, 3, 2, page, d) and s.shape == (2, 3, 2, page)
    assert ref.pack_blocks(fmt, codes, s).tobytes() == b.tobytes()


def test_block_bytes_refusals():
    for args in ((2, 16, 128), (0, 17, 128), (0, 16, 80)):
        with pytest.raises(b4gemv.B4Error):
            b4gemv.kv_block_bytes(*args)
    assert b4gemv.load().b4_kv_block_bytes(0, 16, 128, None) == INV


def step(**kw):
    a = dict(n_req=2, page_size=16, table_width=4, ring_size=8, max_tokens=4, table_stride=4,
             **{n: P * (i + 1) for i, n in enumerate(("tables", "cached", "added", "free_pages", "free_state", "ctx_len",
                                                      "q_starts", "slots", "positions", "free_state_out"))})
    a.update(kw)
    return _lib.KvStep(*[a[n] for n, _ in _lib.KvStep._fields_])


@pytest.mark.parametrize("bad", [dict(n_req=-1), dict(n_req=16385), dict(page_size=24), dict(table_width=-1), dict(ring_size=-1),
                                 dict(max_tokens=-1), dict(table_stride=3), dict(tables=None), dict(cached=None), dict(added=None),
                                 dict(free_pages=None), dict(free_state=None), dict(ctx_len=None), dict(q_starts=None),
                                 dict(slots=None), dict(positions=None), dict(free_state_out=None),
                                 dict(free_state_out=P * 5), dict(free_state_out=P * 5 + 4), dict(free_state_out=P * 5 - 8)])
def test_tables_refusals(bad):
    assert b4gemv.load().b4_kv_tables(ctypes.byref(step(**bad)), None) == INV
    assert b4gemv.load().b4_kv_tables(None, None) == INV


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_append_and_read_refuse_bad_caches(bad):
    lib = b4gemv.load()
    c = cache(**bad)
    assert lib.b4_kv_append(ctypes.byref(c), P, P, 0, 1, 1, 1, 1, P, 4, None) == INV
    assert lib.b4_kv_read(ctypes.byref(c), P, 4, P, P, None) == INV


def test_append_and_read_refusals():
    lib, c = b4gemv.load(), ctypes.byref(cache())
    assert lib.b4_kv_append(None, P, P, 0, 1, 1, 1, 1, P, 4, None) == INV
    for args in ((P, P, 3, P, 4), (P, P, -1, P, 4), (None, P, 0, P, 4), (P, None, 0, P, 4), (P, P, 0, None, 4), (P, P, 0, P, -1),
                 (P + 1, P, 0, P, 4), (P, P + 2, 2, P, 4), (P, P, 0, P + 2, 4)):
        k, v, dt, s, n = args
        assert lib.b4_kv_append(c, k, v, dt, 1, 1, 1, 1, s, n, None) == INV, args
    assert lib.b4_kv_append(c, None, None, 0, 1, 1, 1, 1, None, 0, None) == 0          # nothing to do
    for args in ((None, 4, P, P), (P, -1, P, P), (P, 4, None, P), (P, 4, P, P + 8), (P + 1, 4, P, P)):
        assert lib.b4_kv_read(c, *args, None) == INV, args
    assert lib.b4_kv_read(c, None, 0, None, None, None) == 0


def attn(**kw):
    a = dict(q=P, out=P, lse=None, tables=P, ctx_len=P, q_starts=P, table_stride=4, q_stride_token=1024, q_stride_head=128,
             out_stride_token=1024, out_stride_head=128, table_width=4, n_req=2, total_q=3, max_q=2, heads=8, dtype=0, window=0,
             flags=0, scale=0.1)
    a.update(kw)
    return _lib.KvAttn(*[a[n] for n, _ in _lib.KvAttn._fields_])


BAD_SHAPES = [dict(n_req=-1), dict(total_q=-1), dict(max_q=-1), dict(table_width=-1), dict(table_stride=3), dict(window=-1),
              dict(heads=0), dict(heads=7), dict(heads=130), dict(dtype=2), dict(dtype=-1), dict(flags=2), dict(flags=1, window=3),
              dict(scale=float("inf")), dict(scale=float("nan")), dict(table_width=1 << 27, table_stride=1 << 27)]
BAD_POINTERS = [dict(q=None), dict(out=None), dict(tables=None), dict(ctx_len=None), dict(q_starts=None), dict(q=P + 2),
                dict(out=P + 8), dict(q_stride_token=1028), dict(q_stride_head=132), dict(out_stride_token=1), dict(out_stride_head=4)]


@pytest.mark.parametrize("bad", BAD_SHAPES + BAD_POINTERS)
def test_attention_refusals(bad):
    lib, n = b4gemv.load(), ctypes.c_size_t(0)
    a = ctypes.byref(attn(**bad))
    assert lib.b4_kv_attention(ctypes.byref(cache()), a, P, 1 << 30, None) == INV
    if bad in BAD_SHAPES:
        assert lib.b4_kv_attention_workspace(ctypes.byref(cache()), a, ctypes.byref(n)) == INV


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_attention_refuses_bad_caches(bad):
    lib, n = b4gemv.load(), ctypes.c_size_t(0)
    assert lib.b4_kv_attention(ctypes.byref(cache(**bad)), ctypes.byref(attn()), P, 1 << 30, None) == INV
    assert lib.b4_kv_attention_workspace(ctypes.byref(cache(**bad)), ctypes.byref(attn()), ctypes.byref(n)) == INV


def test_nothing_to_attend_launches_nothing():
    lib = b4gemv.load()
    for empty in (dict(total_q=0), dict(n_req=0)):
        assert lib.b4_kv_attention(ctypes.byref(cache()), ctypes.byref(attn(**empty)), None, 0, None) == 0
