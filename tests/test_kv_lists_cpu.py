"""What the rotated append, the boxes, the choice of pages and attention over lists refuse before anything is launched, and
the table of angles, which the host makes."""
import ctypes
import math

import pytest
import torch

import b4gemv
import kv_lists_ref as ref
from b4gemv import _lib, kv, kvlists
from test_kv_arguments_cpu import Fake, Library, fake_cache

INT, F16, BF16, F32, U8 = torch.int32, torch.float16, torch.bfloat16, torch.float32, torch.uint8


def rotary(dim=64, n_axes=1, index=0):
    r = object.__new__(kvlists.Rotary)
    r.dim, r.n_axes, r.index, r._ref = dim, n_axes, index, None
    return r


# ---- the table of angles --------------------------------------------------------------

@pytest.mark.parametrize("base", [1e4, 1e6, 500000.0, 2.0])
@pytest.mark.parametrize("dim", [16, 48, 128])
def test_turns(base, dim):
    r = b4gemv.Rotary(dim, base=base, device="cpu")
    inv = [base ** (-i / (dim // 2)) for i in range(dim // 2)]
    assert [t % (1 << 64) for t in r.turns.tolist()] == ref.turns(inv)


def test_turns_of_any_frequency():
    inv = [0.0, -1.0, 1e-30, -1e-30, 6.283185307179586, 3.14159, -0.25, 1e9, 7.5, 1e-19, -1e-19, 3e-20, 2.0 ** -60, 1e-17, 0.1, 0.7]
    r = b4gemv.Rotary(32, inv_freq=inv, device="cpu")
    assert [t % (1 << 64) for t in r.turns.tolist()] == ref.turns(inv)


def test_axes():
    r = b4gemv.Rotary(64, sections=(8, 12, 12), device="cpu")
    assert r.n_axes == 3 and r.axes.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    r = b4gemv.Rotary(32, axes=[i % 3 for i in range(16)], device="cpu")
    assert r.n_axes == 3 and r.axes.tolist() == [i % 3 for i in range(16)]
    assert b4gemv.Rotary(32, axes=[0] * 16, device="cpu").axes is None


@pytest.mark.parametrize("bad", [dict(dim=8), dict(dim=24), dict(dim=144), dict(dim=0), dict(dim=32, inv_freq=[1.0] * 15),
                                 dict(dim=32, inv_freq=[math.inf] * 16), dict(dim=32, inv_freq=[math.nan] * 16), dict(dim=32, base=0.0),
                                 dict(dim=32, sections=(8, 7)), dict(dim=32, sections=(20, -4)), dict(dim=32, sections=(8, 8), axes=[0] * 16),
                                 dict(dim=32, axes=[0] * 15), dict(dim=32, axes=[-1] * 16), dict(dim=32, axes=[256] * 16),
                                 dict(dim=32, scale=math.inf)])
def test_tables_refused(bad):
    with pytest.raises(ValueError):
        b4gemv.Rotary(device="cpu", **bad)


def test_turns_refused():
    lib = b4gemv.load()
    one, out = (ctypes.c_double * 1)(1.0), (ctypes.c_uint64 * 1)()
    assert lib.b4_rotary_turns(one, 1, out) == 0 and lib.b4_rotary_turns(None, 0, None) == 0
    assert lib.b4_rotary_turns(one, -1, out) == lib.b4_rotary_turns(None, 1, out) == lib.b4_rotary_turns(one, 1, None) == 1
    one[0] = math.inf
    assert lib.b4_rotary_turns(one, 1, out) == 1


# ---- the wrappers ---------------------------------------------------------------------

def append_args(index=0, n=8):
    t = lambda *shape, dtype=F16: Fake(shape, dtype, index=index)  # noqa: E731
    return dict(rotary=rotary(index=index), q=t(n, 4, 64), k=t(n, 2, 64), v=t(n, 2, 64), positions=t(n, dtype=INT), slots=t(n, dtype=INT),
                out=t(n, 4, 64))


def select_args(index=0, n=8):
    t = lambda *shape, dtype=INT: Fake(shape, dtype, index=index)  # noqa: E731
    return dict(boxes=t(4, 2, 144, dtype=U8), q=t(n, 4, 64, dtype=F16), tables=t(3, 5), ctx_len=t(3), q_starts=t(4), max_q=4, keep=4,
                out=kvlists.KVLists(t(n, 2, 4), t(n)))


def lists_args(index=0, n=8):
    t = lambda *shape, dtype=INT: Fake(shape, dtype, index=index)  # noqa: E731
    return dict(q=t(n, 4, 64, dtype=F16), lists=kvlists.KVLists(t(n, 2, 4), t(n)), out=t(n, 4, 64, dtype=F16), ws=t(1 << 20, dtype=U8))


@pytest.mark.parametrize("index", [0, 1])
@pytest.mark.parametrize("current", [0, 1])
def test_launched_on_the_tensors_device(monkeypatch, index, current):
    lib = Library(monkeypatch, current)
    cache = fake_cache(index)
    kvlists.kv_append_rotary(cache, **append_args(index))
    kvlists.kv_boxes(cache, Fake((4, 2, 144), U8, index=index), Fake((8,), index=index))
    kvlists.kv_select(cache, **select_args(index))
    kvlists.kv_attention_lists(cache, **lists_args(index))
    names = ["b4_kv_append_rotary", "b4_kv_boxes", "b4_kv_select", "b4_kv_attention_lists"]
    assert lib.seen == [(n, index, 100 + index) for n in names]
    a = lists_args(index)
    kvlists.kv_attention_lists_workspace(cache, a["q"], a["lists"])
    assert lib.seen[4][:2] == ("b4_kv_attention_lists_workspace", index)
    assert lib.current == current


@pytest.mark.parametrize("bad", [
    dict(k=Fake((8, 2, 64), F32)), dict(k=Fake((7, 2, 64), F16)), dict(v=Fake((8, 2, 64), F16, stride=(256, 128, 2))), dict(v=Fake((8, 2, 64), F16, index=1)),
    dict(q=Fake((8, 4, 64), BF16)), dict(q=Fake((7, 4, 64), F16)), dict(q=Fake((8, 4, 128), F16)), dict(q=Fake((8, 256), F16)), dict(q=Fake((8, 4, 64), F16, index=1)),
    dict(out=Fake((8, 4, 64), BF16)), dict(out=Fake((8, 4, 64), F32)), dict(out=Fake((8, 5, 64), F16)), dict(out=Fake((8, 4, 64), F16, stride=(512, 128, 2))),
    dict(positions=Fake((8,), torch.int64)), dict(positions=Fake((7,))), dict(positions=Fake((2, 8))), dict(positions=Fake((8,), stride=(2,))),
    dict(positions=Fake((8,), index=1)), dict(slots=Fake((8,), torch.int64)), dict(slots=Fake((9,))), dict(rotary=rotary(dim=128)), dict(rotary=rotary(index=1)),
    dict(rotary=rotary(n_axes=2)), dict(q=None)])
def test_appends_refused(monkeypatch, bad):
    lib = Library(monkeypatch, 0)
    with pytest.raises(ValueError):
        kvlists.kv_append_rotary(fake_cache(0), **{**append_args(), **bad})
    assert not lib.seen


def test_axes_of_positions(monkeypatch):
    lib = Library(monkeypatch, 0)
    for r, p, ok in ((rotary(), Fake((1, 8)), True), (rotary(n_axes=3), Fake((3, 8)), True), (rotary(n_axes=3), Fake((3, 8), stride=(64, 1)), True),
                     (rotary(n_axes=3), Fake((3, 8), stride=(0, 1)), False), (rotary(n_axes=3), Fake((3, 8), stride=(1, 3)), False),
                     (rotary(n_axes=3), Fake((8,)), False), (rotary(n_axes=3), Fake((2, 8)), False)):
        args = {**append_args(), "rotary": r, "positions": p}
        if ok:
            kvlists.kv_append_rotary(fake_cache(0), **args)
        else:
            with pytest.raises(ValueError):
                kvlists.kv_append_rotary(fake_cache(0), **args)
    assert len(lib.seen) == 3
    # keys and values alone; fp32 rows give fp16 or bf16 queries
    assert kvlists.kv_append_rotary(fake_cache(0), **{**append_args(), "q": None, "out": None}) is None
    f = lambda *shape: Fake(shape, F32)  # noqa: E731
    for o in (F16, BF16):
        kvlists.kv_append_rotary(fake_cache(0), **{**append_args(), "q": f(8, 4, 64), "k": f(8, 2, 64), "v": f(8, 2, 64), "out": Fake((8, 4, 64), o)})
    assert len(lib.seen) == 6


@pytest.mark.parametrize("bad", [dict(boxes=Fake((4, 2, 143), U8)), dict(boxes=Fake((5, 2, 144), U8)), dict(boxes=Fake((4, 2, 144), INT)),
                                 dict(boxes=Fake((4, 2, 144), U8, index=1)), dict(boxes=Fake((4, 2, 144), U8, stride=(300, 144, 1))),
                                 dict(slots=Fake((8,), torch.int64))])
def test_boxes_refused(monkeypatch, bad):
    lib = Library(monkeypatch, 0)
    with pytest.raises(ValueError):
        kvlists.kv_boxes(fake_cache(0), **{**dict(boxes=Fake((4, 2, 144), U8), slots=Fake((8,))), **bad})
    if "boxes" in bad:
        with pytest.raises(ValueError):
            kvlists.kv_select(fake_cache(0), **{**select_args(), **bad})
    assert not lib.seen


@pytest.mark.parametrize("bad", [
    dict(q=Fake((8, 4, 64), F32)), dict(q=Fake((8, 3, 64), F16)), dict(q=Fake((8, 4, 128), F16)), dict(q=Fake((8, 4, 64), F16, index=1)),
    dict(tables=Fake((2, 5))), dict(tables=Fake((3, 5), stride=(0, 1))), dict(ctx_len=Fake((3,), torch.int64)), dict(q_starts=Fake((3,))),
    dict(keep=0), dict(first=-1), dict(last=0), dict(first=2, last=3), dict(out=kvlists.KVLists(Fake((8, 2, 5)), Fake((8,)))),
    dict(out=kvlists.KVLists(Fake((8, 2, 4)), Fake((7,)))), dict(out=kvlists.KVLists(Fake((8, 2, 4), torch.int64), Fake((8,))))])
def test_choices_refused(monkeypatch, bad):
    lib = Library(monkeypatch, 0)
    with pytest.raises(ValueError):
        kvlists.kv_select(fake_cache(0), **{**select_args(), **bad})
    assert not lib.seen


@pytest.mark.parametrize("bad", [
    dict(q=Fake((8, 4, 64), F32)), dict(q=Fake((8, 3, 64), F16)), dict(q=Fake((8, 4, 64), F16, index=1)), dict(out=Fake((8, 4, 64), BF16)),
    dict(lists=kvlists.KVLists(Fake((8, 1, 4)), Fake((8,)))), dict(lists=kvlists.KVLists(Fake((7, 2, 4)), Fake((8,)))),
    dict(lists=kvlists.KVLists(Fake((8, 2, 4), stride=(0, 4, 1)), Fake((8,)))), dict(lists=kvlists.KVLists(Fake((8, 2, 4), stride=(4, 0, 1)), Fake((8,)))),
    dict(lists=kvlists.KVLists(Fake((8, 2, 4), stride=(16, 8, 2)), Fake((8,)))), dict(lists=kvlists.KVLists(Fake((8, 2, 4)), Fake((7,)))),
    dict(lists=kvlists.KVLists(Fake((8, 2, 4)), Fake((8,), torch.int64))), dict(lse=Fake((8, 4), F16)), dict(lse=Fake((8, 5), F32)),
    dict(ws=Fake((1 << 20,), U8, index=1)), dict(ws=Fake((1 << 20,), INT))])
def test_lists_refused(monkeypatch, bad):
    lib = Library(monkeypatch, 0)
    with pytest.raises(ValueError):
        kvlists.kv_attention_lists(fake_cache(0), **{**lists_args(), **bad})
    assert not lib.seen


# ---- the library ----------------------------------------------------------------------

def cache(**more):
    return _lib.KvCache(**{**dict(blocks=4096, fmt=0, n_pages=4, page_size=16, kv_heads=2, head_dim=64), **more})


def byref(x):
    return ctypes.byref(x) if x is not None else None


def refused(name, *args):
    return getattr(b4gemv.load(), name)(*args) == 1


def test_library_refuses_appends():
    rot = dict(turns=4096, axes=None, dim=64, n_axes=1, flags=0, scale=1.0)
    rows = dict(q=4096, k=4096, v=4096, q_out=4096, positions=4096, slots=4096, position_stride=8, q_stride_token=256, q_stride_head=64, k_stride_token=128,
                k_stride_head=64, v_stride_token=128, v_stride_head=64, out_stride_token=256, out_stride_head=64, n_tokens=8, heads=4, dtype=0, out_dtype=0)

    def call(c=None, r=None, x=None):
        return refused("b4_kv_append_rotary", byref(cache(**(c or {}))), byref(_lib.RotaryTable(**{**rot, **(r or {})})),
                       byref(_lib.KvRows(**{**rows, **(x or {})})), None)

    for c in (dict(blocks=None), dict(fmt=2), dict(page_size=8), dict(head_dim=96), dict(kv_heads=0)):
        assert call(c=c)
    for r in (dict(turns=None), dict(turns=4100), dict(dim=8), dict(dim=24), dict(dim=80), dict(n_axes=0), dict(n_axes=2), dict(flags=2),
              dict(scale=math.nan), dict(n_axes=2, axes=4096, dim=128)):
        assert call(r=r)
    assert call(r=dict(n_axes=2, axes=4096), x=dict(position_stride=7))
    for x in (dict(n_tokens=-1), dict(heads=-1), dict(dtype=3), dict(out_dtype=2), dict(dtype=0, out_dtype=1), dict(dtype=1, out_dtype=0), dict(k=None), dict(v=None),
              dict(slots=None), dict(positions=None), dict(q=None), dict(q_out=None), dict(q=4097), dict(q_out=4104), dict(out_stride_token=260), dict(slots=4098)):
        assert call(x=x)
    assert not call(x=dict(n_tokens=0))
    assert refused("b4_kv_append_rotary", byref(cache()), None, byref(_lib.KvRows(**rows)), None)


def test_library_refuses_boxes_and_choices():
    n = ctypes.c_size_t()
    lib = b4gemv.load()
    assert lib.b4_kv_box_bytes(64, byref(n)) == 0 and n.value == 144 and lib.b4_kv_box_bytes(128, byref(n)) == 0 and n.value == 272
    assert refused("b4_kv_box_bytes", 96, byref(n)) and refused("b4_kv_box_bytes", 64, None)
    assert b4gemv.kv_box_bytes(128) == 272
    for args in ((4096, -1, 4096), (None, 8, 4096), (4096, 8, None), (4096, 8, 4104), (4098, 8, 4096)):
        assert refused("b4_kv_boxes", byref(cache()), *args, None)
    assert lib.b4_kv_boxes(byref(cache()), None, 0, None, None) == 0
    good = dict(q=4096, boxes=4096, tables=8192, ctx_len=16384, q_starts=20480, lists=24576, seen=28672, table_stride=5, q_stride_token=256, q_stride_head=64,
                table_width=5, n_req=3, total_q=8, max_q=4, heads=4, dtype=0, keep=4, first=1, last=1)
    # lists of 256 bytes and seen of 32 on what the call reads, or on one another
    for at in (8192, 8192 + 56, 8192 - 252, 16384, 16384 + 8, 16384 - 252, 20480, 20480 + 12):
        assert refused("b4_kv_select", byref(cache()), byref(_lib.KvChoice(**{**good, "lists": at})), None), at
    for at in (8192, 8192 + 56, 8192 - 28, 16384, 16384 + 8, 20480 + 12, 24576, 24576 + 252, 24576 - 28):
        assert refused("b4_kv_select", byref(cache()), byref(_lib.KvChoice(**{**good, "seen": at})), None), at
    for bad in (dict(n_req=-1), dict(total_q=-1), dict(max_q=-1), dict(table_width=-1), dict(table_width=49153, table_stride=49153), dict(table_stride=4),
                dict(heads=3), dict(heads=0), dict(heads=130), dict(dtype=2), dict(keep=0), dict(first=-1), dict(last=0), dict(first=3, last=2),
                dict(keep=49153), dict(first=2 ** 31 - 1, last=2 ** 31 - 1), dict(q=None), dict(q=4104), dict(boxes=None), dict(boxes=4104), dict(tables=None), dict(ctx_len=None),
                dict(q_starts=None), dict(lists=None), dict(seen=None), dict(q_stride_token=260)):
        assert refused("b4_kv_select", byref(cache()), byref(_lib.KvChoice(**{**good, **bad})), None), bad
    assert refused("b4_kv_select", byref(cache()), None, None)
    assert lib.b4_kv_select(byref(cache()), byref(_lib.KvChoice(**{**good, "total_q": 0})), None) == 0


def test_library_refuses_lists():
    good = dict(q=4096, out=4096, lse=None, tables=4096, ctx_len=4096, q_starts=None, table_stride=8, q_stride_token=256, q_stride_head=64,
                out_stride_token=256, out_stride_head=64, table_width=4, n_req=0, total_q=8, max_q=0, heads=4, dtype=0, window=0, flags=0, scale=0.125)
    for bad in (dict(window=1), dict(flags=1), dict(total_q=-1), dict(heads=3), dict(heads=130), dict(dtype=2), dict(scale=math.inf), dict(table_stride=3),
                dict(table_width=2 ** 30, table_stride=2 ** 31)):
        assert refused("b4_kv_attention_lists", byref(cache()), byref(_lib.KvAttn(**{**good, **bad})), 1 << 30, 4096, 1 << 40, None), bad
    for bad in (dict(q=None), dict(q=4104), dict(out=None), dict(tables=None), dict(ctx_len=None), dict(q_stride_head=60)):
        assert refused("b4_kv_attention_lists", byref(cache()), byref(_lib.KvAttn(**{**good, **bad})), 4, 4096, 1 << 40, None), bad
    call = lambda stride, ws, size: refused("b4_kv_attention_lists", byref(cache()), byref(_lib.KvAttn(**good)), stride, ws, size, None)  # noqa: E731
    assert call(3, 4096, 1 << 40) and call(4, None, 1 << 40) and call(4, 4104, 1 << 40) and call(4, 4096, 100)
    n = ctypes.c_size_t()
    lib = b4gemv.load()
    assert lib.b4_kv_attention_lists_workspace(byref(cache()), byref(_lib.KvAttn(**good)), byref(n)) == 0 and n.value > 8192
    assert refused("b4_kv_attention_lists_workspace", byref(cache()), byref(_lib.KvAttn(**good)), None)
    assert lib.b4_kv_attention_lists(byref(cache()), byref(_lib.KvAttn(**{**good, "total_q": 0})), 4, None, 0, None) == 0


def test_structures_as_packed():
    assert kvlists._ROWS.size == ctypes.sizeof(_lib.KvRows) and kvlists._CHOICE.size == ctypes.sizeof(_lib.KvChoice)
    x = _lib.KvChoice.from_buffer_copy(kvlists._CHOICE.pack(*range(1, 20)))
    assert [getattr(x, n) for n, _ in x._fields_] == list(range(1, 20))
    x = _lib.KvRows.from_buffer_copy(kvlists._ROWS.pack(*range(1, 20)))
    assert [getattr(x, n) for n, _ in x._fields_] == list(range(1, 20))


def test_module_is_loaded():
    assert kv._torch is torch
