"""What the cache's wrappers check before they launch, on stand-ins for CUDA tensors."""
import math

import pytest
import torch

from b4gemv import kv

INT = torch.int32
kv._load()


class Fake:
    """A tensor on cuda:`index` by its shape, strides and address."""

    def __init__(self, shape, dtype=INT, stride=None, index=0, at=1 << 20):
        self.shape, self.dtype, self.index, self.at = torch.Size(shape), dtype, index, at
        self.strides = tuple(stride) if stride else tuple(math.prod(shape[i + 1:]) for i in range(len(shape)))
        self.device, self.is_cuda = torch.device("cuda", index) if index >= 0 else torch.device("cpu"), index >= 0

    def get_device(self):
        return self.index

    def dim(self):
        return len(self.shape)

    def numel(self):
        return math.prod(self.shape)

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def is_contiguous(self):
        return self.strides == Fake(self.shape).strides

    def data_ptr(self):
        return self.at


@pytest.mark.parametrize("stride", [(0, 1), (3, 1), (4, 1)])
def test_tables_whose_rows_overlap_are_refused(stride):
    """Their rows do not lie where a stride of a row's width would look."""
    with pytest.raises(ValueError):
        kv._table(Fake((3, 5), stride=stride), 0, 3)


def test_table_strides():
    assert kv._table(Fake((3, 5)), 0, 3) == (5, 5)
    assert kv._table(Fake((3, 5), stride=(9, 1)), 0, 2) == (5, 9)
    assert kv._table(Fake((1, 5), stride=(0, 1)), 0, 1) == (5, 5)
    assert kv._table(Fake((3, 5), stride=(0, 1)), 0, 1) == (5, 5)
    assert kv._table(Fake((3, 1), stride=(1, 7)), 0, 3) == (1, 1)
    for t in (Fake((3, 5), stride=(10, 2)), Fake((2, 5)), Fake((15,)), Fake((3, 5), dtype=torch.int64), Fake((3, 5), index=1)):
        with pytest.raises(ValueError):
            kv._table(t, 0, 3)


class Library:
    """Notes the device that is current when an entry point is called."""

    def __init__(self, monkeypatch, current):
        self.current, self.seen = current, []
        monkeypatch.setattr(kv, "load", lambda: self)
        monkeypatch.setattr(kv, "_device", lambda: self.current, raising=False)
        monkeypatch.setattr(kv, "_raw_stream", lambda index: 100 + index)
        monkeypatch.setattr(torch.cuda, "device", lambda index: Current(self, index))

    def __getattr__(self, name):
        def call(*args):
            self.seen.append((name, self.current, args[-1]))
            return 0
        return call


class Current:
    def __init__(self, lib, index):
        self.lib, self.index = lib, index

    def __enter__(self):
        self.before, self.lib.current = self.lib.current, self.index

    def __exit__(self, *_):
        self.lib.current = self.before


def fake_cache(index):
    c = object.__new__(kv.KVCache)
    c.fmt, c.page_size, c.head_dim, c.n_pages, c.kv_heads, c.index, c._ref = 0, 16, 64, 4, 2, index, None
    return c


@pytest.mark.parametrize("index", [0, 1])
@pytest.mark.parametrize("current", [0, 1])
def test_launched_on_the_tensors_device(monkeypatch, index, current):
    lib = Library(monkeypatch, current)
    t = lambda *shape, dtype=INT: Fake(shape, dtype, index=index)  # noqa: E731
    cache, half, f32 = fake_cache(index), torch.float16, torch.float32
    out = kv.KVStep(t(3), t(4), t(8), t(8), t(3))
    kv.kv_tables(16, t(3, 5), t(3), t(3), t(9), t(2), 8, out=out)
    kv.kv_append(cache, t(8, 2, 64, dtype=half), t(8, 2, 64, dtype=half), t(8))
    kv.kv_read(cache, t(8), t(8, 2, 64, dtype=f32), t(8, 2, 64, dtype=f32))
    q = t(8, 4, 64, dtype=half)
    kv.kv_attention(cache, q, t(3, 5), t(3), t(4), 4, out=t(8, 4, 64, dtype=half), ws=t(1 << 20, dtype=torch.uint8))
    kv.kv_attention_workspace(cache, q, t(3, 5), t(3), t(4), 4)
    names = ["b4_kv_tables", "b4_kv_append", "b4_kv_read", "b4_kv_attention"]
    assert lib.seen[:4] == [(n, index, 100 + index) for n in names]
    assert lib.seen[4][:2] == ("b4_kv_attention_workspace", index)
    assert lib.current == current


@pytest.mark.parametrize("bad", [dict(index=-1), dict(index=1), dict(dtype=torch.float32), dict(stride=(2,))])
def test_workspaces_refused(monkeypatch, bad):
    """Of the host, of another device, or counted in something else than bytes."""
    lib = Library(monkeypatch, 0)
    q = Fake((8, 4, 64), torch.float16)
    with pytest.raises(ValueError):
        kv.kv_attention(fake_cache(0), q, Fake((3, 5)), Fake((3,)), Fake((4,)), 4, out=q, ws=Fake((1 << 20,), **{"dtype": torch.uint8, **bad}))
    assert not lib.seen
