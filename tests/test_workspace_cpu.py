"""The GEMVs' package workspace when it grows: graphs that captured the smaller one still write to it."""
import gc
import weakref

import torch

import b4gemv


def test_a_replaced_workspace_is_kept(monkeypatch):
    zeros = torch.zeros
    monkeypatch.setattr(b4gemv, "_WS", {})
    monkeypatch.setattr(torch, "zeros", lambda n, dtype=None, device=None: zeros(n, dtype=dtype))
    small = weakref.ref(b4gemv.workspace("cuda:0", 100))
    assert b4gemv.workspace("cuda:0", 1 << 20) is small()
    large = b4gemv.workspace("cuda:0", 5 << 20)
    gc.collect()
    assert large is not small() and small() is not None and small().numel() == 1 << 20
    assert b4gemv.workspace("cuda:0", 100) is large
