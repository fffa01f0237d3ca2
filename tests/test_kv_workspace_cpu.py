"""The size of the package's attention workspace, without a GPU: it serves every call."""
import ctypes

import pytest

import b4gemv
from b4gemv import _lib, kv


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 7, 8, 9, 16, 17, 48, 64])
def test_most_serves_every_call(head_dim, group):
    most, n = kv._workspace_most(), ctypes.c_size_t(0)
    for page in (16, 32, 64):
        for fmt in (0, 1):
            cache = _lib.KvCache(4096, fmt, 10, page, 2, head_dim)
            for n_req in (1, 3, 1000, 100000):
                for max_q in (0, 1, 2, 3, 4, 5, 8, 32, 48, 4096):
                    for total in (1, n_req * max(max_q, 1), 3000):
                        a = _lib.KvAttn(n_req=n_req, total_q=total, max_q=max_q, heads=2 * group)
                        status = b4gemv.load().b4_kv_attention_workspace(ctypes.byref(cache), ctypes.byref(a), ctypes.byref(n))
                        if total * group <= 0x7fffffff:
                            assert status == 0 and 0 < n.value <= most


@pytest.mark.parametrize("page", [16, 32, 64])
def test_tables_of_the_most_keys(page):
    """2^31 - 64 keys a request at most: the kernels' counts of keys, rounded up to a block, stay in 32 bits."""
    n = ctypes.c_size_t(0)
    cache = _lib.KvCache(4096, 0, 10, page, 2, 128)
    for width, status in (((2 ** 31 - 64) // page, 0), ((2 ** 31 - 64) // page + 1, 1)):
        a = _lib.KvAttn(n_req=1, total_q=1, max_q=1, heads=2, table_width=width, table_stride=width)
        assert b4gemv.load().b4_kv_attention_workspace(ctypes.byref(cache), ctypes.byref(a), ctypes.byref(n)) == status
