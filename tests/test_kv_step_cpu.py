"""What kv_tables refuses of outputs that lie on its inputs, without a GPU: CTAs read the one while the other is written."""
import ctypes

import pytest

import b4gemv
from b4gemv import _lib

READ = {"cached": 50, "added": 50, "free_pages": 80, "free_state": 2}
WRITTEN = {"ctx_len": 50, "q_starts": 51, "slots": 600, "positions": 600, "free_state_out": 3}
AT = {n: 4096 * (i + 1) for i, n in enumerate(list(READ) + list(WRITTEN) + ["tables"])}
WIDTH, STRIDE = 5, 9


def call(**at):
    a = dict(n_req=50, page_size=16, table_width=WIDTH, ring_size=80, max_tokens=600, table_stride=STRIDE, **{**AT, **at})
    return b4gemv.load().b4_kv_tables(ctypes.byref(_lib.KvStep(*[a[n] for n, _ in _lib.KvStep._fields_])), None)


PAIRS = [(o, i) for o in WRITTEN for i in [*READ, *WRITTEN] if o != i]


@pytest.mark.parametrize("o,i", PAIRS)
def test_outputs_on_other_buffers(o, i):
    size = {**READ, **WRITTEN}
    for at in (AT[i], AT[i] + 4 * (size[i] - 1), AT[i] - 4 * (size[o] - 1)):       # from its start, its last value, up to its first
        assert call(**{o: at}) == 1


@pytest.mark.parametrize("name", [*READ, *WRITTEN])
def test_buffers_on_the_tables(name):
    size = {**READ, **WRITTEN}[name]
    last = AT["tables"] + 4 * (49 * STRIDE + WIDTH - 1)
    for at in (AT["tables"], last, AT["tables"] - 4 * (size - 1), AT["tables"] + 4 * (7 * STRIDE + WIDTH - 1)):
        assert call(**{name: at}) == 1
    # between two rows there is room for four values
    if size > 4:
        assert call(**{name: AT["tables"] + 4 * (7 * STRIDE + WIDTH)}) == 1
