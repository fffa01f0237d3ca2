"""kv_tables with buffers of the caller's: those of the last step refused where this step reads them, neighbours taken."""
import pytest
import torch

import b4gemv

pytestmark = pytest.mark.gpu


def test_the_last_steps_buffers(cuda):
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    tab, ring, state = torch.full((300, 4), -1, dtype=torch.int32, device=cuda), torch.arange(900, dtype=torch.int32, device=cuda), t([0, 900, 0])
    one = torch.ones(300, dtype=torch.int32, device=cuda)
    a = b4gemv.kv_tables(16, tab, t([0] * 300), one, ring, state, 300)
    for bad in (dict(cached=a.ctx_len), dict(added=a.q_starts[:300]), dict(free_state=a.free_state), dict(free_pages=a.slots),
                dict(cached=a.positions)):
        args = dict(cached=one, added=one, free_pages=ring, free_state=state)
        args.update(bad)
        with pytest.raises(b4gemv.B4Error):
            b4gemv.kv_tables(16, tab, max_tokens=300, out=a, **args)
    b = b4gemv.kv_tables(16, tab, a.ctx_len, one, ring, a.free_state, 300)
    c = b4gemv.kv_tables(16, tab, b.ctx_len, one, ring, b.free_state, 300, out=a)
    assert c.ctx_len.tolist() == [3] * 300 and c.free_state.tolist() == [300, 600, 0]


def test_neighbours_in_one_buffer(cuda):
    """Outputs and inputs side by side, and outputs between the rows of a wider table."""
    n, width, stride, tokens = 5, 3, 10, 12
    buf = torch.full((400,), 77, dtype=torch.int32, device=cuda)
    tab = buf[:n * stride].view(n, stride)[:, :width]
    tab.fill_(-1)
    ctx, state = buf[stride + width:stride + width + n], buf[2 * stride + width:2 * stride + width + 3]
    at = [n * stride]

    def take(k, values=None):
        x = buf[at[0]:at[0] + k]
        at[0] += k
        if values is not None:
            x.copy_(torch.tensor(values, dtype=torch.int32))
        return x

    cached, added = take(n, [0, 15, 16, 3, 40]), take(n, [2, 1, 1, 0, 5])
    starts, ring, slots = take(n + 1), take(8, [4, 2, 0, 7, 1, 3, 6, 5]), take(tokens)
    free, positions = take(2, [6, 8]), take(tokens)
    step = b4gemv.kv_tables(16, tab, cached, added, ring, free, tokens, out=b4gemv.KVStep(ctx, starts, slots, positions, state))
    assert step.ctx_len.tolist() == [2, 16, 17, 3, 45] and step.q_starts.tolist() == [0, 2, 3, 4, 4, 9]
    # new pages: the first request's first, the third's second; the others have theirs (-1 here, as the test left them)
    assert tab.tolist() == [[6, -1, -1], [-1, -1, -1], [-1, 5, -1], [-1, -1, -1], [-1, -1, -1]]
    assert step.slots.tolist() == [96, 97, -1, 80] + [-1] * 8 and step.free_state.tolist() == [0, 6, 0]
    assert step.positions.tolist() == [0, 1, 15, 16, 40, 41, 42, 43, 44, 0, 0, 0]
    rows = buf[:n * stride].view(n, stride)
    assert rows[0, width:].tolist() == [77] * 7 and rows[3, width:].tolist() == [77] * 7 and bool((buf[at[0]:] == 77).all())
