"""The package's own attention workspace: graphs and other streams hold its address, so it is never replaced."""
import pytest
import torch

import b4gemv
from b4gemv import kv
from test_kv_gpu import F16, INT4, NF4, make

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh(cuda, monkeypatch):
    """As in a process that has not called attention yet."""
    monkeypatch.setattr(kv, "_WS", {})
    return cuda


DECODE, PROMPT = ([700, 90, 2000], [1, 1, 1]), ([900, 300], [700, 40])


def test_not_replaced_by_larger_calls(fresh):
    b4gemv.kv_attention(*make(fresh, INT4, F16, 4, 4, 64, 16, *DECODE))
    ws = kv._WS[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for heads, kvh, d, batch in ((28, 4, 128, DECODE), (32, 2, 128, DECODE), (8, 2, 128, PROMPT), (64, 1, 128, PROMPT)):
        s = make(fresh, NF4, F16, heads, kvh, d, 32, *batch)
        assert b4gemv.kv_attention_workspace(*s) <= ws.numel()
        first = b4gemv.kv_attention(*s)
        side.wait_stream(torch.cuda.current_stream())
        again = b4gemv.kv_attention(*s, stream=side)
        side.synchronize()
        assert torch.equal(first, again)
    assert kv._WS[0] is ws


def test_first_call_on_another_stream(fresh):
    s = make(fresh, INT4, F16, 8, 2, 128, 32, *DECODE)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    first = b4gemv.kv_attention(*s, stream=side)
    side.synchronize()
    with torch.cuda.stream(other):
        again = b4gemv.kv_attention(*s)
    other.synchronize()
    assert torch.equal(first, again)


def test_graph_replayed_after_larger_calls(fresh):
    """Decode captured, prompts run eagerly and their memory handed out again, the graph replayed among them."""
    s = make(fresh, INT4, F16, 8, 2, 128, 32, [9000, 400, 3000], [1, 1, 1])
    out = torch.empty_like(s[1])
    want = b4gemv.kv_attention(*s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b4gemv.kv_attention(*s, out=out)
    prompt = make(fresh, INT4, F16, 8, 2, 128, 32, *PROMPT)
    first = b4gemv.kv_attention(*prompt)
    others = [torch.full((1 << 20,), i, dtype=torch.int32, device=fresh) for i in range(8)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
        assert torch.equal(b4gemv.kv_attention(*prompt), first)
    assert all(bool((x == i).all()) for i, x in enumerate(others))
    del graph


def test_first_call_inside_a_capture_is_refused(fresh):
    s = make(fresh, INT4, F16, 8, 2, 128, 32, *DECODE)
    ws = torch.zeros(b4gemv.kv_attention_workspace(*s), dtype=torch.uint8, device=fresh)
    own = b4gemv.kv_attention(*s, ws=ws)
    out = torch.zeros_like(own)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError):
            b4gemv.kv_attention(*s, out=out)
        b4gemv.kv_attention(*s, out=out, ws=ws)
    assert not kv._WS
    graph.replay()
    assert torch.equal(out, own)
    assert torch.equal(b4gemv.kv_attention(*s), own)
    del graph
