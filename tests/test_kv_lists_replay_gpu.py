"""A captured step of a layer with a choice of pages, replayed far past what is kept, so that boxes are scored and pages left out
in the replays themselves."""
import pytest
import torch

import b4gemv
from test_kv_lists_gpu import Layer, ints

pytestmark = pytest.mark.gpu
INT4, NF4 = 0, 1
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("fmt,dtype,d,pages", [(INT4, F16, 128, 60), (NF4, BF16, 64, 60), (INT4, BF16, 128, 700), (NF4, F16, 64, 1100)])
@pytest.mark.parametrize("prompts,new,steps", [([1, 1, 1], 1, 130), ([300, 40, 95], 1, 40), ([300, 40, 95], 5, 12)])
def test_steps_replayed_past_what_is_kept(cuda, fmt, dtype, d, pages, prompts, new, steps):
    """Of 4 pages of 16: single tokens from the first on and behind prompts, drafts; tables of 700 and 1100 pages are shared by clusters of 8 and
    16 CTAs."""
    keep, page = 4, 16
    layer = Layer(cuda, fmt, dtype, 8, 2, d, page, 3, pages, sum(prompts) + 4, keep, 1, 1)
    g = torch.Generator(device=cuda).manual_seed(d + new)

    def fill():
        for x in (layer.q, layer.k, layer.v):
            x.normal_(generator=g)

    fill()
    layer.added.copy_(ints(prompts, cuda))
    layer.step(max(prompts))                                                             # makes the package's workspace
    torch.cuda.synchronize()
    layer.check(prompts)
    layer.added.fill_(new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(new)
    chosen = 0
    for i in range(1, steps + 1):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        done = [p + i * new for p in prompts]
        if new > 1 or i > steps - 3 or any(n % page in (0, 1) for n in done):
            layer.check(done)
            chosen += any(-(-n // page) > keep for n in done)
        layer.out.fill_(9.0)
    assert chosen >= 8
    assert b4gemv.load().b4_device_error(0) == 0
    del graph
