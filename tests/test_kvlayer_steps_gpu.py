"""A layer's steps at their edges: none of its requests has a token, lengths below 0."""
import pytest
import torch

import b4gemv
from b4gemv.kvlayer import CachedAttention

pytestmark = pytest.mark.gpu


def layer():
    return CachedAttention(b4gemv.FMT_INT4_G128, 256, 2, 1, n_pages=8, max_requests=2, page_size=16, max_context=64)


def test_steps_without_tokens(cuda):
    a, b = layer(), layer()
    x = torch.randn((20, 256), generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).half()
    for added in ([0, 0], [0], []):
        y = a.step(x[:0], added)
        assert y.shape == (0, 256)
    for at, added in ((0, [5, 7]), (12, [1, 1]), (14, [0, 6])):
        n = sum(added)
        assert torch.equal(a.step(x[at:at + n], added), b.step(x[at:at + n], added))
        assert a.step(x[:0], [0, 0]).shape == (0, 256)
    assert a.cached.tolist() == b.cached.tolist() == [6, 14]
    assert a.free_state.tolist() == b.free_state.tolist()


def test_lengths_below_0_are_refused(cuda):
    """The device counts them as 0, so x would have fewer rows than tokens."""
    a = layer()
    with pytest.raises(ValueError):
        a.step(torch.zeros((2, 256), dtype=torch.float16, device=cuda), [3, -1])
    assert a.cached.tolist() == [0, 0]
