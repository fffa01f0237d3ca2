"""Windows far longer than any context are no window, for requests with more queries than tokens too."""
import pytest
import torch

import b4gemv
from test_kv_gpu import F16, INT4, NF4, check_attention, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [INT4, NF4])
@pytest.mark.parametrize("new", [1, 6, 90])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 7, 2 ** 31 - 1])
def test_windows_of_any_length(cuda, fmt, new, window):
    ctx = [0, 1, 3, 40, 133]
    state = make(cuda, fmt, F16, 8, 2, 128, 16, ctx, [new] * 5)
    got = check_attention(cuda, fmt, F16, 8, 2, 128, 16, ctx, [new] * 5, state=state, window=window)
    assert torch.equal(got, b4gemv.kv_attention(*state))
