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
        self.device, self.is_cuda = torch.device("cuda", index), True

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
