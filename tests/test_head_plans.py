"""What the plans of mantle_b200.head do on the host, with stand-ins for CUDA tensors: no GPU needed."""
import pytest
import torch

from mantle_b200 import head as H


class Fake:
    """The shape, strides and type of a CUDA tensor, without its memory."""

    is_cuda = True
    device = torch.device("cuda", 0)

    def __init__(self, shape, dtype=torch.bfloat16, stride=None):
        self.shape, self.dtype = torch.Size(shape), dtype
        self.strides = stride or (shape[1], 1)
        self.on = []

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return self.strides[i]

    def record_stream(self, stream):
        self.on.append(stream)


@pytest.mark.parametrize("shape", [(2 ** 32 + 5, 1), (2 ** 31, 1), (1, 2 ** 32 + 8)])
def test_sizes_past_32_bits_are_refused(shape):
    """A descriptor's sizes are int32: 2^32 + 5 rows must not be taken for five."""
    with pytest.raises(ValueError, match="2147483647"):
        H._rows(Fake(shape), "x", (torch.bfloat16,))
    assert H._rows(Fake((5, 8)), "x", (torch.bfloat16,)) == (1, 8)
