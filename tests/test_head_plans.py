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


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


def test_a_plan_ties_its_memory_to_every_stream_it_runs_on(monkeypatch):
    """Memory of a plan that is dropped while a side stream still runs must not be handed out again before that stream
    is done with it."""
    monkeypatch.setattr(H, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(H, "_current_device", lambda: 0)
    monkeypatch.setattr(H.native, "load", lambda: None)
    plan = H._Plan()
    plan._bind(torch.device("cuda", 0))
    made, given = Fake((4, 8)), Fake((4, 8))
    plan._own([made, None], [given, None])
    launched = []
    plan._fn, plan._args, plan._name = (lambda *a: launched.append(a[-1]) or 0), (), "fake"
    plan._queue(None)  # the stream it was made on: its own
    assert made.on == given.on == []
    side = Stream(9)
    for _ in range(2):
        plan._queue(side)
    assert made.on == given.on == [side]
    other = Stream(11)
    monkeypatch.setattr(H, "_raw_stream", lambda index: 11)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: other)
    plan._queue(None)
    assert made.on == given.on == [side, other] and launched == [7, 9, 9, 11]
