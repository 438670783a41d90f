"""The head at the smallest and the largest sizes that its arguments allow."""
import pytest
import torch

import head_ref as R
from mantle_b200 import head as H
from mantle_b200 import native
from test_gpu_head import BF16, E4M3, F32, check_head, head_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,hidden,n,rank,dtype", [
    (1, 1, 8, 0, 0, BF16), (1, 1, 16, 0, 0, E4M3), (1, 1, 8, 1, 8, BF16), (1, 1, 16, 1, 8, E4M3), (129, 1, 8, 1, 8, BF16),
    (300, 3, 8, 2, 256, BF16), (65, 17, 24, 3, 8, BF16), (17, 33, 48, 2, 72, E4M3),
    (2, native.MAX_VOCAB, 16, 2, 8, BF16), (2, native.MAX_VOCAB, 16, 2, 8, E4M3), (2, native.MAX_VOCAB - 1, 16, 0, 0, E4M3),
    (1 << 20, 24, 16, 0, 0, BF16), (1 << 20, 24, 16, 4096, 8, BF16), (1 << 20, 9, 16, 3, 40, E4M3), (70000, 24, 16, 4096, 8, E4M3),
    (4096, 40, 16, 4096, 256, BF16), (128, 40, 8, 4096, 256, BF16),
])
def test_smallest_and_largest(rows, vocab, hidden, n, rank, dtype):
    s = head_inputs(rows, vocab, hidden, dtype, n, rank)
    for out in (F32, BF16):
        check_head(s, out, where=out)
    if n:
        s.pop("weight")
        s.pop("weight_scales", None)
        s["base"] = torch.randn(rows, vocab, device="cuda:0")
        check_head(s)


def test_one_past_the_largest_is_refused():
    x, w = torch.zeros((1, 16), dtype=BF16, device="cuda:0"), torch.zeros((8, 16), dtype=BF16, device="cuda:0")
    with pytest.raises(native.CudaError, match="vocab"):
        H.HeadPlan(x, w[:1].expand(native.MAX_VOCAB + 1, 16).contiguous())
    with pytest.raises(native.CudaError, match="rows"):
        H.HeadPlan(x.expand((1 << 20) + 1, 16).contiguous(), w)
    with pytest.raises(native.CudaError, match="stride"):
        H.HeadPlan(x.expand(5, 16), w)
