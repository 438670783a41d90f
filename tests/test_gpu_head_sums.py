"""The sums behind the logits, where the definitions' own tolerances would hide a loss: whole numbers, which every sum
holds exactly, and errors measured against the size of the logits."""
import itertools

import pytest
import torch

import head_ref as R
from mantle_b200 import head as H

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def whole(seed, low, high, *shape):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randint(low, high + 1, shape, generator=g).to(F32).to(DEV)


@pytest.mark.parametrize("rows", [1, 20, 64, 100, 128, 129, 300])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_between_an_adapters_products_nothing_is_lost(rows, dtype):
    """u is a whole number of up to 22 bits, B has a single one in a row: the logits are u."""
    k, n, rank, vocab = 256, 3, 24, 200
    x = whole(1, 1, 15, rows, k)           # exact in either type
    a = whole(2, 1, 255, n, rank, k)       # exact in bfloat16; sums up to 256 * 15 * 255, below 2^20, or 2^22 with the gain
    b = torch.zeros(n, vocab, rank, device=DEV)
    v = torch.arange(vocab, device=DEV)
    b[:, v, v % rank] = 1 - 2 * (v % 2).to(F32)
    gain = torch.tensor([1.0, 3.0, -4.0], device=DEV)
    ids = (torch.arange(rows, dtype=torch.int32) % (n + 1) - 1).to(DEV)
    ones = torch.ones(rows, device=DEV) if dtype == E4M3 else None
    want = torch.zeros(rows, vocab, dtype=R.F64, device=DEV)
    for i in range(n):
        at = torch.nonzero(ids == i).view(-1)
        want[at] = (x[at].to(R.F64) @ a[i].to(R.F64).T) @ b[i].to(R.F64).T * gain[i].to(R.F64)
    table = H.Adapters(a.to(BF16), b.to(BF16), gain)
    zero = torch.zeros(vocab, k, device=DEV).to(dtype)
    for kw in (dict(base=torch.zeros(rows, vocab, device=DEV)),
               dict(weight=zero, weight_scales=torch.ones(vocab, device=DEV) if dtype == E4M3 else None)):
        got = H.HeadPlan(x.to(dtype), hidden_scales=ones, adapters=table, adapter_ids=ids, **kw).launch()
        torch.cuda.synchronize()
        assert torch.equal(got.to(R.F64), want)
