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


# widths around the steps (64 and 128 columns) and the rounds (512 and 8192) of either type
WIDTHS = {BF16: (16, 504, 512, 520, 1024, 1032, 4096, 4104, 8192, 16376, 65536),
          E4M3: (16, 112, 128, 144, 4096, 8176, 8192, 8208, 16384, 16400, 65536)}


@pytest.mark.parametrize("rows", [1, 33, 100, 300])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_whole_numbers_of_every_width(rows, dtype):
    """Sums of whole numbers below 2^24 are exact in float32, in any order and cut into any rounds: a step that is left
    out, or taken twice, shows in full."""
    vocab, n, rank = 150, 4, 24
    for k in WIDTHS[dtype]:
        x, w = whole(k, -2, 2, rows, k), whole(k + 1, -3, 3, vocab, k)  # at most 6 * 65536
        ids = (torch.arange(rows, dtype=torch.int32) % (n + 1) - 1).to(DEV)
        a, b = whole(k + 2, -1, 1, n, rank, k), whole(k + 3, -1, 1, n, vocab, rank)  # at most 2 * 65536 * 24 beside them
        plain = x.to(R.F64) @ w.to(R.F64).T
        part = torch.zeros_like(plain)
        for i in range(n):
            at = torch.nonzero(ids == i).view(-1)
            part[at] = (x[at].to(R.F64) @ a[i].to(R.F64).T) @ b[i].to(R.F64).T
        eight = dtype == E4M3
        sx = 2.0 ** whole(k + 4, -3, 3, rows) if eight else None
        sw = 2.0 ** whole(k + 5, -3, 3, vocab) if eight else None
        if eight:  # the scales are powers of two, and so exact; the two parts are summed at their common unit, 2^-6
            plain = plain * sx.to(R.F64)[:, None] * sw.to(R.F64)
            part = part * sx.to(R.F64)[:, None]
        table = H.Adapters(a.to(BF16), b.to(BF16))
        for adapters in (False, True):
            got = H.HeadPlan(x.to(dtype), w.to(dtype), hidden_scales=sx, weight_scales=sw, adapters=table if adapters else None,
                             adapter_ids=ids if adapters else None).launch()
            torch.cuda.synchronize()
            want = plain + part if adapters else plain
            assert float(want.abs().max()) * 2 ** (6 if eight else 0) < 2 ** 24  # exact in float32 itself
            assert torch.equal(got.to(R.F64), want), (k, adapters)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_errors_do_not_grow_with_the_width(dtype):
    """Of a sum in tensor memory every step cuts less than a unit of the last place, 2^-23, half of it on average, and
    always towards zero; the partial sums are no larger than the whole in the mean.  A round of 512 bfloat16 columns has
    32 steps of 16; the sums of `rounds` rounds, and the adapters', round once each, 2^-24 and independently.  With e4m3
    a product has 8 bits and a round is 8192 columns: their sums lose nothing until they pass 2^16 products' units, and
    the figure that the kernel states for 8192 columns is 5.1e-7; four times that is held."""
    rows, vocab = 5, 400
    for k in (512, 1024, 4096, 8192, 16384, 65536):
        g = torch.Generator(device="cpu")
        g.manual_seed(k)
        x, w = (torch.randn(s, k, generator=g, dtype=F32).to(DEV) for s in (rows, vocab))
        if dtype == E4M3:
            (x, sx), (w, sw) = R.to_e4m3_rows(x), R.to_e4m3_rows(w)
            bound = 4 * 5.1e-7
        else:
            x, w, sx, sw = x.to(BF16), w.to(BF16), None, None
            bound = (32 + 1 + (k / 512) ** 0.5) * 2.0 ** -24
        want, _ = R.head(x, w, sx, sw)
        got = H.HeadPlan(x, w, hidden_scales=sx, weight_scales=sw).launch()
        torch.cuda.synchronize()
        error = (got.to(R.F64) - want).square().mean().sqrt() / want.square().mean().sqrt()
        assert float(error) <= bound, (k, float(error), bound)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_a_rows_bits_are_the_same_in_every_batch(dtype):
    from test_gpu_head import head_inputs, head_plan

    s = head_inputs(300, 700, 1040, dtype, 5, 24)
    whole_batch = head_plan(s).launch().clone()
    for rows in (1, 30, 64, 65, 128, 129, 200, 257):
        part = {k: (v[:rows].contiguous() if k in ("hidden", "hidden_scales", "ids") else v) for k, v in s.items()}
        got = head_plan(part).launch()
        torch.cuda.synchronize()
        assert torch.equal(got, whole_batch[:rows]), rows
