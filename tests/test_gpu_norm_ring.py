"""The norm where the other tests do not reach: its largest batches, and every form of the kernel that keeps a ring of rows."""
import itertools

import pytest
import torch

import head_ref as R
from mantle_b200 import head as H

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def test_as_many_rows_as_a_descriptor_can_say():
    rows = 2 ** 31 - 1
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    x = torch.empty((rows, 1), dtype=BF16, device=DEV)
    x[-5000:].normal_(generator=g)
    x[:5000].normal_(generator=g)
    out = torch.empty_like(x)
    H.NormPlan(x, out=out, eps=1.0).launch()
    torch.cuda.synchronize()
    for part in (slice(0, 5000), slice(rows - 5000, rows)):
        y, _ = R.norm(x[part], eps=1.0)
        R.check(out[part], y, y.abs() * R.norm_slack(x[part]), part)


def rand(seed, *shape):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=F32, device=DEV)


def check(x, weight, residual, out_dtype, group, where):
    """A norm against its definition: the sum's rounding, the norm's (norm_slack), the scale's and the output's."""
    o = H.NormPlan(x, weight, residual=residual, out_dtype=out_dtype, scale_group=group).launch()
    torch.cuda.synchronize()
    assert int(o.status.item()) == 0
    y, s = R.norm(x, weight, residual)
    parts = x.to(R.F64).abs() + (0 if residual is None else residual.to(R.F64).abs())
    if residual is not None:
        R.check(o.residual_out, s, parts * 2.0 ** -24, (where, "residual"))
    slack = y.abs() * R.norm_slack(x) + parts * 2.0 ** -24 / (s.square().mean(1, keepdim=True) + 1e-6).sqrt() * weight.to(R.F64).abs()
    if out_dtype is None:
        R.check(o.out, y, slack, (where, "out"))
        return
    g = group or x.shape[1]
    wide = lambda t: t.repeat_interleave(g, 1)[:, :x.shape[1]]
    worst = torch.stack([slack[:, c:c + g].amax(1) for c in range(0, x.shape[1], g)], 1)
    sc = R.scales(y, group)
    R.check(o.scales, sc, worst / R.E4M3_MAX + sc * 2.0 ** -23, (where, "scales"))
    q, scale = o.out.to(R.F64), wide(o.scales.to(R.F64))
    allowed = slack + y.abs() * 2.0 ** -22 + scale * torch.maximum((y / scale).abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** -10))
    assert bool(((q * scale - y).abs() <= allowed * 1.0001 + 1e-37).all()), (where, "out")


# rows: for any number of CTAs an SM that the width allows (up to 1536 threads), three rows and more a CTA, and an odd
# number of rows; the last rows of a CTA come when the copies ahead have ended
@pytest.mark.parametrize("hidden,dtype,per_sm", [
    (1032, BF16, 9), (1288, BF16, 8), (2040, BF16, 6), (2048, BF16, 6), (2048, F32, 6), (2056, BF16, 7), (4104, F32, 3),
    (8192, BF16, 2), (8200, BF16, 1), (11968, BF16, 1), (16376, BF16, 1), (16384, BF16, 1), (8200, F32, 1), (11968, F32, 1), (16384, F32, 1)])
def test_every_form_of_the_ring(hidden, dtype, per_sm):
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    rows = 3 * sms * per_sm + 2 * sms + 5
    x, r = (rand(1, rows, hidden) * 2).to(dtype), rand(2, rows, hidden).to(dtype)
    w = (1 + 0.1 * rand(3, hidden)).to(dtype)
    for residual, (out_dtype, group) in itertools.product((None, r), ((None, 0), (E4M3, 0), (E4M3, 128))):
        check(x, w, residual, out_dtype, group, (residual is not None, out_dtype, group))
    # in place, and rows that are not next to one another
    wide_x, wide_r = torch.zeros((rows, hidden + 16), dtype=dtype, device=DEV), torch.zeros((rows, hidden + 8), dtype=dtype, device=DEV)
    xi, ri = wide_x[:, 8:8 + hidden], wide_r[:, :hidden]
    xi.copy_(x)
    ri.copy_(r)
    H.NormPlan(xi, w, residual=ri, out=xi, residual_out=ri).launch()
    want = H.NormPlan(x, w, residual=r).launch()
    torch.cuda.synchronize()
    assert torch.equal(xi, want.out) and torch.equal(ri, want.residual_out)
    assert not bool(wide_x[:, :8].any()) and not bool(wide_x[:, 8 + hidden:].any()) and not bool(wide_r[:, hidden:].any())
