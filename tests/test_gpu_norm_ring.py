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
