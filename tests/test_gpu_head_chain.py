"""Kernels that start before the one in front has ended: what a chain of them reads is what was written last, call after
call without a wait in between.  And outputs whose offsets pass 32 bits."""
import pytest
import torch

import head_ref as R
from mantle_b200 import head as H
from test_gpu_head import BF16, DEV, E4M3, F32, head_inputs, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,adapters", [(5, 3), (33, 6), (128, 6), (200, 6), (33, 0), (200, 0)])
@pytest.mark.parametrize("captured", [False, True])
def test_norm_and_head_over_and_over(rows, adapters, captured):
    """x, the ids and with them the 8-bit rows, their scales and every table of the adapters change in each round; the
    same rounds with a wait behind every kernel give the reference, bit for bit."""
    vocab, hidden, rounds = 600, 512, 60
    s = head_inputs(rows, vocab, hidden, E4M3, max(1, adapters), 16)
    xs = (rand(7, rounds, rows, hidden) * 3 * (1 + torch.arange(rounds, device=DEV).view(-1, 1, 1) % 7)).to(BF16)
    ids = torch.randint(-1, max(1, adapters), (rounds, rows), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    x = torch.empty_like(xs[0])
    norm = H.NormPlan(x, None, out_dtype=E4M3)
    kw = dict(adapters=H.Adapters(s["a"], s["b"], s["gain"]), adapter_ids=s["ids"]) if adapters else {}
    plan = H.HeadPlan(norm.out, s["weight"], hidden_scales=norm.scales, weight_scales=s["weight_scales"], **kw)

    def step(wait):
        norm.launch()
        wait()
        plan.launch()
        wait()

    want, got = [torch.empty((rounds, rows, vocab), device=DEV) for _ in range(2)]
    for i in range(rounds):
        x.copy_(xs[i])
        s["ids"].copy_(ids[i])
        step(torch.cuda.synchronize)
        want[i].copy_(plan.out)
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph):
            step(lambda: None)
    torch.cuda.synchronize()
    for i in range(rounds):
        x.copy_(xs[i])
        s["ids"].copy_(ids[i])
        if captured:
            graph.replay()
        else:
            step(lambda: None)
        got[i].copy_(plan.out)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [20, 300])
def test_a_base_that_has_just_been_written(rows):
    s = head_inputs(rows, 5000, 256, BF16, 4, 16, beside=True)
    made = []
    for wait in (torch.cuda.synchronize, lambda: None):
        base = s["base"].clone()
        plan = H.HeadPlan(s["hidden"], base=base, adapters=H.Adapters(s["a"], s["b"], s["gain"]), adapter_ids=s["ids"], out=base)
        torch.cuda.synchronize()
        for _ in range(60):
            base.mul_(0.5)
            wait()
            plan.launch()
            wait()
        torch.cuda.synchronize()
        made.append(base)
    assert torch.equal(*made)


@pytest.mark.parametrize("dtype,adapters", [(BF16, 3), (E4M3, 0)])
def test_logits_past_32_bits(dtype, adapters):
    rows, vocab, hidden = 16500, 131080, 16  # 2.2e9 logits
    s = head_inputs(rows, vocab, hidden, dtype, adapters, 8)
    kw = dict(adapters=H.Adapters(s["a"], s["b"], s["gain"]), adapter_ids=s["ids"]) if adapters else {}
    out = torch.empty((rows, vocab + 8), dtype=BF16, device=DEV)[:, :vocab]
    H.HeadPlan(s["hidden"], s["weight"], hidden_scales=s.get("hidden_scales"), weight_scales=s.get("weight_scales"), out_dtype=BF16,
               out=out, **kw).launch()
    torch.cuda.synchronize()
    for part in (slice(0, 40), slice(rows - 150, rows)):
        t = {k: (v[part] if k in ("hidden", "hidden_scales", "ids") else v) for k, v in s.items()}
        want, slack = R.head(**t)
        R.check(out[part], want, slack, part)
