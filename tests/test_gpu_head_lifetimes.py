"""Plans and the streams they run on: memory that outlives its plan's last launch, and what the first launches of two
threads do."""
import threading

import pytest
import torch

import head_ref as R
from mantle_b200 import head as H
from test_gpu_head import BF16, DEV, E4M3, F32, head_inputs, rand

pytestmark = pytest.mark.gpu
SLEEP = 200_000_000  # cycles, about a tenth of a second


def test_a_plan_dropped_while_a_side_stream_runs_it():
    s = head_inputs(300, 2000, 128, E4M3, 6, 16)
    want, slack = R.head(**s)
    side = torch.cuda.Stream()
    out = torch.empty((300, 2000), dtype=F32, device=DEV)
    plan = H.HeadPlan(s["hidden"], s["weight"], hidden_scales=s["hidden_scales"], weight_scales=s["weight_scales"],
                      adapters=H.Adapters(s["a"], s["b"], s["gain"]), adapter_ids=s["ids"], out=out)
    sizes = [plan.workspace.numel()] + [t.numel() * t.element_size() for t in s.values()]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
    plan.launch(stream=side)
    del plan
    s.clear()
    junk = [torch.full((n,), 255, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(3)]  # runs at once
    torch.cuda.synchronize()
    R.check(out, want, slack)
    del junk


def test_one_shot_forms_on_a_busy_side_stream():
    x, w = rand(1, 500, 1024).to(BF16), rand(2, 700, 1024).to(BF16)
    y, _ = R.norm(x)
    want, slack = R.head(x, w)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
    o = H.norm_rows(x, stream=side)
    logits = H.head_logits(x, w, stream=side)
    sizes = [t.numel() * t.element_size() for t in (x, w)]
    del x, w
    junk = [torch.full((n,), 255, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(3)]
    torch.cuda.synchronize()
    R.check(o.out, y, y.abs() * R.norm_slack(y))
    R.check(logits, want, slack)
    del junk


def test_first_launches_of_two_threads():
    """One kernel with two sizes of shared memory: afterwards either runs."""
    made = [head_inputs(rows, 1000, 256, BF16, 3, 16, seed=rows) for rows in (96, 128, 20, 32)]
    want = [R.head(**s) for s in made]
    plans = [H.HeadPlan(s["hidden"], s["weight"], adapters=H.Adapters(s["a"], s["b"], s["gain"]), adapter_ids=s["ids"]) for s in made]
    torch.cuda.synchronize()
    failed = []

    def run(plan):
        try:
            st = torch.cuda.Stream()
            for _ in range(50):
                plan.launch(stream=st)
            st.synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=run, args=(p,)) for p in plans]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for p, (w, slack) in zip(plans, want):
        p.launch()
        torch.cuda.synchronize()
        R.check(p.out, w, slack)
