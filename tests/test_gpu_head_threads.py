"""Plans launched from threads that have not used the GPU before."""
import threading

import pytest
import torch

import head_ref as R
from test_gpu_head import BF16, head_inputs, head_plan

pytestmark = pytest.mark.gpu


def in_a_thread(work):
    failed = []

    def run():
        try:
            work()
        except Exception as e:
            failed.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert not failed, failed


def test_a_threads_first_call_is_a_launch():
    """The driver's tensor maps want a context that is current on the calling thread."""
    s = head_inputs(20, 1000, 256, BF16, 3, 16)
    plan = head_plan(s)
    stream = torch.cuda.current_stream()
    torch.cuda.synchronize()
    in_a_thread(lambda: plan.launch(stream=stream))
    torch.cuda.synchronize()
    want, slack = R.head(**s)
    R.check(plan.out, want, slack)


def test_a_threads_first_call_is_a_captured_launch():
    s = head_inputs(20, 1000, 256, BF16, 3, 16)
    plan = head_plan(s)
    plan.launch()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    with torch.cuda.stream(side):
        graph.capture_begin(capture_error_mode="relaxed")
        try:
            in_a_thread(lambda: plan.launch(stream=side))
        finally:
            graph.capture_end()
    plan.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    want, slack = R.head(**s)
    R.check(plan.out, want, slack)
