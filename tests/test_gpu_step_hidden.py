"""BatchSampler.step and step_hidden where the other tests do not reach: other streams, refusals, statuses."""
import numpy as np
import pytest
import torch

from mantle_b200 import head as H
from mantle_b200 import native, sampler

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
SLEEP = 200_000_000  # cycles, about a tenth of a second


def rand(seed, *shape):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=F32).to(DEV)


def started(rows, vocab, **kw):
    b = sampler.BatchSampler(rows, vocab, 256, [7], **{"device": DEV, **kw})
    for i in range(rows):
        b.set_row(i, sampler.SamplerConfig(seed=i, temperature=0.9, top_k=20, top_p=0.95), [i, i + 1])
    return b


def generators(rows):
    return [np.random.default_rng(i).random for i in range(rows)]


@pytest.mark.parametrize("hidden_state", [False, True])
def test_steps_on_a_busy_side_stream(hidden_state):
    """The tokens are this step's, not the ones that the step before left in pinned memory."""
    rows, vocab, hidden = 8, 2000, 64
    x, w = rand(1, rows, hidden).to(BF16), rand(2, vocab, hidden).to(BF16)
    plan = H.HeadPlan(x, w)
    logits = plan.launch()
    side = torch.cuda.Stream()
    got_by, ref_by = started(rows, vocab), started(rows, vocab)
    got_rng, ref_rng = generators(rows), generators(rows)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(SLEEP)
        got, ended = (got_by.step_hidden(plan, got_rng, stream=side) if hidden_state
                      else got_by.step(logits, got_rng, stream=side))
        ref, ref_ended = ref_by.step(logits, ref_rng)
        assert np.array_equal(got, ref) and np.array_equal(ended, ref_ended)
    got_by.close()
    ref_by.close()


@pytest.mark.parametrize("post", [dict(logit_scale=-1.0), dict(logit_scale=float("nan")), dict(logit_scale=float("inf")),
                                  dict(logit_softcap=float("inf")), dict(logit_softcap=float("-inf"))])
def test_a_refused_step_has_launched_nothing(post):
    """The norm in front would add x to the residual once more on the retry."""
    rows, vocab, hidden = 8, 2000, 64
    x, r, w = rand(1, rows, hidden).to(BF16), rand(2, rows, hidden).to(BF16), rand(3, vocab, hidden).to(BF16)
    norm = H.NormPlan(x, residual=r, residual_out=r)
    plan = H.HeadPlan(norm.out, w)
    norm.out.fill_(3.0)
    plan.out.fill_(5.0)
    r0 = r.clone()
    by, ref_by = started(rows, vocab), started(rows, vocab)
    rng, ref_rng = generators(rows), generators(rows)
    with pytest.raises(native.CudaError):
        by.step_hidden_async(plan, np.zeros(rows), norm=norm, **post)
    with pytest.raises(native.CudaError):
        by.step_async(plan.out, np.zeros(rows), **post)
    torch.cuda.synchronize()
    assert torch.equal(r, r0) and bool((norm.out == 3.0).all()) and bool((plan.out == 5.0).all())
    got, _ = by.step_hidden(plan, rng, norm=norm)
    assert torch.equal(r, (x.float() + r0.float()).to(BF16))
    ref, _ = ref_by.step(plan.out, ref_rng)
    assert np.array_equal(got, ref)
    by.close()
    ref_by.close()


@pytest.mark.parametrize("which", ["norm", "head"])
def test_a_wait_that_ran_out_is_the_steps_error(which):
    """The mark that such a wait leaves in a plan's status word, put there by hand."""
    rows, vocab, hidden = 8, 2000, 64
    x, w = rand(1, rows, hidden).to(BF16), rand(2, vocab, hidden).to(BF16)
    norm = H.NormPlan(x)
    plan = H.HeadPlan(norm.out, w)
    by = started(rows, vocab)
    rng = generators(rows)
    by.step_hidden(plan, rng, norm=norm)
    assert by.results()[2] == 0
    bad = {"norm": norm, "head": plan}[which]
    bad.status.fill_(native.STATUS_TIMEOUT)
    with pytest.raises(RuntimeError, match="ran out"):
        by.step_hidden(plan, rng, norm=norm)
    assert by.results()[2] & native.STATUS_TIMEOUT
    with pytest.raises(RuntimeError, match="ran out"):
        bad.check()
    norm.check()  # said once
    plan.check()
    by.close()
    by = started(rows, vocab)
    by.step_hidden(plan, rng, norm=norm)
    by.close()


def test_status_words_of_the_one_shot_forms():
    x, w = rand(1, 8, 64).to(BF16), rand(2, 100, 64).to(BF16)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = H.norm_rows(x, status=word)
    assert o.status is word and int(H.norm_rows(x).status.item()) == 0
    H.head_logits(o.out, w, status=word)
    assert int(word.item()) == 0
    for bad in (word.float(), word.cpu(), torch.zeros(2, dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError, match="status"):
            H.norm_rows(x, status=bad)


def test_a_sampler_without_a_device_number_stays_on_its_device():
    """"cuda" means the device that is current when the sampler is made, then and later."""
    by = started(4, 100, device="cuda")
    assert by.device == torch.device("cuda", torch.cuda.current_device())
    plan = H.HeadPlan(rand(1, 4, 64).to(BF16), rand(2, 100, 64).to(BF16))
    other = type("Plan", (), dict(device=torch.device("cuda", 5), batch=plan.batch, workspace=None, workspace_bytes=0,
                                  use_on=lambda self, stream: None))()
    with pytest.raises(ValueError, match="not on"):
        by.step_hidden_async(other, np.zeros(4))
    by.step_hidden(plan, generators(4))
    by.close()
