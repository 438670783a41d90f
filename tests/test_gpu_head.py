"""The norm, the head projection and the adapters (include/mantle_head.h) against their definitions in 64 bits."""
import itertools

import numpy as np
import pytest
import torch

import head_ref as R
from mantle_b200 import head as H
from mantle_b200 import native, sampler

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def rand(seed, *shape):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=F32).to(DEV)


# ---------------------------------------------------------------------------------------
# norm


def check_norm(x, weight=None, residual=None, out_dtype=None, group=0, eps=1e-6, offset=0.0, plan=None, where=""):
    y, s = R.norm(x, weight, residual, eps, offset)
    plan = plan or H.NormPlan(x, weight, residual=residual, eps=eps, weight_offset=offset, out_dtype=out_dtype, scale_group=group)
    o = plan.launch()
    torch.cuda.synchronize()
    parts = x.to(R.F64).abs() + (0 if residual is None else residual.to(R.F64).abs())
    if residual is not None:
        R.check(o.residual_out, s, parts * 2.0 ** -24, (where, "residual"))
    # y's error: relative, and what the rounding of s leaves where x and residual cancel
    rel = R.norm_slack(x)
    w = (torch.ones(x.shape[1], dtype=R.F64, device=x.device) if weight is None else weight.to(R.F64)) + offset
    slack = y.abs() * rel + parts * 2.0 ** -24 / (s.square().mean(1, keepdim=True) + eps).sqrt() * w.abs()
    if o.out.dtype != E4M3:
        R.check(o.out, y, slack, (where, "out"))
        return o
    sc = R.scales(y, group)
    g = group or x.shape[1]
    wide = lambda t: t.repeat_interleave(g, 1)[:, :x.shape[1]]
    worst = torch.stack([slack[:, c:c + g].amax(1) for c in range(0, x.shape[1], g)], 1)
    R.check(o.scales, sc, worst / R.E4M3_MAX + sc * 2.0 ** -23, (where, "scales"))
    # an e4m3 value is off by half a step: 2^-4 of itself, or 2^-10 below the normal range
    q, scale = o.out.to(R.F64), wide(o.scales.to(R.F64))
    allowed = slack + y.abs() * 2.0 ** -22 + scale * torch.maximum((y / scale).abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** -10))
    assert bool(((q * scale - y).abs() <= allowed * 1.0001 + 1e-37).all()), (where, "out")
    return o


@pytest.mark.parametrize("hidden", [1, 7, 8, 31, 127, 128, 129, 248, 256, 257, 1000, 1024, 4096, 5001, 8192, 16384, 32767, 32768])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_over_sizes(hidden, dtype):
    for rows, residual, quant, group in itertools.product((1, 3, 301), (False, True), (False, True), (0, 128)):
        if group and not quant or rows * hidden > 4 << 20:
            continue
        x = (rand(hidden + rows, rows, hidden) * 3).to(dtype)
        r = rand(hidden + rows + 1, rows, hidden).to(dtype) if residual else None
        w = (1 + 0.2 * rand(5, hidden)).to(dtype)
        check_norm(x, w, r, E4M3 if quant else None, group, where=(rows, residual, quant, group))


@pytest.mark.parametrize("quant,group", [(False, 0), (True, 0), (True, 128)])
def test_norm_strides_offsets_and_weights(quant, group):
    for dtype, hidden, pad, shift in itertools.product((F32, BF16), (264, 1000, 2049), (0, 8, 3), (0, 8, 1)):
        wide = rand(1, 9, hidden + pad + shift + 5).to(dtype)
        x = wide[:, shift:shift + hidden]
        r = rand(2, 9, hidden + 2 * pad + shift).to(dtype)[:, shift:shift + hidden]
        for weight in (None, rand(3, hidden), rand(3, hidden).to(BF16), rand(3, hidden + 1)[1:]):
            out = torch.full((11, hidden + pad + 16), 7.0, device=DEV).to(E4M3 if quant else dtype)
            plan = H.NormPlan(x, weight, residual=r, eps=1e-5, weight_offset=1.0, out_dtype=E4M3 if quant else None,
                              scale_group=group, out=out[1:10, 8:8 + hidden])
            check_norm(x, weight, r, eps=1e-5, offset=1.0, group=group, plan=plan, where=(dtype, hidden, pad, shift))
            rim = out.float()
            rim[1:10, 8:8 + hidden] = 7.0
            assert bool((rim == 7.0).all())  # nothing beside the rows was written


@pytest.mark.parametrize("hidden,dtype", [(2048, BF16), (2056, F32), (4096, BF16), (8192, BF16), (8184, BF16), (4104, F32)])
def test_norm_of_many_long_rows(hidden, dtype):
    """Enough rows for the kernel that keeps a ring of them, an odd number for each of its CTAs."""
    rows = 148 * 17 + 5
    x, r = (rand(1, rows, hidden) * 2).to(dtype), rand(2, rows, hidden).to(dtype)
    w = (1 + 0.1 * rand(3, hidden)).to(dtype)
    for residual, quant, group in itertools.product((False, True), (False, True), (0, 128)):
        if group and not quant:
            continue
        o = check_norm(x, w, r if residual else None, E4M3 if quant else None, group, where=(residual, quant, group))
    xi, ri = x.clone(), r.clone()
    got = H.NormPlan(xi, w, residual=ri, out=xi, residual_out=ri)
    got.launch()
    want = H.NormPlan(x, w, residual=r).launch()
    torch.cuda.synchronize()
    assert torch.equal(xi, want.out) and torch.equal(ri, want.residual_out) and int(got.status.item()) == 0


def test_norm_in_place():
    for dtype in (F32, BF16):
        x0, r0 = (rand(1, 50, 1032) * 2).to(dtype), rand(2, 50, 1032).to(dtype)
        w = rand(3, 1032).to(dtype)
        want = H.NormPlan(x0, w, residual=r0).launch()
        x, r = x0.clone(), r0.clone()
        got = H.NormPlan(x, w, residual=r, out=x, residual_out=r).launch()
        torch.cuda.synchronize()
        assert torch.equal(got.out, want.out) and torch.equal(got.residual_out, want.residual_out)
        x = x0.clone()
        o = torch.empty_like(x)
        H.NormPlan(x, w, residual=r0, out=o, residual_out=x).launch()
        torch.cuda.synchronize()
        assert torch.equal(o, want.out) and torch.equal(x, want.residual_out)


def test_norm_rows_of_zeros_infinities_and_nan():
    for hidden, dtype in itertools.product((256, 1024, 1001), (F32, BF16)):
        x = rand(1, 6, hidden).to(dtype)
        x[0] = 0
        x[1, 200] = float("inf")
        x[2, 200] = float("nan")
        x[3] = 1e-30
        for quant, group in ((False, 0), (True, 0), (True, 128)):
            o = H.NormPlan(x, eps=1e-6, out_dtype=E4M3 if quant else None, scale_group=group).launch()
            torch.cuda.synchronize()
            y = o.out.float()
            if quant:
                g = group or hidden
                y = y * o.scales.repeat_interleave(g, 1)[:, :hidden]
                nan_cols = slice(128, 256) if group else slice(0, hidden)
                assert bool(torch.isnan(y[1, nan_cols]).all())
                assert bool((y[1, :128] == 0).all()) == bool(group)
                assert bool((o.scales[0] == R.SCALE_MIN).all())
            else:
                # 1 / sqrt(inf) is 0: zeros, and NaN where the infinity stood
                assert bool(torch.isnan(y[1, 200])) and bool((y[1, :200] == 0).all())
            assert bool((y[0] == 0).all()) and bool(torch.isnan(y[2]).all()) and bool(torch.isfinite(y[3:]).all())


# ---------------------------------------------------------------------------------------
# head


def head_inputs(rows, vocab, hidden, dtype=BF16, adapters=0, rank=0, beside=False, out=F32, seed=0):
    s = {}
    x = rand(seed + 1, rows, hidden)
    w = rand(seed + 2, vocab, hidden) * (3 / hidden ** 0.5)
    if dtype == E4M3:
        s["hidden"], s["hidden_scales"] = R.to_e4m3_rows(x)
        if not beside:
            s["weight"], s["weight_scales"] = R.to_e4m3_rows(w)
    else:
        s["hidden"] = x.to(BF16)
        if not beside:
            s["weight"] = w.to(BF16)
    if beside:
        s["base"] = rand(seed + 3, rows, vocab).to(out)
    if adapters:
        s["a"] = (rand(seed + 4, adapters, rank, hidden) / hidden ** 0.5).to(BF16)
        s["b"] = (rand(seed + 5, adapters, vocab, rank) / rank ** 0.5).to(BF16)
        s["gain"] = 0.5 + rand(seed + 6, adapters).abs()
        g = torch.Generator(device="cpu")
        g.manual_seed(seed + 7)
        s["ids"] = torch.randint(-1, adapters, (rows,), generator=g, dtype=torch.int32).to(DEV)
    return s


def head_plan(s, out_dtype=F32, **kw):
    ad = H.Adapters(s["a"], s["b"], s.get("gain")) if "a" in s else None
    return H.HeadPlan(s["hidden"], s.get("weight"), hidden_scales=s.get("hidden_scales"), weight_scales=s.get("weight_scales"),
                      adapters=ad, adapter_ids=s.get("ids"), base=s.get("base"), out_dtype=out_dtype, **kw)


def check_head(s, out_dtype=F32, plan=None, where=""):
    want, slack = R.head(**s)
    plan = plan or head_plan(s, out_dtype)
    got = plan.launch()
    torch.cuda.synchronize()
    assert int(plan.status.item()) == 0, where
    R.check(got, want, slack, where)
    return got


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 100, 128, 129, 200, 256, 257, 300, 513])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_head_over_rows(rows, dtype):
    for vocab, hidden in ((1, 64), (15, 16), (128, 128), (1000, 272), (2500, 1040)):
        check_head(head_inputs(rows, vocab, hidden, dtype), where=(vocab, hidden))


@pytest.mark.parametrize("rows", [1, 7, 16, 40, 129, 256, 300, 600])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_head_with_adapters(rows, dtype):
    for vocab, hidden, n, rank in ((1, 64, 1, 8), (300, 128, 3, 8), (1111, 336, 5, 24), (2500, 528, 40, 16), (999, 64, 7, 64),
                                   (130, 256, 2, 256)):
        for out in (F32, BF16):
            check_head(head_inputs(rows, vocab, hidden, dtype, n, rank), out, where=(vocab, hidden, n, rank, out))


@pytest.mark.parametrize("rows", [1, 16, 90, 260, 520])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_adapters_beside_a_projection(rows, dtype):
    for vocab, hidden, n, rank in ((1, 64, 1, 8), (1000, 128, 3, 40), (4097, 512, 20, 16)):
        for out in (F32, BF16):
            s = head_inputs(rows, vocab, hidden, dtype, n, rank, beside=True, out=out)
            got = check_head(s, out, where=(vocab, hidden, n, rank, out)).clone()
            base = s["base"].clone()
            plan = head_plan({**s, "base": base}, out, out=base)  # in place
            plan.launch()
            torch.cuda.synchronize()
            assert torch.equal(base, got)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("rows,vocab,hidden,n,rank", [
    (3, 40, 65536, 2, 8),        # the widest row: rounds of either type
    (128, 300, 64, 200, 32),     # nearly every row its own adapter: several segments of steps a tile, rows in place
    (300, 700, 64, 400, 32),     # the same with sorted rows
    (1000, 260, 64, 1, 16),      # one adapter over several tiles of rows
    (40, 64, 64, 4096, 8),       # the largest table
    (2100, 130, 128, 5, 24),     # more rows than one pass of the sort's threads
])
def test_head_at_the_ends_of_its_ranges(rows, vocab, hidden, n, rank, dtype):
    s = head_inputs(rows, vocab, hidden, dtype, n, rank)
    check_head(s)
    s["ids"].copy_(torch.arange(rows, dtype=torch.int32) % (n + 1) - 1)
    check_head(s)
    s.pop("weight")
    s.pop("weight_scales", None)
    s["base"] = rand(9, rows, vocab)
    check_head(s)


def test_two_graphs_of_two_plans_and_more_rows_than_stay_in_place():
    """The sorted form captured, ids changed between replays, beside another graph on another stream."""
    made = []
    for i in range(2):
        s = head_inputs(200 + 90 * i, 900, 128, (BF16, E4M3)[i], 12, 16, seed=20 * i)
        plan = head_plan(s)
        plan.launch()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plan.launch()
        made.append((s, plan, g, torch.cuda.Stream()))
    for turn in range(3):
        for i, (s, plan, g, st) in enumerate(made):
            rows = s["ids"].shape[0]
            s["ids"].copy_(torch.randint(-1, 12, (rows,), generator=torch.Generator().manual_seed(turn + 7 * i), dtype=torch.int32))
        torch.cuda.synchronize()
        for s, plan, g, st in made:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, plan, g, st in made:
            want, slack = R.head(**s)
            R.check(plan.out, want, slack, turn)


def test_ids_that_mean_no_adapter():
    s = head_inputs(70, 900, 128, BF16, 4, 16)
    plain = head_plan({k: s[k] for k in ("hidden", "weight")}).launch()
    plan = head_plan(s)
    for ids in ([-1] * 70, [4] * 70, [-2 ** 31, 2 ** 31 - 1] * 35):
        s["ids"].copy_(torch.tensor(ids, dtype=torch.int64).to(torch.int32))
        got = plan.launch()
        torch.cuda.synchronize()
        assert torch.equal(got, plain)
    s["ids"].fill_(3)  # all on one
    check_head(s, plan=plan)
    s["ids"].copy_(torch.arange(70, dtype=torch.int32) % 6 - 1)
    check_head(s, plan=plan)


def test_a_row_does_not_depend_on_its_batch():
    for dtype in (BF16, E4M3):
        s = head_inputs(150, 700, 256, dtype, 6, 16)
        whole = head_plan(s).launch().clone()
        order = torch.randperm(150, generator=torch.Generator().manual_seed(3)).to(DEV)
        t = dict(s)
        for k in ("hidden", "hidden_scales", "ids"):
            if k in s:
                t[k] = (s[k].view(torch.uint8) if s[k].dtype == E4M3 else s[k])[order].contiguous()
                t[k] = t[k].view(E4M3) if s[k].dtype == E4M3 else t[k]
        shuffled = head_plan(t).launch().clone()
        torch.cuda.synchronize()
        assert torch.equal(shuffled, whole[order])


def test_a_bad_row_spoils_only_itself():
    s = head_inputs(40, 500, 128, BF16, 3, 8)
    clean = head_plan(s).launch().clone()
    s["hidden"][11, 5] = float("nan")
    s["hidden"][20, 7] = float("inf")
    got = head_plan(s).launch()
    torch.cuda.synchronize()
    keep = torch.ones(40, dtype=torch.bool, device=DEV)
    keep[11] = keep[20] = False
    assert torch.equal(got[keep], clean[keep])
    assert bool(torch.isnan(got[11]).all()) and not bool(torch.isfinite(got[20]).any())


def test_head_strides_and_alignment():
    for dtype, shift, pad in itertools.product((BF16, E4M3), (0, 1, 16), (0, 16, 5)):
        for adapters in (0, 3):
            s = head_inputs(37, 333, 160, dtype, adapters, 16)
            raw = torch.zeros((40, 160 + pad + shift + 3), device=DEV).to(BF16).to(dtype)
            view = raw[1:38, shift:shift + 160]
            view.copy_(s["hidden"])
            s["hidden"] = view
            wraw = torch.zeros((340, 160 + 16), device=DEV).to(BF16).to(dtype)
            wraw[2:335, :160].copy_(s["weight"])
            s["weight"] = wraw[2:335, :160]
            out = torch.full((39, 333 + 9), 5.0, device=DEV)
            plan = head_plan(s, out=out[1:38, 4:337])
            check_head(s, plan=plan, where=(dtype, shift, pad, adapters))
            out[1:38, 4:337] = 5.0
            assert bool((out == 5.0).all())


def test_other_stream_and_a_captured_step():
    s = head_inputs(48, 3000, 256, BF16, 8, 16)
    x = (rand(90, 48, 256) * 2).to(BF16)
    norm = H.NormPlan(x, None, out=s["hidden"])
    plan = head_plan(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the first launches of a kernel set its attributes: outside the capture
        norm.launch()
        plan.launch()
    side.synchronize()
    check_head(s, plan=plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm.launch()
        plan.launch()
    for turn in range(3):
        x.copy_((rand(91 + turn, 48, 256) * 2).to(BF16))
        s["ids"].copy_(torch.randint(-1, 8, (48,), generator=torch.Generator().manual_seed(turn), dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, slack = R.head(**s)
        R.check(plan.out, want, slack, turn)
        y, _ = R.norm(x)
        R.check(s["hidden"], y, y.abs() * R.norm_slack(x), turn)


def test_two_plans_on_two_streams():
    plans = [(s, head_plan(s)) for s in (head_inputs(30, 20000, 512, BF16, 5, 16, seed=10 * i) for i in range(2))]
    streams = [torch.cuda.Stream() for _ in plans]
    torch.cuda.synchronize()
    for _ in range(20):
        for (s, plan), st in zip(plans, streams):
            plan.launch(stream=st)
    torch.cuda.synchronize()
    for s, plan in plans:
        want, slack = R.head(**s)
        R.check(plan.out, want, slack)


def test_norm_head_sampler_in_a_row():
    """The decode step: norm with the residual to 8 bits, head with adapters, sampler; the sampler's tokens are the
    oracle's on the logits that the head wrote, and the logits the definition's on the 8-bit values."""
    import oracle_lib as O

    rows, vocab, hidden = 24, 5003, 512
    x, r = (rand(1, rows, hidden) * 2).to(BF16), rand(2, rows, hidden).to(BF16)
    s = head_inputs(rows, vocab, hidden, E4M3, 6, 16)
    norm = H.NormPlan(x, 1 + 0.1 * rand(3, hidden), residual=r, out_dtype=E4M3)
    s["hidden"], s["hidden_scales"] = norm.out, norm.scales.view(-1)
    plan = head_plan(s)
    rng = np.random.default_rng(4)
    params = np.zeros(rows, dtype=native.PARAMS_DTYPE)
    for i in range(rows):
        params[i] = sampler.new_sampler_params(sampler.SamplerConfig(temperature=0.8, top_k=30, top_p=0.95), rng.random())
    batch = sampler.BatchPlan(plan.out, sampler.params_to_device(params, DEV), 30)
    norm.launch()
    plan.launch()
    out = batch.launch()
    torch.cuda.synchronize()
    want, slack = R.head(**s)
    R.check(plan.out, want, slack)
    ref = O.sample_rows(plan.out.cpu().numpy(), params)
    assert np.array_equal(out.next.cpu().numpy(), ref["next"])


def test_decode_loop_from_the_hidden_state():
    """BatchSampler.step_hidden: the tokens are those of a BatchSampler that is fed the head's logits, step after step."""
    rows, vocab, hidden = 20, 4001, 256
    s = head_inputs(rows, vocab, hidden, BF16, 5, 8)
    x, r = rand(1, rows, hidden).to(BF16), rand(2, rows, hidden).to(BF16)
    norm = H.NormPlan(x, rand(3, hidden).to(BF16), residual=r, weight_offset=1.0, out=s["hidden"])
    plan = head_plan(s)
    both = [sampler.BatchSampler(rows, vocab, 64, [7], device=DEV) for _ in range(2)]
    for i in range(rows):
        cfg = sampler.SamplerConfig(seed=i, temperature=0.9, top_k=20, top_p=0.95, repeat_penalty=1.2, repeat_last_n=16)
        for b in both:
            b.set_row(i, cfg, [i, i + 1])
    rngs = [[np.random.default_rng(i).random for i in range(rows)] for _ in both]
    for turn in range(6):
        x.copy_(rand(100 + turn, rows, hidden).to(BF16))
        s["ids"].copy_(torch.randint(-1, 5, (rows,), generator=torch.Generator().manual_seed(turn), dtype=torch.int32))
        got, ended = both[0].step_hidden(plan, rngs[0], norm=norm)
        check_norm(x, norm.keep[1], r, offset=1.0, plan=norm, where=turn)  # (runs the norm again, to the same place)
        want, slack = R.head(**s)
        R.check(plan.out, want, slack, turn)
        ref, ref_ended = both[1].step(plan.out, rngs[1])
        assert np.array_equal(got, ref) and np.array_equal(ended, ref_ended)
    other = head_plan(head_inputs(rows, vocab + 1, hidden, BF16))
    for bad in (dict(head=other), dict(head=plan, norm=H.NormPlan(x)), dict(head=plan, norm=H.NormPlan(x, out_dtype=E4M3))):
        with pytest.raises(native.CudaError):
            both[0].step_hidden_async(uniforms=np.zeros(rows), **bad)
    with pytest.raises(ValueError):
        both[0].step_hidden_async(plan, np.zeros(rows + 1))
    for b in both:
        b.close()


def test_an_adapter_is_replaced():
    s = head_inputs(30, 700, 128, BF16, 4, 16)
    ad = H.Adapters(s["a"], s["b"], s["gain"])
    plan = H.HeadPlan(s["hidden"], s["weight"], adapters=ad, adapter_ids=s["ids"])
    t = head_inputs(30, 700, 128, BF16, 4, 16, seed=50)
    s["b"] = s["b"].clone()
    ad.replace(2, t["a"][1], t["b"][1], 1.75)
    s["b"][2] = t["b"][1]
    check_head(s, plan=plan)
    assert torch.equal(s["a"][2], t["a"][1]) and float(s["gain"][2]) == 1.75
    with pytest.raises(ValueError):
        ad.replace(4, t["a"][1], t["b"][1], 1.0)
    with pytest.raises(ValueError):
        ad.replace(1, t["a"][1], t["b"][1])


def test_plans_refuse_what_they_cannot_run():
    s = head_inputs(8, 100, 64, BF16, 2, 8)
    x = s["hidden"]
    ad = H.Adapters(s["a"], s["b"])
    for args, kw in (((x,), {}), ((x, s["weight"]), dict(base=torch.zeros(8, 100, device=DEV))),
                     ((x, s["weight"][:, :32]), {}), ((x, s["weight"]), dict(adapters=ad)),
                     ((x, s["weight"]), dict(adapter_ids=s["ids"])), ((x, s["weight"]), dict(adapters=ad, adapter_ids=s["ids"].long())),
                     ((x, s["weight"]), dict(adapters=ad, adapter_ids=s["ids"][:7])), ((x, s["weight"][:50]), dict(adapters=ad, adapter_ids=s["ids"])),
                     ((x, s["weight"]), dict(out_dtype=torch.float16)), ((x, s["weight"]), dict(out=torch.zeros(8, 99, device=DEV))),
                     ((x, s["weight"]), dict(hidden_scales=torch.ones(8, device=DEV))), ((x.float(), s["weight"]), {}),
                     ((x.to(E4M3), s["weight"].to(E4M3)), {})):
        with pytest.raises(ValueError):
            H.HeadPlan(*args, **kw)
    with pytest.raises(native.CudaError, match="16 bytes"):  # rows of W that TMA cannot read
        H.HeadPlan(x[:, :56].contiguous(), torch.zeros(100, 60, device=DEV, dtype=BF16)[:, :56])
    with pytest.raises(native.CudaError, match="multiple of 8"):
        H.HeadPlan(x[:, :60].contiguous(), torch.zeros(100, 60, device=DEV, dtype=BF16))
    wide = torch.zeros(8, 200, device=DEV, dtype=BF16)
    with pytest.raises(ValueError, match="overlaps"):
        H.NormPlan(wide[:, :64], out=wide[:, 32:96])
    with pytest.raises(ValueError, match="overlaps"):
        H.HeadPlan(wide[:, :64], s["weight"], out_dtype=BF16, out=wide[:, 100:])
    with pytest.raises(ValueError):
        H.NormPlan(wide, residual=wide.float())
    with pytest.raises(native.CudaError, match="MAX_HIDDEN"):
        H.NormPlan(torch.zeros(1, 32769, device=DEV)).launch()
