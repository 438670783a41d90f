"""What stands between a model's last layer and the sampler: the norm with the residual's addition
(in 8 bits where asked), the head projection, and the low-rank adapters that the requests of a batch
bring with them -- as cases to measure, with their plain forms.

Kinds of a case:
  norm   s = x + residual;  y = s * rsqrt(mean(s^2) + eps) * (weight + offset);  out = y, or y in e4m3
         with one scale a row (group 0) or a scale for every `group` columns
  head   out[r][v] = sum_k x[r][k] W[v][k]  (x and W bf16, or e4m3 with a scale a row)
         + g[a] * sum_j B[a][v][j] * sum_k x[r][k] A[a][j][k]  for a row r that uses adapter a;
         with beside = True a given `base` takes the place of the projection
  step   both in a row: norm, 8-bit output, head with adapters
"""
import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
DEV = "cuda"


def _norm(name, rows, hidden, dtype="bf16", residual=True, out="same", group=0, offset=0.0):
    return dict(name=name, kind="norm", rows=rows, hidden=hidden, dtype=dtype, residual=residual, out=out, group=group,
                offset=offset)


def _head(name, rows, vocab, hidden, dtype="bf16", out="f32", adapters=0, rank=0, beside=False, kind="head"):
    return dict(name=name, kind=kind, rows=rows, vocab=vocab, hidden=hidden, dtype=dtype, out=out, adapters=adapters,
                rank=rank, beside=beside)


def listed():
    return [
        # one request, one token: latency
        _norm("norm_token", 1, 1024),
        # a decode batch whose head reads 8 bits
        _norm("norm_batch_8bit", 64, 4096, out="e4m3"),
        # a prompt's rows
        _norm("norm_prompt", 4096, 1024),
        # many long rows, a scale for every 128 columns, weights stored as offsets from one
        _norm("norm_prompt_groups", 16384, 8192, out="e4m3", group=128, offset=1.0),
        # 32-bit activations whose rows start off the 16-byte boundary
        _norm("norm_f32_odd", 777, 5001, dtype="f32", residual=False),
        # one token of one request: the head's weights are all there is to read
        _head("head_token", 1, 151936, 1024),
        # a decode batch of requests with sixteen adapters among them
        _head("head_decode_adapters", 64, 151936, 1024, adapters=16, rank=16),
        # a large decode batch on 8-bit weights
        _head("head_8bit", 256, 128256, 4096, dtype="e4m3"),
        # a ragged one: odd vocabulary, odd batch, the smallest rank
        _head("head_8bit_odd_adapters", 33, 50001, 2048, dtype="e4m3", adapters=8, rank=8),
        # scoring: every row of a full batch, many adapters (the largest)
        _head("head_scores", 4096, 151936, 1024, adapters=64, rank=16),
        # adapters added to the logits of one vocabulary shard that another projection made
        _head("adapters_beside", 512, 32768, 4096, adapters=32, rank=64, beside=True),
        # the decode step in front of the sampler: norm, 8 bits, head, adapters
        _head("step_8bit", 128, 128256, 4096, dtype="e4m3", out="bf16", adapters=32, rank=16, kind="step"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "head", "head", "head", "step"])
    if kind == "norm":
        while True:
            rows, hidden = _log(rng, 1, 16384), _log(rng, 1, 16384)
            if rng.random() < 0.5:
                hidden = max(8, hidden // 64 * 64)
            if rows * hidden <= 16384 * 8192 // 2:
                break
        out = rng.choice(["same", "e4m3"])
        return dict(kind=kind, rows=rows, hidden=hidden, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    residual=rng.random() < 0.7, out=out, group=rng.choice([0, 128]) if out == "e4m3" else 0,
                    offset=rng.choice([0.0, 1.0]))
    while True:
        rows, vocab, hidden = _log(rng, 1, 4096), _log(rng, 1000, 262144), max(64, _log(rng, 64, 8192) // 16 * 16)
        adapters = 0 if kind == "head" and rng.random() < 0.3 else _log(rng, 1, 64)
        rank = 8 * rng.randint(1, 8) if adapters else 0
        if (vocab * hidden <= 128256 * 4096 and rows * vocab <= 2048 * 151936
                and rows * vocab * (hidden + adapters * rank) <= 4096 * 151936 * 1024
                and vocab * adapters * rank <= 64 * 16 * 151936):
            break
    return dict(kind=kind, rows=rows, vocab=vocab, hidden=hidden,
                dtype="e4m3" if kind == "step" else rng.choice(["bf16", "e4m3"]),
                out="bf16" if kind == "step" else rng.choice(["f32", "f32", "bf16"]), adapters=adapters, rank=rank,
                beside=bool(kind == "head" and adapters and rng.random() < 0.25))


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_ADAPTER_SHARE = 0.875  # the rest of the rows use none


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _in_8_bits(t):
    """e4m3 with one scale a row, as stored weights come."""
    scale = (t.abs().amax(1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (t / scale[:, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _norm_inputs(g, case, dtype):
    rows, hidden = case["rows"], case["hidden"]
    x = _rand(g, rows, hidden)
    # a few channels of a trained model's hidden state are far larger than the rest
    x[:, torch.randint(0, hidden, (max(1, hidden // 256),), generator=g, device=DEV)] *= 20.0
    s = {"x": x.to(dtype), "weight": (1.0 - case.get("offset", 0.0) + 0.2 * _rand(g, hidden)).to(dtype),
         "residual": (3.0 * _rand(g, rows, hidden)).to(dtype) if case.get("residual", True) else None}
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "norm":
        s.update(_norm_inputs(g, case, _TYPES[case["dtype"]]))
    else:
        rows, vocab, hidden, n, rank = (case[k] for k in ("rows", "vocab", "hidden", "adapters", "rank"))
        eight = case["dtype"] == "e4m3"
        if case["kind"] == "step":
            s.update(_norm_inputs(g, case, torch.bfloat16))
        elif eight:
            s["hidden"], s["hidden_scales"] = _in_8_bits(_rand(g, rows, hidden))
        else:
            s["hidden"] = _rand(g, rows, hidden).to(torch.bfloat16)
        if case["beside"]:
            s["base"] = 3.0 * _rand(g, rows, vocab)
            s["base"] = s["base"].to(_TYPES[case["out"]])
        elif eight:
            s["head"], s["head_scales"] = _in_8_bits(_rand(g, vocab, hidden).mul_(3.0 / math.sqrt(hidden)))
        else:
            s["head"] = _rand(g, vocab, hidden).mul_(3.0 / math.sqrt(hidden)).to(torch.bfloat16)
        if n:
            s["a"] = _rand(g, n, rank, hidden).div_(math.sqrt(hidden)).to(torch.bfloat16)
            s["b"] = _rand(g, n, vocab, rank).mul_(0.5 / math.sqrt(rank)).to(torch.bfloat16)
            s["gain"] = 0.5 + 1.5 * torch.rand(n, generator=g, device=DEV)
            ids = torch.randint(0, n, (rows,), generator=g, device=DEV, dtype=torch.int32)
            s["ids"] = torch.where(torch.rand(rows, generator=g, device=DEV) < _ADAPTER_SHARE, ids, torch.full_like(ids, -1))
    if own:
        from mantle_b200 import head as H

        if case["kind"] in ("norm", "step"):
            eight = case["kind"] == "step" or case["out"] == "e4m3"
            s["norm_plan"] = H.NormPlan(s["x"], s["weight"], residual=s["residual"], eps=EPS,
                                        weight_offset=case.get("offset", 0.0),
                                        out_dtype=torch.float8_e4m3fn if eight else None,
                                        scale_group=case.get("group", 0))
        if case["kind"] != "norm":
            hidden, scales = ((s["norm_plan"].out, s["norm_plan"].scales) if case["kind"] == "step"
                              else (s["hidden"], s.get("hidden_scales")))
            s["head_plan"] = H.HeadPlan(hidden, s.get("head"), hidden_scales=scales, weight_scales=s.get("head_scales"),
                                        adapters=H.Adapters(s["a"], s["b"], s["gain"]) if case["adapters"] else None,
                                        adapter_ids=s.get("ids"), base=s.get("base"), out_dtype=_TYPES[case["out"]])
    return s


def _plain_norm(s, case, eight, group):
    x = s["x"].float()
    out = {}
    if s["residual"] is not None:
        x = x + s["residual"].float()
        out["residual"] = x.to(s["x"].dtype)
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * (s["weight"].float() + case.get("offset", 0.0))
    if not eight:
        out["out"] = y.to(s["x"].dtype)
        return out
    rows, hidden = y.shape
    group = group or hidden
    groups = -(-hidden // group)
    wide = torch.nn.functional.pad(y, (0, groups * group - hidden)).view(rows, groups, group)
    out["scales"] = (wide.abs().amax(2) / E4M3_MAX).clamp_min(SCALE_MIN)
    q = (wide / out["scales"][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows, groups * group)[:, :hidden]
    out["out"] = q.to(torch.float8_e4m3fn)
    return out


def _plain_head(s, case, hidden, hidden_scales):
    x = hidden.float()
    if hidden_scales is not None:
        x = x * hidden_scales.view(-1, 1)
    if case["beside"]:
        out = s["base"].float()
    else:
        w = s["head"].float()
        if "head_scales" in s:
            w = w * s["head_scales"][:, None]
        out = x @ w.T
    n, rank = case["adapters"], case["rank"]
    if n:
        # all adapters' products at once; a row keeps its own adapter's part
        u = (x @ s["a"].float().view(n * rank, -1).T).view(-1, n, rank)
        mine = s["ids"][:, None] == torch.arange(n, device=u.device, dtype=torch.int32)
        u = torch.where(mine[:, :, None], u * s["gain"][:, None], torch.zeros_like(u))
        out = out + u.view(-1, n * rank) @ s["b"].permute(0, 2, 1).reshape(n * rank, -1).float()
    return out.to(_TYPES[case["out"]])


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        got = {}
        if kind != "head":
            o = s["norm_plan"].launch()
            got = {"residual": o.residual_out} if kind == "step" else {"out": o.out, "residual": o.residual_out, "scales": o.scales}
        if kind != "norm":
            got["logits"] = s["head_plan"].launch()
        return got
    if kind == "norm":
        return _plain_norm(s, case, case["out"] == "e4m3", case["group"])
    if kind == "head":
        return {"logits": _plain_head(s, case, s["hidden"], s.get("hidden_scales"))}
    o = _plain_norm(s, case, True, 0)
    return {"residual": o["residual"], "logits": _plain_head(s, case, o["out"], o["scales"])}


def exact(case, seed):
    """The definitions in 64 bits.  Nothing is rounded at the end; inside a step the 8-bit values between
    norm and head are part of the definition."""
    s = prepare(case, seed)
    d = torch.float64
    got = {}
    if case["kind"] != "head":
        t = s["x"].to(d)
        if s["residual"] is not None:
            t += s["residual"].to(d)
            got["residual"] = t
        w = s["weight"].to(d) + case.get("offset", 0.0)
        y = t / (t.pow(2).sum(1, keepdim=True) / t.shape[1] + EPS).sqrt() * w
        if case["kind"] == "norm" and case["out"] != "e4m3":
            got["out"] = y
            return got
        group = case.get("group", 0) or y.shape[1]
        q, scales = torch.empty_like(y), []
        for c in range(0, y.shape[1], group):
            part = y[:, c:c + group]
            scales.append((part.abs().amax(1) / 448.0).clamp_min(2.0 ** -126))
            q[:, c:c + group] = part / scales[-1][:, None]
        if case["kind"] == "norm":
            got["out"], got["scales"] = q, torch.stack(scales, 1)
            return got
        x = q.to(torch.float8_e4m3fn).to(d) * scales[0][:, None]
    else:
        x = s["hidden"].to(d)
        if "hidden_scales" in s:
            x = x * s["hidden_scales"].to(d)[:, None]
    if case["beside"]:
        out = s["base"].to(d)
    else:
        out = x @ (s["head"].to(d).T if "head_scales" not in s else (s["head"].to(d) * s["head_scales"].to(d)[:, None]).T)
    for a in range(case["adapters"]):
        rows = torch.nonzero(s["ids"] == a).view(-1)
        if rows.numel():
            out[rows] += s["gain"][a].to(d) * (x[rows] @ s["a"][a].to(d).T) @ s["b"][a].to(d).T
    got["logits"] = out
    return got


def work(case):
    """Bytes: every input read once (of the adapters those that the rows are expected to use), every output written once."""
    rows, hidden = case["rows"], case["hidden"]
    size = {"f32": 4, "bf16": 2, "e4m3": 1, "same": 0}
    nbytes, flops = 0.0, 0.0
    if case["kind"] != "head":
        e = 2 if case["kind"] == "step" else size[case["dtype"]]
        nbytes += rows * hidden * e * (3 if case.get("residual", True) else 1) + hidden * e
        flops += 8.0 * rows * hidden
        if case["kind"] == "norm":
            nbytes += rows * hidden * (e if case["out"] == "same" else 1)
            if case["out"] == "e4m3":
                nbytes += 4 * rows * (-(-hidden // case["group"]) if case["group"] else 1)
            return {"bytes": nbytes, "flops": flops}
    else:
        nbytes += rows * hidden * size[case["dtype"]] + (4 * rows if case["dtype"] == "e4m3" else 0)
    vocab, n, rank = case["vocab"], case["adapters"], case["rank"]
    nbytes += rows * vocab * size[case["out"]] * (2 if case["beside"] else 1)
    if not case["beside"]:
        nbytes += vocab * hidden * size[case["dtype"]] + (4 * vocab if case["dtype"] == "e4m3" else 0)
        flops += 2.0 * rows * vocab * hidden
    if n:
        used = n * (1.0 - (1.0 - _ADAPTER_SHARE / n) ** rows)
        nbytes += used * rank * (hidden + vocab) * 2 + 4 * rows
        flops += 2.0 * _ADAPTER_SHARE * rows * rank * (hidden + vocab)
    return {"bytes": nbytes, "flops": flops}
