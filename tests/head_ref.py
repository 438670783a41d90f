"""The norm, the head projection and the adapters from their definitions in 64 bits, and how far a result
in fewer bits may be from them: shared by the CPU and GPU tests."""
import torch

F64 = torch.float64
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}


def to_e4m3_rows(t):
    """A float32 matrix as e4m3 with one scale a row."""
    scale = (t.abs().amax(1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (t / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def norm(x, weight=None, residual=None, eps=1e-6, offset=0.0):
    """(y, s): the normed rows and the sums, unrounded."""
    s = x.to(F64)
    if residual is not None:
        s = s + residual.to(F64)
    w = (torch.ones(x.shape[1], dtype=F64, device=x.device) if weight is None else weight.to(F64)) + offset
    return s / (s.square().mean(1, keepdim=True) + eps).sqrt() * w, s


def norm_slack(x, residual=None, weight=None, offset=0.0):
    """How far the float32 y may be from the exact one, relative to |y|, and beside it as an absolute part:
    s is rounded once (2^-24 of |x| + |r|, which cancellation can make large against s), the sum of n squares of
    rounded values has at most n + 2 roundings of its positive terms, halved by the root; root, division, two
    products and weight + offset round once each, and the products' factors are s and w + offset."""
    n = x.shape[1]
    return (n / 2 + 10) * 2.0 ** -24


def scales(y, group):
    n = y.shape[1]
    g = group or n
    return torch.stack([(y[:, c:c + g].abs().amax(1) / E4M3_MAX).clamp_min(SCALE_MIN) for c in range(0, n, g)], 1)


def head(hidden, weight=None, hidden_scales=None, weight_scales=None, a=None, b=None, gain=None, ids=None, base=None):
    """(out, slack): the logits, and the largest distance a float32 computation may have from them.

    A step of the tensor cores adds 16 (32 with 8 bits) exact products to a float32 sum; its rounding, and what
    it drops when it lines the products up, is at most 2^-22 of the sum of the terms' sizes.  Between the
    adapter's products u is two bfloat16, so it is off by 2^-8 * 2^-8 of itself beside its own sum's error.
    """
    x = hidden.to(F64)
    if hidden_scales is not None:
        x = x * hidden_scales.to(F64).view(-1, 1)
    rows, k = x.shape
    steps = k / 16 + 8
    if base is not None:
        out = base.to(F64).clone()
        size = out.abs()
    else:
        w = weight.to(F64)
        if weight_scales is not None:
            w = w * weight_scales.to(F64).view(-1, 1)
        out = x @ w.T
        size = x.abs() @ w.abs().T
    slack = size * (steps * 2.0 ** -22)
    if a is not None:
        used = 0
        for i in range(a.shape[0]):
            at = torch.nonzero(ids == i).view(-1)
            if not at.numel():
                continue
            used += 1
            g = 1.0 if gain is None else gain[i].to(F64)
            ai, bi = a[i].to(F64), b[i].to(F64)
            u = g * (x[at] @ ai.T)
            u_size = (x[at].abs() @ ai.abs().T) * abs(g)
            out[at] += u @ bi.T
            slack[at] += (u.abs() * 2.0 ** -16 + u_size * (steps * 2.0 ** -22)) @ bi.abs().T
            slack[at] += (u.abs() @ bi.abs().T) * ((a.shape[1] / 8 + 8) * 2.0 ** -22)
        # every adapter in the batch is one more step of every sum that its window covers
        slack += (size + slack) * (used * a.shape[1] / 8 * 2.0 ** -24)
    return out, slack


def check(got, want, slack, where=""):
    """got within slack, and one rounding to its type, of want; NaN where want is NaN."""
    got64 = got.to(F64)
    assert torch.equal(torch.isnan(got64), torch.isnan(want)), where
    off = (got64 - want).abs()
    allowed = slack + HALF_STEP[got.dtype] * (want.abs() + slack) + 1e-37
    bad = torch.nonzero(off > allowed)
    assert not bad.numel(), (where, bad[:4].tolist(), float((off / allowed).nan_to_num(0.0).max()),
                             [(float(got64[tuple(i)]), float(want[tuple(i)])) for i in bad[:4]])
