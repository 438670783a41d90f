"""include/mantle_head.h without a GPU: exports, struct layouts, and the refusals, which come before any device call;
the Python side's own checks; the test's definitions against elementary sums."""
import ctypes as C
import os
import re

import pytest
import torch

import head_ref as R
from mantle_b200 import head as H
from mantle_b200 import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INV = native.CUDA_ERROR_INVALID_VALUE


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(ROOT, "include", "mantle_head.h")).read()
    names = re.findall(r"\bint\s+(mantle\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S))
    assert len(names) >= 4 and sorted(names) == sorted(n for n in native.HEAD_EXPORTS)
    lib = native.load()
    for n in names:
        assert hasattr(lib, n)


def test_struct_layouts_match_the_header():
    assert C.sizeof(native.NormBatch) == 128
    assert native.NormBatch.x_stride.offset == 56 and native.NormBatch.rows.offset == 96
    assert C.sizeof(native.HeadBatch) == 152
    assert native.HeadBatch.hidden_stride.offset == 88 and native.HeadBatch.rows.offset == 120


def norm_batch(**kw):
    b = native.NormBatch()
    b.x, b.out, b.x_stride, b.out_stride, b.rows, b.hidden = 0x1000, 0x2000, 64, 64, 4, 64
    b.dtype = b.out_dtype = b.weight_dtype = native.DTYPE_BF16
    b.eps = 1e-6
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def head_batch(**kw):
    b = native.HeadBatch()
    b.hidden_rows, b.weight, b.out = 0x1000, 0x2000, 0x3000
    b.hidden_stride = b.weight_stride = 64
    b.rows, b.vocab, b.hidden, b.out_stride = 4, 100, 64, 100
    b.dtype, b.out_dtype = native.DTYPE_BF16, native.DTYPE_F32
    for k, v in kw.items():
        setattr(b, k, v)
    return b


ADAPTERS = dict(adapter_a=0x10000, adapter_b=0x20000, adapter_ids=0x30000, n_adapters=3, rank=16)
EIGHT = dict(dtype=native.DTYPE_E4M3, hidden_scales=0x40000, weight_scales=0x50000)


@pytest.mark.parametrize("change", [
    dict(x=0), dict(out=0), dict(rows=0), dict(rows=-1), dict(hidden=0), dict(hidden=32769, x_stride=32769, out_stride=32769),
    dict(dtype=2), dict(dtype=7), dict(out_dtype=native.DTYPE_F32), dict(weight=0x5000, weight_dtype=2), dict(weight=0x5001),
    dict(out_scale=0x6000), dict(out_dtype=native.DTYPE_E4M3), dict(scale_group=128),
    dict(out_dtype=native.DTYPE_E4M3, out_scale=0x6000, scale_stride=0),
    dict(out_dtype=native.DTYPE_E4M3, out_scale=0x6000, scale_stride=1, scale_group=64),
    dict(out_dtype=native.DTYPE_E4M3, out_scale=0x6000, scale_stride=1, scale_group=128, hidden=129, x_stride=129, out_stride=129),
    dict(residual_out=0x7000, residual_out_stride=64), dict(residual=0x7000, residual_stride=63),
    dict(residual=0x7000, residual_stride=64, residual_out=0x8000, residual_out_stride=63), dict(residual=0x7001, residual_stride=64),
    dict(x_stride=63), dict(out_stride=63), dict(x=0x1001), dict(out=0x2001),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(weight_offset=float("nan")),
])
def test_norm_refuses(change):
    lib = native.load()
    assert lib.mantleCudaNormRows(C.byref(norm_batch(**change)), None) == INV
    assert lib.mantleCudaSamplerLastError().startswith(b"norm: ")
    assert lib.mantleCudaNormRows(None, None) == INV


@pytest.mark.parametrize("change", [
    dict(hidden_rows=0), dict(out=0), dict(rows=0), dict(rows=(1 << 20) + 1), dict(vocab=0),
    dict(vocab=native.MAX_VOCAB + 1, out_stride=native.MAX_VOCAB + 1), dict(hidden=0), dict(hidden=60), dict(hidden=65544, hidden_stride=65544, weight_stride=65544),
    dict(dtype=native.DTYPE_F32), dict(out_dtype=native.DTYPE_E4M3), dict(reserved=1), dict(weight=0), dict(base=0x9000, base_stride=100),
    dict(weight=0, base=0x9000, base_stride=100), dict(weight=0, base=0x9000, base_stride=99, **ADAPTERS),
    dict(hidden_scales=0x9000), dict(weight_scales=0x9000), dict(dtype=native.DTYPE_E4M3), dict(EIGHT, weight_scales=0),
    dict(EIGHT, hidden_scales=0), dict(EIGHT, hidden=72, hidden_stride=80, weight_stride=80),
    dict(hidden_stride=63), dict(out_stride=99), dict(weight_stride=56), dict(weight_stride=68), dict(weight=0x2008), dict(weight_stride=1 << 37),
    dict(hidden_rows=0x1001), dict(out=0x3002), dict(status=0x9001), dict(n_adapters=-1), dict(ADAPTERS, n_adapters=4097),
    dict(ADAPTERS, adapter_a=0), dict(ADAPTERS, adapter_b=0), dict(ADAPTERS, adapter_ids=0), dict(ADAPTERS, adapter_ids=0x30002),
    dict(ADAPTERS, rank=0), dict(ADAPTERS, rank=12), dict(ADAPTERS, rank=264), dict(ADAPTERS, adapter_a=0x10008), dict(ADAPTERS, adapter_b=0x20010),
    dict(ADAPTERS, adapter_gain=0x9001),
])
def test_head_refuses(change):
    lib = native.load()
    n, c = C.c_size_t(7), C.c_int(7)
    b = head_batch(**change)
    assert lib.mantleCudaHeadRows(C.byref(b), 0x100000, 1 << 30, None) == INV
    assert lib.mantleCudaSamplerLastError().startswith(b"head: ")
    assert lib.mantleCudaHeadWorkspaceBytes(C.byref(b), C.byref(n)) == INV
    assert lib.mantleCudaHeadLaunches(C.byref(b), C.byref(c)) == INV
    assert n.value == 7 and c.value == 7


def test_head_workspace():
    lib = native.load()
    n, c = C.c_size_t(7), C.c_int(7)
    assert lib.mantleCudaHeadWorkspaceBytes(C.byref(head_batch()), C.byref(n)) == 0 and n.value == 0
    assert lib.mantleCudaHeadLaunches(C.byref(head_batch()), C.byref(c)) == 0 and c.value == 1
    assert lib.mantleCudaHeadWorkspaceBytes(C.byref(head_batch(hidden_rows=0x1002)), C.byref(n)) == 0 and n.value >= 4 * 64 * 2
    b = head_batch(**ADAPTERS)
    assert lib.mantleCudaHeadWorkspaceBytes(C.byref(b), C.byref(n)) == 0 and n.value > 0
    for ws, size in ((None, n.value), (0x100000, n.value - 1), (0x100080, n.value)):
        assert lib.mantleCudaHeadRows(C.byref(b), ws, size, None) == INV
    assert lib.mantleCudaHeadRows(None, None, 0, None) == INV
    assert lib.mantleCudaHeadWorkspaceBytes(C.byref(b), None) == INV and lib.mantleCudaHeadLaunches(C.byref(b), None) == INV


def test_python_refuses_tensors_off_the_gpu():
    x = torch.zeros(3, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        H.NormPlan(x)
    with pytest.raises(ValueError):
        H.HeadPlan(x, x)
    with pytest.raises(ValueError):
        H.Adapters(torch.zeros(2, 8, 16, dtype=torch.bfloat16), torch.zeros(2, 5, 8, dtype=torch.bfloat16))


def test_overlap():
    t = torch.zeros(100)
    assert H._overlap(t[:50], t[49:]) and not H._overlap(t[:50], t[50:])
    m = torch.zeros(10, 10)
    assert H._overlap(m[:, :5], m[:, 5:])  # spans, not elements: interleaved columns count as overlapping
    assert not H._overlap(m[:5], m[5:]) and not H._overlap(m[:0], m)


def test_definitions_against_elementary_sums():
    g = torch.Generator().manual_seed(1)
    x, r, w = (torch.randn(s, generator=g) for s in ((3, 5), (3, 5), (5,)))
    y, s = R.norm(x, w, r, 1e-6, 1.0)
    for i in range(3):
        sums = [float(x[i, k]) + float(r[i, k]) for k in range(5)]
        d = (sum(v * v for v in sums) / 5 + 1e-6) ** 0.5
        for k in range(5):
            assert abs(float(y[i, k]) - sums[k] / d * (float(w[k]) + 1)) < 1e-12
    x, w = torch.randn(4, 6, generator=g), torch.randn(7, 6, generator=g)
    a, b = torch.randn(2, 3, 6, generator=g), torch.randn(2, 7, 3, generator=g)
    ids, gain = torch.tensor([1, -1, 0, 2]), torch.tensor([0.5, 2.0])
    out, slack = R.head(x, w, a=a, b=b, gain=gain, ids=ids)
    for i in range(4):
        for v in range(7):
            t = sum(float(x[i, k]) * float(w[v, k]) for k in range(6))
            n = int(ids[i])
            if 0 <= n < 2:
                t += float(gain[n]) * sum(float(b[n, v, j]) * sum(float(a[n, j, k]) * float(x[i, k]) for k in range(6)) for j in range(3))
            assert abs(float(out[i, v]) - t) < 1e-12
    assert bool((slack > 0).all())


def test_pack_and_step_refusals():
    lib = native.load()
    n = C.c_size_t(7)
    for args in ((0, 10, 8), (1, 0, 8), (1, 10, 0), (1, 10, 12), (1, 10, 264), (4097, 10, 8), (1, native.MAX_VOCAB + 1, 8)):
        assert lib.mantleCudaAdapterPackBytes(*args, C.byref(n)) == INV
        assert lib.mantleCudaAdapterPack(0x1000, *args, 0x2000, None) == INV
    assert n.value == 7
    assert lib.mantleCudaAdapterPackBytes(2, 257, 24, C.byref(n)) == 0 and n.value == 2 * 2 * 512 * 16 * 2
    assert lib.mantleCudaAdapterPack(None, 1, 10, 8, 0x2000, None) == INV
    assert lib.mantleCudaAdapterPack(0x1000, 1, 10, 8, None, None) == INV
    assert lib.mantleCudaAdapterPack(0x1008, 1, 10, 8, 0x2000, None) == INV
    assert lib.mantleCudaAdapterPack(0x1000, 1, 10, 8, 0x2040, None) == INV
    assert lib.mantleBatchSamplerStepHidden(None, None, C.byref(head_batch()), None, 0, None, 0.0, 0.0, None) == INV
