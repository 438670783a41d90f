"""What stands between a model's last layer and the sampler, over the C-ABI of include/mantle_head.h:
the norm with the residual's addition (NormPlan, norm_rows), the head projection and the low-rank
adapters of a batch's requests (HeadPlan, Adapters, head_logits).

    norm = NormPlan(x, weight, residual=residual, out_dtype=torch.float8_e4m3fn)
    head = HeadPlan(norm.out, w8, hidden_scales=norm.scales, weight_scales=w8_scales,
                    adapters=Adapters(a, b, gain), adapter_ids=ids)
    while ...:                                  # x, residual, ids change in place
        norm.launch()
        logits = head.launch()                  # -> sampler.BatchPlan, sampler.BatchSampler.step

A plan binds a descriptor to device tensors, as sampler.BatchPlan does: built once, launched many times,
captured into a CUDA graph where wanted.  It owns its outputs and its workspace, so two plans may run at the
same time; two launches of one plan may not.  It may be launched on any stream of its device and dropped at once: its
memory, and the inputs' that it keeps, is handed out again only when the streams it ran on are done.  (Not so for a
captured graph, which the caller keeps the plan for.)  A stream other than the one that made the plan and its inputs
waits for that one first, as with any kernel: the caller orders them.  torch supplies device memory and streams; all arithmetic
happens in the CUDA library.
"""
import ctypes as C

import torch

from . import native

_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_DTYPES = {torch.float32: native.DTYPE_F32, torch.bfloat16: native.DTYPE_BF16, torch.float8_e4m3fn: native.DTYPE_E4M3}

_INT32_MAX = 2 ** 31 - 1


def _check(lib, code, where):
    if code != 0:
        err = native.CudaError(code, where)
        if code == native.CUDA_ERROR_INVALID_VALUE:
            msg = lib.mantleCudaSamplerLastError()
            err.args = (err.args[0] + (": " + msg.decode() if msg else ""),)
        raise err


def _rows(t, name, dtypes, device=None, shape=None):
    """A 2-D CUDA tensor with unit column stride: its dtype code and row stride."""
    if not t.is_cuda or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("%s must be a 2-D CUDA tensor with unit column stride" % name)
    if t.dtype not in dtypes:
        raise ValueError("%s must be %s" % (name, " or ".join(str(d).replace("torch.", "") for d in dtypes)))
    if max(t.shape) > _INT32_MAX:  # ctypes would keep the low bits
        raise ValueError("%s has more than %d rows or columns" % (name, _INT32_MAX))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s must be %s, is %s" % (name, tuple(shape), tuple(t.shape)))
    # one row has no stride of its own to speak of
    return _DTYPES[t.dtype], (t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1]))


def _vector(t, name, n, dtypes, device):
    if t.device != device or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or t.dtype not in dtypes:
        raise ValueError("%s must be a contiguous vector of %d %s on %s"
                         % (name, n, " or ".join(str(d).replace("torch.", "") for d in dtypes), device))


def _overlap(a, b):
    """Whether the spans of two tensors' elements meet."""
    def span(t):
        last = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _same(a, b):
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and a.stride() == b.stride()


class _Plan:
    def _bind(self, device):
        self.device = device
        self._index = device.index
        self.lib = native.load()
        self._streams = {_raw_stream(self._index)}  # those that the memory below is tied to

    def _own(self, made, given):
        """What the plan reads and writes: its own tensors, and the caller's, which it keeps alive."""
        self.keep = given
        self._memory = [t for t in made + given if t is not None]

    def use_on(self, stream):
        """Ties the plan's memory to `stream` before it is used there: what is dropped while the stream still runs is not
        handed out again until it is done.  (Streams that torch does not own may end before the memory does: not those.)"""
        if stream.cuda_stream not in self._streams:
            self._tie(stream)

    def _tie(self, stream):
        self._streams.add(stream.cuda_stream)
        if not isinstance(stream, torch.cuda.ExternalStream):
            for t in self._memory:
                t.record_stream(stream)

    def _queue(self, stream):
        # the stream that is current on the plan's device, whatever device is current
        s = _raw_stream(self._index) if stream is None else stream.cuda_stream
        if s not in self._streams:
            self.use_on(torch.cuda.current_stream(self._index) if stream is None else stream)
        if _current_device() == self._index:
            rc = self._fn(*self._args, s)
        else:
            with torch.cuda.device(self._index):
                rc = self._fn(*self._args, s)
        if rc:
            _check(self.lib, rc, self._name)

    def check(self):
        """Raises where a wait inside one of the launches so far ran out, whose outputs are then not valid, and clears
        that mark.  Waits for the device's current stream: launches on others have to be done before."""
        with torch.cuda.device(self._index):
            bits = int(self.status.item())
            if bits:
                self.status.zero_()
                raise RuntimeError("%s: a wait inside the kernel ran out (status %d)" % (self._name, bits))

    def _status(self, status):
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=self.device)
        else:
            _vector(status, "status", 1, (torch.int32,), self.device)
        self.status = status
        return status.data_ptr()


class NormOutputs:
    __slots__ = ("out", "scales", "residual_out", "status")


class NormPlan(_Plan):
    """s = x + residual; out = s / sqrt(mean(s^2) + eps) * (weight + weight_offset), row by row.

    x            [rows, hidden] float32 or bfloat16 CUDA tensor, unit column stride, hidden up to 32768
    weight       optional [hidden] float32 or bfloat16
    residual     optional, like x; residual_out receives s rounded to x's type (made here unless given; x or
                 residual themselves may be given)
    out_dtype    None: x's type (out may be x itself).  torch.float8_e4m3fn: 8 bits, `scales` [rows, 1] float32 for
                 scale_group 0, [rows, ceil(hidden / 128)] for scale_group 128; value = out * scale.  HeadPlan reads
                 scale_group 0; groups are for a reader of the caller's
    out, scales, residual_out   made here unless given.  Apart from what is said above, nothing that is written may
                 overlap anything else, by the spans of the tensors: interleaved columns of one buffer count as overlapping
    status       optional [1] int32 on the device, made here unless given: not 0 once a wait inside a launch has run out
                 (check() says so; several plans may share one)
    """

    def __init__(self, x, weight=None, residual=None, eps=1e-6, weight_offset=0.0, out_dtype=None, scale_group=0,
                 out=None, scales=None, residual_out=None, status=None):
        dtype, x_stride = _rows(x, "x", (torch.float32, torch.bfloat16))
        dev = x.device
        self._bind(dev)
        rows, hidden = x.shape
        out_dtype = x.dtype if out_dtype is None else out_dtype
        if out_dtype not in (x.dtype, torch.float8_e4m3fn):
            raise ValueError("out_dtype must be x's type or float8_e4m3fn")
        b = native.NormBatch()
        b.x, b.x_stride, b.rows, b.hidden, b.dtype = x.data_ptr(), x_stride, rows, hidden, dtype
        if weight is not None:
            _vector(weight, "weight", hidden, (torch.float32, torch.bfloat16), dev)
            b.weight, b.weight_dtype = weight.data_ptr(), _DTYPES[weight.dtype]
        if residual is not None:
            _, b.residual_stride = _rows(residual, "residual", (x.dtype,), dev, x.shape)
            b.residual = residual.data_ptr()
            if residual_out is None:
                residual_out = torch.empty((rows, hidden), dtype=x.dtype, device=dev)
            _, b.residual_out_stride = _rows(residual_out, "residual_out", (x.dtype,), dev, x.shape)
            b.residual_out = residual_out.data_ptr()
        elif residual_out is not None:
            raise ValueError("residual_out without residual")
        if out is None:
            out = torch.empty((rows, hidden), dtype=out_dtype, device=dev)
        b.out_dtype, b.out_stride = _rows(out, "out", (out_dtype,), dev, x.shape)
        b.out = out.data_ptr()
        if out_dtype == torch.float8_e4m3fn:
            groups = -(-hidden // scale_group) if scale_group > 0 else 1
            if scales is None:
                scales = torch.empty((rows, groups), dtype=torch.float32, device=dev)
            _, b.scale_stride = _rows(scales, "scales", (torch.float32,), dev, (rows, groups))
            b.out_scale = scales.data_ptr()
        elif scales is not None:
            raise ValueError("scales go with out_dtype float8_e4m3fn")
        b.scale_group, b.eps, b.weight_offset = scale_group, eps, weight_offset
        writes = [(n, t) for n, t in (("out", out), ("residual_out", residual_out), ("scales", scales)) if t is not None]
        reads = [(n, t) for n, t in (("x", x), ("residual", residual), ("weight", weight)) if t is not None]
        for i, (n, t) in enumerate(writes):
            for m, u in writes[i + 1:]:
                if _overlap(t, u):
                    raise ValueError("%s overlaps %s" % (n, m))
            for m, u in reads:
                # a row's elements are read before any of them is written, and no other row's are touched
                in_place = (n, m) in (("out", "x"), ("residual_out", "x"), ("residual_out", "residual")) and _same(t, u)
                if _overlap(t, u) and not in_place:
                    raise ValueError("%s overlaps %s" % (n, m))
        b.status = self._status(status)
        self.rows, self.hidden = rows, hidden
        self.out, self.scales, self.residual_out = out, scales, residual_out
        self._own([out, scales, residual_out, self.status], [x, weight, residual])
        self.batch = b
        self._args = (C.byref(b),)
        self._fn, self._name = self.lib.mantleCudaNormRows, "mantleCudaNormRows"
        o = NormOutputs()
        o.out, o.scales, o.residual_out, o.status = out, scales, residual_out, self.status
        self._outputs = o

    def launch(self, stream=None):
        """Queues the norm on `stream` (default: the device's current stream).  Does not synchronise."""
        self._queue(stream)
        return self._outputs


def norm_rows(x, weight=None, stream=None, **kw):
    """One-shot form of NormPlan.  Its outputs carry `status`, which is not 0 where a wait inside the kernel ran out."""
    with torch.cuda.device(x.device), torch.cuda.stream(stream):  # outputs belong to the stream that writes them
        plan = NormPlan(x, weight, **kw)
        if stream is not None:  # made here, but what the caller gave may belong to another
            plan._tie(stream)
        return plan.launch()


class Adapters:
    """A table of low-rank adapters of one projection: row r's part is gain[i] * (x[r] a[i]^T) b[i]^T.

    a     [n, rank, hidden] bfloat16     b     [n, vocab, rank] bfloat16, both contiguous
    gain  optional [n] float32 (alpha / rank, usually)
    rank is a multiple of 8; adapters of smaller rank are padded with zeros.  Everything in a and b is finite; an
    adapter that is not spoils the rows that use it, and no others.
    b is copied into the layout the projection reads (on the current stream, once); a and gain are kept as they are:
    replace() writes into the caller's own tensors, and what the caller writes there is used from then on.
    """

    def __init__(self, a, b, gain=None):
        for t, name in ((a, "a"), (b, "b")):
            if not t.is_cuda or t.dim() != 3 or t.dtype != torch.bfloat16 or not t.is_contiguous():
                raise ValueError("%s must be a contiguous 3-D bfloat16 CUDA tensor" % name)
        if a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or a.device != b.device:
            raise ValueError("a is [n, rank, hidden] and b [n, vocab, rank], on one device")
        if gain is not None:
            _vector(gain, "gain", a.shape[0], (torch.float32,), a.device)
        self.lib = native.load()
        self.a, self.gain, self.device = a, gain, a.device
        self.n, self.rank, self.hidden, self.vocab = a.shape[0], a.shape[1], a.shape[2], b.shape[1]
        n = C.c_size_t(0)
        _check(self.lib, self.lib.mantleCudaAdapterPackBytes(1, self.vocab, self.rank, C.byref(n)), "mantleCudaAdapterPackBytes")
        self._one = n.value
        self.packed = torch.empty(self.n * self._one, dtype=torch.uint8, device=a.device)
        self._pack(b, 0, self.n)

    def _pack(self, b, first, n):
        with torch.cuda.device(self.device):
            rc = self.lib.mantleCudaAdapterPack(b.data_ptr(), n, self.vocab, self.rank, self.packed.data_ptr() + first * self._one,
                                                torch.cuda.current_stream().cuda_stream)
        _check(self.lib, rc, "mantleCudaAdapterPack")

    def replace(self, i, a, b, gain=None):
        """Puts another adapter, a [rank, hidden] and b [vocab, rank], in the place of adapter i, on the current
        stream of the table's device.  gain is a number, given exactly when the table has gains."""
        if not 0 <= i < self.n:
            raise ValueError("no adapter %d in a table of %d" % (i, self.n))
        if (gain is None) != (self.gain is None):
            raise ValueError("gain is needed exactly when the table has gains")
        for t, name, shape in ((a, "a", (self.rank, self.hidden)), (b, "b", (self.vocab, self.rank))):
            if t.device != self.device or tuple(t.shape) != shape or t.dtype != torch.bfloat16 or not t.is_contiguous():
                raise ValueError("%s must be a contiguous %s bfloat16 tensor on %s" % (name, shape, self.device))
        if b.data_ptr() % 16:
            raise ValueError("b must start on 16 bytes")
        if gain is not None and not (isinstance(gain, torch.Tensor) and gain.dim() == 0):
            gain = float(gain)  # what is no number is refused before anything is written
        self.a[i].copy_(a)
        if gain is not None:
            self.gain[i].fill_(gain)
        self._pack(b, i, 1)


class HeadPlan(_Plan):
    """logits[r] = hidden[r] weight^T, and the adapter's part of the row's request.

    hidden         [rows, hidden] bfloat16, or float8_e4m3fn with hidden_scales (rows values)
    weight         [vocab, hidden] of the same type, with weight_scales (vocab values) where it is float8_e4m3fn;
                   rows on 16 bytes
    base           instead of weight: [rows, vocab] of out_dtype, to which the adapters' part is added (out may be base)
    adapters, adapter_ids   a table and the [rows] int32 ids of the requests' adapters; an id outside the table: none
    out_dtype      float32 or bfloat16
    out, status    as in NormPlan
    """

    def __init__(self, hidden, weight=None, hidden_scales=None, weight_scales=None, adapters=None, adapter_ids=None,
                 base=None, out_dtype=None, out=None, status=None):
        dtype, b_stride = _rows(hidden, "hidden", (torch.bfloat16, torch.float8_e4m3fn))
        dev = hidden.device
        self._bind(dev)
        rows, k = hidden.shape
        b = native.HeadBatch()
        b.hidden_rows, b.hidden_stride, b.rows, b.hidden, b.dtype = hidden.data_ptr(), b_stride, rows, k, dtype
        if (weight is None) == (base is None):
            raise ValueError("one of weight and base is needed")
        eight = hidden.dtype == torch.float8_e4m3fn
        if out_dtype is None:
            out_dtype = torch.float32 if base is None else base.dtype
        if out_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("out_dtype must be float32 or bfloat16")

        def scales(t, n, name):
            if t is not None and t.dim() == 2 and t.shape[1] == 1 and t.is_contiguous():
                t = t.view(-1)
            if t is None:
                raise ValueError("%s are needed with float8_e4m3fn" % name)
            _vector(t, name, n, (torch.float32,), dev)
            return t.data_ptr()

        if weight is not None:
            _, b.weight_stride = _rows(weight, "weight", (hidden.dtype,), dev)
            if weight.shape[1] != k:
                raise ValueError("weight has %d columns, hidden %d" % (weight.shape[1], k))
            b.weight, vocab = weight.data_ptr(), weight.shape[0]
        else:
            _, b.base_stride = _rows(base, "base", (out_dtype,), dev)
            if base.shape[0] != rows:
                raise ValueError("base has %d rows, hidden %d" % (base.shape[0], rows))
            b.base, vocab = base.data_ptr(), base.shape[1]
        if eight:
            b.hidden_scales = scales(hidden_scales, rows, "hidden_scales")
            if weight is not None:
                b.weight_scales = scales(weight_scales, vocab, "weight_scales")
        if (hidden_scales is not None and not eight) or (weight_scales is not None and not (eight and weight is not None)):
            raise ValueError("scales go with float8_e4m3fn")
        if (adapters is None) != (adapter_ids is None):
            raise ValueError("adapters and adapter_ids go together")
        if adapters is not None:
            if adapters.device != dev or adapters.hidden != k or adapters.vocab != vocab:
                raise ValueError("the adapters are for another projection: [%d, %d] on %s"
                                 % (adapters.vocab, adapters.hidden, adapters.device))
            _vector(adapter_ids, "adapter_ids", rows, (torch.int32,), dev)
            b.adapter_a, b.adapter_b = adapters.a.data_ptr(), adapters.packed.data_ptr()
            b.adapter_gain = None if adapters.gain is None else adapters.gain.data_ptr()
            b.adapter_ids, b.n_adapters, b.rank = adapter_ids.data_ptr(), adapters.n, adapters.rank
        if out is None:
            out = torch.empty((rows, vocab), dtype=out_dtype, device=dev)
        b.out_dtype, b.out_stride = _rows(out, "out", (out_dtype,), dev, (rows, vocab))
        b.out, b.vocab = out.data_ptr(), vocab
        reads = [hidden, weight, base, hidden_scales, weight_scales, adapter_ids]
        reads += [adapters.a, adapters.packed, adapters.gain] if adapters is not None else []
        for t in reads:
            if t is not None and _overlap(out, t) and not (t is base and _same(out, base)):
                raise ValueError("out overlaps an input")
        b.status = self._status(status)
        n = C.c_size_t(0)
        with torch.cuda.device(dev):
            _check(self.lib, self.lib.mantleCudaHeadWorkspaceBytes(C.byref(b), C.byref(n)), "mantleCudaHeadWorkspaceBytes")
            c = C.c_int(0)
            _check(self.lib, self.lib.mantleCudaHeadLaunches(C.byref(b), C.byref(c)), "mantleCudaHeadLaunches")
        self.workspace_bytes = n.value
        self.workspace = torch.empty(n.value, dtype=torch.uint8, device=dev) if n.value else None
        self.kernels_per_launch = c.value
        self.rows, self.vocab, self.out = rows, vocab, out
        self._own([out, self.workspace, self.status], reads)
        self.batch = b
        self._args = (C.byref(b), None if self.workspace is None else self.workspace.data_ptr(), n.value)
        self._fn, self._name = self.lib.mantleCudaHeadRows, "mantleCudaHeadRows"

    def launch(self, stream=None):
        """Queues the projection on `stream` (default: the device's current stream) and returns the logits.
        Does not synchronise."""
        self._queue(stream)
        return self.out


def head_logits(hidden, weight=None, stream=None, **kw):
    """One-shot form of HeadPlan.  Pass `status` to learn of a wait inside the kernel that ran out."""
    with torch.cuda.device(hidden.device), torch.cuda.stream(stream):
        plan = HeadPlan(hidden, weight, **kw)
        if stream is not None:
            plan._tie(stream)
        return plan.launch()
