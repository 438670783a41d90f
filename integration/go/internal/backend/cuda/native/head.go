//go:build cuda

// Package native: cgo binding of what stands in front of the device-side sampler
// (libmantle_cuda_sampler, mantle_head.h): the final norm, the head projection and the low-rank
// adapters of a batch's requests, and the decode step that runs them in a row.
//
// Conventions as in sampler.go: a file-local preamble that forward-declares the C symbols, Go
// functions that check their arguments and return samplerErr(code), which carries
// mantleCudaSamplerLastError().  Written without a Go toolchain at hand and not compiled; the same
// symbols are exercised from C++ and Python.
package native

/*
#include <stdint.h>
#include <stddef.h>
typedef void* cudaStream_t;

typedef struct MantleNormBatch {
	const void* x;
	const void* residual;
	void* residual_out;
	const void* weight;
	void* out;
	float* out_scale;
	int32_t* status;
	int64_t x_stride, residual_stride, residual_out_stride, out_stride, scale_stride;
	int32_t rows, hidden, dtype, weight_dtype, out_dtype, scale_group;
	float eps, weight_offset;
} MantleNormBatch;

typedef struct MantleHeadBatch {
	const void* hidden_rows;
	const void* weight;
	const void* base;
	const float* hidden_scales;
	const float* weight_scales;
	const void* adapter_a;
	const void* adapter_b;
	const float* adapter_gain;
	const int32_t* adapter_ids;
	void* out;
	int32_t* status;
	int64_t hidden_stride, weight_stride, base_stride, out_stride;
	int32_t rows, vocab, hidden, dtype, out_dtype, n_adapters, rank, reserved;
} MantleHeadBatch;

typedef struct MantleBatchSampler MantleBatchSampler;

extern int mantleCudaNormRows(const MantleNormBatch* b, cudaStream_t s);
extern int mantleCudaHeadRows(const MantleHeadBatch* b, void* ws, size_t wsBytes, cudaStream_t s);
extern int mantleCudaHeadWorkspaceBytes(const MantleHeadBatch* b, size_t* bytes);
extern int mantleCudaHeadLaunches(const MantleHeadBatch* b, int* launches);
extern int mantleCudaAdapterPackBytes(int n, int vocab, int rank, size_t* bytes);
extern int mantleCudaAdapterPack(const void* b, int n, int vocab, int rank, void* packed, cudaStream_t s);
extern int mantleBatchSamplerStepHidden(MantleBatchSampler* s, const MantleNormBatch* norm, const MantleHeadBatch* head,
	void* ws, size_t wsBytes, const double* uniforms, float logitScale, float logitSoftcap, cudaStream_t stream);

static int normRowsW(const MantleNormBatch* b, cudaStream_t s) { return mantleCudaNormRows(b, s); }
static int headRowsW(const MantleHeadBatch* b, void* ws, size_t n, cudaStream_t s) { return mantleCudaHeadRows(b, ws, n, s); }
static int headWorkspaceBytesW(const MantleHeadBatch* b, size_t* n) { return mantleCudaHeadWorkspaceBytes(b, n); }
static int headLaunchesW(const MantleHeadBatch* b, int* n) { return mantleCudaHeadLaunches(b, n); }
static int adapterPackBytesW(int n, int vocab, int rank, size_t* bytes) { return mantleCudaAdapterPackBytes(n, vocab, rank, bytes); }
static int adapterPackW(const void* b, int n, int vocab, int rank, void* packed, cudaStream_t s) {
	return mantleCudaAdapterPack(b, n, vocab, rank, packed, s);
}
static int batchStepHiddenW(MantleBatchSampler* s, const MantleNormBatch* norm, const MantleHeadBatch* head, void* ws, size_t n,
	const double* u, float scale, float cap, cudaStream_t st) {
	return mantleBatchSamplerStepHidden(s, norm, head, ws, n, u, scale, cap, st);
}
*/
import "C"

import (
	"fmt"
	"unsafe"
)

// Element types of mantle_head.h.
const (
	HeadF32  = 0
	HeadBF16 = 1
	HeadE4M3 = 2
)

// NormBatch describes mantleCudaNormRows: out = (x + residual) / rms * (weight + WeightOffset).
type NormBatch struct {
	X, Residual, ResidualOut, Weight, Out, OutScale, Status           DeviceBuffer
	XStride, ResidualStride, ResidualOutStride, OutStride, ScaleStride int64
	Rows, Hidden, DType, WeightDType, OutDType, ScaleGroup            int
	Eps, WeightOffset                                                 float32
}

func (b *NormBatch) c() C.MantleNormBatch {
	return C.MantleNormBatch{
		x: b.X.ptr, residual: b.Residual.ptr, residual_out: b.ResidualOut.ptr, weight: b.Weight.ptr, out: b.Out.ptr,
		out_scale: (*C.float)(b.OutScale.ptr), status: (*C.int32_t)(b.Status.ptr),
		x_stride: C.int64_t(b.XStride), residual_stride: C.int64_t(b.ResidualStride),
		residual_out_stride: C.int64_t(b.ResidualOutStride), out_stride: C.int64_t(b.OutStride),
		scale_stride: C.int64_t(b.ScaleStride), rows: C.int32_t(b.Rows), hidden: C.int32_t(b.Hidden),
		dtype: C.int32_t(b.DType), weight_dtype: C.int32_t(b.WeightDType), out_dtype: C.int32_t(b.OutDType),
		scale_group: C.int32_t(b.ScaleGroup), eps: C.float(b.Eps), weight_offset: C.float(b.WeightOffset),
	}
}

// NormRows queues the norm on the stream.
func NormRows(b *NormBatch, stream Stream) error {
	if b == nil || b.X.ptr == nil || b.Out.ptr == nil {
		return fmt.Errorf("norm: nil batch or buffer")
	}
	cb := b.c()
	return samplerErr(C.normRowsW(&cb, stream.ptr))
}

// HeadBatch describes mantleCudaHeadRows: the logits of a batch, and the low-rank adapters of its requests.
type HeadBatch struct {
	Hidden, Weight, Base, HiddenScales, WeightScales           DeviceBuffer
	AdapterA, AdapterB, AdapterGain, AdapterIDs, Out, Status    DeviceBuffer
	HiddenStride, WeightStride, BaseStride, OutStride           int64
	Rows, Vocab, HiddenSize, DType, OutDType, NAdapters, Rank   int
}

func (b *HeadBatch) c() C.MantleHeadBatch {
	return C.MantleHeadBatch{
		hidden_rows: b.Hidden.ptr, weight: b.Weight.ptr, base: b.Base.ptr,
		hidden_scales: (*C.float)(b.HiddenScales.ptr), weight_scales: (*C.float)(b.WeightScales.ptr),
		adapter_a: b.AdapterA.ptr, adapter_b: b.AdapterB.ptr, adapter_gain: (*C.float)(b.AdapterGain.ptr),
		adapter_ids: (*C.int32_t)(b.AdapterIDs.ptr), out: b.Out.ptr, status: (*C.int32_t)(b.Status.ptr),
		hidden_stride: C.int64_t(b.HiddenStride), weight_stride: C.int64_t(b.WeightStride),
		base_stride: C.int64_t(b.BaseStride), out_stride: C.int64_t(b.OutStride), rows: C.int32_t(b.Rows),
		vocab: C.int32_t(b.Vocab), hidden: C.int32_t(b.HiddenSize), dtype: C.int32_t(b.DType),
		out_dtype: C.int32_t(b.OutDType), n_adapters: C.int32_t(b.NAdapters), rank: C.int32_t(b.Rank),
	}
}

// HeadWorkspaceBytes says how much device workspace HeadRows needs for this batch (0 when none).
func HeadWorkspaceBytes(b *HeadBatch) (int64, error) {
	if b == nil {
		return 0, fmt.Errorf("head: nil batch")
	}
	cb := b.c()
	var n C.size_t
	if err := samplerErr(C.headWorkspaceBytesW(&cb, &n)); err != nil {
		return 0, err
	}
	return int64(n), nil
}

// HeadLaunches says how many kernels HeadRows launches for this batch.
func HeadLaunches(b *HeadBatch) (int, error) {
	if b == nil {
		return 0, fmt.Errorf("head: nil batch")
	}
	cb := b.c()
	var n C.int
	if err := samplerErr(C.headLaunchesW(&cb, &n)); err != nil {
		return 0, err
	}
	return int(n), nil
}

// HeadRows queues the projection and the adapters on the stream.
func HeadRows(b *HeadBatch, workspace DeviceBuffer, stream Stream) error {
	if b == nil || b.Hidden.ptr == nil || b.Out.ptr == nil {
		return fmt.Errorf("head: nil batch or buffer")
	}
	cb := b.c()
	return samplerErr(C.headRowsW(&cb, workspace.ptr, C.size_t(workspace.nbytes), stream.ptr))
}

// AdapterPackBytes is the size of n adapters' packed second factor.
func AdapterPackBytes(n, vocab, rank int) (int64, error) {
	var bytes C.size_t
	if err := samplerErr(C.adapterPackBytesW(C.int(n), C.int(vocab), C.int(rank), &bytes)); err != nil {
		return 0, err
	}
	return int64(bytes), nil
}

// AdapterPack lays the second factor of n adapters, [n][vocab][rank] bfloat16, out as HeadRows reads it.
func AdapterPack(b DeviceBuffer, n, vocab, rank int, packed DeviceBuffer, stream Stream) error {
	if b.ptr == nil || packed.ptr == nil {
		return fmt.Errorf("adapter pack: nil buffer")
	}
	return samplerErr(C.adapterPackW(b.ptr, C.int(n), C.int(vocab), C.int(rank), packed.ptr, stream.ptr))
}

// StepHidden queues norm (nil: none), head and one sampling step on the logits that the head writes.
func (s *BatchSampler) StepHidden(norm *NormBatch, head *HeadBatch, workspace DeviceBuffer, uniforms []float64, post HeadPost, stream Stream) error {
	if head == nil || len(uniforms) == 0 || len(uniforms) != s.rows {
		return fmt.Errorf("batch sampler step: nil head or %d uniforms for %d rows", len(uniforms), s.rows)
	}
	ch := head.c()
	var cn C.MantleNormBatch
	var np *C.MantleNormBatch
	if norm != nil {
		cn = norm.c()
		np = &cn
	}
	return samplerErr(C.batchStepHiddenW(s.p, np, &ch, workspace.ptr, C.size_t(workspace.nbytes),
		(*C.double)(unsafe.Pointer(&uniforms[0])), C.float(post.Scale), C.float(post.Softcap), stream.ptr))
}
