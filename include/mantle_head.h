/*
 * C-ABI of what stands between a model's last layer and the sampler (sm_100a): the norm with the
 * residual's addition, the head projection, and the low-rank adapters that the requests of a batch
 * bring with them.  The output of mantleCudaHeadRows is the `logits` of a MantleSampleBatch.
 *
 * Conventions are those of mantle_cuda_sampler.h: a cudaError_t as int, cudaErrorInvalidValue for
 * bad arguments before anything is launched (mantleCudaSamplerLastError() says which), work queued on
 * `stream`, no allocation, no synchronisation, every buffer the caller's, the current device the one
 * that owns the buffers.  Both calls may be captured into a CUDA graph.
 */
#ifndef MANTLE_HEAD_H
#define MANTLE_HEAD_H

#include <stddef.h>
#include <stdint.h>

#include "mantle_cuda_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* In addition to MANTLE_DTYPE_F32 and MANTLE_DTYPE_BF16: 8 bits, 4 of exponent and 3 of mantissa,
 * largest value 448, no infinity; a float32 scale beside it says what one stands for. */
#define MANTLE_DTYPE_E4M3 2

/* Largest row the norm takes: a row lives in the registers of one CTA. */
#define MANTLE_NORM_MAX_HIDDEN 32768
/* The one group size with a scale for every group of columns. */
#define MANTLE_NORM_GROUP 128

/*
 * For every row r:
 *
 *     s = x[r] + residual[r]                                  (float32; s = x[r] without a residual)
 *     residual_out[r] = s                                     (rounded to x's type, where wanted)
 *     y = s * (1 / sqrt(mean(s * s) + eps)) * (weight + weight_offset)
 *     out[r] = y                                              (rounded once)
 *
 * or, where out_dtype is MANTLE_DTYPE_E4M3, with one scale for the row (scale_group 0) or one for every
 * MANTLE_NORM_GROUP columns (the last group may be shorter):
 *
 *     out_scale = max(max|y| / 448, 2^-126);   out = y / out_scale, rounded to 8 bits
 *
 * The norm is taken of the float32 sum, not of the rounded residual_out.  Sums are float32, so a row
 * whose squares pass float32's range gives zeros, and a NaN or an infinity in a row makes NaN of what it
 * reaches (in 8 bits: of its whole group, scale included).
 *
 *   x, residual, residual_out   [rows][*_stride] of `dtype` (float32 or bfloat16)
 *   weight       [hidden] of weight_dtype (float32 or bfloat16); NULL: ones (weight_offset still added)
 *   out          [rows][out_stride] of out_dtype: dtype itself, or MANTLE_DTYPE_E4M3
 *   out_scale    [rows][scale_stride] float32, given exactly when out_dtype is MANTLE_DTYPE_E4M3;
 *                1 value a row for scale_group 0, ceil(hidden / scale_group) else
 *
 *   status       optional: as in MantleHeadBatch
 *
 * Strides are in elements.  residual_out may be x or residual itself, out may be x itself (same type and
 * stride); apart from that no output may overlap an input or another output.  hidden, strides and
 * addresses may be odd: rows that do not start on 16 bytes take element-wise loads.
 */
typedef struct MantleNormBatch {
    const void* x;
    const void* residual;
    void* residual_out;
    const void* weight;
    void* out;
    float* out_scale;
    int32_t* status;
    int64_t x_stride;
    int64_t residual_stride;
    int64_t residual_out_stride;
    int64_t out_stride;
    int64_t scale_stride;
    int32_t rows;
    int32_t hidden;
    int32_t dtype;
    int32_t weight_dtype;
    int32_t out_dtype;
    int32_t scale_group;
    float eps;
    float weight_offset;
} MantleNormBatch;

int mantleCudaNormRows(const MantleNormBatch* batch, mantleCudaStream_t stream);

/*
 * The head projection of a batch, and the low-rank adapters of its requests:
 *
 *     x^[r][k] = hidden_rows[r][k]              (bfloat16), or times hidden_scales[r] (e4m3)
 *     W^[v][k] = weight[v][k]                   (bfloat16), or times weight_scales[v] (e4m3)
 *     out[r][v] = sum_k x^[r][k] * W^[v][k]
 *               + gain[a] * sum_j b[a][v][j] * (sum_k x^[r][k] * a[a][j][k]),     a = adapter_ids[r]
 *
 * rounded once.  An id outside [0, n_adapters) means no adapter.  With `base` given and no weight, base[r][v]
 * takes the place of the projection: adapters beside a projection that something else computed; out may be
 * base itself (same type and stride).
 *
 *   hidden_rows  [rows][hidden_stride] of `dtype`: MANTLE_DTYPE_BF16 or MANTLE_DTYPE_E4M3
 *   hidden_scales, weight_scales   [rows] and [vocab] float32, given exactly when dtype is MANTLE_DTYPE_E4M3
 *                (weight_scales only with a weight)
 *   weight       [vocab][weight_stride] of `dtype`; starts on 16 bytes, weight_stride a multiple of 16 bytes
 *   base         [rows][base_stride] of out_dtype, instead of weight
 *   adapter_a    [n_adapters][rank][hidden] bfloat16, contiguous, on 16 bytes
 *   adapter_b    what mantleCudaAdapterPack made of [n_adapters][vocab][rank] bfloat16; on 128 bytes
 *   adapter_gain [n_adapters] float32, or NULL: ones
 *   adapter_ids  [rows] int32, on the device: may change between launches, and between replays of a graph
 *   rank         a multiple of 8, up to MANTLE_HEAD_MAX_RANK; adapters of smaller rank are padded with zeros
 *   out          [rows][out_stride], out_dtype MANTLE_DTYPE_F32 or MANTLE_DTYPE_BF16; columns past vocab are
 *                left as they are
 *   hidden       a multiple of 8 for bfloat16, of 16 for e4m3
 *   status       optional: one int32 that MANTLE_SAMPLE_STATUS_TIMEOUT is OR-ed into when a wait inside the
 *                kernel ran out (two seconds; the output is then not valid)
 *
 * Sums are float32; between the adapter's two products a value keeps its 24 bits (16 where the logits are bfloat16, of
 * 8 bits themselves).  The factors of an adapter have to be finite: an infinity or NaN in its `b` is packed as the largest
 * finite value (rows of several adapters share a step of the tensor cores, where an infinity times another row's zero
 * would be NaN), so that what is not finite spoils the rows that use the adapter, and no others.
 *
 * `workspace`: mantleCudaHeadWorkspaceBytes() bytes on 256 bytes, needed with adapters or where hidden_rows do
 * not start on 16 bytes each, else NULL is fine.  Its contents mean nothing between calls; two calls that may
 * overlap on the GPU (two streams, two graphs) need one each.
 */
#define MANTLE_HEAD_MAX_RANK 256
#define MANTLE_HEAD_MAX_ADAPTERS 4096

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
    int64_t hidden_stride;
    int64_t weight_stride;
    int64_t base_stride;
    int64_t out_stride;
    int32_t rows;
    int32_t vocab;
    int32_t hidden;
    int32_t dtype;
    int32_t out_dtype;
    int32_t n_adapters;
    int32_t rank;
    int32_t reserved;
} MantleHeadBatch;

/*
 * Lays `b` of n adapters, [n][vocab][rank] bfloat16, contiguous and on 16 bytes, out as mantleCudaHeadRows reads it,
 * once, when they are loaded.  An adapter's part of `packed` (on 128 bytes) is mantleCudaAdapterPackBytes(1, ...) bytes
 * long, and n of them stand one after the other, so that one can be replaced.
 */
int mantleCudaAdapterPackBytes(int n, int vocab, int rank, size_t* bytes);
int mantleCudaAdapterPack(const void* b, int n, int vocab, int rank, void* packed, mantleCudaStream_t stream);

int mantleCudaHeadRows(const MantleHeadBatch* batch, void* workspace, size_t workspace_bytes,
                       mantleCudaStream_t stream);

/* Bytes of workspace mantleCudaHeadRows needs for this batch (0 when none). */
int mantleCudaHeadWorkspaceBytes(const MantleHeadBatch* batch, size_t* bytes);

/* Kernels one mantleCudaHeadRows of this batch launches. */
int mantleCudaHeadLaunches(const MantleHeadBatch* batch, int* launches);

#ifdef __cplusplus
}
#endif

#endif /* MANTLE_HEAD_H */
