// What stands between a model's last layer and the sampler: the norm with the residual's addition
// (norm_rows.cuh) and the head projection with the adapters of a batch's requests (head_prepare.cuh,
// head_rows.cuh).  The C-ABI of include/mantle_head.h.

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "../../include/mantle_head.h"
#include "device_info.cuh"
#include "mbarrier.cuh"
#include "sampler_internal.h"

namespace {

typedef uint16_t bf16_raw;  // a bfloat16's bits

int device_sms() { return device_info().sms; }

}  // namespace

#include "norm_rows.cuh"
#include "head_prepare.cuh"
#include "head_rows.cuh"

namespace {

constexpr int kInvalid = (int)cudaErrorInvalidValue;
constexpr int kMaxHeadHidden = 65536;
constexpr int kMaxHeadRows = 1 << 20;
// Up to how many rows a CTA works alone.  64 rows of bfloat16, 151 936 x 1024: 65 us alone, 70 as pairs; 128 rows of e4m3,
// 128 256 x 4096: 110 alone, 106 as pairs; 256 rows of the same: 154 and 141.
constexpr int ALONE_ROWS = 64;

// The packed B of an adapter covers whole tiles of a pair.
int padded_vocab(int vocab) { return (vocab + 2 * VT - 1) / (2 * VT) * (2 * VT); }

int refuse(const char* why) {
    mantle_internal_set_last_error(why);
    return kInvalid;
}

bool on(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

size_t size_of(int dtype) { return dtype == MANTLE_DTYPE_F32 ? 4 : dtype == MANTLE_DTYPE_BF16 ? 2 : 1; }

// nullptr: the batch is in order
const char* norm_fault(const MantleNormBatch* b) {
    if (!b) return "norm: no batch";
    if (!b->x || !b->out) return "norm: x and out are needed";
    if (b->rows <= 0) return "norm: rows must be positive";
    if (b->hidden <= 0 || b->hidden > MANTLE_NORM_MAX_HIDDEN) return "norm: hidden must be 1 to MANTLE_NORM_MAX_HIDDEN";
    if (b->dtype != MANTLE_DTYPE_F32 && b->dtype != MANTLE_DTYPE_BF16) return "norm: dtype must be float32 or bfloat16";
    if (b->weight && b->weight_dtype != MANTLE_DTYPE_F32 && b->weight_dtype != MANTLE_DTYPE_BF16)
        return "norm: weight_dtype must be float32 or bfloat16";
    const bool quant = b->out_dtype == MANTLE_DTYPE_E4M3;
    if (!quant && b->out_dtype != b->dtype) return "norm: out_dtype must be dtype or e4m3";
    if (quant != (b->out_scale != nullptr)) return "norm: out_scale goes with an e4m3 output, and only with one";
    if (b->scale_group != 0 && (!quant || b->scale_group != MANTLE_NORM_GROUP))
        return "norm: scale_group must be 0, or MANTLE_NORM_GROUP with an e4m3 output";
    if (b->residual_out && !b->residual) return "norm: residual_out without residual";
    if (b->x_stride < b->hidden || b->out_stride < b->hidden || (b->residual && b->residual_stride < b->hidden) ||
        (b->residual_out && b->residual_out_stride < b->hidden))
        return "norm: a stride is smaller than hidden";
    const int groups = b->scale_group ? (b->hidden + b->scale_group - 1) / b->scale_group : 1;
    if (quant && b->scale_stride < groups) return "norm: scale_stride is smaller than the number of scales of a row";
    if (!(b->eps >= 0.0f) || std::isinf(b->eps) || !std::isfinite(b->weight_offset))
        return "norm: eps must be finite and not negative, weight_offset finite";
    const size_t e = size_of(b->dtype);
    if (!on(b->x, e) || !on(b->residual, e) || !on(b->residual_out, e) || !on(b->out, size_of(b->out_dtype)) ||
        !on(b->out_scale, 4) || !on(b->status, 4) || (b->weight && !on(b->weight, size_of(b->weight_dtype))))
        return "norm: an address is not a multiple of its element size";
    return nullptr;
}

const char* head_fault(const MantleHeadBatch* b) {
    if (!b) return "head: no batch";
    if (!b->hidden_rows || !b->out) return "head: hidden_rows and out are needed";
    if (b->rows <= 0 || b->rows > kMaxHeadRows) return "head: rows must be 1 to 1048576";
    if (b->vocab <= 0 || b->vocab > MANTLE_SAMPLE_MAX_VOCAB) return "head: vocab must be 1 to MANTLE_SAMPLE_MAX_VOCAB";
    if (b->dtype != MANTLE_DTYPE_BF16 && b->dtype != MANTLE_DTYPE_E4M3) return "head: dtype must be bfloat16 or e4m3";
    if (b->out_dtype != MANTLE_DTYPE_F32 && b->out_dtype != MANTLE_DTYPE_BF16)
        return "head: out_dtype must be float32 or bfloat16";
    const bool eight = b->dtype == MANTLE_DTYPE_E4M3;
    const int64_t e = (int64_t)size_of(b->dtype);
    if (b->hidden <= 0 || b->hidden > kMaxHeadHidden || b->hidden * e % 16)
        return "head: hidden must be 1 to 65536, a multiple of 8 (bfloat16) or 16 (e4m3)";
    if (b->reserved) return "head: reserved must be 0";
    if ((b->weight != nullptr) == (b->base != nullptr)) return "head: one of weight and base is needed";
    if (eight != (b->hidden_scales != nullptr)) return "head: hidden_scales go with e4m3, and only with it";
    if ((eight && b->weight) != (b->weight_scales != nullptr)) return "head: weight_scales go with an e4m3 weight, and only with one";
    if (b->hidden_stride < b->hidden || b->out_stride < b->vocab || (b->weight && b->weight_stride < b->hidden) ||
        (b->base && b->base_stride < b->vocab))
        return "head: a stride is smaller than a row";
    if (b->weight && (!on(b->weight, 16) || b->weight_stride * e % 16))
        return "head: weight and its rows must start on 16 bytes";
    if (b->weight_stride > ((int64_t)1 << 36) || b->hidden_stride > ((int64_t)1 << 36)) return "head: a stride is too large";
    const size_t o = size_of(b->out_dtype);
    if (!on(b->hidden_rows, (size_t)e) || !on(b->out, o) || !on(b->base, o) || !on(b->hidden_scales, 4) ||
        !on(b->weight_scales, 4) || !on(b->status, 4) || !on(b->adapter_ids, 4) || !on(b->adapter_gain, 4))
        return "head: an address is not a multiple of its element size";
    if (b->n_adapters < 0 || b->n_adapters > MANTLE_HEAD_MAX_ADAPTERS)
        return "head: n_adapters must be 0 to MANTLE_HEAD_MAX_ADAPTERS";
    if (b->n_adapters) {
        if (!b->adapter_a || !b->adapter_b || !b->adapter_ids) return "head: adapters need adapter_a, adapter_b and adapter_ids";
        if (b->rank <= 0 || b->rank > MANTLE_HEAD_MAX_RANK || b->rank % 8)
            return "head: rank must be a multiple of 8, up to MANTLE_HEAD_MAX_RANK";
        if (!on(b->adapter_a, 16) || !on(b->adapter_b, 128)) return "head: adapter_a must start on 16 bytes, adapter_b on 128";
    } else if (b->base) {
        return "head: base without adapters";
    }
    return nullptr;
}

// Everything about a batch that follows from its sizes: the tiling, what runs, and where in the workspace things lie.
struct HeadLayout {
    bool eight, adapters;
    bool sorted;  // rows in the order of their adapters
    bool copied;  // x is read from the workspace's copy
    bool pair;    // two CTAs to a tile
    int tile_cols, row_tiles, v_tiles, w_steps, chunks, slot_bound, box_bound, u_rows, parts;
    int stages, stage_bytes, grid;
    size_t smem;
    size_t perm, slots, boxes, tile_first, n_boxes, u, xs, total;
};

HeadLayout head_layout(const MantleHeadBatch* b) {
    HeadLayout l = {};
    const size_t e = size_of(b->dtype);
    l.eight = b->dtype == MANTLE_DTYPE_E4M3;
    l.adapters = b->n_adapters > 0;
    const bool aligned = on(b->hidden_rows, 16) && b->hidden_stride * (int64_t)e % 16 == 0;
    const bool weight = b->weight != nullptr;
    l.pair = b->rows > ALONE_ROWS;
    const int ctas = l.pair ? 2 : 1, step = 16 * ctas;
    l.row_tiles = (b->rows + MAX_COLS - 1) / MAX_COLS;
    l.tile_cols = ((b->rows + l.row_tiles - 1) / l.row_tiles + step - 1) / step * step;
    l.row_tiles = (b->rows + l.tile_cols - 1) / l.tile_cols;
    l.v_tiles = (b->vocab + VT * ctas - 1) / (VT * ctas);
    l.w_steps = weight ? (int)((b->hidden * e + STEP_BYTES - 1) / STEP_BYTES) : 0;
    const long long work = l.row_tiles == 1 ? (b->vocab + UNIT * ctas - 1) / (UNIT * ctas) : (long long)l.v_tiles * l.row_tiles;
    l.grid = (int)std::min<long long>(device_info().sms / ctas, work) * ctas;
    // 128 rows of e4m3, 128 256 x 4096, 32 adapters: 143 us in place, 154 sorted; up to 256 rows, where windows of whole tiles
    // cost a step 256 cycles, the two were even
    l.sorted = l.adapters && b->rows > HERE_ROWS;
    l.copied = weight && (l.sorted || !aligned);  // beside a projection x is only read by the shrink kernels
    const bool own_round = l.adapters && (l.eight || !weight);
    const size_t fixed = 1024 + sizeof(HeadCtl) + (own_round ? ZERO_BYTES : 0);
    l.stage_bytes = A_BYTES + l.tile_cols / ctas * STEP_BYTES;
    l.stages = (int)std::min<size_t>(MAX_STAGES, ((size_t)232448 - fixed) / (size_t)l.stage_bytes);
    l.smem = fixed + (size_t)l.stages * (size_t)l.stage_bytes;

    auto take = [&](size_t bytes) {
        const size_t at = l.total;
        l.total += (bytes + 255) & ~(size_t)255;
        return at;
    };
    if (l.adapters) {
        l.chunks = (b->rank + U_RANKS - 1) / U_RANKS;
        l.parts = u_parts(b->out_dtype == MANTLE_DTYPE_BF16);
        l.slot_bound = std::min(b->rows, b->n_adapters);
        if (l.sorted) {
            // a piece per adapter in use and one per tile's end; each box holds a row at least, and a piece of n rows
            // touches at most n / WINDOW + 2 boxes
            l.slot_bound = std::min(b->rows, l.slot_bound + l.row_tiles);
            l.box_bound = std::min(b->rows, b->rows / WINDOW + 2 * l.slot_bound);
            l.perm = take((size_t)b->rows * 4);
            l.boxes = take((size_t)l.box_bound * sizeof(HeadBox));
            l.n_boxes = take(4);
        }
        l.u_rows = l.sorted ? l.box_bound * WINDOW : l.slot_bound * l.tile_cols;
        l.slots = take((size_t)l.slot_bound * sizeof(HeadSlot));
        l.tile_first = take((size_t)(l.row_tiles + 1) * 4);
        l.u = take((size_t)l.chunks * (size_t)l.u_rows * u_bytes(l.parts));
    }
    if (l.copied) l.xs = take((size_t)b->rows * (size_t)b->hidden * e);
    return l;
}

// cuTensorMapEncodeTiled, asked from the driver: the library does not link libcuda.
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::atomic<EncodeTiled> g_encode;

EncodeTiled encode_fn() {
    EncodeTiled f = g_encode.load(std::memory_order_acquire);
    if (f) return f;
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
        return nullptr;
    f = reinterpret_cast<EncodeTiled>(p);
    g_encode.store(f, std::memory_order_release);
    return f;
}

// A thread that has made no call of the runtime yet has no current context, and the driver's own calls want one.  (Where one
// is current, the runtime's or the caller's, it is left alone.)
bool bind_context() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

// Tiles of `box` from a [d2][d1][d0] array with row strides in bytes; what lies outside reads as zero.
bool encode(CUtensorMap* m, const void* p, bool eight, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
    const EncodeTiled f = encode_fn();
    const cuuint32_t steps[3] = {1, 1, 1};
    auto call = [&] {
        return f(m, eight ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(p),
                 dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    if (!f) return false;
    CUresult r = call();
    if ((r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) && bind_context()) r = call();
    return r == CUDA_SUCCESS;
}
bool encode_rows(CUtensorMap* m, const void* p, bool eight, long long rows, long long cols, long long stride_bytes, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)(STEP_BYTES / (eight ? 1 : 2)), (cuuint32_t)box_rows};
    return encode(m, p, eight, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Plain 128-byte rows (packed B, u): [d2][d1] of them, `box_rows` a copy.
bool encode_plain(CUtensorMap* m, const void* p, long long d1, long long d2, int box_rows) {
    const cuuint64_t dims[3] = {64, (cuuint64_t)d1, (cuuint64_t)d2}, strides[2] = {128, 128 * (cuuint64_t)d1};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    return encode(m, p, false, d2 ? 3 : 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <class... Args>
int launch(void (*kern)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t stream, bool pair, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    // every kernel here waits for what is in front of it by itself (griddepcontrol.wait), after its own set-up
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    if (pair) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = 2;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    return (int)cudaLaunchKernelEx(&cfg, kern, args...);
}

template <bool E4M3, bool OUT16, int GROUPS>
int launch_head_as(const HeadArgs& a, const HeadMaps& maps, const HeadLayout& l, cudaStream_t stream) {
    static std::atomic<int> granted[kMaxDevices];
    const auto kern = head_rows_kernel<E4M3, OUT16, GROUPS>;
    const int rc = ensure_smem(kern, l.smem, granted);
    if (rc) return rc;
    return launch<HeadArgs, HeadMaps>(kern, dim3((unsigned)l.grid), HEAD_NT, l.smem, stream, l.pair, a, maps);
}

template <bool E4M3, bool OUT16>
int launch_head(const HeadArgs& a, const HeadMaps& maps, const HeadLayout& l, cudaStream_t stream) {
    if (l.tile_cols <= 32) return launch_head_as<E4M3, OUT16, 1>(a, maps, l, stream);
    if (l.tile_cols <= 64) return launch_head_as<E4M3, OUT16, 2>(a, maps, l, stream);
    if (l.tile_cols <= 128) return launch_head_as<E4M3, OUT16, 4>(a, maps, l, stream);
    return launch_head_as<E4M3, OUT16, 8>(a, maps, l, stream);
}

}  // namespace

const char* mantle_internal_norm_fault(const MantleNormBatch* b) { return norm_fault(b); }

extern "C" int mantleCudaNormRows(const MantleNormBatch* b, mantleCudaStream_t stream_) {
    const char* fault = norm_fault(b);
    if (fault) return refuse(fault);
    NormArgs a = {};
    a.x = b->x;
    a.residual = b->residual;
    a.residual_out = b->residual_out;
    a.weight = b->weight;
    a.out = b->out;
    a.scale = b->out_scale;
    a.x_stride = b->x_stride;
    a.residual_stride = b->residual_stride;
    a.residual_out_stride = b->residual_out_stride;
    a.out_stride = b->out_stride;
    a.scale_stride = b->scale_stride;
    a.rows = b->rows;
    a.hidden = b->hidden;
    a.group = b->scale_group;
    a.weight_f32 = b->weight_dtype == MANTLE_DTYPE_F32;
    a.eps = b->eps;
    a.offset = b->weight_offset;
    a.status = b->status;
    const bool quant = b->out_dtype == MANTLE_DTYPE_E4M3;
    const int64_t e = (int64_t)size_of(b->dtype);
    auto rows_on_16 = [&](const void* p, int64_t stride) { return !p || (on(p, 16) && stride * e % 16 == 0); };
    const bool vec = b->hidden % 8 == 0 && rows_on_16(b->x, b->x_stride) && rows_on_16(b->residual, b->residual_stride) &&
                     rows_on_16(b->residual_out, b->residual_out_stride) && on(b->weight, 16) &&
                     (quant ? on(b->out, 8) && b->out_stride % 8 == 0 : rows_on_16(b->out, b->out_stride));
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return b->dtype == MANTLE_DTYPE_F32 ? launch_norm<float>(a, quant, vec, stream) : launch_norm<bf16_raw>(a, quant, vec, stream);
}

extern "C" int mantleCudaAdapterPackBytes(int n, int vocab, int rank, size_t* bytes) {
    if (!bytes || n <= 0 || n > MANTLE_HEAD_MAX_ADAPTERS || vocab <= 0 || vocab > MANTLE_SAMPLE_MAX_VOCAB || rank <= 0 ||
        rank > MANTLE_HEAD_MAX_RANK || rank % 8)
        return refuse("adapter pack: n, vocab or rank is out of range");
    *bytes = (size_t)n * ((rank + U_RANKS - 1) / U_RANKS) * (size_t)padded_vocab(vocab) * U_RANKS * 2;
    return 0;
}

extern "C" int mantleCudaAdapterPack(const void* b, int n, int vocab, int rank, void* packed, mantleCudaStream_t stream_) {
    size_t bytes = 0;
    const int rc = mantleCudaAdapterPackBytes(n, vocab, rank, &bytes);
    if (rc) return rc;
    if (!b || !packed || !on(b, 16) || !on(packed, 128))
        return refuse("adapter pack: b must start on 16 bytes, packed on 128");
    const int grid = (int)std::min<size_t>((bytes / 16 + 255) / 256, (size_t)device_info().sms * 16);
    adapter_pack_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream_)>>>(
        static_cast<const bf16_raw*>(b), n, vocab, rank, padded_vocab(vocab), static_cast<bf16_raw*>(packed));
    return (int)cudaGetLastError();
}

extern "C" int mantleCudaHeadWorkspaceBytes(const MantleHeadBatch* b, size_t* bytes) {
    const char* fault = bytes ? head_fault(b) : "head: no place for the size";
    if (fault) return refuse(fault);
    *bytes = head_layout(b).total;
    return 0;
}

extern "C" int mantleCudaHeadLaunches(const MantleHeadBatch* b, int* launches) {
    const char* fault = launches ? head_fault(b) : "head: no place for the count";
    if (fault) return refuse(fault);
    const HeadLayout l = head_layout(b);
    *launches = 1 + (l.adapters || l.copied ? 1 : 0) + (l.sorted ? 1 : 0);
    return 0;
}

extern "C" int mantleCudaHeadRows(const MantleHeadBatch* b, void* workspace, size_t workspace_bytes,
                                  mantleCudaStream_t stream_) {
    const char* fault = head_fault(b);
    if (fault) return refuse(fault);
    const HeadLayout l = head_layout(b);
    if (l.total && (!workspace || workspace_bytes < l.total || !on(workspace, 256)))
        return refuse("head: the workspace is missing, too small or not on 256 bytes");
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    char* ws = static_cast<char*>(workspace);
    const int64_t e = (int64_t)size_of(b->dtype);

    HeadArgs a = {};
    a.rows = b->rows;
    a.vocab = b->vocab;
    a.w_steps = l.w_steps;
    a.tile_cols = l.tile_cols;
    a.row_tiles = l.row_tiles;
    a.v_tiles = l.v_tiles;
    a.front_is_ours = l.adapters || l.copied;
    a.slots_on = l.adapters;
    a.sorted = l.sorted;
    a.copied = l.copied;
    a.chunks = l.chunks;
    a.u_rows = l.u_rows;
    a.u_box = l.sorted ? WINDOW / 2 : l.tile_cols / (l.pair ? 2 : 1);
    const int padded = padded_vocab(b->vocab);
    a.b_rows = padded / 4;
    a.stages = l.stages;
    a.stage_bytes = l.stage_bytes;
    a.pack_bytes = B_BYTES + l.tile_cols / (l.pair ? 2 : 1) * u_bytes(l.parts);
    a.pack = l.stage_bytes / a.pack_bytes;
    a.x_scales = b->hidden_scales;
    a.w_scales = b->weight_scales;
    a.base = b->base;
    a.out = b->out;
    a.base_stride = b->base_stride;
    a.out_stride = b->out_stride;
    a.status = b->status;

    HeadPrep p = {};
    p.x = b->hidden_rows;
    p.x_scales = b->hidden_scales;
    p.a = static_cast<const bf16_raw*>(b->adapter_a);
    p.gain = b->adapter_gain;
    p.ids = b->adapter_ids;
    p.x_stride = b->hidden_stride;
    p.rows = b->rows;
    p.hidden = b->hidden;
    p.e4m3 = l.eight;
    p.vec = on(b->hidden_rows, 16) && b->hidden_stride * e % 16 == 0;
    p.n_adapters = b->n_adapters;
    p.rank = b->rank;
    p.u_rows = l.u_rows;
    p.parts = l.parts;
    p.tile_cols = l.tile_cols;
    p.row_tiles = l.row_tiles;
    p.units = l.sorted ? l.box_bound : l.slot_bound;
    p.copy_ctas = l.copied ? std::min((b->rows + SHRINK_WARPS - 1) / SHRINK_WARPS, 2 * device_info().sms) : 0;
    if (l.adapters) {
        p.slots = reinterpret_cast<HeadSlot*>(ws + l.slots);
        p.tile_first = reinterpret_cast<int*>(ws + l.tile_first);
        p.u = reinterpret_cast<bf16_raw*>(ws + l.u);
        a.slots = p.slots;
        a.tile_first = p.tile_first;
    }
    if (l.sorted) {
        p.perm = reinterpret_cast<int*>(ws + l.perm);
        p.boxes = reinterpret_cast<HeadBox*>(ws + l.boxes);
        p.n_boxes = reinterpret_cast<int*>(ws + l.n_boxes);
        a.perm = p.perm;
    }
    if (l.copied) p.xs = ws + l.xs;

    HeadMaps maps;
    memset(&maps, 0, sizeof maps);
    bool ok = true;
    const int x_rows = l.tile_cols / (l.pair ? 2 : 1);
    if (b->weight) {
        for (int m = 0; m < 4; m++)
            ok = ok && encode_rows(&maps.w[m], b->weight, l.eight, b->vocab, b->hidden, b->weight_stride * e, VT >> m);
        ok = ok && (p.xs ? encode_rows(&maps.x, p.xs, l.eight, b->rows, b->hidden, b->hidden * e, x_rows)
                         : encode_rows(&maps.x, b->hidden_rows, l.eight, b->rows, b->hidden, b->hidden_stride * e, x_rows));
    }
    if (l.adapters) {
        const long long per_adapter = (long long)l.chunks * a.b_rows;
        for (int m = 0; m < 4; m++) ok = ok && encode_plain(&maps.b[m], b->adapter_b, per_adapter, b->n_adapters, (VT >> m) / 4);
        ok = ok && encode_plain(&maps.u, p.u, (long long)l.chunks * u_lines(l.u_rows, l.parts), 0, u_lines(a.u_box, l.parts));
    }
    if (!ok) return refuse("head: the driver refused a tensor map");

    int rc = 0;
    if (l.sorted) {
        rc = launch<HeadPrep>(head_sort_kernel, dim3(1), SORT_NT, ((size_t)b->n_adapters + 1) * 4, stream, false, p);
        if (rc) return rc;
    }
    if (l.adapters || l.copied) {
        const dim3 grid((unsigned)(p.units + p.copy_ctas), (unsigned)std::max(1, l.chunks),
                        (unsigned)(l.adapters && !l.sorted ? (b->rows + 31) / 32 : 1));
        rc = l.sorted ? launch<HeadPrep>(head_shrink_kernel, grid, SHRINK_NT, 0, stream, false, p)
                      : launch<HeadPrep>(head_shrink_here_kernel, grid, SHRINK_NT, 0, stream, false, p);
        if (rc) return rc;
    }
    if (b->out_dtype == MANTLE_DTYPE_BF16)
        return l.eight ? launch_head<true, true>(a, maps, l, stream) : launch_head<false, true>(a, maps, l, stream);
    return l.eight ? launch_head<true, false>(a, maps, l, stream) : launch_head<false, false>(a, maps, l, stream);
}
