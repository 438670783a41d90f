// The root-mean-square norm with the residual's addition, rounded to the type of its input or to
// 8 bits with scales.  Part of head_kernels.cu.
//
//   s = x + residual;  y = s / sqrt(mean(s^2) + eps) * (weight + offset);  out = y, or y / scale in e4m3
//
// Bound by HBM (by launch latency for a few rows): every operand is read once and every output written
// once.  A row lives in the registers of the threads that own it -- a warp, or a CTA -- from its load
// to its last store, so the second use of s (the scaling) and the third (the 8 bits, which need the
// largest |y| first) cost no traffic.  s, the sum of squares and y are float32; the only roundings are
// the stores.
#pragma once

namespace {

struct NormArgs {
    const void* x;
    const void* residual;
    void* residual_out;
    const void* weight;
    void* out;
    float* scale;
    long long x_stride, residual_stride, residual_out_stride, out_stride, scale_stride;
    int rows, hidden, group;
    int weight_f32;
    float eps, offset;
    int* status;
};

constexpr int NORM_NT = 512;  // threads of a row at most; times 8 eights MANTLE_NORM_MAX_HIDDEN columns

constexpr float E4M3_MAX = 448.0f;
constexpr float E4M3_SCALE_MIN = 1.17549435e-38f;  // 2^-126: its reciprocal is finite

// max that keeps a NaN, as the definition's max does
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// two values to e4m3, the first in the low byte; past 448 saturates (a rounding error above the
// row's own maximum), NaN stays NaN
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

__device__ __forceinline__ void eight_of(const uint4& u, float v[8]) {
    v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
    v[4] = bf16_lo(u.z), v[5] = bf16_hi(u.z), v[6] = bf16_lo(u.w), v[7] = bf16_hi(u.w);
}
__device__ __forceinline__ void load8(const bf16_raw* p, float v[8]) { eight_of(*reinterpret_cast<const uint4*>(p), v); }
__device__ __forceinline__ void load8(const float* p, float v[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void store8(bf16_raw* p, const float v[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float v[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float load1(const bf16_raw* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(bf16_raw* p, float v) { *p = (bf16_raw)(pack_bf16(v, 0.0f) & 0xffffu); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }

// Sum or NaN-keeping maximum over the threads of a row: a warp, or the CTA (`part`: one float a warp).
template <bool WARP_ROW, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    if (WARP_ROW) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? part[lane] : 0.0f;  // of both: sums start at 0, no maximum of |y| is below it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    return v;
}

// What a thread holds of a row: VPT times eight columns.  VEC: every row of every operand starts on 16 bytes and hidden
// is a multiple of 8; the eights are then contiguous, else single columns, the row's threads apart.
template <int VPT, bool VEC>
struct NormCols {
    int t, tpr, hidden;
    __device__ __forceinline__ int at(int j, int e) const { return VEC ? (j * tpr + t) * 8 + e : (j * 8 + e) * tpr + t; }
    __device__ __forceinline__ bool has(int j, int e = 0) const { return at(j, e) < hidden; }
};

// The row's factors, asked for before the sum of squares is known so that they arrive meanwhile, as far as registers
// reach.  bfloat16 weights of whole eights stay packed until they are used.
template <int VPT, bool VEC>
struct NormWeight {
    static constexpr bool EARLY = VPT <= (VEC ? 4 : 2);
    uint4 raw[VEC && EARLY ? VPT : 1];
    float one[!VEC && EARLY ? VPT : 1][8];
    __device__ __forceinline__ void load(const NormArgs& a, const NormCols<VPT, VEC>& c) {
        if (!EARLY) return;
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if constexpr (!EARLY) {
            } else if constexpr (VEC) {
                if (a.weight && !a.weight_f32 && c.has(j)) raw[j] = *reinterpret_cast<const uint4*>(static_cast<const bf16_raw*>(a.weight) + c.at(j, 0));
            } else {
                singles(a, c, j, one[j]);
            }
        }
    }
    // eight single columns: the type is asked for once, so that the loads go out together
    template <typename P>
    __device__ __forceinline__ void singles_of(const P* p, const NormCols<VPT, VEC>& c, int j, float w[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = c.has(j, e) ? load1(p + c.at(j, e)) : 1.0f;
    }
    __device__ __forceinline__ void singles(const NormArgs& a, const NormCols<VPT, VEC>& c, int j, float w[8]) const {
        if (!a.weight) {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = 1.0f;
        } else if (a.weight_f32) {
            singles_of(static_cast<const float*>(a.weight), c, j, w);
        } else {
            singles_of(static_cast<const bf16_raw*>(a.weight), c, j, w);
        }
    }
    __device__ __forceinline__ void get(const NormArgs& a, const NormCols<VPT, VEC>& c, int j, float w[8]) const {
        if constexpr (VEC) {
            if (!a.weight || !c.has(j)) {
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = 1.0f;
            } else if (a.weight_f32) {
                load8(static_cast<const float*>(a.weight) + c.at(j, 0), w);
            } else if constexpr (EARLY) {
                eight_of(raw[j], w);
            } else {
                load8(static_cast<const bf16_raw*>(a.weight) + c.at(j, 0), w);
            }
        } else if constexpr (EARLY) {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = one[j][e];
        } else {
            singles(a, c, j, w);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] += a.offset;
    }
};
// The same held ready over many rows.
template <int VPT>
struct NormWeightHeld {
    float held[VPT][8];
    __device__ __forceinline__ void load(const NormArgs& a, const NormCols<VPT, true>& c) {
        NormWeight<VPT, true> weight;
        weight.load(a, c);
#pragma unroll
        for (int j = 0; j < VPT; j++) weight.get(a, c, j, held[j]);
    }
    __device__ __forceinline__ void get(const NormArgs&, const NormCols<VPT, true>&, int j, float w[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = held[j][e];
    }
};

// From the row's s, in registers, to its outputs: the sum of squares, y in the place of s, the scales, the stores.
// `after_sum` runs once every thread of the row holds its part of s.
template <typename T, bool QUANT, int VPT, bool VEC, bool WARP_ROW, class W, class F>
__device__ __forceinline__ void norm_finish(const NormArgs& a, long long row, const NormCols<VPT, VEC>& c, float s[VPT][8],
                                            const W& weight, float (*part)[32], uint32_t* group_max, F after_sum) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
#pragma unroll
        for (int e = 0; e < 8; e++) sum = __fmaf_rn(s[j][e], s[j][e], sum);
    }
    sum = row_reduce<WARP_ROW, false>(sum, part[0]);
    after_sum();
    const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)a.hidden), a.eps));
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        float w[8];
        weight.get(a, c, j, w);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // past the row s is 0 and w is finite: 0, or NaN where the whole row is
            s[j][e] = (s[j][e] * rstd) * w[e];
        }
    }

    if constexpr (!QUANT) {
        T* out = static_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if constexpr (VEC) {
                if (c.has(j)) store8(out + c.at(j, 0), s[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c.has(j, e)) store1(out + c.at(j, e), s[j][e]);
            }
        }
    } else {
        uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.out_stride;
        float* scales = a.scale + row * a.scale_stride;
        // Multiplying by the scale's reciprocal differs from dividing in the last float32 bit only: two rounding
        // errors of 2^-24 before one of 2^-4.
        if (a.group == 0) {
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < VPT; j++) {
#pragma unroll
                for (int e = 0; e < 8; e++) m = max_nan(m, fabsf(s[j][e]));
            }
            m = row_reduce<WARP_ROW, true>(m, part[1]);
            const float scale = max_nan(__fdiv_rn(m, E4M3_MAX), E4M3_SCALE_MIN), inv = __frcp_rn(scale);
            if (c.t == 0) scales[0] = scale;
#pragma unroll
            for (int j = 0; j < VPT; j++) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] *= inv;
            }
        } else if constexpr (VEC) {
            // sixteen neighbouring threads hold the 128 columns of a group
#pragma unroll
            for (int j = 0; j < VPT; j++) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) m = max_nan(m, fabsf(s[j][e]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float scale = max_nan(__fdiv_rn(m, E4M3_MAX), E4M3_SCALE_MIN), inv = __frcp_rn(scale);
                if (c.t % 16 == 0 && c.has(j)) scales[c.at(j, 0) / MANTLE_NORM_GROUP] = scale;
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] *= inv;
            }
        } else {
            // the bits of non-negative floats order like integers, NaN above all
            const int groups = (a.hidden + MANTLE_NORM_GROUP - 1) / MANTLE_NORM_GROUP;
            for (int g = threadIdx.x; g < groups; g += blockDim.x) group_max[g] = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; j++) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(s[j][e])));
                    // a warp's 32 columns start on a multiple of 32: one group
                    if ((threadIdx.x & 31) == 0 && c.has(j, e)) atomicMax(&group_max[c.at(j, e) / MANTLE_NORM_GROUP], m);
                }
            }
            __syncthreads();
            for (int g = threadIdx.x; g < groups; g += blockDim.x) {
                const float scale = max_nan(__fdiv_rn(__uint_as_float(group_max[g]), E4M3_MAX), E4M3_SCALE_MIN);
                scales[g] = scale;
                group_max[g] = __float_as_uint(__frcp_rn(scale));
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; j++) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c.has(j, e)) s[j][e] *= __uint_as_float(group_max[c.at(j, e) / MANTLE_NORM_GROUP]);
            }
        }
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if constexpr (VEC) {
                if (c.has(j))
                    *reinterpret_cast<uint2*>(out + c.at(j, 0)) =
                        make_uint2(pack_e4m3(s[j][0], s[j][1]) | pack_e4m3(s[j][2], s[j][3]) << 16,
                                   pack_e4m3(s[j][4], s[j][5]) | pack_e4m3(s[j][6], s[j][7]) << 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c.has(j, e)) out[c.at(j, e)] = (uint8_t)pack_e4m3(s[j][e], 0.0f);
            }
        }
    }
}

// One row for a warp or a CTA.
template <typename T, bool QUANT, int VPT, bool VEC, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 128 : NORM_NT) norm_rows_kernel(const NormArgs a) {
    __shared__ float part[2][32];
    __shared__ uint32_t group_max[VEC || !QUANT ? 1 : MANTLE_NORM_MAX_HIDDEN / MANTLE_NORM_GROUP];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long row = WARP_ROW ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP_ROW && row >= a.rows) return;
    const NormCols<VPT, VEC> c = {WARP_ROW ? (int)(threadIdx.x & 31) : (int)threadIdx.x, WARP_ROW ? 32 : (int)blockDim.x, a.hidden};
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* res_out = a.residual_out ? static_cast<T*>(a.residual_out) + row * a.residual_out_stride : nullptr;
    constexpr bool EARLY = VPT <= 4;
    float s[VPT][8], r[EARLY ? VPT : 1][8];
    // all loads before the first use, as far as registers reach
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        if constexpr (VEC) {
#pragma unroll
            for (int e = 0; e < 8; e++) s[j][e] = 0.0f;
            if (c.has(j)) load8(x + c.at(j, 0), s[j]);
            if (EARLY && res && c.has(j)) load8(res + c.at(j, 0), r[EARLY ? j : 0]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                s[j][e] = c.has(j, e) ? load1(x + c.at(j, e)) : 0.0f;
                if (EARLY && res) r[EARLY ? j : 0][e] = c.has(j, e) ? load1(res + c.at(j, e)) : 0.0f;
            }
        }
    }
    NormWeight<VPT, VEC> weight;
    weight.load(a, c);
    if (res) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if constexpr (VEC) {
                if (!c.has(j)) continue;
                if (!EARLY) load8(res + c.at(j, 0), r[0]);
            } else if (!EARLY) {
#pragma unroll
                for (int e = 0; e < 8; e++) r[0][e] = c.has(j, e) ? load1(res + c.at(j, e)) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) s[j][e] += r[EARLY ? j : 0][e];
            if (!res_out) continue;
            if constexpr (VEC) {
                store8(res_out + c.at(j, 0), s[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c.has(j, e)) store1(res_out + c.at(j, e), s[j][e]);
            }
        }
    }
    norm_finish<T, QUANT, VPT, VEC, WARP_ROW>(a, row, c, s, weight, part, group_max, [] {});
}

// Many long rows: CTAs that stay, each with a ring of rows of x and residual in shared memory that bulk copies fill ahead.
// In registers alone an SM holds no more bytes in flight than its threads have room for beside the row they work on,
// and none at all between a CTA's end and the next one's first load (16 384 x 8192 bfloat16 with residual, to 8 bits:
// 243 us so; here 148 at 1965 MHz, 99 % of the measured copy bandwidth, and 167 after a second or two, when the card's
// 1000 W hold the clock at 1730 MHz).  The row's factors stay in registers as they are used: with them packed, and a
// test for the row's end at every value, instruction issue was the bound (36 instructions a value, 170 us).
constexpr int NORM_RING = 2;          // (four deep measured the same)
constexpr int NORM_STREAM_NT = 512;  // threads at most

template <typename T, bool QUANT, int VPT>
__global__ void __launch_bounds__(VPT == 1 ? NORM_STREAM_NT / 2 : NORM_STREAM_NT, VPT == 1 ? 6 : VPT == 2 ? 2 : 1) norm_stream_kernel(const NormArgs a) {
    extern __shared__ __align__(128) char ring[];  // [NORM_RING][x, residual][row_bytes]
    __shared__ float part[2][2][32];               // a row's, and the next one's
    __shared__ uint64_t full[NORM_RING];
    const uint32_t row_bytes = (uint32_t)a.hidden * sizeof(T), operands = a.residual ? 2 : 1;
    const NormCols<VPT, true> c = {(int)threadIdx.x, (int)blockDim.x, a.hidden};
    if (threadIdx.x == 0) {
        for (int i = 0; i < NORM_RING; i++) mbar_init(&full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    auto fetch = [&](long long row, int slot) {  // one thread
        const uint32_t bar = smem_u32(&full[slot]), dst = smem_u32(ring) + (uint32_t)slot * operands * row_bytes;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(operands * row_bytes) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(dst), "l"(static_cast<const T*>(a.x) + row * a.x_stride), "r"(row_bytes), "r"(bar) : "memory");
        if (a.residual)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(dst + row_bytes), "l"(static_cast<const T*>(a.residual) + row * a.residual_stride), "r"(row_bytes), "r"(bar) : "memory");
    };
    NormWeightHeld<VPT> weight;
    weight.load(a, c);
    if (threadIdx.x == 0)
        for (int i = 0; i < NORM_RING; i++)
            if ((long long)blockIdx.x + (long long)i * gridDim.x < a.rows) fetch((long long)blockIdx.x + (long long)i * gridDim.x, i);
    int slot = 0, odd = 0;
    uint32_t turn = 0;  // parity of the slot's phase
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        // a copy that does not come in two seconds: the CTA says so and gives up together, when its other copies are in
        if (!__syncthreads_and(mbar_wait(&full[slot], turn))) {
            if (threadIdx.x == 0) {
                if (a.status) atomicOr(a.status, MANTLE_SAMPLE_STATUS_TIMEOUT);
                for (int i = 1; i < NORM_RING && row + (long long)i * gridDim.x < a.rows; i++)
                    mbar_wait(&full[(slot + i) % NORM_RING], turn ^ (slot + i >= NORM_RING), 100000000ull);
            }
            return;
        }
        const T* x = reinterpret_cast<const T*>(ring + (size_t)slot * operands * row_bytes);
        float s[VPT][8];
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if (c.has(j)) {
                load8(x + c.at(j, 0), s[j]);
                if (a.residual) {
                    float r[8];
                    load8(x + a.hidden + c.at(j, 0), r);
#pragma unroll
                    for (int e = 0; e < 8; e++) s[j][e] += r[e];
                    if (a.residual_out) store8(static_cast<T*>(a.residual_out) + row * a.residual_out_stride + c.at(j, 0), s[j]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] = 0.0f;
            }
        }
        norm_finish<T, QUANT, VPT, true, false>(a, row, c, s, weight, part[odd], nullptr, [&] {
            // behind the sum's barrier every thread has taken its part of the slot
            const long long ahead = row + (long long)NORM_RING * gridDim.x;
            if (threadIdx.x == 0 && ahead < a.rows) fetch(ahead, slot);
        });
        odd ^= 1;
        if (++slot == NORM_RING) slot = 0, turn ^= 1;
    }
}

// Every norm kernel waits for what is in front of it by itself, so that its launch overlaps that kernel's end.
int launch_norm_kernel(void (*kern)(NormArgs), const NormArgs& a, int grid, int threads, size_t smem, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T, bool QUANT, int VPT>
int launch_norm_stream(const NormArgs& a, int threads, int per_sm, size_t smem, cudaStream_t stream) {
    static std::atomic<int> granted[kMaxDevices];
    const auto kern = norm_stream_kernel<T, QUANT, VPT>;
    const int rc = ensure_smem(kern, smem, granted);
    if (rc) return rc;
    return launch_norm_kernel(kern, a, std::min(a.rows, device_sms() * per_sm), threads, smem, stream);
}

template <typename T, bool QUANT, bool VEC>
int launch_norm_as(const NormArgs& a, cudaStream_t stream) {
    const int eights = (a.hidden + 7) / 8;
    const bool many = a.rows > 2 * device_sms();
    // A warp a row, four to a CTA: short rows, and rows of up to 1024 columns where there are many.  (Not where
    // element-wise rows need the CTA's group maxima.)
    if (VEC || !QUANT) {
        const int grid = (a.rows - 1) / 4 + 1;  // (rows + 3 may pass 2^31)
        if (eights <= 32) return launch_norm_kernel(norm_rows_kernel<T, QUANT, 1, VEC, true>, a, grid, 128, 0, stream);
        if (many && eights <= 64) return launch_norm_kernel(norm_rows_kernel<T, QUANT, 2, VEC, true>, a, grid, 128, 0, stream);
        if (many && eights <= 128) return launch_norm_kernel(norm_rows_kernel<T, QUANT, 4, VEC, true>, a, grid, 128, 0, stream);
    }
    if constexpr (VEC) {
        // The ring: where a CTA gets several rows, and a row is worth a bulk copy.  One eight a thread up to 2048
        // columns, two up to 8192 (16 384 x 8192: 193 us with four and 256 threads, 170 with two and 512), four above.
        // Up to 2048 columns in bfloat16 alone, against a CTA a row: 32 768 x 1280 39 us and 49, 8192 x 1280 with
        // residual 16.4 and 18.8; not with a residual from some ten thousand rows on (32 768 x 1536: 76 and 70), nor in
        // float32 (32 768 x 1536: 78 and 61).
        const size_t row = (a.residual ? 2 : 1) * (size_t)a.hidden * sizeof(T), room = (size_t)device_info().per_sm;
        const int vpt = eights <= 256 ? 1 : eights <= 2 * NORM_STREAM_NT ? 2 : 4, threads = ((eights + vpt - 1) / vpt + 31) / 32 * 32;
        // as many CTAs as are resident: up to 42 registers a thread, 64 with two eights, 128 with four; 2 KB of an SM's
        // room are not theirs
        const int per_sm = (int)std::min<size_t>((size_t)((vpt == 1 ? 1536 : vpt == 2 ? 1024 : 512) / threads), room / (NORM_RING * row + 2048));
        const bool worth = vpt > 1 || (sizeof(T) == 2 && eights > 128 && (!a.residual || a.rows <= 16384));
        if (worth && eights <= 4 * NORM_STREAM_NT && per_sm >= 1 && a.rows >= 3ll * device_sms() * per_sm) {
            if constexpr (sizeof(T) == 2) {
                if (vpt == 1) return launch_norm_stream<T, QUANT, 1>(a, threads, per_sm, NORM_RING * row, stream);
            }
            if (vpt == 2) return launch_norm_stream<T, QUANT, 2>(a, threads, per_sm, NORM_RING * row, stream);
            return launch_norm_stream<T, QUANT, 4>(a, threads, per_sm, NORM_RING * row, stream);
        }
    }
    // A CTA a row.  Few rows: as few eights a thread as 512 threads allow, the shortest path through the kernel.  Many
    // rows: up to four, more bytes in flight for the same threads.  (2048 columns stand on the line: two for whole eights,
    // 32 768 rows with residual 91 us and 114, four for single columns, 4096 rows 15.5 and 17.7.)
    int vpt = 1;
    while (eights > vpt * NORM_NT || (vpt < 4 && many && eights >= vpt * 128 + VEC)) vpt *= 2;
    const int threads = ((eights + vpt - 1) / vpt + 31) / 32 * 32;
    if (vpt == 1) return launch_norm_kernel(norm_rows_kernel<T, QUANT, 1, VEC, false>, a, a.rows, threads, 0, stream);
    if (vpt == 2) return launch_norm_kernel(norm_rows_kernel<T, QUANT, 2, VEC, false>, a, a.rows, threads, 0, stream);
    if (vpt == 4) return launch_norm_kernel(norm_rows_kernel<T, QUANT, 4, VEC, false>, a, a.rows, threads, 0, stream);
    return launch_norm_kernel(norm_rows_kernel<T, QUANT, 8, VEC, false>, a, a.rows, threads, 0, stream);
}

template <typename T>
int launch_norm(const NormArgs& a, bool quant, bool vec, cudaStream_t stream) {
    if (quant) return vec ? launch_norm_as<T, true, true>(a, stream) : launch_norm_as<T, true, false>(a, stream);
    return vec ? launch_norm_as<T, false, true>(a, stream) : launch_norm_as<T, false, false>(a, stream);
}

}  // namespace
