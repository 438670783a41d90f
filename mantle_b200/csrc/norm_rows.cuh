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

__device__ __forceinline__ void load8(const bf16_raw* p, float v[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
    v[4] = bf16_lo(u.z), v[5] = bf16_hi(u.z), v[6] = bf16_lo(u.w), v[7] = bf16_hi(u.w);
}
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

// T: float or bf16_raw.  QUANT: out in e4m3.  VPT: eights of columns a thread holds.  VEC: every row of every
// operand starts on 16 bytes and hidden is a multiple of 8; a thread's eights are then contiguous, else it
// holds single columns a row's threads apart.
template <typename T, bool QUANT, int VPT, bool VEC, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 128 : NORM_NT) norm_rows_kernel(const NormArgs a) {
    __shared__ float part[2][32];
    __shared__ uint32_t group_max[VEC || !QUANT ? 1 : MANTLE_NORM_MAX_HIDDEN / MANTLE_NORM_GROUP];
    const int tpr = WARP_ROW ? 32 : (int)blockDim.x;
    const int t = WARP_ROW ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
    const long long row = WARP_ROW ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP_ROW && row >= a.rows) return;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* res_out = a.residual_out ? static_cast<T*>(a.residual_out) + row * a.residual_out_stride : nullptr;

    float s[VPT][8];
    // column of element e of eight j
    auto col = [&](int j, int e) { return VEC ? (j * tpr + t) * 8 + e : (j * 8 + e) * tpr + t; };
    float sum = 0.0f;
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if (col(j, 0) < a.hidden) {
                load8(x + col(j, 0), s[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] = 0.0f;
            }
        }
        if (res) {
#pragma unroll
            for (int j = 0; j < VPT; j++) {
                if (col(j, 0) >= a.hidden) continue;
                float r[8];
                load8(res + col(j, 0), r);
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] += r[e];
            }
        }
        if (res_out) {
#pragma unroll
            for (int j = 0; j < VPT; j++)
                if (col(j, 0) < a.hidden) store8(res_out + col(j, 0), s[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = col(j, e);
                s[j][e] = 0.0f;
                if (c < a.hidden) {
                    s[j][e] = load1(x + c);
                    if (res) s[j][e] += load1(res + c);
                    if (res_out) store1(res_out + c, s[j][e]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; j++) {
#pragma unroll
        for (int e = 0; e < 8; e++) sum = __fmaf_rn(s[j][e], s[j][e], sum);
    }
    sum = row_reduce<WARP_ROW, false>(sum, part[0]);
    const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)a.hidden), a.eps));

    // y in the place of s
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = 1.0f;
        if (a.weight) {
            if constexpr (VEC) {
                if (col(j, 0) < a.hidden) {
                    if (a.weight_f32) load8(static_cast<const float*>(a.weight) + col(j, 0), w);
                    else load8(static_cast<const bf16_raw*>(a.weight) + col(j, 0), w);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int c = col(j, e);
                    if (c < a.hidden)
                        w[e] = a.weight_f32 ? load1(static_cast<const float*>(a.weight) + c)
                                            : load1(static_cast<const bf16_raw*>(a.weight) + c);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = (s[j][e] * rstd) * (w[e] + a.offset);
            s[j][e] = col(j, e) < a.hidden ? y : 0.0f;  // past the row: nothing that a maximum would see
        }
    }

    if constexpr (!QUANT) {
        T* out = static_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            if constexpr (VEC) {
                if (col(j, 0) < a.hidden) store8(out + col(j, 0), s[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (col(j, e) < a.hidden) store1(out + col(j, e), s[j][e]);
            }
        }
        return;
    }

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
        if (t == 0) scales[0] = scale;
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
            if (t % 16 == 0 && col(j, 0) < a.hidden) scales[col(j, 0) / MANTLE_NORM_GROUP] = scale;
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
                if ((threadIdx.x & 31) == 0 && col(j, e) < a.hidden) atomicMax(&group_max[col(j, e) / MANTLE_NORM_GROUP], m);
            }
        }
        __syncthreads();
        for (int g = threadIdx.x; g < groups; g += blockDim.x)
            scales[g] = max_nan(__fdiv_rn(__uint_as_float(group_max[g]), E4M3_MAX), E4M3_SCALE_MIN);
#pragma unroll
        for (int j = 0; j < VPT; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (col(j, e) >= a.hidden) continue;
                const float m = __uint_as_float(group_max[col(j, e) / MANTLE_NORM_GROUP]);
                s[j][e] *= __frcp_rn(max_nan(__fdiv_rn(m, E4M3_MAX), E4M3_SCALE_MIN));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; j++) {
        if constexpr (VEC) {
            if (col(j, 0) < a.hidden)
                *reinterpret_cast<uint2*>(out + col(j, 0)) =
                    make_uint2(pack_e4m3(s[j][0], s[j][1]) | pack_e4m3(s[j][2], s[j][3]) << 16,
                               pack_e4m3(s[j][4], s[j][5]) | pack_e4m3(s[j][6], s[j][7]) << 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (col(j, e) < a.hidden) out[col(j, e)] = (uint8_t)pack_e4m3(s[j][e], 0.0f);
        }
    }
}

template <typename T, bool QUANT, int VPT, bool VEC>
int launch_norm_vpt(const NormArgs& a, int threads, cudaStream_t stream) {
    norm_rows_kernel<T, QUANT, VPT, VEC, false><<<a.rows, threads, 0, stream>>>(a);
    return (int)cudaGetLastError();
}

template <typename T, bool QUANT, bool VEC>
int launch_norm_as(const NormArgs& a, cudaStream_t stream) {
    const int eights = (a.hidden + 7) / 8;
    // rows of a warp go four to a CTA; not so where element-wise rows need the CTA's group maxima
    if (eights <= 32 && (VEC || !QUANT)) {
        norm_rows_kernel<T, QUANT, 1, VEC, true><<<(a.rows + 3) / 4, 128, 0, stream>>>(a);
        return (int)cudaGetLastError();
    }
    // Few rows: as few eights a thread as 512 threads allow, the shortest path through the kernel.  Many rows: up to
    // four, more bytes in flight for the same threads.
    int vpt = 1;
    while (eights > vpt * NORM_NT || (vpt < 4 && a.rows > 2 * device_sms() && eights >= vpt * 128)) vpt *= 2;
    const int threads = ((eights + vpt - 1) / vpt + 31) / 32 * 32;
    if (vpt == 1) return launch_norm_vpt<T, QUANT, 1, VEC>(a, threads, stream);
    if (vpt == 2) return launch_norm_vpt<T, QUANT, 2, VEC>(a, threads, stream);
    if (vpt == 4) return launch_norm_vpt<T, QUANT, 4, VEC>(a, threads, stream);
    return launch_norm_vpt<T, QUANT, 8, VEC>(a, threads, stream);
}

template <typename T>
int launch_norm(const NormArgs& a, bool quant, bool vec, cudaStream_t stream) {
    if (quant) return vec ? launch_norm_as<T, true, true>(a, stream) : launch_norm_as<T, true, false>(a, stream);
    return vec ? launch_norm_as<T, false, true>(a, stream) : launch_norm_as<T, false, false>(a, stream);
}

}  // namespace
