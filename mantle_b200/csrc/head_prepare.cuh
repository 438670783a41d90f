// What the head projection needs to know about a batch's adapters, worked out on the device: which rows
// use which adapter, and each row's rank-long product with its adapter's first factor.
// Part of head_kernels.cu.
//
// The projection (head_rows.cuh) adds an adapter to a tile of rows as a few more steps of its matrix product:
//
//     D[v][row] += sum_j B[a][v][j] * u[row][j],     u[row][j] = gain[a] * sum_k x^[row][k] A[a][j][k]
//
// on a window of neighbouring columns of D, with zeros in u for the columns there that belong to rows of other
// adapters; a slot is one such step.  A row's result depends neither on where it stands in the tile nor on what
// stands beside it: a column of D only ever sees its own column of the operands, and adding zeros to it changes
// nothing.
//
// Two forms.  Up to HERE_ROWS rows, one kernel: rows stay where they are, and an adapter's window is the whole
// tile, zeros and all; the projection does not wait for this kernel before it reads x and W, and meets its results only
// when it comes to the adapters.  (It starts at once on the SMs that have no CTA of this kernel: the two do not fit on
// one SM together, 34 KB here beside a ring that fills the rest.)  More rows: head_sort_kernel puts the rows in an
// order in which those of one adapter stand together, and head_shrink_kernel copies x in that order, so that a window
// covers an adapter's own rows and little else.
#pragma once

namespace {

constexpr int WINDOW = 32;         // sorted: windows start and end on a multiple of 32 columns of their tile
constexpr int U_RANKS = 16;        // ranks of one step of the tensor cores: a chunk
// Bfloat16 that hold a value of u, side by side.  Three keep the 24 bits of its float32; two keep 16, which adds a
// 256th to what the rounding of bfloat16 logits takes.
__host__ __device__ constexpr int u_parts(bool out16) { return out16 ? 2 : 3; }
__host__ __device__ constexpr int u_bytes(int parts) { return parts * 2 * U_RANKS; }  // a row of u of one chunk
// That many rows of u, whole eights, in rows of 128 bytes, as tensor maps count them.
__host__ __device__ constexpr int u_lines(int rows, int parts) { return rows / 8 * (8 * u_bytes(parts) / 128); }
constexpr int HERE_ROWS = 128;
constexpr int SORT_NT = 1024;
constexpr int SHRINK_NT = 512;
constexpr int SHRINK_WARPS = SHRINK_NT / 32;

// One step's worth of columns: adapter `adapter` on columns [col, col + n) of its row tile, with the rows of u
// from u_row on.  16 bytes, read as one int4.
struct __align__(16) HeadSlot {
    int adapter, col, n, u_row;
};
// WINDOW rows of u: sorted places [place, place + WINDOW), of which [first, last) use the adapter.
struct __align__(16) HeadBox {
    int adapter, place, first, last;
};

struct HeadPrep {
    // in
    const void* x;
    const float* x_scales;
    const bf16_raw* a;
    const float* gain;
    const int32_t* ids;
    long long x_stride;  // elements
    int rows, hidden, e4m3, vec;  // vec: rows of x start on 16 bytes
    int n_adapters, rank;
    int u_rows, parts;   // rows of u of one chunk of ranks; see u_parts
    int tile_cols, row_tiles;
    int units, copy_ctas;  // CTAs of the shrink kernel: slots or boxes at most; and those that copy x
    // workspace
    int* perm;        // [rows] sorted place -> row
    HeadSlot* slots;
    HeadBox* boxes;
    int* tile_first;  // [row_tiles + 1] first slot of a tile
    int* n_boxes;     // [1]
    bf16_raw* u;      // [chunks][u_rows / 8][parts * 2][8][8], see u_at
    void* xs;         // [rows][hidden] contiguous, sorted
};

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Exclusive sum of `v` over the CTA's threads; *total gets the whole.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += w;
    }
    __syncthreads();  // warp_sums may still be read from the call before
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    int w = warp_sums[lane];  // SORT_NT / 32 = 32 of them
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += x;
    }
    *total = __shfl_sync(0xffffffffu, w, 31);
    const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
    return before + s - v;
}

// One CTA: counts the rows of every adapter, gives each adapter its run of places (rows without one come
// last), and cuts the runs into slots, at the ends of tiles, and boxes.  Shared memory: n_adapters + 1 counts.
__global__ void __launch_bounds__(SORT_NT) head_sort_kernel(const HeadPrep p) {
    extern __shared__ int bins[];  // [n_adapters + 1]: counts, then next free places, then ends of runs
    __shared__ int warp_sums[32];
    const int n = p.n_adapters, tid = threadIdx.x;
    pdl_wait();
    pdl_trigger();
    for (int b = tid; b <= n; b += SORT_NT) bins[b] = 0;
    __syncthreads();
    for (int r = tid; r < p.rows; r += SORT_NT) {
        const int id = p.ids[r];
        atomicAdd(&bins[id >= 0 && id < n ? id : n], 1);
    }
    __syncthreads();
    int carry = 0;
    for (int b0 = 0; b0 <= n; b0 += SORT_NT) {
        const int b = b0 + tid, v = b <= n ? bins[b] : 0;
        int total;
        const int at = carry + block_scan(v, warp_sums, &total);
        if (b <= n) bins[b] = at;
        carry += total;
    }
    __syncthreads();
    for (int r = tid; r < p.rows; r += SORT_NT) {
        const int id = p.ids[r];
        p.perm[atomicAdd(&bins[id >= 0 && id < n ? id : n], 1)] = r;
    }
    __syncthreads();  // bins[b] is now the end of run b, and its start the end of run b - 1

    int slot_carry = 0, box_carry = 0;
    for (int b0 = 0; b0 < n; b0 += SORT_NT) {
        const int b = b0 + tid;
        const int lo = b < n ? (b ? bins[b - 1] : 0) : 0, hi = b < n ? bins[b] : 0;
        auto cut = [&](int at) { return min(hi, (at / p.tile_cols + 1) * p.tile_cols); };  // end of the piece that starts at `at`
        int n_slots = 0, n_boxes = 0;
        for (int at = lo; at < hi;) {
            const int end = cut(at), tile0 = at / p.tile_cols * p.tile_cols;
            const int c0 = (at - tile0) / WINDOW, c1 = (end - tile0 + WINDOW - 1) / WINDOW;
            n_slots++;
            n_boxes += c1 - c0;
            at = end;
        }
        int slot_total, box_total;
        int slot = slot_carry + block_scan(n_slots, warp_sums, &slot_total);
        int box = box_carry + block_scan(n_boxes, warp_sums, &box_total);
        for (int at = lo; at < hi;) {
            const int end = cut(at), tile = at / p.tile_cols, tile0 = tile * p.tile_cols;
            const int c0 = (at - tile0) / WINDOW, c1 = (end - tile0 + WINDOW - 1) / WINDOW;
            HeadSlot s = {b, c0 * WINDOW, (c1 - c0) * WINDOW, box * WINDOW};
            p.slots[slot] = s;
            // the first slot of a tile is the one whose predecessor -- the place before it, if that has an adapter --
            // lies in another tile; rows with adapters are gapless from place 0 on
            if (at == tile0) p.tile_first[tile] = slot;
            for (int c = c0; c < c1; c++) {
                HeadBox x = {b, tile0 + c * WINDOW, at, end};
                p.boxes[box++] = x;
            }
            slot++;
            at = end;
        }
        slot_carry += slot_total;
        box_carry += box_total;
    }
    // tiles from the first place without an adapter on that no slot starts: empty
    __syncthreads();
    const int with = n ? bins[n - 1] : 0;
    const int last_tile = (with + p.tile_cols - 1) / p.tile_cols;
    for (int t = last_tile + tid; t <= p.row_tiles; t += SORT_NT) p.tile_first[t] = slot_carry;
    if (tid == 0) *p.n_boxes = box_carry;
}

__device__ __forceinline__ void mma_16x8x16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// two e4m3 (exact in f16, and from there in bfloat16) to two bfloat16
__device__ __forceinline__ uint32_t e4m3x2_to_bf16x2(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    float lo, hi;
    asm("{.reg .b16 l, u; mov.b32 {l, u}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, u;}" : "=f"(lo), "=f"(hi) : "r"(h));
    return pack_bf16(lo, hi);
}

// Eight neighbouring values of one row of x as four bfloat16 pairs.
__device__ __forceinline__ uint4 x_eight(const HeadPrep& p, const char* row, int k) {
    if (p.e4m3) {
        uint32_t w[2];
        if (p.vec) {
            const uint2 u = *reinterpret_cast<const uint2*>(row + k);
            w[0] = u.x, w[1] = u.y;
        } else {
            const uint8_t* q = reinterpret_cast<const uint8_t*>(row) + k;
#pragma unroll
            for (int i = 0; i < 2; i++) w[i] = q[4 * i] | q[4 * i + 1] << 8 | q[4 * i + 2] << 16 | (uint32_t)q[4 * i + 3] << 24;
        }
        return make_uint4(e4m3x2_to_bf16x2(w[0] & 0xffff), e4m3x2_to_bf16x2(w[0] >> 16), e4m3x2_to_bf16x2(w[1] & 0xffff),
                          e4m3x2_to_bf16x2(w[1] >> 16));
    }
    const bf16_raw* q = reinterpret_cast<const bf16_raw*>(row) + k;
    if (p.vec) return *reinterpret_cast<const uint4*>(q);
    return make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16,
                      q[6] | (uint32_t)q[7] << 16);
}

// The copy of x, in sorted order where there is one: one warp a row.
__device__ __forceinline__ void copy_rows(const HeadPrep& p, int first, int step) {
    const int lane = threadIdx.x & 31, esz = p.e4m3 ? 1 : 2;
    const long long bytes = (long long)p.hidden * esz;  // a multiple of 16
    for (int r = first; r < p.rows; r += step) {
        const int from = p.perm ? p.perm[r] : r;
        const char* src = static_cast<const char*>(p.x) + (long long)from * p.x_stride * esz;
        char* dst = static_cast<char*>(p.xs) + r * bytes;
        if (p.vec) {
            for (long long i = lane * 16; i < bytes; i += 512)
                *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(src + i);
        } else if (p.e4m3) {
            for (long long i = lane; i < bytes; i += 32) dst[i] = src[i];
        } else {
            for (long long i = lane * 2; i < bytes; i += 64)
                *reinterpret_cast<bf16_raw*>(dst + i) = *reinterpret_cast<const bf16_raw*>(src + i);
        }
    }
}

// One chunk of ranks (from j0) of 32 rows' products with one adapter's A: rows[i] is the row of x of place i, -1 none.
// The warps share out the columns of x and add their sums up in shared memory.  The order of the columns within
// a step is free in a dot product, so each lane takes eight neighbours of its row, one 16-byte load, as two
// steps' operands.  On return thread i * 16 + j holds place i, rank j0 + j.
typedef float ShrinkSums[SHRINK_WARPS][32][U_RANKS];
__device__ __forceinline__ float shrink32(const HeadPrep& p, int adapter, int j0, const int* rows, ShrinkSums& sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int esz = p.e4m3 ? 1 : 2;
    const char* row[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = rows[g + 8 * i];
        row[i] = r >= 0 ? static_cast<const char*>(p.x) + (long long)r * p.x_stride * esz : nullptr;
    }
    const bf16_raw* arow = p.a + ((long long)adapter * p.rank + j0 + g) * p.hidden;
    const bool both = j0 + 8 < p.rank;  // (the rank may end after eight)
    const int mine = rows[threadIdx.x >> 4];
    float factor = p.gain ? p.gain[adapter] : 1.0f;
    if (p.e4m3 && mine >= 0) factor *= p.x_scales[mine];
    float d[2][2][4] = {};
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll 4
    for (int k = warp * 32 + q * 8; k < p.hidden + q * 8; k += SHRINK_WARPS * 32) {  // the same count for a warp's lanes
        const bool in = k < p.hidden;
        uint4 x[4], w[2];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = in && row[i] ? x_eight(p, row[i], k) : none;
        w[0] = in ? *reinterpret_cast<const uint4*>(arow + k) : none;
        w[1] = in && both ? *reinterpret_cast<const uint4*>(arow + 8ll * p.hidden + k) : none;
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                mma_16x8x16(d[m][n], x[2 * m].x, x[2 * m + 1].x, x[2 * m].y, x[2 * m + 1].y, w[n].x, w[n].y);
                mma_16x8x16(d[m][n], x[2 * m].z, x[2 * m + 1].z, x[2 * m].w, x[2 * m + 1].w, w[n].z, w[n].w);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < 2; m++) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
            sums[warp][m * 16 + g][n * 8 + q * 2] = d[m][n][0], sums[warp][m * 16 + g][n * 8 + q * 2 + 1] = d[m][n][1];
            sums[warp][m * 16 + g + 8][n * 8 + q * 2] = d[m][n][2], sums[warp][m * 16 + g + 8][n * 8 + q * 2 + 1] = d[m][n][3];
        }
    }
    __syncthreads();
    const int i = threadIdx.x >> 4, j = threadIdx.x & 15;
    if (mine < 0) return 0.0f;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < SHRINK_WARPS; w++) v += sums[w][i][j];
    return v * factor;
}

// u lies in memory as the tensor cores read it from shared memory without swizzle: blocks of 8 rows by 8 values (16
// bytes a row), two for each part to a group of 8 rows -- leading parts of ranks 0-7 and 8-15 of the chunk, then the next --
// so that any run of rows is one contiguous copy.
__device__ __forceinline__ bf16_raw* u_at(const HeadPrep& p, int rank_at, int u_row) {
    return p.u + ((long long)(rank_at / U_RANKS) * p.u_rows + (u_row & ~7)) * (u_bytes(p.parts) / 2) +
           (rank_at % U_RANKS / 8) * 64 + (u_row & 7) * 8 + rank_at % 8;
}

// v in its parts, each the rounding of what those before it leave (an infinity or NaN stays in the leading part alone).
// In two, float32 logits of adapters on a base were off by 4.9e-7 of their size where float32 sums are by 1.3e-7; in
// three by 1.0e-7.
__device__ __forceinline__ void store_u(const HeadPrep& p, int rank_at, int u_row, float v) {
    bf16_raw* u = u_at(p, rank_at, u_row);
    for (int i = 0; i < p.parts; i++) {
        const uint32_t part = pack_bf16(v, 0.0f) & 0xffffu;
        u[128 * i] = (bf16_raw)part;
        v = (part & 0x7f80u) == 0x7f80u ? 0.0f : v - __uint_as_float(part << 16);
    }
}

// Sorted form.  CTAs [0, units) x [0, chunks): one chunk of ranks of one box.  CTAs from `units` on: the copy of x.
__global__ void __launch_bounds__(SHRINK_NT) head_shrink_kernel(const HeadPrep p) {
    __shared__ ShrinkSums sums;
    __shared__ int rows[WINDOW];
    pdl_wait();
    pdl_trigger();
    if ((int)blockIdx.x >= p.units) {
        if (blockIdx.y == 0)
            copy_rows(p, ((int)blockIdx.x - p.units) * SHRINK_WARPS + (int)(threadIdx.x >> 5), p.copy_ctas * SHRINK_WARPS);
        return;
    }
    if ((int)blockIdx.x >= *p.n_boxes) return;
    const HeadBox box = p.boxes[blockIdx.x];
    if (threadIdx.x < WINDOW) {
        const int at = box.place + (int)threadIdx.x;
        rows[threadIdx.x] = at >= box.first && at < box.last ? p.perm[at] : -1;
    }
    __syncthreads();
    const int j0 = blockIdx.y * U_RANKS;
    const float v = shrink32(p, box.adapter, j0, rows, sums);
    store_u(p, j0 + (int)(threadIdx.x & 15), (int)blockIdx.x * WINDOW + (int)(threadIdx.x >> 4), v);
}

// Form for up to HERE_ROWS rows.  CTAs [0, units) x [0, chunks) x [0, rows / 32): a chunk of ranks of up to 32 rows of one adapter -- the
// blockIdx.x-th of those in use, in the order of their first rows -- and zeros for the others.  CTAs from `units` on:
// the copy of x, where its rows do not start on 16 bytes.
__global__ void __launch_bounds__(SHRINK_NT) head_shrink_here_kernel(const HeadPrep p) {
    __shared__ ShrinkSums sums;
    __shared__ __align__(16) int ids[HERE_ROWS];
    __shared__ int mine[HERE_ROWS], first_of[HERE_ROWS];
    __shared__ int counts[2 * (HERE_ROWS / 32)];  // of its first HERE_ROWS threads' warps, twice
    pdl_wait();
    pdl_trigger();  // not before: the projection reads W and x as soon as it starts
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if ((int)blockIdx.x >= p.units) {
        if (blockIdx.y == 0 && blockIdx.z == 0)
            copy_rows(p, ((int)blockIdx.x - p.units) * SHRINK_WARPS + warp, p.copy_ctas * SHRINK_WARPS);
        return;
    }
    // the adapters in use: a row is its adapter's first if no row before it has the same
    if (tid < HERE_ROWS) {
        const int id = tid < p.rows ? p.ids[tid] : -1;
        ids[tid] = id >= 0 && id < p.n_adapters ? id : -1;
        mine[tid] = -1;
    }
    __syncthreads();
    if (tid < HERE_ROWS) {
        const int id = ids[tid];
        bool first = id >= 0;
#pragma unroll 4
        for (int r = 0; r < p.rows; r += 4) {  // (behind the last row: no adapter)
            const int4 v = *reinterpret_cast<const int4*>(ids + r);
            first = first && !(r < tid && v.x == id) && !(r + 1 < tid && v.y == id) && !(r + 2 < tid && v.z == id) && !(r + 3 < tid && v.w == id);
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, first);
        if (lane == 0) counts[warp] = __popc(votes);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        int at = __popc(votes & ((1u << lane) - 1));
        for (int w = 0; w < warp; w++) at += counts[w];
        if (first) first_of[at] = tid;
    }
    __syncthreads();
    int in_use = 0;
    for (int w = 0; w < HERE_ROWS / 32; w++) in_use += counts[w];
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
        if (tid < in_use) {
            HeadSlot s = {ids[first_of[tid]], 0, p.tile_cols, tid * p.tile_cols};
            p.slots[tid] = s;
        }
        if (tid < 2) p.tile_first[tid] = tid ? in_use : 0;
    }
    if ((int)blockIdx.x >= in_use) return;
    const int adapter = ids[first_of[blockIdx.x]], j0 = blockIdx.y * U_RANKS, u_row = (int)blockIdx.x * p.tile_cols;
    if (tid < HERE_ROWS) {
        const bool use = ids[tid] == adapter;
        const uint32_t votes = __ballot_sync(0xffffffffu, use);
        if (lane == 0) counts[HERE_ROWS / 32 + warp] = __popc(votes);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        int at = __popc(votes & ((1u << lane) - 1));
        for (int w = 0; w < warp; w++) at += counts[HERE_ROWS / 32 + w];
        if (use) mine[at] = tid;
    }
    for (int i = (int)blockIdx.z * SHRINK_NT + tid; i < p.tile_cols * U_RANKS; i += SHRINK_NT * (int)gridDim.z)
        if (ids[i / U_RANKS] != adapter) store_u(p, j0 + i % U_RANKS, u_row + i / U_RANKS, 0.0f);
    __syncthreads();
    int n = 0;
    for (int w = 0; w < HERE_ROWS / 32; w++) n += counts[HERE_ROWS / 32 + w];
    const int i = (int)blockIdx.z * 32;
    if (i >= n) return;
    const float v = shrink32(p, adapter, j0, mine + i, sums);
    if (i + (tid >> 4) < n) store_u(p, j0 + (tid & 15), u_row + mine[i + (tid >> 4)], v);
}

// Two factors as they are packed: an infinity or NaN as the largest finite value.  A step of the tensor cores multiplies
// every factor of its adapter with the zeros that u has for the other rows of the window, and zero times infinity would
// reach those.
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t two) {
    if ((two & 0x7f80u) == 0x7f80u) two = (two & 0xffff8000u) | 0x7f7fu;
    if ((two & 0x7f800000u) == 0x7f800000u) two = (two & 0x8000ffffu) | 0x7f7f0000u;
    return two;
}

// B of the adapters as the tensor cores read it, so that any run of 8 vocabulary rows of a chunk of 16 ranks is one
// contiguous copy: [n][chunks][padded / 8][2][8][8], blocks of 8 vocabulary rows by 8 ranks; zeros behind the
// vocabulary and the rank.  (From [vocab][rank] rows of 32 bytes the copies ran at a few requests a microsecond: 16
// adapters of rank 16 cost 64 rows 58 us more than their bytes take.)  One thread, one row of a block.
__global__ void __launch_bounds__(256) adapter_pack_kernel(const bf16_raw* b, int n, int vocab, int rank, int padded, bf16_raw* packed) {
    const int chunks = (rank + U_RANKS - 1) / U_RANKS;
    const long long total = (long long)n * chunks * padded * 2;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const int in_group = (int)(t % 16);
        const long long group = t / 16;
        const long long v = group % (padded / 8) * 8 + in_group % 8, above = group / (padded / 8);
        const int k = (int)(above % chunks) * U_RANKS + in_group / 8 * 8;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (v < vocab && k < rank) w = *reinterpret_cast<const uint4*>(b + (above / chunks * vocab + v) * rank + k);
        w = make_uint4(finite_bf16x2(w.x), finite_bf16x2(w.y), finite_bf16x2(w.z), finite_bf16x2(w.w));
        reinterpret_cast<uint4*>(packed)[t] = w;
    }
}

}  // namespace
