// The head projection and its adapters as one matrix product on the tensor cores.
// Part of head_kernels.cu.
//
//     D[v][row] = sum_k W[v][k] x[row][k]  +  sum over the tile's slots of  sum_j B[a][v][j] u[row][j]
//
// The vocabulary is the product's long side, so it takes the 128 lanes of the accumulator, and the batch's
// rows its columns (16 to 256 of them): one row costs a sixteenth of 256, and a store of the finished tile
// writes 32 neighbouring columns of a row of logits per warp.  W and B pass through the SM once per tile of
// rows, whatever the number of rows.
//
// One CTA per SM, persistent over its tiles.  Warp 4 moves operands with TMA into a ring of stages (a stage: 128
// rows of W, 128 bytes wide, and the same slice of x; or 32 ranks of one adapter's B and its window of u), warp 5
// issues tcgen05.mma from it, warps 0-3 read finished accumulators out of tensor memory and write them while
// the next tile is computed into the other half.
//
// u comes as two bfloat16, leading part and remainder, side by side in a row of 128 bytes: two products with
// the same B, which cost no more bytes, keep 16 bits of it.
//
// With 8-bit operands the projection's accumulator has to be scaled by row and column before the adapters'
// part is added, so the two have accumulators of their own (128 rows a tile at most).
#pragma once

namespace {

constexpr int VT = 128;            // vocabulary rows of a tile
constexpr int STEP_BYTES = 128;    // bytes of a row that one stage holds
constexpr int A_BYTES = VT * STEP_BYTES;
constexpr int MAX_COLS = 256;
constexpr int MAX_STAGES = 12;
constexpr int UNIT = 16;           // vocabulary rows by which single-tile batches are shared out
constexpr int HEAD_NT = 192;
constexpr int ZERO_BYTES = MAX_COLS * 32;

struct HeadCtl {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int abort;
    int row_of[MAX_COLS];
    float scale_of[MAX_COLS];
};

struct HeadArgs {
    int rows, vocab, w_steps, tile_cols, row_tiles, v_tiles;
    int slots_on, rank, chunks, u_chunk_rows;
    int stages, stage_bytes;
    const int* perm;
    const HeadSlot* slots;
    const int* tile_first;
    const float* x_scales;
    const float* w_scales;
    const void* base;
    void* out;
    long long base_stride, out_stride;
    int out_bf16;
    int* status;
};

struct HeadMaps {
    CUtensorMap w, w16, x, b, b16, u;
};

// ---- the instructions

__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

// Shared-memory matrix descriptor of a K-major operand: rows of 128, 64 or 32 bytes, swizzled by the same
// width, eight rows to a group and the groups one after the other.
enum : uint64_t { SWIZZLE_128 = 2, SWIZZLE_64 = 4, SWIZZLE_32 = 6 };
template <uint64_t SWIZZLE>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    constexpr uint64_t row = SWIZZLE == SWIZZLE_128 ? 128 : SWIZZLE == SWIZZLE_64 ? 64 : 32;
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (row * 8 >> 4) << 32 | (uint64_t)1 << 46 | SWIZZLE << 61;
}
// Instruction descriptor: float32 accumulator, 128 x n; bfloat16 operands, or e4m3.
__device__ __forceinline__ uint32_t shape_bf16(int n) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(VT >> 4) << 24;
}
__device__ __forceinline__ uint32_t shape_e4m3(int n) {
    return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(VT >> 4) << 24;
}
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}"
                 ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((int)add) : "memory");
}
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;}"
                 ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((int)add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_load16(uint32_t addr, float v[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

// A wait that ends: when the phase completes (true), when another role gave up, or after two seconds (false,
// and then everybody gives up).
__device__ __forceinline__ bool head_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 8; i++)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
        if (global_ns() - t0 > WAIT_LIMIT_NS) {
            *abort = 1;
            return false;
        }
    }
}

// A barrier of the 128 threads that write results, and whether all of them are still in order.
__device__ __forceinline__ bool epilogue_agree(bool ok) {
    int all;
    asm volatile("{.reg .pred p, q; setp.ne.b32 p, %1, 0; bar.red.and.pred q, 1, 128, p; selp.b32 %0, 1, 0, q;}"
                 : "=r"(all) : "r"((int)ok) : "memory");
    return all != 0;
}

// The tiles of this CTA, one after the other.  One tile of rows: the vocabulary is shared out in equal runs of
// 16-row units, so that every SM streams the same bytes (151 936 columns are 1187 tiles of 128: eight for each of
// 148 SMs, and three left over); a run's last tile may be short.  Several tiles of rows: whole tiles, those of the
// same vocabulary rows next to each other, so that W comes from HBM once and from L2 after that.
struct HeadTiles {
    int unit, unit_end, t, n_tiles, row_tiles;
    __device__ explicit HeadTiles(const HeadArgs& a) {
        row_tiles = a.row_tiles;
        const long long units = (a.vocab + UNIT - 1) / UNIT;
        unit = (int)(units * blockIdx.x / gridDim.x);
        unit_end = (int)(units * (blockIdx.x + 1) / gridDim.x);
        t = blockIdx.x;
        n_tiles = a.v_tiles * a.row_tiles;
    }
    // false: no more
    __device__ bool next(int* v0, int* v_rows, int* row_tile) {
        if (row_tiles == 1) {
            if (unit >= unit_end) return false;
            *v0 = unit * UNIT;
            *v_rows = min(VT / UNIT, unit_end - unit) * UNIT;
            *row_tile = 0;
            unit += VT / UNIT;
            return true;
        }
        if (t >= n_tiles) return false;
        *v0 = t / row_tiles * VT;
        *v_rows = VT;
        *row_tile = t % row_tiles;
        t += gridDim.x;
        return true;
    }
};

// ---- the kernel

template <bool E4M3>
__global__ void __launch_bounds__(HEAD_NT, 1) head_rows_kernel(const HeadArgs a, const __grid_constant__ HeadMaps maps) {
    extern __shared__ char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    char* const ring = raw + (base - smem_u32(raw));
    const uint32_t zeros = base + (uint32_t)(a.stages * a.stage_bytes);
    const bool zero_first = a.slots_on && (E4M3 || a.w_steps == 0);
    HeadCtl& ctl = *reinterpret_cast<HeadCtl*>(ring + a.stages * a.stage_bytes + (zero_first ? ZERO_BYTES : 0));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // columns of tensor memory: two accumulators of 256, the adapters' part in the second 128 of each with e4m3
    const uint32_t acc_of[2] = {0u, 256u};
    const uint32_t slot_acc = E4M3 && a.w_steps ? 128u : 0u;

    if (zero_first) {
        for (int i = threadIdx.x; i < ZERO_BYTES / 16; i += HEAD_NT)
            reinterpret_cast<uint4*>(ring + a.stages * a.stage_bytes)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; s++) {
            mbar_init(&ctl.full[s], 1);
            mbar_init(&ctl.empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&ctl.acc_full[i], 1);
            mbar_init(&ctl.acc_empty[i], 4);
        }
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ctl.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = ctl.tmem;
    HeadTiles tiles(a);
    int v0, v_rows, row_tile;

    if (warp == 4) {
        if (lane == 0) {
            // fills of the ring, counted from the start; stage fill % stages
            int fill = 0, stage = 0;
            uint32_t phase = 1;  // of `empty`: the first round passes
            bool ok = true, waited = false;
            auto take = [&]() { ok = head_wait(&ctl.empty[stage], phase, &ctl.abort); return ok; };
            auto advance = [&]() {
                fill++;
                if (++stage == a.stages) stage = 0, phase ^= 1;
            };
            auto load_w = [&](int s) {
                const uint32_t dst = base + (uint32_t)(stage * a.stage_bytes);
                mbar_expect(&ctl.full[stage], (uint32_t)((v_rows + a.tile_cols) * STEP_BYTES));
                const int x = s * (E4M3 ? STEP_BYTES : STEP_BYTES / 2);
                if (v_rows == VT) {
                    tma_2d(dst, &maps.w, x, v0, &ctl.full[stage]);
                } else {
                    for (int i = 0; i < v_rows; i += UNIT) tma_2d(dst + i * STEP_BYTES, &maps.w16, x, v0 + i, &ctl.full[stage]);
                }
            };
            auto load_x = [&](int s, int st) {
                tma_2d(base + (uint32_t)(st * a.stage_bytes + A_BYTES), &maps.x, s * (E4M3 ? STEP_BYTES : STEP_BYTES / 2),
                       row_tile * a.tile_cols, &ctl.full[st]);
            };
            while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
                int s = 0;
                if (!waited) {
                    // W does not come from the kernels in front: the ring fills with it while they still run
                    const int ahead = min(a.stages, a.w_steps);
                    for (; s < ahead; s++) {
                        load_w(s);
                        advance();
                    }
                    pdl_wait();
                    asm volatile("fence.proxy.async.global;" ::: "memory");
                    for (int i = 0; i < ahead; i++) load_x(i, i);
                    waited = true;
                }
                for (; s < a.w_steps; s++) {
                    if (!take()) break;
                    load_w(s);
                    load_x(s, stage);
                    advance();
                }
                if (!ok || !a.slots_on) continue;
                const int end = a.tile_first[row_tile + 1];
                for (int i = a.tile_first[row_tile]; i < end && ok; i++) {
                    const HeadSlot slot = a.slots[i];
                    for (int c = 0; c < a.chunks; c++) {
                        if (!take()) break;
                        const uint32_t dst = base + (uint32_t)(stage * a.stage_bytes);
                        uint64_t* bar = &ctl.full[stage];
                        mbar_expect(bar, (uint32_t)(v_rows * U_CHUNK * 2 + slot.n * U_ROW * 2));
                        if (v_rows == VT) {
                            tma_3d(dst, &maps.b, c * U_CHUNK, v0, slot.adapter, bar);
                        } else {
                            for (int r = 0; r < v_rows; r += UNIT)
                                tma_3d(dst + r * U_CHUNK * 2, &maps.b16, c * U_CHUNK, v0 + r, slot.adapter, bar);
                        }
                        for (int r = 0; r < slot.n; r += WINDOW)
                            tma_2d(dst + A_BYTES + r * U_ROW * 2, &maps.u, 0, c * a.u_chunk_rows + slot.u_row + r, bar);
                        advance();
                    }
                }
            }
            // every copy has landed before the CTA may end, whether its stage was used or not
            if (ok) {
                for (int i = 0; i < a.stages; i++) {  // (a stage never filled counts as empty)
                    if (!take()) break;
                    advance();
                }
            }
            if (!ok) {
                const int outstanding = min(fill, a.stages);
                for (int i = fill - outstanding; i < fill; i++)
                    mbar_wait(&ctl.full[i % a.stages], (uint32_t)(i / a.stages) & 1, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            int stage = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            if (a.slots_on) pdl_wait();  // the slots come from the kernel in front
            auto take = [&]() {
                ok = head_wait(&ctl.full[stage], phase, &ctl.abort);
                tmem_fence_after();
                return ok;
            };
            auto advance = [&]() {
                mma_commit(&ctl.empty[stage]);
                if (++stage == a.stages) stage = 0, phase ^= 1;
            };
            const uint32_t shape = E4M3 ? shape_e4m3(a.tile_cols) : shape_bf16(a.tile_cols);
            for (; ok && tiles.next(&v0, &v_rows, &row_tile); it++) {
                const int buf = it & 1;
                ok = head_wait(&ctl.acc_empty[buf], ((it >> 1) & 1) ^ 1, &ctl.abort);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t acc = tmem + acc_of[buf];
                // the slots' windows cover a tile in part only: zero times zero first
                if (zero_first)
                    mma_bf16(acc + slot_acc, operand<SWIZZLE_32>(zeros), operand<SWIZZLE_32>(zeros), shape_bf16(a.tile_cols), false);
                for (int s = 0; s < a.w_steps; s++) {
                    if (!take()) break;
                    const uint32_t src = base + (uint32_t)(stage * a.stage_bytes);
#pragma unroll
                    for (int k = 0; k < STEP_BYTES; k += 32) {
                        const uint64_t wd = operand<SWIZZLE_128>(src + k), xd = operand<SWIZZLE_128>(src + A_BYTES + k);
                        if (E4M3) mma_e4m3(acc, wd, xd, shape, s > 0 || k > 0);
                        else mma_bf16(acc, wd, xd, shape, s > 0 || k > 0);
                    }
                    advance();
                }
                if (ok && a.slots_on) {
                    const int end = a.tile_first[row_tile + 1];
                    for (int i = a.tile_first[row_tile]; i < end && ok; i++) {
                        const HeadSlot slot = a.slots[i];
                        const uint32_t d = acc + slot_acc + (uint32_t)slot.col, n_shape = shape_bf16(slot.n);
                        for (int c = 0; c < a.chunks; c++) {
                            if (!take()) break;
                            const uint32_t src = base + (uint32_t)(stage * a.stage_bytes);
                            const int steps = (min(U_CHUNK, a.rank - c * U_CHUNK) + 15) / 16;
                            for (int k = 0; k < steps; k++) {
                                const uint64_t bd = operand<SWIZZLE_64>(src + k * 32);
                                mma_bf16(d, bd, operand<SWIZZLE_128>(src + A_BYTES + k * 32), n_shape, true);
                                mma_bf16(d, bd, operand<SWIZZLE_128>(src + A_BYTES + U_CHUNK * 2 + k * 32), n_shape, true);
                            }
                            advance();
                        }
                    }
                }
                if (ok) mma_commit(&ctl.acc_full[buf]);
            }
            if (!ok) {  // what was issued ends before tensor memory is given back
                mma_commit(&ctl.drain);
                mbar_wait(&ctl.drain, 0, 100000000ull);
            }
        }
        __syncwarp();
    } else {
        bool ok = true;
        pdl_wait();
        for (int it = 0; ok && tiles.next(&v0, &v_rows, &row_tile); it++) {
            const int buf = it & 1, place0 = row_tile * a.tile_cols, cols = min(a.tile_cols, a.rows - place0);
            for (int c = threadIdx.x; c < a.tile_cols; c += 128) {
                const int row = c < cols ? (a.perm ? a.perm[place0 + c] : place0 + c) : 0;
                ctl.row_of[c] = row;
                if (E4M3 && a.w_steps) ctl.scale_of[c] = a.x_scales[row];
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const int v = v0 + (int)threadIdx.x;
            const bool mine = (int)threadIdx.x < v_rows && v < a.vocab;
            const float w_scale = E4M3 && a.w_steps && mine ? a.w_scales[v] : 1.0f;
            ok = head_wait(&ctl.acc_full[buf], (it >> 1) & 1, &ctl.abort);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                tmem_fence_after();
                const uint32_t acc = tmem + acc_of[buf] + ((uint32_t)(warp * 32) << 16);
                for (int c0 = 0; c0 < cols; c0 += 16) {
                    float d[16];
                    tmem_load16(acc + c0, d);
                    if (E4M3 && a.w_steps) {
#pragma unroll
                        for (int i = 0; i < 16; i++) d[i] *= ctl.scale_of[c0 + i] * w_scale;
                        if (a.slots_on) {
                            float e[16];
                            tmem_load16(acc + slot_acc + c0, e);
#pragma unroll
                            for (int i = 0; i < 16; i++) d[i] += e[i];
                        }
                    }
                    if (mine) {
                        if (a.base) {
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                if (c0 + i >= cols) break;
                                const long long at = (long long)ctl.row_of[c0 + i] * a.base_stride + v;
                                d[i] += a.out_bf16 ? load1(static_cast<const bf16_raw*>(a.base) + at)
                                                   : load1(static_cast<const float*>(a.base) + at);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            if (c0 + i >= cols) break;
                            const long long at = (long long)ctl.row_of[c0 + i] * a.out_stride + v;
                            if (a.out_bf16) store1(static_cast<bf16_raw*>(a.out) + at, d[i]);
                            else store1(static_cast<float*>(a.out) + at, d[i]);
                        }
                    }
                    __syncwarp();
                }
                tmem_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl.acc_empty[buf]);
            ok = epilogue_agree(ok);  // the tables are free, and the four warps go on together or not at all
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && ctl.abort && a.status) atomicOr(a.status, MANTLE_SAMPLE_STATUS_TIMEOUT);
    if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace
