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
// One CTA per SM, persistent over its tiles.  Warp 8 moves operands with TMA into a ring of stages (a stage: 128
// rows of W, 128 bytes wide, and the same slice of x; or some adapters' B, 16 or 32 ranks wide, and their windows of
// u), warp 9 issues tcgen05.mma from it, warps 0-7 read accumulators out of tensor memory, add them up in
// registers and write the finished tile while the next one is computed.
//
// Rounds.  A float32 accumulator in tensor memory is cut, not rounded, at every step, so its error grows with the
// number of steps, always towards zero (measured with bfloat16 operands: 2.3e-7 of the result after 256 columns,
// 9.1e-6 after 8192).  A tile is therefore computed in rounds of 512 columns, each in a fresh one of two
// accumulators, and the rounds are added with ordinary float32 sums (5e-7 at any width).  With e4m3 operands the
// products are short and the cut costs nothing that shows (5.1e-7 after 8192 columns): a round is 8192 columns.
//
// u comes as two bfloat16, leading part and remainder, side by side: two products with the same B, which cost no more
// bytes, keep 16 bits of it.  With 8-bit operands the projection's rounds are scaled by row and column, and the
// adapters have a round of their own.
#pragma once

namespace {

constexpr int VT = 128;            // vocabulary rows of a tile
constexpr int STEP_BYTES = 128;    // bytes of a row that one stage holds
constexpr int A_BYTES = VT * STEP_BYTES;
constexpr int MAX_COLS = 256;
constexpr int MAX_STAGES = 12;
constexpr int UNIT = 16;           // vocabulary rows by which single-tile batches are shared out
constexpr int ROUND_BF16 = 8;      // steps of a round
constexpr int ROUND_E4M3 = 64;
constexpr int WRITERS = 256;       // threads that read accumulators and write results
constexpr int HEAD_NT = WRITERS + 64;
constexpr int ZERO_BYTES = MAX_COLS * 32;
constexpr int MAX_PACK = 4;        // adapters' steps in one stage

struct HeadCtl {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int abort;
    long long out_of[MAX_COLS], base_of[MAX_COLS];  // a column's row, as a distance in bytes
    float scale_of[MAX_COLS];
};

struct HeadArgs {
    int rows, vocab, w_steps, tile_cols, row_tiles, v_tiles;
    int slots_on, sorted, copied;  // adapters; perm and x come from the kernel in front
    int rank, u_cols, u_rows, u_box;  // u_box: rows of u of one copy
    int stages, stage_bytes;
    const int* perm;
    const HeadSlot* slots;
    const int* tile_first;
    const float* x_scales;
    const float* w_scales;
    const void* base;
    void* out;
    long long base_stride, out_stride;
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
__device__ __forceinline__ uint64_t operand_format(int row_bytes) {
    const uint64_t swizzle = row_bytes == 128 ? 2 : row_bytes == 64 ? 4 : 6;
    return (uint64_t)1 << 16 | (uint64_t)(row_bytes * 8 >> 4) << 32 | (uint64_t)1 << 46 | swizzle << 61;
}
__device__ __forceinline__ uint64_t operand(uint64_t format, uint32_t addr) { return format | (uint64_t)((addr >> 4) & 0x3fff); }
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

// A barrier of the threads that write results, and whether all of them are still in order.
__device__ __forceinline__ bool writers_agree(bool ok) {
    int all;
    asm volatile("{.reg .pred p, q; setp.ne.b32 p, %1, 0; bar.red.and.pred q, 1, 256, p; selp.b32 %0, 1, 0, q;}"
                 : "=r"(all) : "r"((int)ok) : "memory");
    return all != 0;
}

// The tiles of this CTA, one after the other.  One tile of rows: the vocabulary is shared out in equal runs of
// 16-row units, so that every SM streams the same bytes (151 936 columns are 1187 tiles of 128: eight for each of
// 148 SMs, and three left over); a run's short tile comes first, where the ring is filling anyway.  Several tiles of
// rows: whole tiles, those of the same vocabulary rows next to each other, so that W comes from HBM once and from
// L2 after that.
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
            const int odd = (unit_end - unit) % (VT / UNIT), n = odd ? odd : VT / UNIT;
            *v0 = unit * UNIT;
            *v_rows = n * UNIT;
            *row_tile = 0;
            unit += n;
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

// The adapters' steps of a tile, packed into stages as they come: up to the stage's room for B and for u.
struct HeadPacks {
    const HeadSlot* slots;
    int at, end, chunk, chunks, most, room, row_bytes;
    __device__ HeadPacks(const HeadArgs& a, int row_tile) {
        slots = a.slots;
        at = a.tile_first[row_tile];
        end = a.tile_first[row_tile + 1];
        chunk = 0;
        chunks = (a.rank + a.u_cols - 1) / a.u_cols;
        row_bytes = a.u_cols * 4;
        most = A_BYTES / (VT * a.u_cols * 2);
        room = a.stage_bytes - A_BYTES;
    }
    // The steps of the next stage; 0: no more.
    __device__ int next(HeadSlot slot[MAX_PACK], int chunk_of[MAX_PACK], int* u_bytes) {
        int n = 0;
        *u_bytes = 0;
#pragma unroll
        for (int i = 0; i < MAX_PACK; i++) {
            if (i < most && n == i && at < end) {
                const HeadSlot s = slots[at];
                if (*u_bytes + s.n * row_bytes <= room) {
                    slot[i] = s;
                    chunk_of[i] = chunk;
                    *u_bytes += s.n * row_bytes;
                    n++;
                    if (++chunk == chunks) chunk = 0, at++;
                }
            }
        }
        return n;
    }
};

// ---- the kernel

template <bool OUT16>
struct OutType {
    typedef float type;
};
template <>
struct OutType<true> {
    typedef bf16_raw type;
};

// GROUPS: a tile has up to 32 * GROUPS columns.  (The writers' part is unrolled over them, its sums being registers;
// unrolled to 256 columns for every batch, a single row spent its time on fetching instructions: 88 against 58 us.)
template <bool E4M3, bool OUT16, int GROUPS>
__global__ void __launch_bounds__(HEAD_NT, 1) head_rows_kernel(const HeadArgs a, const __grid_constant__ HeadMaps maps) {
    extern __shared__ char raw[];
    constexpr int STEP_COLS = E4M3 ? STEP_BYTES : STEP_BYTES / 2;
    constexpr int ROUND = E4M3 ? ROUND_E4M3 : ROUND_BF16;
    constexpr int OUT_BYTES = OUT16 ? 2 : 4;
    using Out = typename OutType<OUT16>::type;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    char* const ring = raw + (base - smem_u32(raw));
    const uint32_t zeros = base + (uint32_t)(a.stages * a.stage_bytes);
    // the adapters have a round of their own, or are the end of the projection's last one
    const bool own_round = a.slots_on && (E4M3 || a.w_steps == 0);
    HeadCtl& ctl = *reinterpret_cast<HeadCtl*>(ring + a.stages * a.stage_bytes + (own_round ? ZERO_BYTES : 0));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (own_round) {
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
            mbar_init(&ctl.acc_empty[i], WRITERS / 32);
        }
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == WRITERS / 32 + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ctl.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = ctl.tmem;
    HeadTiles tiles(a);
    int v0, v_rows, row_tile;
    // what the kernels in front wrote may be read from here on (each thread asks once, where it first needs it)
    bool behind = false;
    auto wait_for_front = [&]() {
        if (!behind) pdl_wait();
        behind = true;
    };

    if (warp == WRITERS / 32) {
        if (lane == 0) {
            // fills of the ring, counted from the start; stage fill % stages
            int fill = 0, stage = 0;
            uint32_t phase = 1;  // of `empty`: the first round passes
            bool ok = true;
            auto take = [&]() { ok = head_wait(&ctl.empty[stage], phase, &ctl.abort); return ok; };
            auto advance = [&]() {
                fill++;
                if (++stage == a.stages) stage = 0, phase ^= 1;
            };
            auto load_w = [&](int s) {
                const uint32_t dst = base + (uint32_t)(stage * a.stage_bytes);
                mbar_expect(&ctl.full[stage], (uint32_t)((v_rows + a.tile_cols) * STEP_BYTES));
                if (v_rows == VT) {
                    tma_2d(dst, &maps.w, s * STEP_COLS, v0, &ctl.full[stage]);
                } else {
                    for (int i = 0; i < v_rows; i += UNIT) tma_2d(dst + i * STEP_BYTES, &maps.w16, s * STEP_COLS, v0 + i, &ctl.full[stage]);
                }
            };
            auto load_x = [&](int s, int st) {
                tma_2d(base + (uint32_t)(st * a.stage_bytes + A_BYTES), &maps.x, s * STEP_COLS, row_tile * a.tile_cols, &ctl.full[st]);
            };
            while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
                int s = 0;
                if (a.copied && !behind) {
                    // W does not come from the kernels in front: the ring fills with it while they still run
                    const int ahead = min(a.stages, a.w_steps);
                    for (; s < ahead; s++) {
                        load_w(s);
                        advance();
                    }
                    wait_for_front();
                    asm volatile("fence.proxy.async.global;" ::: "memory");
                    for (int i = 0; i < ahead; i++) load_x(i, i);
                }
                for (; s < a.w_steps; s++) {
                    if (!take()) break;
                    load_w(s);
                    load_x(s, stage);
                    advance();
                }
                if (!ok || !a.slots_on) continue;
                if (!behind) {
                    wait_for_front();
                    asm volatile("fence.proxy.async.global;" ::: "memory");
                }
                HeadPacks packs(a, row_tile);
                HeadSlot slot[MAX_PACK];
                int chunk[MAX_PACK], u_bytes;
                while (const int n = packs.next(slot, chunk, &u_bytes)) {
                    if (!take()) break;
                    const uint32_t dst = base + (uint32_t)(stage * a.stage_bytes);
                    uint64_t* bar = &ctl.full[stage];
                    mbar_expect(bar, (uint32_t)(n * v_rows * a.u_cols * 2 + u_bytes));
                    uint32_t u_dst = dst + A_BYTES;
#pragma unroll
                    for (int i = 0; i < MAX_PACK; i++) {
                        if (i >= n) continue;
                        const uint32_t b_dst = dst + (uint32_t)(i * VT * a.u_cols * 2);
                        if (v_rows == VT) {
                            tma_3d(b_dst, &maps.b, chunk[i] * a.u_cols, v0, slot[i].adapter, bar);
                        } else {
                            for (int r = 0; r < v_rows; r += UNIT)
                                tma_3d(b_dst + r * a.u_cols * 2, &maps.b16, chunk[i] * a.u_cols, v0 + r, slot[i].adapter, bar);
                        }
                        for (int r = 0; r < slot[i].n; r += a.u_box)
                            tma_2d(u_dst + r * a.u_cols * 4, &maps.u, 0, chunk[i] * a.u_rows + slot[i].u_row + r, bar);
                        u_dst += (uint32_t)(slot[i].n * a.u_cols * 4);
                    }
                    advance();
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
    } else if (warp == WRITERS / 32 + 1) {
        if (lane == 0) {
            int stage = 0, round = 0;
            uint32_t phase = 0;
            bool ok = true;
            auto take = [&]() {
                ok = head_wait(&ctl.full[stage], phase, &ctl.abort);
                tmem_fence_after();
                return ok;
            };
            auto advance = [&]() {
                mma_commit(&ctl.empty[stage]);
                if (++stage == a.stages) stage = 0, phase ^= 1;
            };
            uint32_t acc = 0;
            auto begin_round = [&]() {
                ok = head_wait(&ctl.acc_empty[round & 1], ((round >> 1) & 1) ^ 1, &ctl.abort);
                tmem_fence_after();
                acc = tmem + (uint32_t)(round & 1) * MAX_COLS;
                return ok;
            };
            auto end_round = [&]() { mma_commit(&ctl.acc_full[round++ & 1]); };
            const uint32_t shape = E4M3 ? shape_e4m3(a.tile_cols) : shape_bf16(a.tile_cols);
            const uint64_t wide = operand_format(128), zero = operand(operand_format(32), zeros);
            const uint64_t b_format = operand_format(a.u_cols * 2), u_format = operand_format(a.u_cols * 4);
            while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
                for (int s = 0; s < a.w_steps; s++) {
                    const bool first = s % ROUND == 0;
                    if (first && !begin_round()) break;
                    if (!take()) break;
                    const uint32_t src = base + (uint32_t)(stage * a.stage_bytes);
#pragma unroll
                    for (int k = 0; k < STEP_BYTES; k += 32) {
                        const uint64_t wd = operand(wide, src + k), xd = operand(wide, src + A_BYTES + k);
                        if (E4M3) mma_e4m3(acc, wd, xd, shape, !first || k > 0);
                        else mma_bf16(acc, wd, xd, shape, !first || k > 0);
                    }
                    advance();
                    if (s % ROUND == ROUND - 1 || s == a.w_steps - 1) {
                        if (!(a.slots_on && !own_round && s == a.w_steps - 1)) end_round();
                    }
                }
                if (!ok || !a.slots_on) continue;
                wait_for_front();
                HeadPacks packs(a, row_tile);
                if (own_round) {
                    if (packs.at == packs.end) continue;
                    if (!begin_round()) break;
                    // the slots' windows may cover a tile in part only: zero times zero first
                    mma_bf16(acc, zero, zero, shape_bf16(a.tile_cols), false);
                }
                HeadSlot slot[MAX_PACK];
                int chunk[MAX_PACK], u_bytes;
                while (const int n = packs.next(slot, chunk, &u_bytes)) {
                    if (!take()) break;
                    const uint32_t src = base + (uint32_t)(stage * a.stage_bytes);
                    uint32_t u_src = src + A_BYTES;
#pragma unroll
                    for (int i = 0; i < MAX_PACK; i++) {
                        if (i >= n) continue;
                        const uint32_t d = acc + (uint32_t)slot[i].col, n_shape = shape_bf16(slot[i].n);
                        const uint32_t b_src = src + (uint32_t)(i * VT * a.u_cols * 2);
                        for (int k = 0; k < a.u_cols && chunk[i] * a.u_cols + k < a.rank; k += 16) {
                            const uint64_t bd = operand(b_format, b_src + k * 2);
                            mma_bf16(d, bd, operand(u_format, u_src + k * 2), n_shape, true);
                            mma_bf16(d, bd, operand(u_format, u_src + (a.u_cols + k) * 2), n_shape, true);
                        }
                        u_src += (uint32_t)(slot[i].n * a.u_cols * 4);
                    }
                    advance();
                }
                if (ok) end_round();
            }
            if (!ok) {  // what was issued ends before tensor memory is given back
                mma_commit(&ctl.drain);
                mbar_wait(&ctl.drain, 0, 100000000ull);
            }
        }
        __syncwarp();
    } else {
        // a warp reads the 32 lanes of tensor memory that its number allows, and every other sixteen columns of them
        const int quarter = warp & 3, half = warp >> 2;
        const int w_rounds = (a.w_steps + ROUND - 1) / ROUND;
        bool ok = true;
        int round = 0;
        if (a.sorted) wait_for_front();
        while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
            const int place0 = row_tile * a.tile_cols, cols = min(a.tile_cols, a.rows - place0);
            {
                const int c = threadIdx.x;
                const int row = c < cols ? (a.sorted ? a.perm[place0 + c] : place0 + c) : 0;
                ctl.out_of[c] = row * a.out_stride * OUT_BYTES;
                if (a.base) ctl.base_of[c] = row * a.base_stride * OUT_BYTES;
                if (E4M3 && a.w_steps) ctl.scale_of[c] = a.x_scales[row];
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const int v = v0 + quarter * 32 + lane;
            const bool mine = quarter * 32 + lane < v_rows && v < a.vocab;
            const float w_scale = E4M3 && a.w_steps && mine ? a.w_scales[v] : 1.0f;
            float sum[GROUPS][16];
#pragma unroll
            for (int j = 0; j < GROUPS; j++) {
#pragma unroll
                for (int i = 0; i < 16; i++) sum[j][i] = 0.0f;
            }
            if (a.base && mine) {
                const char* from = static_cast<const char*>(a.base) + (long long)v * OUT_BYTES;
#pragma unroll
                for (int j = 0; j < GROUPS; j++) {
                    const int c0 = j * 32 + half * 16;
                    if (c0 < cols) {
#pragma unroll
                        for (int i = 0; i < 16; i++)  // (a column past the last reads its row 0: not stored)
                            sum[j][i] = load1(reinterpret_cast<const Out*>(from + ctl.base_of[c0 + i]));
                    }
                }
            }
            int rounds = w_rounds;
            if (own_round) {
                wait_for_front();
                rounds += a.tile_first[row_tile] < a.tile_first[row_tile + 1];
            }
            for (int r = 0; r < rounds && ok; r++, round++) {
                // one lane of a warp watches the barrier
                int landed = 1;
                if (lane == 0) landed = head_wait(&ctl.acc_full[round & 1], (round >> 1) & 1, &ctl.abort);
                ok = __shfl_sync(0xffffffffu, landed, 0);
                if (ok) {
                    tmem_fence_after();
                    const uint32_t acc = tmem + (uint32_t)(round & 1) * MAX_COLS + ((uint32_t)(quarter * 32) << 16);
                    const bool scaled = E4M3 && r < w_rounds;
#pragma unroll
                    for (int j = 0; j < GROUPS; j++) {
                        const int c0 = j * 32 + half * 16;
                        if (c0 < cols) {
                            float d[16];
                            tmem_load16(acc + c0, d);
                            if (scaled) {
#pragma unroll
                                for (int i = 0; i < 16; i++) d[i] *= ctl.scale_of[c0 + i] * w_scale;
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) sum[j][i] += d[i];
                        }
                    }
                    tmem_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl.acc_empty[round & 1]);
            }
            if (ok && mine) {
                char* to = static_cast<char*>(a.out) + (long long)v * OUT_BYTES;
#pragma unroll
                for (int j = 0; j < GROUPS; j++) {
                    const int c0 = j * 32 + half * 16;
                    if (c0 < cols) {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (c0 + i < cols) store1(reinterpret_cast<Out*>(to + ctl.out_of[c0 + i]), sum[j][i]);
                    }
                }
            }
            __syncwarp();
            ok = writers_agree(ok);  // the tables are free, and the warps go on together or not at all
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && ctl.abort && a.status) atomicOr(a.status, MANTLE_SAMPLE_STATUS_TIMEOUT);
    if (warp == WRITERS / 32 + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace
