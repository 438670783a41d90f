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
// rows of W, 128 bytes wide, and the same slice of x; or some adapters' B, 16 ranks wide, and their windows of u),
// warp 9 issues tcgen05.mma from it, warps 0-7 read accumulators out of tensor memory, add them up in registers
// and write the finished tile while the next one is computed.
//
// Pairs.  W comes from HBM once, but x from L2 for every 128 vocabulary rows: at 256 rows that is twice W's bytes,
// and what L2 can hand out (about 10 TB/s) bounds the kernel long before HBM or the tensor cores do.  From 65 rows
// on two CTAs therefore compute 256 vocabulary rows together (cta_group::2): each holds its own 128 rows of W and
// of the accumulator, and half of x.  The even CTA of a pair issues the products; copies of both complete on its
// barriers.
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
constexpr int UNIT = 16;           // vocabulary rows of a CTA by which single-tile batches are shared out
constexpr int B_BYTES = VT * U_RANKS * 2;  // one adapter's B of one chunk and a whole tile
constexpr int ROUND_BF16 = 8;      // steps of a round
constexpr int ROUND_E4M3 = 64;
constexpr int WRITERS = 256;       // threads that read accumulators and write results
constexpr int HEAD_NT = WRITERS + 64;
constexpr int ZERO_BYTES = VT * 32;
constexpr int MAX_PACK = A_BYTES / B_BYTES;  // adapters' steps in one stage

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
    int chunks, u_rows, u_box;        // u_box: rows of u of one copy
    int b_rows;                       // 128-byte rows of one chunk of an adapter's B
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
    CUtensorMap w, w16, x, b, b16, u;  // (b, b16 and u: plain 128-byte rows)
};

// ---- the instructions

__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// The address of `bar` in the pair's even CTA (PAIR), or in this one.
template <bool PAIR>
__device__ __forceinline__ uint32_t lead_bar(uint64_t* bar) {
    uint32_t at = smem_u32(bar);
    if (PAIR) asm volatile("mapa.shared::cluster.u32 %0, %0, 0;" : "+r"(at));
    return at;
}
template <bool PAIR>
__device__ __forceinline__ void lead_arrive(uint64_t* bar) {
    if (PAIR) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_bar<true>(bar)) : "memory");
    else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Copies to this CTA's shared memory that complete on a barrier of the pair's even CTA (bar: lead_bar's).
template <bool PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// Shared-memory matrix descriptors of K-major operands.  W and x: rows of 128 bytes, swizzled, 1024 bytes from eight
// rows to the next eight.  B and u: blocks of 8 rows by 16 bytes, 128 bytes from one block of a row to the next, and
// `group` bytes from eight rows to the next eight.
constexpr uint64_t SWIZZLED_ROWS = (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
__device__ constexpr uint64_t blocks(int group) { return (uint64_t)(128 >> 4) << 16 | (uint64_t)(group >> 4) << 32 | (uint64_t)1 << 46; }
__device__ __forceinline__ uint64_t operand(uint64_t format, uint32_t addr) { return format | (uint64_t)((addr >> 4) & 0x3fff); }
// Instruction descriptor: float32 accumulator, 128 (a pair: 256) x n; bfloat16 operands, or e4m3.
template <bool PAIR>
__device__ __forceinline__ uint32_t shape_bf16(int n) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(VT * (PAIR ? 2 : 1) >> 4) << 24;
}
template <bool PAIR>
__device__ __forceinline__ uint32_t shape_e4m3(int n) {
    return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(VT * (PAIR ? 2 : 1) >> 4) << 24;
}
template <bool PAIR, bool E4M3>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
#define MANTLE_MMA(GROUP, KIND)                                                                                          \
    asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;}" \
                 ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((int)add) : "memory")
    if (PAIR && E4M3) MANTLE_MMA("2", "f8f6f4");
    else if (PAIR) MANTLE_MMA("2", "f16");
    else if (E4M3) MANTLE_MMA("1", "f8f6f4");
    else MANTLE_MMA("1", "f16");
#undef MANTLE_MMA
}
// Arrives on `bar` -- of both CTAs of a pair -- when the products issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// All threads of the CTA, or of the pair.
template <bool PAIR>
__device__ __forceinline__ void sync_all() {
    if (PAIR) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
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
template <bool PAIR>
struct HeadTiles {
    int unit, unit_end, t, n_tiles, row_tiles, rank;
    __device__ explicit HeadTiles(const HeadArgs& a) {
        const int index = PAIR ? blockIdx.x / 2 : blockIdx.x, count = PAIR ? gridDim.x / 2 : gridDim.x;
        rank = PAIR ? blockIdx.x & 1 : 0;
        row_tiles = a.row_tiles;
        const long long units = (a.vocab + UNIT * CTAS - 1) / (UNIT * CTAS);
        unit = (int)(units * index / count);
        unit_end = (int)(units * (index + 1) / count);
        t = index;
        n_tiles = a.v_tiles * a.row_tiles;
    }
    // This CTA's part of the next tile; false: no more.
    __device__ bool next(int* v0, int* v_rows, int* row_tile) {
        if (row_tiles == 1) {
            if (unit >= unit_end) return false;
            const int odd = (unit_end - unit) % (VT / UNIT), n = odd ? odd : VT / UNIT;
            *v_rows = n * UNIT;
            *v0 = unit * (UNIT * CTAS) + rank * *v_rows;
            *row_tile = 0;
            unit += n;
            return true;
        }
        if (t >= n_tiles) return false;
        *v0 = (t / row_tiles * CTAS + rank) * VT;
        *v_rows = VT;
        *row_tile = t % row_tiles;
        t += PAIR ? gridDim.x / 2 : gridDim.x;
        return true;
    }
    static constexpr int CTAS = PAIR ? 2 : 1;
};

// The adapters' steps of a tile, packed into stages as they come: up to the stage's room for B and for u.
template <bool PAIR>
struct HeadPacks {
    const HeadSlot* slots;
    int at, end, chunk, chunks, room;
    __device__ HeadPacks(const HeadArgs& a, int row_tile) {
        slots = a.slots;
        at = a.tile_first[row_tile];
        end = a.tile_first[row_tile + 1];
        chunk = 0;
        chunks = a.chunks;
        room = a.stage_bytes - A_BYTES;
    }
    // The steps of the next stage, and the bytes of u that this CTA holds of them; 0: no more.
    __device__ int next(HeadSlot slot[MAX_PACK], int chunk_of[MAX_PACK], int* u_bytes) {
        int n = 0;
        *u_bytes = 0;
#pragma unroll
        for (int i = 0; i < MAX_PACK; i++) {
            if (n == i && at < end) {
                const HeadSlot s = slots[at];
                const int bytes = s.n / (PAIR ? 2 : 1) * U_BYTES;
                if (*u_bytes + bytes <= room) {
                    slot[i] = s;
                    chunk_of[i] = chunk;
                    *u_bytes += bytes;
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
    constexpr bool PAIR = GROUPS >= 4;
    constexpr int CTAS = PAIR ? 2 : 1;
    const bool lead = !PAIR || (blockIdx.x & 1) == 0;
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
            mbar_init(&ctl.acc_empty[i], WRITERS / 32 * CTAS);
        }
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == WRITERS / 32 + 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ctl.tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ctl.tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
        tmem_fence_before();
    }
    sync_all<PAIR>();
    tmem_fence_after();
    const uint32_t tmem = ctl.tmem;
    HeadTiles<PAIR> tiles(a);
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
            // the even CTA of a pair awaits the bytes of both; a barrier counts them in any order
            auto expect = [&](int bytes) { if (lead) mbar_expect(&ctl.full[stage], (uint32_t)bytes * CTAS); };
            const int x_rows = a.tile_cols / CTAS, half = PAIR ? blockIdx.x & 1 : 0;
            auto load_w = [&](int s) {
                const uint32_t dst = base + (uint32_t)(stage * a.stage_bytes), bar = lead_bar<PAIR>(&ctl.full[stage]);
                expect((v_rows + x_rows) * STEP_BYTES);
                if (v_rows == VT) {
                    tma_2d<PAIR>(dst, &maps.w, s * STEP_COLS, v0, bar);
                } else {
                    for (int i = 0; i < v_rows; i += UNIT) tma_2d<PAIR>(dst + i * STEP_BYTES, &maps.w16, s * STEP_COLS, v0 + i, bar);
                }
            };
            auto load_x = [&](int s, int st) {
                tma_2d<PAIR>(base + (uint32_t)(st * a.stage_bytes + A_BYTES), &maps.x, s * STEP_COLS, row_tile * a.tile_cols + half * x_rows,
                             lead_bar<PAIR>(&ctl.full[st]));
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
                HeadPacks<PAIR> packs(a, row_tile);
                HeadSlot slot[MAX_PACK];
                int chunk[MAX_PACK], u_bytes;
                while (const int n = packs.next(slot, chunk, &u_bytes)) {
                    if (!take()) break;
                    const uint32_t dst = base + (uint32_t)(stage * a.stage_bytes), bar = lead_bar<PAIR>(&ctl.full[stage]);
                    expect(n * v_rows * U_RANKS * 2 + u_bytes);
                    uint32_t u_dst = dst + A_BYTES;
#pragma unroll
                    for (int i = 0; i < MAX_PACK; i++) {
                        if (i >= n) continue;
                        const uint32_t b_dst = dst + (uint32_t)(i * B_BYTES);
                        const int row = chunk[i] * a.b_rows + v0 / 4;  // four vocabulary rows to 128 bytes
                        if (v_rows == VT) {
                            tma_3d<PAIR>(b_dst, &maps.b, 0, row, slot[i].adapter, bar);
                        } else {
                            for (int r = 0; r < v_rows / 4; r += UNIT / 4)
                                tma_3d<PAIR>(b_dst + r * 128, &maps.b16, 0, row + r, slot[i].adapter, bar);
                        }
                        const int u_n = slot[i].n / CTAS, u_row = chunk[i] * a.u_rows + slot[i].u_row + half * u_n;
                        for (int r = 0; r < u_n; r += a.u_box)  // two rows of u to 128 bytes
                            tma_2d<PAIR>(u_dst + r * U_BYTES, &maps.u, 0, (u_row + r) / 2, bar);
                        u_dst += (uint32_t)(u_n * U_BYTES);
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
        if (lane == 0 && lead) {
            int stage = 0, round = 0;
            uint32_t phase = 0;
            bool ok = true;
            auto take = [&]() {
                ok = head_wait(&ctl.full[stage], phase, &ctl.abort);
                tmem_fence_after();
                return ok;
            };
            auto advance = [&]() {
                mma_commit<PAIR>(&ctl.empty[stage]);
                if (++stage == a.stages) stage = 0, phase ^= 1;
            };
            uint32_t acc = 0;
            auto begin_round = [&]() {
                ok = head_wait(&ctl.acc_empty[round & 1], ((round >> 1) & 1) ^ 1, &ctl.abort);
                tmem_fence_after();
                acc = tmem + (uint32_t)(round & 1) * MAX_COLS;
                return ok;
            };
            auto end_round = [&]() { mma_commit<PAIR>(&ctl.acc_full[round++ & 1]); };
            const uint32_t shape = E4M3 ? shape_e4m3<PAIR>(a.tile_cols) : shape_bf16<PAIR>(a.tile_cols);
            const uint64_t zero = operand(blocks(U_RANKS * 16), zeros);
            while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
                for (int s = 0; s < a.w_steps; s++) {
                    const bool first = s % ROUND == 0;
                    if (first && !begin_round()) break;
                    if (!take()) break;
                    const uint32_t src = base + (uint32_t)(stage * a.stage_bytes);
#pragma unroll
                    for (int k = 0; k < STEP_BYTES; k += 32) {
                        mma<PAIR, E4M3>(acc, operand(SWIZZLED_ROWS, src + k), operand(SWIZZLED_ROWS, src + A_BYTES + k), shape, !first || k > 0);
                    }
                    advance();
                    if (s % ROUND == ROUND - 1 || s == a.w_steps - 1) {
                        if (!(a.slots_on && !own_round && s == a.w_steps - 1)) end_round();
                    }
                }
                if (!ok || !a.slots_on) continue;
                wait_for_front();
                HeadPacks<PAIR> packs(a, row_tile);
                if (own_round) {
                    if (packs.at == packs.end) continue;
                    if (!begin_round()) break;
                    // the slots' windows may cover a tile in part only: zero times zero first
                    mma<PAIR, false>(acc, zero, zero, shape_bf16<PAIR>(a.tile_cols), false);
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
                        const uint32_t d = acc + (uint32_t)slot[i].col, n_shape = shape_bf16<PAIR>(slot[i].n);
                        const uint64_t bd = operand(blocks(U_RANKS * 16), src + (uint32_t)(i * B_BYTES));
                        mma<PAIR, false>(d, bd, operand(blocks(U_BYTES * 8), u_src), n_shape, true);
                        mma<PAIR, false>(d, bd, operand(blocks(U_BYTES * 8), u_src + 256), n_shape, true);
                        u_src += (uint32_t)(slot[i].n / CTAS * U_BYTES);
                    }
                    advance();
                }
                if (ok) end_round();
            }
            if (!ok) {  // what was issued ends before tensor memory is given back
                mma_commit<PAIR>(&ctl.drain);
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
                if (lane == 0) lead_arrive<PAIR>(&ctl.acc_empty[round & 1]);
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
    sync_all<PAIR>();  // a pair's products read both CTAs' shared memory, and their ends arrive in both
    if (threadIdx.x == 0 && ctl.abort && a.status) atomicOr(a.status, MANTLE_SAMPLE_STATUS_TIMEOUT);
    if (warp == WRITERS / 32 + 1) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

}  // namespace
