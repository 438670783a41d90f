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
// One CTA per SM, persistent over its tiles.  Warps 8 and 11 move operands with TMA into a ring of stages: warp 8 what
// depends on the vocabulary (128 rows of W, 128 bytes wide; or some adapters' B, 16 ranks wide), warp 11 what depends on
// the batch (the same slice of x, or the windows of u).  Warp 9 issues tcgen05.mma from the ring, warps 0-7 read
// accumulators out of tensor memory, add them up in registers and write the finished tile while the next one is
// computed.  Warp 10 works out, a lane each, what every step of the tile's adapters copies and multiplies, ahead of the
// three that issue: an instruction that starts a copy or a product costs its warp some hundred cycles, and what
// stands around it comes on top (one adapter's step of 64 rows took a single copying warp 490 cycles; it has 4 KB of
// B, which HBM delivers in 170).
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
// Shorter rounds cost the writers more than they give: 256 columns halve the error again (4.3e-7 to 2.2e-7 after 1024
// columns) and take 4096 rows of 151 936 x 1024 from 1232 to 1666 us; and one length for every batch keeps a row's bits
// the same in all of them.
//
// u comes as bfloat16 side by side, its parts of 8 bits each: three products with the same B cost no more of its bytes
// and keep the 24 bits of float32 (64 rows with 16 adapters: 90 us, 85 with two parts and 16 bits).  Bfloat16 logits take
// two.  With 8-bit operands the projection's rounds are scaled by row and column, and the adapters have a round of their own.
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
constexpr int HEAD_NT = WRITERS + 128;
constexpr int ZERO_BYTES = VT * 32;
constexpr int SEGMENT = 96;        // adapters' steps that are worked out at a time; a multiple of 2, 3 and 4

struct __align__(16) HeadCtl {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2], steps_full[2], steps_empty[2], drain;
    uint32_t tmem;
    int abort;
    int n_steps[2], more[2];  // of a segment, and whether the tile has another
    int4 steps[2][SEGMENT];   // a step: row of its B in 128-byte rows, adapter, row of its u, first column and columns
    long long out_of[MAX_COLS], base_of[MAX_COLS];  // a column's row, as a distance in bytes
    float scale_of[MAX_COLS];
};

struct HeadArgs {
    int rows, vocab, w_steps, tile_cols, row_tiles, v_tiles;
    int front_is_ours;                // prepare kernels of the same call stand in front
    int slots_on, sorted, copied;     // adapters; perm comes from the kernels in front; x does
    int chunks, u_rows, u_box;        // u_box: rows of u of one copy
    int pack, pack_bytes;             // adapters' steps in one stage, and the room of each
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
    CUtensorMap w[4], x, b[4], u;  // w and b: copies of 128, 64, 32 and 16 vocabulary rows; b and u: plain 128-byte rows
};

// ---- the instructions
//
// Warps 8, 9 and 11 run as whole warps, all lanes with the same values, and only the instructions that act take a predicate
// (`on`, true in one lane): the operands then live in the uniform registers that these instructions want.  As the
// code of a single thread every stage's four products took 515 cycles to issue, whatever their size: that alone was
// as long as W takes to come from HBM.

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_on(uint32_t bar, bool on) {
    asm volatile("{.reg .pred q; setp.ne.b32 q, %1, 0; @q mbarrier.arrive.shared::cta.b64 _, [%0];}" ::"r"(bar), "r"((int)on) : "memory");
}
// Announces the bytes of a stage's copies, and that these are all; the next one: that there are more to come.
__device__ __forceinline__ void mbar_expect_on(uint32_t bar, uint32_t bytes, bool on) {
    asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;}" ::"r"(bar), "r"(bytes), "r"((int)on) : "memory");
}
__device__ __forceinline__ void mbar_expect_more_on(uint32_t bar, uint32_t bytes, bool on) {
    asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; @q mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;}" ::"r"(bar), "r"(bytes), "r"((int)on) : "memory");
}
// The address of a barrier in the pair's even CTA (PAIR), or in this one.
template <bool PAIR>
__device__ __forceinline__ uint32_t lead_bar(uint32_t bar) {
    if (PAIR) asm volatile("mapa.shared::cluster.u32 %0, %0, 0;" : "+r"(bar));
    return bar;
}
template <bool PAIR>
__device__ __forceinline__ void lead_arrive(uint64_t* bar) {
    if (PAIR) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_bar<true>(smem_u32(bar))) : "memory");
    else mbar_arrive(bar);
}
// Copies to this CTA's shared memory that complete on a barrier of the pair's even CTA (bar: lead_bar's).
template <bool PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, bool on) {
    if (PAIR)
        asm volatile("{.reg .pred q; setp.ne.b32 q, %5, 0; @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];}"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "r"((int)on) : "memory");
    else
        asm volatile("{.reg .pred q; setp.ne.b32 q, %5, 0; @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];}"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "r"((int)on) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar, bool on) {
    if (PAIR)
        asm volatile("{.reg .pred q; setp.ne.b32 q, %6, 0; @q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];}"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"((int)on) : "memory");
    else
        asm volatile("{.reg .pred q; setp.ne.b32 q, %6, 0; @q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];}"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"((int)on) : "memory");
}

// Shared-memory matrix descriptors of K-major operands.  W and x: rows of 128 bytes, swizzled, 1024 bytes from eight
// rows to the next eight.  B and u: blocks of 8 rows by 16 bytes, 128 bytes from one block of a row to the next, and
// `group` bytes from eight rows to the next eight.
// (As two words: the low one holds the address and the distance of blocks, the high one all that does not change.)
constexpr uint32_t SWIZZLED_ROWS_LO = 1u << 16, SWIZZLED_ROWS_HI = 1024u >> 4 | 1u << 14 | 2u << 29;
constexpr uint32_t BLOCKS_LO = 128u >> 4 << 16, B_BLOCKS_HI = 256u >> 4 | 1u << 14;
__device__ constexpr uint32_t u_blocks_hi(int parts) { return 8u * u_bytes(parts) >> 4 | 1u << 14; }
__device__ __forceinline__ uint32_t operand_lo(uint32_t format, uint32_t addr) { return format | ((addr >> 4) & 0x3fff); }
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
__device__ __forceinline__ void mma(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t shape, bool add, bool on) {
#define MANTLE_MMA(GROUP, KIND)                                                                                                  \
    asm volatile("{.reg .pred p, q; .reg .b64 a, b; setp.ne.b32 p, %6, 0; setp.ne.b32 q, %7, 0; mov.b64 a, {%1, %2}; mov.b64 b, {%3, %4}; " \
                 "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], a, b, %5, p;}"                                        \
                 ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(shape), "r"((int)add), "r"((int)on) : "memory")
    if (PAIR && E4M3) MANTLE_MMA("2", "f8f6f4");
    else if (PAIR) MANTLE_MMA("2", "f16");
    else if (E4M3) MANTLE_MMA("1", "f8f6f4");
    else MANTLE_MMA("1", "f16");
#undef MANTLE_MMA
}
// Arrives on `bar` -- of both CTAs of a pair -- when the products issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar, bool on) {
    if (PAIR)
        asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;}"
                     ::"r"(bar), "h"((uint16_t)3), "r"((int)on) : "memory");
    else
        asm volatile("{.reg .pred q; setp.ne.b32 q, %1, 0; @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];}"
                     ::"r"(bar), "r"((int)on) : "memory");
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

// The same for all lanes of a warp together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 8; i++)
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *abort)) return false;
        if (__any_sync(0xffffffffu, global_ns() - t0 > WAIT_LIMIT_NS)) {
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
    constexpr int PARTS = u_parts(OUT16), U_BYTES = u_bytes(PARTS);
    constexpr uint32_t U_BLOCKS_HI = u_blocks_hi(PARTS);
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
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (own_round) {
        for (int i = threadIdx.x; i < ZERO_BYTES / 16; i += HEAD_NT)
            reinterpret_cast<uint4*>(ring + a.stages * a.stage_bytes)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; s++) {
            mbar_init(&ctl.full[s], 2);  // the announcements of warps 8 and 11
            mbar_init(&ctl.empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&ctl.acc_full[i], 1);
            mbar_init(&ctl.acc_empty[i], WRITERS / 32 * CTAS);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&ctl.steps_full[i], 1);
            mbar_init(&ctl.steps_empty[i], lead ? 3 : 2);
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
    // Launched before the kernel in front has ended, so that all this overlaps its end.  That kernel is this call's own
    // (which starts no earlier than what was in front of it has ended) or, without prepare kernels, anybody's.
    if (!a.front_is_ours) pdl_wait();
    HeadTiles<PAIR> tiles(a);
    int v0, v_rows, row_tile;
    // what the kernels in front wrote may be read from here on (each thread asks once, where it first needs it)
    bool behind = false;
    auto wait_for_front = [&]() {
        if (!behind) pdl_wait();
        behind = true;
    };
    const uint32_t full0 = smem_u32(ctl.full), empty0 = smem_u32(ctl.empty);  // barriers of stage 0, 8 bytes each
    if (warp == WRITERS / 32 || warp == WRITERS / 32 + 3) {
        const bool v_side = warp == WRITERS / 32;  // W and B; else x and u
        const bool on = lane == 0, on_lead = on && lead;
        const int x_rows = a.tile_cols / CTAS, half = PAIR ? blockIdx.x & 1 : 0;
        const uint32_t stage_bytes = (uint32_t)a.stage_bytes;
        int filled = 0, stage = 0, segment = 0;  // filled: stages in use so far
        uint32_t phase = 1, dst = base;          // phase of `empty`: the first round passes
        bool ok = true;
        auto take = [&]() { return ok = warp_wait(empty0 + 8 * stage, phase, &ctl.abort); };
        auto advance = [&]() {
            filled = max(filled, ++stage);
            dst += stage_bytes;
            if (stage == a.stages) stage = 0, phase ^= 1, dst = base;
        };
        // v_rows vocabulary rows in as few copies as their sizes allow
        auto copy_w = [&](int x, uint32_t bar) {
            if (v_rows == VT) {
                tma_2d<PAIR>(dst, &maps.w[0], x, v0, bar, on);
                return;
            }
#pragma unroll 1
            for (int m = 1, v = 0; m < 4; m++) {
                if (v_rows & VT >> m) {
                    tma_2d<PAIR>(dst + v * STEP_BYTES, &maps.w[m], x, v0 + v, bar, on);
                    v += VT >> m;
                }
            }
        };
        auto copy_b = [&](int row, int adapter, uint32_t to, uint32_t bar) {  // four vocabulary rows to 128 bytes
            if (v_rows == VT) {
                tma_3d<PAIR>(to, &maps.b[0], 0, row, adapter, bar, on);
                return;
            }
#pragma unroll 1
            for (int m = 1, r = 0; m < 4; m++) {
                if (v_rows & VT >> m) {
                    tma_3d<PAIR>(to + r * 128, &maps.b[m], 0, row + r, adapter, bar, on);
                    r += (VT >> m) / 4;
                }
            }
        };
        auto fence_front = [&]() {
            if (!behind) {
                wait_for_front();
                asm volatile("fence.proxy.async.global;" ::: "memory");
            }
        };
        // W and B do not come from the kernels in front: their copies start while those still run
        if (!v_side && a.copied) fence_front();
        while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
            // the even CTA of a pair awaits the bytes of both; a barrier counts them in any order
            const uint32_t bytes = (uint32_t)((v_side ? v_rows : x_rows) * STEP_BYTES * CTAS);
#pragma unroll 1
            for (int s = 0; s < a.w_steps; s++) {
                if (!take()) break;
                const uint32_t bar = lead_bar<PAIR>(full0 + 8 * stage);
                mbar_expect_on(full0 + 8 * stage, bytes, on_lead);
                if (v_side) copy_w(s * STEP_COLS, bar);
                else tma_2d<PAIR>(dst + A_BYTES, &maps.x, s * STEP_COLS, row_tile * a.tile_cols + half * x_rows, bar, on);
                advance();
            }
            if (!ok || !a.slots_on) continue;
            if (!v_side) fence_front();
            bool more = true;
            for (; ok && more; segment++) {
                const int table = segment & 1;
                ok = warp_wait(smem_u32(&ctl.steps_full[table]), (segment >> 1) & 1, &ctl.abort);
                if (!ok) break;
                const int n = __shfl_sync(0xffffffffu, ctl.n_steps[table], 0);
                more = __shfl_sync(0xffffffffu, ctl.more[table], 0);
                int place = 0;  // of a step in its stage
                uint32_t to = 0, bar = 0;
                int4 step = ctl.steps[table][0];
#pragma unroll 1
                for (int i = 0; i < n; i++) {
                    const int4 next = ctl.steps[table][min(i + 1, SEGMENT - 1)];
                    if (place == 0) {
                        if (!take()) break;
                        to = dst;
                        bar = lead_bar<PAIR>(full0 + 8 * stage);
                    }
                    if (v_side) {
                        mbar_expect_more_on(full0 + 8 * stage, (uint32_t)(v_rows * U_RANKS * 2 * CTAS), on_lead);
                        copy_b(step.x + v0 / 4, step.y, to, bar);
                    } else {
                        const int u_n = __shfl_sync(0xffffffffu, (step.w >> 16) / CTAS, 0);
                        mbar_expect_more_on(full0 + 8 * stage, (uint32_t)(u_n * U_BYTES * CTAS), on_lead);
#pragma unroll 1
                        for (int r = 0; r < u_n; r += a.u_box)  // eight rows of u to a whole number of 128 bytes
                            tma_2d<PAIR>(to + B_BYTES + r * U_BYTES, &maps.u, 0, u_lines(step.z + half * u_n + r, PARTS), bar, on);
                    }
                    to += (uint32_t)a.pack_bytes;
                    if (++place == a.pack || i == n - 1) {
                        mbar_arrive_on(full0 + 8 * stage, on_lead);
                        place = 0;
                        advance();
                    }
                    step = next;
                }
                if (ok) mbar_arrive_on(smem_u32(&ctl.steps_empty[table]), on);
            }
        }
        // every copy has landed before the CTA may end, whether its stage was used or not
        if (ok) {
            for (int i = 0; i < a.stages; i++) {  // (a stage never filled counts as empty)
                if (!take()) break;
                advance();
            }
        }
        if (!ok && on) {
            // the last fill of every stage in use: of this turn of the ring before `stage`, of the turn before from there on
            for (int i = 0; i < filled; i++)
                mbar_wait(&ctl.full[i], (i < stage ? phase : phase ^ 1) ^ 1, 100000000ull);
        }
        __syncwarp();
    } else if (warp == WRITERS / 32 + 1) {
        if (lead) {
            const bool on = lane == 0;
            const uint32_t acc_full0 = smem_u32(ctl.acc_full), acc_empty0 = smem_u32(ctl.acc_empty);
            int stage = 0, round = 0, segment = 0;
            uint32_t phase = 0, src = base;
            bool ok = true;
            auto take = [&]() {
                ok = warp_wait(full0 + 8 * stage, phase, &ctl.abort);
                tmem_fence_after();
                return ok;
            };
            auto advance = [&]() {
                mma_commit<PAIR>(empty0 + 8 * stage, on);
                src += (uint32_t)a.stage_bytes;
                if (++stage == a.stages) stage = 0, phase ^= 1, src = base;
            };
            uint32_t acc = 0;
            auto begin_round = [&]() {
                ok = warp_wait(acc_empty0 + 8 * (round & 1), ((round >> 1) & 1) ^ 1, &ctl.abort);
                tmem_fence_after();
                acc = tmem + (uint32_t)(round & 1) * MAX_COLS;
                return ok;
            };
            auto end_round = [&]() {
                mma_commit<PAIR>(acc_full0 + 8 * (round & 1), on);
                round++;
            };
            const uint32_t shape = E4M3 ? shape_e4m3<PAIR>(a.tile_cols) : shape_bf16<PAIR>(a.tile_cols);
            while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
                for (int s0 = 0; s0 < a.w_steps; s0 += ROUND) {
                    if (!begin_round()) break;
                    const int s1 = min(s0 + ROUND, a.w_steps);
#pragma unroll 1
                    for (int s = s0; s < s1; s++) {
                        if (!take()) break;
                        const uint32_t w_lo = operand_lo(SWIZZLED_ROWS_LO, src), x_lo = operand_lo(SWIZZLED_ROWS_LO, src + A_BYTES);
#pragma unroll
                        for (int k = 0; k < STEP_BYTES / 32; k++)
                            mma<PAIR, E4M3>(acc, w_lo + 2 * k, SWIZZLED_ROWS_HI, x_lo + 2 * k, SWIZZLED_ROWS_HI, shape, k > 0 || s > s0, on);
                        advance();
                    }
                    if (!ok) break;
                    if (s1 < a.w_steps || !a.slots_on || own_round) end_round();
                }
                if (!ok || !a.slots_on) continue;
                if (own_round) {
                    if (!begin_round()) break;
                    // the slots' windows may cover a tile in part only, or not at all: zero times zero first
                    const uint32_t lo = operand_lo(BLOCKS_LO, zeros);
                    mma<PAIR, false>(acc, lo, B_BLOCKS_HI, lo, B_BLOCKS_HI, shape_bf16<PAIR>(a.tile_cols), false, on);
                }
                bool more = true;
                for (; ok && more; segment++) {
                    const int table = segment & 1;
                    ok = warp_wait(smem_u32(&ctl.steps_full[table]), (segment >> 1) & 1, &ctl.abort);
                    if (!ok) break;
                    const int n = __shfl_sync(0xffffffffu, ctl.n_steps[table], 0);
                    more = __shfl_sync(0xffffffffu, ctl.more[table], 0);
                    int place = 0;
                    uint32_t at = 0;
                    int window = ctl.steps[table][0].w;
#pragma unroll 1
                    for (int i = 0; i < n; i++) {
                        const int next = ctl.steps[table][min(i + 1, SEGMENT - 1)].w;
                        if (place == 0) {
                            if (!take()) break;
                            at = src;
                        }
                        window = __shfl_sync(0xffffffffu, window, 0);
                        const uint32_t d = acc + (uint32_t)(window & 0xffff), n_shape = shape_bf16<PAIR>(window >> 16);
                        const uint32_t b_lo = operand_lo(BLOCKS_LO, at), u_lo = operand_lo(BLOCKS_LO, at + B_BYTES);
#pragma unroll
                        for (int part = 0; part < PARTS; part++)
                            mma<PAIR, false>(d, b_lo, B_BLOCKS_HI, u_lo + part * (256 >> 4), U_BLOCKS_HI, n_shape, true, on);
                        at += (uint32_t)a.pack_bytes;
                        if (++place == a.pack || i == n - 1) {
                            place = 0;
                            advance();
                        }
                        window = next;
                    }
                    if (ok) mbar_arrive_on(smem_u32(&ctl.steps_empty[table]), on);
                }
                if (ok) end_round();
            }
            if (!ok) {  // what was issued ends before tensor memory is given back
                mma_commit<PAIR>(smem_u32(&ctl.drain), on);
                if (on) mbar_wait(&ctl.drain, 0, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == WRITERS / 32 + 2) {
        if (a.slots_on) {
            wait_for_front();
            bool ok = true;
            int segment = 0;
            while (ok && tiles.next(&v0, &v_rows, &row_tile)) {
                const int first = a.tile_first[row_tile], total = (a.tile_first[row_tile + 1] - first) * a.chunks;
                int at = 0;
                do {  // (a tile without adapters: one segment of nothing)
                    const int table = segment & 1, n = min(SEGMENT, total - at);
                    int free = 1;
                    if (lane == 0) free = head_wait(&ctl.steps_empty[table], ((segment >> 1) & 1) ^ 1, &ctl.abort);
                    ok = __shfl_sync(0xffffffffu, free, 0);
                    if (!ok) break;
                    for (int i = lane; i < n; i += 32) {
                        const HeadSlot slot = a.slots[first + (at + i) / a.chunks];
                        const int chunk = (at + i) % a.chunks;
                        ctl.steps[table][i] = make_int4(chunk * a.b_rows, slot.adapter, chunk * a.u_rows + slot.u_row, slot.col | slot.n << 16);
                    }
                    at += n;
                    if (lane == 0) {
                        ctl.n_steps[table] = n;
                        ctl.more[table] = at < total;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl.steps_full[table]);
                    segment++;
                } while (at < total);
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
            const int rounds = w_rounds + own_round;
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
