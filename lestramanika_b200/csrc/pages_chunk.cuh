// pages_chunk.cuh - attention of many rows over the paged cache, on the
// sm_100a tensor cores (tcgen05, accumulators in TMEM).
//
// A CTA takes 256 consecutive rows of one (sequence, KV head), a row being a
// (token, query head of the group) pair, as two 128-row tiles A and B that
// share every tile of keys; with several pieces a CTA takes one piece of the
// keys and leaves (maximum, sum, O) for the merge.
//   warps 21, 22 look pages up and ask for the rows of K and of V: BF16 pages with TMA
//               tensor copies of a cell's 16 rows straight into the operands'
//               layout (128-byte swizzle), 8-bit pages with bulk copies of the
//               codes into the place of their operands, and their scales;
//   warps 16-19 turn a tile's codes in place into 16-bit operands (K-major K,
//               MN-major V); of BF16 pages they only clear V rows that no row
//               sees, or that are not finite and not seen by all;
//   warp 20     one lane issues tcgen05.mma: S_X = Q_X K^T, O_X += P_X V,
//               P_X read from TMEM, in the order PV_A, S_A, PV_B, S_B so that one
//               tile's softmax runs under the other's products;
//   warps 0-7, 8-15  softmax of tile A, B: two threads share a row, one for each
//               half of a tile's keys. They mask, keep the running maximum
//               (which moves only when a score passes it by 2^8: the two
//               warps of 32 rows vote, and only then read each other's half) and
//               write P over S.
// 8-bit codes become F16 numbers code * 2^(e - E), exact for e - E down to -24
// (int8) or -15 (E4M3), see pages_decode.cuh: K has one E for 32 keys of a tile, which the
// softmax undoes in the factor it applies anyway;
// V has a running one per 32 elements, which a tile may pass by 2^5 (int8) or 2^7 (E4M3)
// before it moves, and moving it rescales O. Elements keep the order that is cheapest to unpack;
// Q is written, and O read, in the same order. BF16 pages are copied and
// multiplied as they are.
//
// BF16 rows: q is exact in one operand (as F16 it is scaled to a row maximum near
// 2^15); P is rounded to F16 (2^-12) or, on BF16 pages, to BF16 (2^-9).
// F32 rows: q and P are sums of two F16 (22 bits) or three BF16 (24 bits)
// numbers with a product each, which keeps F32 accuracy at two or three times
// the products.
//
// What bounds it, by a tile of 128 keys and 256 rows: the products take 2048
// tensor cycles a part of q and p at D = 128 (1.1 us at 1.9 GHz), the softmax of both tiles
// the issue slots of about 2 us, under which the products run: 2.25 us with BF16 rows on BF16
// pages, 2.6 on 8-bit ones, whose codes four warps turn over meanwhile; F32 rows 4.9 and 8.1 (two and three
// operands, tiles of 64 keys). Twins, 128 rows or fewer: 1.5 and 2.0. An item of 256 rows adds about 10 us
// that nothing hides, one CTA filling an SM: page ids and q (3 us), the first
// keys and softmax (5 us), the epilogue (3 us).
// Measured (us): 2048 tokens on 8192, 32 / 8 heads, E4M3: 383 (808 TFLOP/s); 4 prompts of 2048, 32 / 32 heads,
// BF16: 236 to 243 (583 to 566, by GPU); 2 ragged ones up to 4001, window 1000, F32, D = 64, int8: 118;
// 8 x 16 tokens on ragged contexts up to 4096, int8: 35.
// Registers: 80 a softmax thread; 8-bit pages, D = 64 and F32 rows spill 196 bytes of them.
//
// Every wait is bounded; one that gives up records an error, and the CTA
// lets its MMAs drain and frees its TMEM before it ends.
#pragma once
#include <cuda.h>

#include "pages_decode.cuh"
#include "tcgen05.cuh"

namespace pages {

using namespace tc;

template <int KV, int D, int ROWS>
struct ChunkTile {
    static constexpr bool BF = KV == BF16;
    static constexpr int NP = ROWS == PICKLE_CUDA_ROW_BF16 ? 1 : BF ? 3 : 2;      // operands a q or p is split into
    // The tensor cores cut their sums off instead of rounding them, always towards 0, once a product: the small parts of
    // P get sums of their own where TMEM has room (1.3e-6 without, D = 64 after 1000 keys).
    static constexpr bool APART = NP == 2 && D == 64;
    static constexpr int TILES = NP == 3 && D == 128 ? 1 : 2;                      // 128-row tiles
    static constexpr int BN = NP > 1 && D == 128 ? 64 : 128;                       // keys of a tile
    static constexpr int ROWS_CTA = TILES * 128;
    static constexpr int Q_HALF = 128 * 128, Q_TILE = Q_HALF * (D / 64);           // bytes: 64 columns, a tile
    static constexpr int KV_HALF = BN * 128, KV_TILE = KV_HALF * (D / 64);
    static constexpr int SMEM_KV = TILES * NP * Q_TILE;
    static constexpr int STAGE = 2 * KV_TILE;
    static constexpr int AUX = BF ? 3040 : 6656;                                  // barriers and words, below
    static constexpr int FIT = (232448 - AUX - SMEM_KV) / STAGE;
    static constexpr int STAGES = FIT >= 4 ? 4 : 2;
    static constexpr int SMEM_AUX = SMEM_KV + STAGES * STAGE;
    static constexpr int SMEM = SMEM_AUX + AUX;                                    // from a 1024-byte boundary on
    // Codes land where their operands will be: row r's D codes in the upper half of what row r (D = 128) or its cell
    // (D = 64) becomes, and are turned over in place.
    PCU_DEV static int raw_at(int r) { return D == 128 ? KV_HALF + r * 128 : r / CELL * (CELL * 128) + CELL * 64 + r % CELL * 64; }
    static_assert(FIT >= 2, "the ring needs two stages");
    static_assert(STAGES * STAGE >= 16 * 4096, "the epilogue's staging reuses the ring");
};

constexpr int CHUNK_THREADS = 768;
constexpr int CHUNK_STAGE_WARP = 16, CHUNK_MMA_WARP = 20, CHUNK_LOAD_WARP = 21;
// Registers a thread after the split: 16 softmax, 4 staging, 4 other warps; 32 * (16 * 80 + 4 * 72 + 4 * 88) = 61440, what
// 768 threads of 80 were launched with.
// Barrier `id` of 64 threads; whether any of them says so.
PCU_DEV bool bar_any(int id, bool x) {
    uint32_t y;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(y) : "r"(id), "r"((uint32_t)x) : "memory");
    return y != 0;
}
// The lowest n bits, n of any size or sign.
PCU_DEV uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
PCU_DEV void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
PCU_DEV void bulk_g2s_at(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// Bytes that a phase of the barrier waits for, besides its arrivals.
PCU_DEV void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
PCU_DEV void sts128(uint32_t to, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
PCU_DEV uint4 lds128(uint32_t from) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    return v;
}

template <int N>
PCU_DEV void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
PCU_DEV void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 16-bit operands (BF16 or F16), F32 accumulation, M = 128, A K-major, B K-major or MN-major.
__host__ __device__ constexpr uint32_t chunk_idesc(bool bf, int n, int b_mn) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

PCU_DEV void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// P's TMEM columns of k-step ks (16 keys, 8 columns), part p of tile x. They lie over S, of which 32 columns are read
// again just before their P is written: one part packs a half's keys at its start, two parts share the 32 columns of
// their own keys; a third has columns of its own.
template <int BN, int NP>
PCU_DEV uint32_t p_column(int x, int ks, int p) {
    if (p == 2) return 384 + x * 64 + ks * 8;
    if (NP == 1) return x * 128 + ks / (BN / 32) * (BN / 2) + ks % (BN / 32) * 8;
    return x * 128 + (ks >> 1) * 32 + p * 16 + (ks & 1) * 8;
}

// Where a row's element d lies in the operand order of 8-bit pages: eights of the upper 64 elements change places
// pairwise (the two halves of a 16-code chunk are then stored without bank conflicts), and an I8 four is
// (0, 2, 1, 3), as two logic operations unpack it.
template <int KV, int D>
__host__ __device__ constexpr int operand_pos(int d) {
    if (KV == BF16) return d;
    const int eight = (d >> 3) ^ (D == 128 && d >= 64 ? 1 : 0), i = d & 3;
    return eight * 8 + (d & 4) + (KV == I8 ? (i == 1 ? 2 : i == 2 ? 1 : i) : i);
}

template <int KV, int D, int ROWS>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
pages_chunk_kernel(const __grid_constant__ CUtensorMap tm, const AttnArgs a) {
    using T = ChunkTile<KV, D, ROWS>;
    constexpr bool BF = T::BF;
    constexpr int NP = T::NP, BN = T::BN, STAGES = T::STAGES, NB = D / 32;
    constexpr float P_SHIFT = BF ? 0.f : 7.f, GROW = 8.f;
    constexpr int SLACK = Slack<KV>::value;
    enum { Q_FULL = 0, S_FULL = 2, P_FULL = 4, O_DONE = 6, DRAIN = 8, K_FULL = 9, K_EMPTY = K_FULL + STAGES,
           V_FULL = K_EMPTY + STAGES, V_EMPTY = V_FULL + STAGES, RAW_K = V_EMPTY + STAGES, RAW_V = RAW_K + STAGES,
           N_BARS = RAW_V + STAGES };
    static_assert(N_BARS * 8 <= 320, "barriers");
    // What the loading warp tells the others of a tile outlives the tile's K: K's stage is free once its S is made,
    // while the softmax of that S still runs.
    constexpr int INFO = 4 * STAGES;
    constexpr int NCT = BN / CELL;                 // cells of a tile
    constexpr int HOLES = 64;
    extern __shared__ __align__(1024) unsigned char base[];
    // Of a tile: K's reference exponents (a quarter of the keys each), V's (a byte per 32 elements), the keys of each cell
    // that some row sees (bit 16: and that lie on a bad page), whether there are any of those. Scales: the tile's
    // scale bytes, a word a key. qexp: what a row of q was scaled by, as an exponent.
    struct Aux {
        uint64_t bars[N_BARS];
        uint32_t km[INFO][4], vref[INFO], need[2][INFO][NCT];
        int bad[INFO];
        uint32_t scale[BF ? 1 : STAGES][2][BF ? 4 : BN];
        unsigned char qexp[256];
        uint32_t tmem, twin_vref;
        int abort;
        // Keys that are not finite: 8-bit K or V with a scale of 255, V of BF16 pages where not all rows see all keys. 0
        // times one would be no 0, so it counts as 0 in the products, and the epilogue makes NaN of the rows that see
        // it. Cells with such keys in tiles that some row does not see whole (at most 7 tiles of 128 keys), as (first
        // position, keys); everyone: there is one that all rows see.
        uint2 hole[HOLES];
        int n_holes, everyone;
    };
    static_assert(sizeof(Aux) <= T::AUX, "the words behind the operands");
    Aux& aux = *reinterpret_cast<Aux*>(base + T::SMEM_AUX);
    auto& s_km = aux.km;
    auto& s_vref = aux.vref;
    auto& s_need = aux.need;
    auto& s_bad = aux.bad;
    auto& s_scale = aux.scale;
    int& s_abort = aux.abort;

    const View& w = a.w;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    griddep_launch_dependents();
    const int b = blockIdx.x / w.HK, hk = blockIdx.x % w.HK;
    const int qb = gridDim.y - 1 - blockIdx.y, split = blockIdx.z;       // later rows (more keys) first
    int row0, n, kv;
    const int chunk = piece_steps<BN>(a, lane);
    if (!seq_bounds(w, b, row0, n, kv)) return;
    if (qb * T::ROWS_CTA >= n * a.G) return;
    const ChunkWork cw = chunk_work<BN, T::ROWS_CTA>(a, row0, n, kv, qb, chunk);
    if (split > 0 && split >= cw.pieces) return;
    const int t0 = split * chunk, t1 = min(cw.span.n, t0 + chunk), n_tiles = t1 - t0;
    // Tile A ends with an earlier position than the block: the key tiles it has to see.
    const bool has_b = T::TILES == 2 && cw.r0 + 128 < cw.R;
    // Rows for one tile only: both work on it, A on the even tiles of keys and B on the odd ones, so that one's softmax
    // still runs under the other's products; their results are joined in the epilogue.
    const bool twin = T::TILES == 2 && !has_b && n_tiles > 1;
    const int last_a = cw.pos0 + min(cw.R - 1, cw.r0 + 127) / a.G;
    const int seen_a = last_a < 0 ? 0 : last_a / BN + 1;
    const int reach_a = max(0, min(n_tiles, min(cw.span.sunk, seen_a) + max(0, seen_a - cw.span.lo) - t0));
    const int n_a = twin ? (n_tiles + 1) / 2 : reach_a, n_b = twin ? n_tiles / 2 : has_b ? n_tiles : 0;
    const int n_all = twin ? n_tiles : max(n_a, n_b);
    auto tile_of = [&](int x, int i) { return twin ? 2 * i + x : i; };      // tile x's i-th tile of keys
    // Keys `keys` of the cell at position key0, of the tile from j0 on, are not finite.
    auto hole = [&](int j0, int key0, uint32_t keys) {
        if (!keys) return;
        const bool edge = j0 + BN - 1 > cw.pos0 + cw.r0 / a.G || (a.window > 0 && j0 <= cw.last - a.window && j0 + BN - 1 >= a.sinks);
        const int k = edge ? atomicAdd(&aux.n_holes, 1) : HOLES;
        if (k < HOLES) aux.hole[k] = make_uint2((uint32_t)key0, keys);
        else aux.everyone = 1;
    };
    // Tiles [edge_a, edge_b) of this piece lie at or before the block's first position and, with a window, inside all of its
    // rows' windows: they need no second look.
    auto tile_at = [&](int step) { return (step < cw.span.lo ? min(step, cw.span.sunk) : step - cw.span.lo + cw.span.sunk) - t0; };
    const int edge_a = a.window > 0 ? tile_at(max(0, cw.last - a.window + BN) / BN) : 0;
    const int edge_b = tile_at(max(0, cw.pos0 + cw.r0 / a.G + 1) / BN);
    auto on_edge = [&](int j) { return j < edge_a || j >= edge_b; };

    // Softmax warps: 16 of their tile's q rows each, D / 8 lanes a row. The first QA of the QSTEPS loads are on their
    // way while barriers and TMEM are set up (asked for after that, four by four, q was there 3 us later).
    constexpr int LPR = D / 8, QSTEPS = 16 * LPR / 32, QA = ROWS == PICKLE_CUDA_ROW_F32 && QSTEPS > 4 ? 4 : QSTEPS;
    const int qx = warp >> 3;                                      // their tile of rows
    const bool takes_q = warp < CHUNK_STAGE_WARP && (qx ? has_b && n_b > 0 : n_a > 0);
    const int q_row = (warp & 7) * 16 + lane / LPR;                // first of the lane's rows
    RawRow8<ROWS> q_raw[QA];
    auto ask_q = [&](int s0) {
        #pragma unroll
        for (int k = 0; k < QA; ++k) {
            const int q = cw.r0 + qx * 128 + q_row + (s0 + k) * (32 / LPR), t = div_group(q, a);
            q_raw[k].clear();
            if (q < cw.R)
                q_raw[k].load(a.q, (size_t)(cw.row0 + t) * a.q_stride + (size_t)(hk * a.G + q - t * a.G) * D + 8 * (lane % LPR));
        }
    };
    if (takes_q) ask_q(0);

    // Loading warps: lane c < NCT looks after cell c of a tile. need: its keys that some row sees; a page id is asked for two
    // tiles before it is used, and the cell's bytes are asked for in L2 a tile before they are copied.
    const uint32_t cpp = w.page_size / CELL;
    struct Cell {
        uint32_t at, need;
    };
    auto ask = [&](int j, int& id) {
        Cell x{0u, 0u};
        id = 0;
        if (j < n_all && lane < NCT) {
            const int k0 = cw.span.step(t0 + j) * BN + lane * CELL;
            x.need = bits_below(cw.last + 1 - k0) & 0xffffu;
            if (k0 < cw.span.lo_key) x.need &= ~bits_below(cw.span.lo_key - k0) | bits_below(a.sinks - k0);
            if (x.need) {
                const uint32_t cell = (uint32_t)k0 / CELL, page = cell / cpp;
                id = w.table[(size_t)b * w.table_stride + page];
                x.at = cell - page * cpp;
            }
        }
        return x;
    };
    // With its page's id: the cell in the pool; on a bad page none of its keys is there.
    auto look = [&](Cell x, int id) {
        if (x.need) {
            if ((unsigned)id < (unsigned)w.n_pages) {
                x.at += ((uint32_t)id * w.HK + hk) * cpp;
            } else {
                x.need = 0x10000u;
                record_error(w.err, PCU_DEVERR_ARG);
            }
        }
        return x;
    };
    auto want = [](const Cell& x) { return (x.need & 0xffffu) != 0; };
    auto cell_at = [&](const Cell& x) { return w.pool + (size_t)x.at * cell_bytes(KV, D); };
    // The first tiles' pages are looked up, and the first tile asked for in L2, while the rest is set up.
    Cell x0{0u, 0u}, x1{0u, 0u}, far{0u, 0u};
    int id2 = 0;
    if (warp >= CHUNK_LOAD_WARP && warp <= CHUNK_LOAD_WARP + 1) {
        int id0, id1;
        x0 = ask(0, id0);
        x1 = ask(1, id1);
        far = ask(2, id2);
        x0 = look(x0, id0);
        x1 = look(x1, id1);
        if (warp > CHUNK_LOAD_WARP && want(x0)) bulk_prefetch_l2(cell_at(x0), cell_bytes(KV, D));
    }

    const uint32_t base_u32 = smem_u32(base);
    if (base_u32 & 1023u) {                        // the operands' swizzle goes by address bits
        record_error(w.err, PCU_DEVERR_ARG);
        return;
    }
    uint64_t* bars = aux.bars;
    if (tid == CHUNK_THREADS - 32) {               // of a warp that has nothing else to do here
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bars[Q_FULL + x], 8);
            mbar_init(&bars[S_FULL + x], 2);      // the products, and the thread that saw the tile's words
            mbar_init(&bars[P_FULL + x], 8);
            mbar_init(&bars[O_DONE + x], 2);
        }
        mbar_init(&bars[DRAIN], 1);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bars[K_FULL + s], BF ? 1 : 4);       // BF16: the TMA copies themselves
            mbar_init(&bars[V_FULL + s], 4);
            mbar_init(&bars[K_EMPTY + s], 2);       // by the softmax of the tiles that read it: see there
            mbar_init(&bars[V_EMPTY + s], 2);
            mbar_init(&bars[RAW_K + s], 1);
            mbar_init(&bars[RAW_V + s], 1);
        }
        mbar_fence_init();
        s_abort = 0;
        aux.n_holes = aux.everyone = 0;
    }
    if (warp == CHUNK_MMA_WARP) tmem_alloc(&aux.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = aux.tmem;
    auto aborted = [&]() { return *(volatile int*)&s_abort != 0; };
    auto fail = [&](int code) { record_error(w.err, code); *(volatile int*)&s_abort = 1; };

    if (warp >= CHUNK_MMA_WARP) {
        regs_up<88>();
        if (warp == CHUNK_MMA_WARP) {
          if (lane == 0) {
            // ---------------- MMA issue ----------------
            // One instance of each product's code. A commit holds the tensor pipe up for about 100 cycles, so only S (and
            // the last O) has one: the softmax that waits for it passes on that K, and the V before, are free.
            const uint32_t id_s = chunk_idesc(BF, BN, 0), id_o = chunk_idesc(BF, D, 1);
            const uint64_t q_desc = smem_desc(base_u32, 16, 1024), k_desc = smem_desc(base_u32 + T::SMEM_KV, 16, 1024);
            const uint64_t v_desc = smem_desc(base_u32 + T::SMEM_KV + T::KV_TILE, T::KV_HALF, 1024);
            bool ok = true;
            int k_ready = -1, v_ready = -1;
            auto wait_tile = [&](int bar, int& ready, int j) {
                if (ok && j > ready) {
                    ok = mbar_wait(&bars[bar + j % STAGES], (j / STAGES) & 1);
                    ready = j;
                }
                tc_fence_after();
            };
            #pragma unroll 1
            for (int i = -1; ok && i < max(n_a, n_b); ++i) {
                #pragma unroll 1
                for (int x = 0; x < 2 && ok; ++x) {
                    const int n_x = x ? n_b : n_a;
                    if (i >= 0 && i < n_x) {
                        const int j = tile_of(x, i);
                        const uint64_t vd = v_desc + (((j % STAGES) * T::STAGE) >> 4);
                        wait_tile(V_FULL, v_ready, j);
                        ok = ok && mbar_wait(&bars[P_FULL + x], i & 1);
                        if (!ok) break;
                        tc_fence_after();
                        #pragma unroll
                        for (int p = 0; p < NP; ++p)
                            #pragma unroll
                            for (int k = 0; k < BN / 16; ++k)
                                mma_bf16_ts(tmem + 256 + x * D + (T::APART && p > 0 ? 128 : 0), tmem + p_column<BN, NP>(x, k, p),
                                            vd + (k * 16 * 128 >> 4), id_o, i > 0 || (p > 0 && !T::APART) || k > 0);
                        if (i + 1 == n_x) {
                            mma_commit(&bars[O_DONE + x]);
                            mbar_arrive(&bars[O_DONE + x]);
                        }
                        // Twins: this tile's next S needs the K two tiles on, too late a sign for the V that follows it.
                        if (twin) {
                            mma_commit(&bars[V_EMPTY + j % STAGES]);
                            mbar_arrive(&bars[V_EMPTY + j % STAGES]);
                        }
                    }
                    if (i + 1 < n_x) {
                        const int j = tile_of(x, i + 1), xq = twin ? 0 : x;
                        if (i < 0) ok = mbar_wait(&bars[Q_FULL + xq], 0);
                        wait_tile(K_FULL, k_ready, j);
                        if (!ok) break;
                        const uint64_t qd = q_desc + ((xq * NP * T::Q_TILE) >> 4), kd = k_desc + (((j % STAGES) * T::STAGE) >> 4);
                        #pragma unroll
                        for (int p = 0; p < NP; ++p)
                            #pragma unroll
                            for (int ks = 0; ks < D / 16; ++ks)
                                mma_bf16(tmem + x * 128, qd + ((p * T::Q_TILE + (ks / 4) * T::Q_HALF + (ks % 4) * 32) >> 4),
                                         kd + (((ks / 4) * T::KV_HALF + (ks % 4) * 32) >> 4), id_s, p > 0 || ks > 0);
                        mma_commit(&bars[S_FULL + x]);
                        mbar_arrive(&bars[S_FULL + x]);
                    }
                }
            }
            if (!ok) fail(PCU_DEVERR_MMA_WAIT);
            mma_commit(&bars[DRAIN]);
            if (!mbar_wait(&bars[DRAIN], 0)) record_error(w.err, PCU_DEVERR_DRAIN_WAIT);
          }
        } else if (warp <= CHUNK_LOAD_WARP + 1) {
            const int v = warp - CHUNK_LOAD_WARP;          // K or V: a copy costs its issuer some 80 cycles
            // ---------------- pages -> shared memory ----------------
            bool ok = true;
            auto wait = [&](int bar, int phase) { ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars[bar], phase & 1) && !aborted()); };
            // 8-bit: scale words of keys 32 q + lane of the next tile; V's reference exponents.
            uint32_t ks[BN / 32], vs[BN / 32], ev = 0;
            auto scales = [&](const Cell& x) {
                #pragma unroll
                for (int q = 0; q < BN / 32; ++q) {
                    const uint32_t at = __shfl_sync(0xffffffffu, x.at, 2 * q + lane / CELL);
                    const uint32_t need = __shfl_sync(0xffffffffu, x.need, 2 * q + lane / CELL);
                    const int r = lane % CELL;
                    const unsigned char* cell = w.pool + (size_t)at * cell_bytes(KV, D);
                    ks[q] = vs[q] = 0;
                    if ((need >> r) & 1) {
                        if (D == 128) {
                            ks[q] = *reinterpret_cast<const uint32_t*>(cell + k_scale(D, r));
                            vs[q] = *reinterpret_cast<const uint32_t*>(cell + v_scale(D, r));
                        } else {
                            ks[q] = *reinterpret_cast<const uint16_t*>(cell + k_scale(D, r));
                            vs[q] = *reinterpret_cast<const uint16_t*>(cell + v_scale(D, r));
                        }
                    }
                }
            };
            if (!BF) scales(x0);
            int issued = 0;                        // tiles asked for
            #pragma unroll 1
            for (int j = 0; j < n_all; ++j) {
                const int i = j % INFO, st = j % STAGES;
                if (v && want(x1)) bulk_prefetch_l2(cell_at(x1), cell_bytes(KV, D));
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, want(x0))) * CELL * D * elem_bytes(KV);
                const int bad = __any_sync(0xffffffffu, x0.need >> 16);
                if (j >= STAGES) wait((v ? V_EMPTY : K_EMPTY) + st, j / STAGES - 1);
                if (!ok) break;
                const uint32_t dst = base_u32 + T::SMEM_KV + st * T::STAGE + v * T::KV_TILE + (BF ? lane * CELL * 128 : T::raw_at(lane * CELL));
                uint64_t* bar = &bars[(v ? RAW_V : BF ? K_FULL : RAW_K) + st];
                // BF16: two boxes of 64 columns and 16 rows for each of a cell's K and V. 8-bit: a cell's codes, where
                // staging turns them over; they are asked for before the scales, which come from the same cells, are looked at.
                auto copy = [&]() {
                    __syncwarp();
                    if (want(x0)) {
                        if constexpr (BF) {
                            for (int h = 0; h < D / 64; ++h)
                                tma_load_2d(dst + h * T::KV_HALF, &tm, 64 * h, (int)(x0.at * 2 * CELL + v * CELL), bar);
                        } else {
                            bulk_g2s_at(dst, cell_at(x0) + (v ? v_row(KV, D, 0) : 0), CELL * D, bar);
                        }
                    }
                    ++issued;
                };
                if (!BF) {
                    if (lane == 0 && bytes) mbar_expect_tx(bar, bytes);
                    copy();
                }
                uint32_t km[BN / 32], vm = 0;
                if (!BF && v == 0) {
                    // K: one reference for 32 keys. V: a reference moves where the tile's largest exponent passes it by
                    // more than the slack. A second time around without scales of 255.
                    uint32_t top[NB];
                    #pragma unroll 1
                    for (;;) {
                        uint32_t most = 0;
                        #pragma unroll
                        for (int q = 0; q < BN / 32; ++q) {
                            uint32_t m = ks[q] & 255u;
                            #pragma unroll
                            for (int k = 1; k < NB; ++k) m = max(m, (ks[q] >> (8 * k)) & 255u);
                            km[q] = __reduce_max_sync(0xffffffffu, m);
                            most = max(most, km[q]);
                        }
                        #pragma unroll
                        for (int k = 0; k < NB; ++k) {
                            uint32_t m = 0;
                            #pragma unroll
                            for (int q = 0; q < BN / 32; ++q) m = max(m, (vs[q] >> (8 * k)) & 255u);
                            top[k] = __reduce_max_sync(0xffffffffu, m);
                            most = max(most, top[k]);
                        }
                        if (most != 255u) break;
                        #pragma unroll
                        for (int q = 0; q < BN / 32; ++q) {
                            const uint32_t k255 = __vcmpeq4(ks[q], 0xffffffffu), v255 = __vcmpeq4(vs[q], 0xffffffffu);
                            const uint32_t keys = __ballot_sync(0xffffffffu, (k255 | v255) != 0);
                            ks[q] &= ~k255;
                            vs[q] &= ~v255;
                            const int j0 = cw.span.step(t0 + j) * BN;
                            if (lane < 2) hole(j0, j0 + 32 * q + CELL * lane, (keys >> (CELL * lane)) & 0xffffu);
                        }
                    }
                    #pragma unroll
                    for (int k = 0; k < NB; ++k) {
                        const uint32_t old = (ev >> (8 * k)) & 255u;
                        vm |= (top[k] > old + SLACK ? top[k] : old) << (8 * k);
                    }
                    ev = vm;
                }
                if (lane < NCT) s_need[v][i][lane] = x0.need;
                if (!BF) {
                    #pragma unroll
                    for (int q = 0; q < BN / 32; ++q)
                        s_scale[st][v][32 * q + lane] = v ? vs[q] & ~__vcmpeq4(vs[q], 0xffffffffu) : ks[q];
                }
                if (v == 0 && lane == 0) {
                    s_bad[i] = bad;
                    if (!BF) {
                        s_vref[i] = ev;
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) s_km[i][k] = km[k * (BN / 32) / 4];
                    }
                }
                __syncwarp();
                if (BF) {
                    if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
                    copy();
                } else {
                    if (lane == 0) mbar_arrive(bar);
                    scales(x1);
                }
                x0 = x1;
                x1 = look(far, id2);
                far = ask(j + 3, id2);
            }
            if (!ok || aborted()) {
                // What was asked for must land before shared memory goes away: the last STAGES tiles cover it.
                for (int j = max(0, issued - STAGES); j < issued; ++j)
                    if (!mbar_wait(&bars[(v ? RAW_V : BF ? K_FULL : RAW_K) + j % STAGES], (j / STAGES) & 1) && lane == 0)
                        record_error(w.err, PCU_DEVERR_DRAIN_WAIT);
                if (!ok && lane == 0) fail(PCU_DEVERR_EMPTY_WAIT);
            }
        }
    } else if (warp >= CHUNK_STAGE_WARP) {
        regs_down<72>();
        // ---------------- codes -> operands ----------------
        constexpr int KPW = BN / 4;                                 // keys of a tile that this warp turns over
        const int sw = warp - CHUNK_STAGE_WARP;
        bool ok = true;
        auto wait = [&](int bar, int phase) { ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars[bar], phase & 1) && !aborted()); };
        auto full = [&](int bar, int j) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[bar + j % STAGES]);
        };
        // The keys of row r's cell that some row sees, of tile j.
        auto need_of = [&](int v, int j, int r) { return s_need[v][j % INFO][r / CELL]; };
        if constexpr (BF) {
            for (int j = 0; j < n_all; ++j) {
                wait(RAW_V + j % STAGES, j / STAGES);
                if (!ok) break;
                // Rows that no row of the call sees may hold anything, and 0 times a NaN is no 0: a lane a row.
                if (lane < KPW) {
                    const int r = sw * KPW + lane;
                    const uint32_t at = base_u32 + T::SMEM_KV + (j % STAGES) * T::STAGE + T::KV_TILE + r * 128;
                    bool no = !((need_of(1, j, r) >> (r % CELL)) & 1), inf = false;
                    if (on_edge(j)) {
                        // Nor may a row that is not finite reach rows that do not see it.
                        #pragma unroll
                        for (int i = 0; i < D / 8; ++i) inf |= bf16x8_bad(lds128(at + (i >> 3) * T::KV_HALF + ((i + lane) & 7) * 16));
                        inf = inf && !no;
                        no |= inf;
                        const uint32_t keys = __ballot_sync(KPW == 32 ? 0xffffffffu : 0xffffu, inf);
                        const int j0 = cw.span.step(t0 + j) * BN;
                        if (lane < KPW / CELL) hole(j0, j0 + sw * KPW + CELL * lane, (keys >> (CELL * lane)) & 0xffffu);
                    }
                    if (no) {
                        #pragma unroll
                        for (int i = 0; i < D / 8; ++i)
                            sts128(at + (i >> 3) * T::KV_HALF + (i & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
                    }
                }
                full(V_FULL, j);
            }
        } else {
            // A lane takes the 32 codes of a scale: D / 32 lanes a row. One loop body serves K (even steps) and V.
            constexpr int LPR = D / 32, RPS = 32 / LPR, NI = KPW / RPS;
            static_assert(NI >= 2, "two steps are in flight");
            const int k32 = lane % LPR, row0_l = lane / LPR;
            #pragma unroll 1
            for (int step = 0; step < 2 * n_all; ++step) {
                const int j = step >> 1, v = step & 1, i = j % INFO;
                wait((v ? RAW_V : RAW_K) + j % STAGES, j / STAGES);
                if (!ok) break;
                const uint32_t tile = base_u32 + T::SMEM_KV + (j % STAGES) * T::STAGE + v * T::KV_TILE;
                const uint32_t dst = tile + (k32 >> 1) * T::KV_HALF;
                const int ref = v ? (int)((s_vref[i] >> (8 * k32)) & 255u) : (int)s_km[i][sw];
                const unsigned char* sc = reinterpret_cast<const unsigned char*>(&s_scale[j % STAGES][v][sw * KPW]) + k32;
                bool whole = true;
                #pragma unroll
                for (int c = 0; c < KPW / CELL; ++c) whole = whole && (s_need[v][i][sw * (KPW / CELL) + c] & 0xffffu) == 0xffffu;
                #pragma unroll 1
                for (int q0 = 0; q0 < NI; q0 += 2) {
                    uint4 x[2][2];
                    uint32_t f[2], cc[2];
                    // Odd rows take their two chunks in the other order: eight lanes then read eight different banks.
                    #pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int row = (q0 + q) * RPS + row0_l, odd = row & 1;
                        const uint32_t from = tile + T::raw_at(sw * KPW + row) + k32 * 32;
                        x[q][0] = lds128(from + odd * 16);
                        x[q][1] = lds128(from + (odd ^ 1) * 16);
                        const float ff = rel_scale(sc[4 * row], ref);
                        f[q] = f16x2(ff, ff);
                        cc[q] = KV == I8 ? as_u32(__hmul2(as_half2(f[q]), __floats2half2_rn(-1152.f, -1152.f))) : 0u;
                    }
                    if (!whole) {
                        // Rows that no row of the call sees may hold anything, E4M3's NaN too.
                        #pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int r = sw * KPW + (q0 + q) * RPS + row0_l;
                            if (!((need_of(v, j, r) >> (r % CELL)) & 1)) x[q][0] = x[q][1] = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    __syncwarp();                  // a cell is read before any of it is written over
                    #pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int row = (q0 + q) * RPS + row0_l, r = sw * KPW + row;
                        #pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int c = 2 * k32 + (h ^ (row & 1));            // chunk of 16 codes
                            uint4 lo, hi;
                            codes_row<KV>(x[q][h].x, f[q], cc[q], lo.x, lo.y);
                            codes_row<KV>(x[q][h].y, f[q], cc[q], lo.z, lo.w);
                            codes_row<KV>(x[q][h].z, f[q], cc[q], hi.x, hi.y);
                            codes_row<KV>(x[q][h].w, f[q], cc[q], hi.z, hi.w);
                            // The upper chunks' halves change places, for the stores' banks.
                            const uint32_t to = dst + r * 128 + ((((2 * c) & 7) ^ (c >> 2) ^ (r & 7)) << 4);
                            sts128(to, lo);
                            sts128(to ^ 16, hi);
                        }
                    }
                }
                full(v ? V_FULL : K_FULL, j);
            }
        }
        if (!ok && lane == 0) fail(PCU_DEVERR_EMPTY_WAIT);
    } else {
        // ---------------- softmax: two threads per row of tile X, one for each half of the keys ----------------
        const int x = warp >> 3, hf = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tm = tmem + x * 128 + lane_off, o_tm = tmem + 256 + x * D + lane_off;
        const int n_x = x ? n_b : n_a;
        const int xr = twin ? 0 : x;                               // tile of rows
        const int r = cw.r0 + xr * 128 + row;                      // row of the sequence's KV head
        const bool live = r < cw.R && (xr == 0 || has_b);
        const int tok = div_group(r, a), head = hk * a.G + r - tok * a.G;
        const int p = live ? cw.pos0 + tok : -1;
        bool ok = true;
        if (takes_q) {
            // q into shared memory, in the operand order.
            const int i0 = 8 * (lane % LPR);
            #pragma unroll
            for (int s0 = 0; s0 < QSTEPS; s0 += QA) {
                if (s0) ask_q(s0);
                #pragma unroll
                for (int k = 0; k < QA; ++k) {
                    const int r_t = q_row + (s0 + k) * (32 / LPR);                // row of the tile
                    const Row8 v = q_raw[k].row();
                    float qs = 1.f;
                    if (!BF) {
                        uint32_t m = max(amax_bits(v.a), amax_bits(v.b));
                        #pragma unroll
                        for (int y = 1; y < LPR; y <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, y));
                        const uint32_t e = min(268u - (m >> 23), 254u);
                        qs = __uint_as_float(e << 23);
                        if (lane % LPR == 0) aux.qexp[x * 128 + r_t] = (unsigned char)e;
                    }
                    const float e[8] = {v.a.x * qs, v.a.y * qs, v.a.z * qs, v.a.w * qs, v.b.x * qs, v.b.y * qs, v.b.z * qs, v.b.w * qs};
                    constexpr int o1 = KV == I8 ? 2 : 1, o2 = KV == I8 ? 1 : 2;
                    uint32_t q0[NP], q1[NP], q2[NP], q3[NP];
                    split_parts<BF, NP>(e[0], e[o1], q0);
                    split_parts<BF, NP>(e[o2], e[3], q1);
                    split_parts<BF, NP>(e[4], e[4 + o1], q2);
                    split_parts<BF, NP>(e[4 + o2], e[7], q3);
                    const int c = operand_pos<KV, D>(i0) >> 3;                   // 16-byte chunk of the row
                    const uint32_t to = base_u32 + x * NP * T::Q_TILE + (c >> 3) * T::Q_HALF + r_t * 128 + (((c & 7) ^ (r_t & 7)) << 4);
                    #pragma unroll
                    for (int y = 0; y < NP; ++y) sts128(to + y * T::Q_TILE, make_uint4(q0[y], q1[y], q2[y], q3[y]));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[Q_FULL + x]);
        }
        // Positions of the tile's first and last rows: tiles of keys that all of them see need no mask.
        const int p_first = cw.pos0 + (cw.r0 + xr * 128) / a.G;
        const int p_last = cw.pos0 + min(cw.R - 1, cw.r0 + xr * 128 + 127) / a.G;
        // The two warps of 32 rows: barrier 1 + 4 x + quadrant.
        const int pair = 1 + x * 4 + (warp & 3);
        // A key tile that one tile of rows reads alone is passed on twice.
        auto pass_on = [&](int bar, int k) {
            const int j = tile_of(x, k);
            mbar_arrive(&bars[bar + j % STAGES]);
            if (twin || k >= (x ? n_a : n_b)) mbar_arrive(&bars[bar + j % STAGES]);
        };
        // Which of the 32 keys from position k0 on the row sees: at or before its own, inside its window or among the sinks.
        auto visible = [&](int k0) {
            const int hi = max(p, -1) - k0, sk = a.sinks - k0;
            const int lo = (a.window > 0 ? max(max(p, -1) - a.window, -1) : -1) - k0;
            return bits_below(hi + 1) & (~bits_below(lo + 1) | bits_below(sk));
        };
        float m_run = -INFINITY, l_run = 0.f, rf = a.scale_log2;
        uint32_t vref = 0;                     // V's references that O is relative to
        for (int i = 0; i < n_x; ++i) {
            const int s = tile_of(x, i) % INFO;
            ok = __all_sync(0xffffffffu, mbar_wait(&bars[S_FULL + x], i & 1));
            tc_fence_after();
            // S(i) is made, so its K is free, and so is the V of tile i - 1, whose products came before.
            if ((warp & 7) == 0 && lane == 0) {
                pass_on(K_EMPTY, i);
                if (i > 0 && !twin) pass_on(V_EMPTY, i - 1);
            }
            if (!BF && i == 0) rf = a.scale_log2 / __uint_as_float((uint32_t)aux.qexp[xr * 128 + row] << 23);
            const int j0 = cw.span.step(t0 + tile_of(x, i)) * BN;
            const bool bad = *(volatile int*)&s_bad[s] != 0;
            const bool masked = j0 + BN - 1 > p_first ||
                                (a.window > 0 && j0 <= p_last - a.window && j0 + BN - 1 >= a.sinks) || bad;
            // Columns [c0, c0 + 32) of the row's scores, those that it does not see as -inf. S is read twice, for the
            // maximum and for P, 32 columns at a time: registers and code stay small.
            auto scores = [&](int c0, float (&sc)[32]) {
                tmem_ld32(s_tm + c0, sc);
                if (masked) {
                    // Visible columns as bits; two instructions a column then.
                    uint32_t see = visible(j0 + c0);
                    if (bad) see &= (s_need[0][s][c0 / 16] & 0xffffu) | s_need[0][s][c0 / 16 + 1] << 16;
                    #pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(see & (1u << c))) sc[c] = -INFINITY;
                }
            };
            // The factor of a quarter of the keys; never 0, a masked score is -inf times it.
            auto factor = [&](int k) {
                const uint32_t e = BF ? 0u : s_km[s][k];
                return BF ? rf : fmaxf(rf * __uint_as_float(e << 23), 1.2e-38f);
            };
            constexpr int QN = BN / 4 < 32 ? BN / 4 : 32;             // columns under one factor
            auto half_max = [&](int h) {
                float m = -INFINITY;
                #pragma unroll 1
                for (int c0 = h * (BN / 2); c0 < (h + 1) * (BN / 2); c0 += 32) {
                    float sc[32];
                    scores(c0, sc);
                    #pragma unroll
                    for (int k = 0; k < 32; k += QN) {
                        float a0 = sc[k], a1 = sc[k + 1];
                        #pragma unroll
                        for (int c = 2; c < QN - 2; c += 4) {
                            a0 = fmax3(a0, sc[k + c], sc[k + c + 1]);
                            a1 = fmax3(a1, sc[k + c + 2], sc[k + c + 3]);
                        }
                        m = fmaxf(m, fmax3(fmaxf(a0, a1), sc[k + QN - 2], sc[k + QN - 1]) * factor((c0 + k) / (BN / 4)));
                    }
                }
                return m;
            };
            // Both halves' S is read before either's P is written over it.
            float m_tile = half_max(hf);
            float alpha = 1.0f;
            bool grow = false;
            if (bar_any(pair, m_tile > m_run + GROW || !ok)) {
                m_tile = fmaxf(m_tile, half_max(hf ^ 1));
                grow = m_tile > m_run + GROW;
                if (grow) {
                    alpha = ex2(m_run - m_tile);
                    m_run = m_tile;
                }
                // Either warp's give-up ends both.
                if (bar_any(pair, !ok)) {
                    ok = false;
                    break;
                }
            }
            const float nm = m_run == -INFINITY ? 0.f : P_SHIFT - m_run;
            const uint32_t vnow = BF ? 0u : s_vref[s];
            if (i > 0 && __any_sync(0xffffffffu, grow || vnow != vref)) {
                // This half's columns of O. S_FULL_X(i) implies PV_X(i - 1) is complete, and PV_X(i) waits for P_FULL.
                #pragma unroll 1
                for (int y = hf * (D / 64); y < (hf + 1) * (D / 64) + (T::APART ? 1 : 0); ++y) {
                    // (Apart: one step for the large part, one for the small.)
                    const int c = T::APART ? hf : y, at = c * 32 + (T::APART && y > hf ? 128 : 0);
                    float o[32];
                    tmem_ld32(o_tm + at, o);
                    const float g = BF ? alpha : alpha * rel_scale((vref >> (8 * c)) & 255, (vnow >> (8 * c)) & 255);
                    #pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] *= g;
                    tmem_st32(o_tm + at, o);
                }
            }
            float2 sm2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            #pragma unroll 1
            for (int c0 = hf * (BN / 2); c0 < (hf + 1) * (BN / 2); c0 += 32) {
                float sc[32];
                scores(c0, sc);
                uint32_t pk[NP][16];
                #pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float ff = factor((c0 + c / QN * QN) / (BN / 4));
                    const float2 e = ffma2(make_float2(sc[c], sc[c + 1]), make_float2(ff, ff), make_float2(nm, nm));
                    const float2 pp = make_float2(ex2(e.x), ex2(e.y));
                    sm2[(c >> 1) & 1] = fadd2(sm2[(c >> 1) & 1], pp);
                    uint32_t parts[NP];
                    split_parts<BF, NP>(pp.x, pp.y, parts);
                    #pragma unroll
                    for (int k = 0; k < NP; ++k) pk[k][c >> 1] = parts[k];
                }
                #pragma unroll
                for (int k = 0; k < NP; ++k) tmem_st16(tmem + lane_off + p_column<BN, NP>(x, c0 / 16, k), pk[k]);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bars[P_FULL + x]);
            }
            const float2 t = fadd2(sm2[0], sm2[1]);
            l_run = l_run * alpha + (t.x + t.y);
            vref = vnow;
        }
        // ---------------- epilogue ----------------
        // The ring becomes the output's staging once both tiles' products are done.
        // This tile of rows may end before the other: its last V goes on as well.
        if (ok && n_x > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[O_DONE + x], 0));
        if (ok && n_x > 0 && !twin && (warp & 7) == 0 && lane == 0) pass_on(V_EMPTY, n_x - 1);
        if (ok && (x ? n_a : n_b) > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[O_DONE + (x ^ 1)], 0));
        ok = __all_sync(0xffffffffu, ok && !aborted());
        if (n_x > 0 && (*(volatile int*)&aux.n_holes | *(volatile int*)&aux.everyone)) {
            bool sees_one = *(volatile int*)&aux.everyone != 0;
            for (int k = 0; k < min(HOLES, *(volatile int*)&aux.n_holes); ++k)
                sees_one |= (visible((int)aux.hole[k].x) & aux.hole[k].y) != 0;
            if (sees_one) l_run = __uint_as_float(0x7fc00000u);
        }
        // Each thread's maximum and sum: [tile][half][row], in the place of q.
        float2* s_ml = reinterpret_cast<float2*>(base);
        asm volatile("bar.sync 9, 512;" ::: "memory");             // all 16 warps are past the products
        if (ok) s_ml[(x * 2 + hf) * 128 + row] = make_float2(m_run, l_run);
        if (tid == 256) aux.twin_vref = vref;                      // tile B's, the same for all of its rows
        asm volatile("bar.sync 9, 512;" ::: "memory");
        if (ok && (x == 0 || has_b)) {
            tc_fence_after();
            l_run += s_ml[(x * 2 + (hf ^ 1)) * 128 + row].y;
            // Twins: A joins both. f_a, f_b: factors of the two outputs.
            float f_a = 1.f, f_b = 0.f;
            const uint32_t vref_b = aux.twin_vref;
            if (twin) {
                const float2 b0 = s_ml[2 * 128 + row], b1 = s_ml[3 * 128 + row];
                const float M = fmaxf(m_run, b0.x), Mz = M == -INFINITY ? 0.f : M;
                f_a = ex2(m_run - Mz);
                f_b = ex2(b0.x - Mz);
                l_run = l_run * f_a + (b0.y + b1.y) * f_b;
                m_run = M;
            }
            const bool whole = cw.pieces <= 1;
            const float inv = whole ? 1.0f / (l_run == 0.f ? 1.0f : l_run) : 1.0f;
            const size_t rows = (size_t)w.n_tok * a.H;
            if (!whole && live && hf == 0)
                *reinterpret_cast<float2*>(a.ws_ml + 2 * (split * rows + (size_t)(cw.row0 + tok) * a.H + head)) = make_float2(m_run, l_run);
            const uint32_t stage = base_u32 + T::SMEM_KV + warp * 4096;
            const int wr0 = cw.r0 + x * 128 + (warp & 3) * 32;         // the warp's first row
            // 32 columns a time through the warp's stage, 128 bytes a row of floats or 64 of BF16 numbers.
            #pragma unroll 1
            for (int c = hf * (D / 64); c < (hf + 1) * (D / 64); ++c) {
                float o[32];
                if (n_x > 0) {
                    tmem_ld32(o_tm + c * 32, o);
                    if (T::APART) {
                        float small[32];
                        tmem_ld32(o_tm + 128 + c * 32, small);
                        #pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] += small[k];
                    }
                } else {
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                }
                auto v_scale_of = [&](uint32_t ref) {
                    const uint32_t e = (ref >> (8 * c)) & 255u;
                    return BF ? 1.0f : __uint_as_float(e << 23);
                };
                const float ga = inv * f_a * (n_x > 0 ? v_scale_of(vref) : 1.0f);
                #pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= ga;
                if (twin) {
                    float ob[32];
                    tmem_ld32(o_tm + D + c * 32, ob);            // O_B: the same lanes, the next columns
                    if (T::APART) {
                        float small[32];
                        tmem_ld32(o_tm + D + 128 + c * 32, small);
                        #pragma unroll
                        for (int k = 0; k < 32; ++k) ob[k] += small[k];
                    }
                    const float gb = inv * f_b * v_scale_of(vref_b);
                    #pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = fmaf(ob[k], gb, o[k]);
                }
                // Columns are in the operand order: eights of the upper elements change places, fours may be (0, 2, 1, 3).
                const int swap = KV != BF16 && D == 128 ? c >> 1 : 0;
                constexpr int n1 = KV == I8 ? 2 : 1, n2 = KV == I8 ? 1 : 2;          // where elements 1 and 2 of a four lie
                const bool f32 = ROWS == PICKLE_CUDA_ROW_F32 || !whole;
                __syncwarp();
                if (f32) {
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        sts128(stage + lane * 128 + (((i ^ (swap << 1)) ^ (lane & 7)) << 4),
                               make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + n1]), __float_as_uint(o[4 * i + n2]),
                                          __float_as_uint(o[4 * i + 3])));
                } else {
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sts128(stage + lane * 128 + (((i ^ swap) ^ (lane & 7)) << 4),
                               make_uint4(bf16x2(o[8 * i], o[8 * i + n1]), bf16x2(o[8 * i + n2], o[8 * i + 3]),
                                          bf16x2(o[8 * i + 4], o[8 * i + 4 + n1]), bf16x2(o[8 * i + 4 + n2], o[8 * i + 7])));
                }
                __syncwarp();
                const int lpr = f32 ? 8 : 4, rps = 32 / lpr;           // lanes a row, rows a step
                #pragma unroll 4
                for (int i = 0; i < lpr; ++i) {
                    const int rr = rps * i + lane / lpr, ch = lane % lpr, q = wr0 + rr;
                    const uint4 v = lds128(stage + rr * 128 + ((ch ^ (rr & 7)) << 4));
                    if (q < cw.R) {
                        const int t = div_group(q, a), tk = cw.row0 + t, hd = hk * a.G + q - t * a.G;
                        if (f32) {
                            float* to = whole ? reinterpret_cast<float*>(a.out) + (size_t)tk * a.out_stride + hd * D
                                              : a.ws_o + (split * rows + (size_t)tk * a.H + hd) * D;
                            *reinterpret_cast<uint4*>(to + c * 32 + 4 * ch) = v;
                        } else {
                            __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)tk * a.out_stride + hd * D;
                            *reinterpret_cast<uint4*>(to + c * 32 + 8 * ch) = v;
                        }
                    }
                }
            }
        }
        if (!ok && lane == 0) fail(PCU_DEVERR_FULL_WAIT);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == CHUNK_MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace pages
