// pages_chunk.cuh - attention of many rows over the paged cache, on the
// sm_100a tensor cores (tcgen05, accumulators in TMEM).
//
// A CTA takes 256 consecutive rows of one (sequence, KV head), a row being a
// (token, query head of the group) pair, as two 128-row tiles A and B that
// share every tile of keys; with several pieces a CTA takes one piece of the
// keys and leaves (maximum, sum, O) for the merge.
//   warps 8-11  bring a tile of keys from its pages into shared memory as
//               16-bit numbers in the layout the MMAs read (K-major K,
//               MN-major V, 128-byte swizzle);
//   warp 12     one lane issues tcgen05.mma: S_X = Q_X K^T, O_X += P_X V,
//               P_X read from TMEM, in the order PV_A, S_A, PV_B, S_B so that one
//               tile's softmax runs under the other's products;
//   warps 0-3, 4-7  softmax of tile A, B: a thread owns a row. It masks, keeps
//               the running maximum (O is rescaled only when it grows by more
//               than 2^8) and writes P over S.
// 8-bit codes become F16 numbers code * 2^(e - E), exact but for elements
// 2^-24 below the reference: K has one E for the keys that a staging warp
// brings of a tile, which the softmax undoes in the factor it applies anyway;
// V has a running one per 32 elements, 2^7 of slack below F16's largest number, and
// moving it rescales O. Elements keep the order that is cheapest to unpack;
// Q is written, and O read, in the same order. BF16 pages are copied and
// multiplied as they are.
//
// BF16 rows: q is exact in one operand (as F16 it is scaled to a row maximum near
// 2^15); P is rounded to F16 (2^-12) or, on BF16 pages, to BF16 (2^-9).
// F32 rows: q and P are sums of two F16 (22 bits) or three BF16 (24 bits)
// numbers with a product each, which keeps F32 accuracy at two or three times
// the products.
//
// Every wait is bounded; one that gives up records an error, and the CTA
// lets its MMAs drain and frees its TMEM before it ends.
#pragma once
#include "pages_decode.cuh"
#include "tcgen05.cuh"

namespace pages {

using namespace tc;

template <int KV, int D, int ROWS>
struct ChunkTile {
    static constexpr bool BF = KV == BF16;
    static constexpr int NP = ROWS == PICKLE_CUDA_ROW_BF16 ? 1 : BF ? 3 : 2;      // operands a q or p is split into
    static constexpr int TILES = NP == 3 && D == 128 ? 1 : 2;                      // 128-row tiles
    static constexpr int BN = NP > 1 && D == 128 ? 64 : 128;                       // keys of a tile
    static constexpr int ROWS_CTA = TILES * 128;
    static constexpr int Q_HALF = 128 * 128, Q_TILE = Q_HALF * (D / 64);           // bytes: 64 columns, a tile
    static constexpr int KV_HALF = BN * 128, KV_TILE = KV_HALF * (D / 64);
    static constexpr int SMEM_KV = TILES * NP * Q_TILE;
    static constexpr int STAGE = 2 * KV_TILE;
    static constexpr int FIT = (232448 - 1024 - 1024 - SMEM_KV) / STAGE;
    static constexpr int STAGES = FIT > 4 ? 4 : FIT;
    static constexpr int SMEM_BAR = SMEM_KV + STAGES * STAGE;
    static constexpr int SMEM = SMEM_BAR + 1024 + 1024;                            // barriers and words; alignment
    static_assert(STAGES >= 2, "the ring needs two stages");
    static_assert(STAGES * STAGE >= 8 * 4096, "the epilogue's staging reuses the ring");
};

constexpr int CHUNK_THREADS = 512;
constexpr int CHUNK_STAGE_WARP = 8, CHUNK_MMA_WARP = 12;
// Registers a thread after the split: 8 softmax, 4 staging, 4 other warps; 32 * (8 * 176 + 4 * 112 + 4 * 48) = 65536,
// what 512 threads of 128 were launched with.
// The lowest n bits, n of any size or sign.
PCU_DEV uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
PCU_DEV void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
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

// 64 consecutive 32-bit columns of this thread's TMEM lane, waited for.
PCU_DEV void tmem_ld64(uint32_t taddr, float* v) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
    #pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// 128 consecutive 32-bit columns of this thread's TMEM lane, two loads in flight together.
PCU_DEV void tmem_ld2x64(uint32_t taddr, float* v) {
    uint32_t r[128];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%128];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
        "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
        "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
        "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%129];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
          "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
          "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
          "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
          "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
          "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
          "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
          "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
          "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
        : "r"(taddr), "r"(taddr + 64)
        : "memory");
    #pragma unroll
    for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(r[i]);
}

PCU_DEV void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
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
__global__ void __launch_bounds__(CHUNK_THREADS, 1) pages_chunk_kernel(const AttnArgs a) {
    using T = ChunkTile<KV, D, ROWS>;
    constexpr bool BF = T::BF;
    constexpr int NP = T::NP, BN = T::BN, STAGES = T::STAGES, NB = D / 32;
    constexpr float P_SHIFT = BF ? 0.f : 7.f, GROW = 8.f;
    constexpr int SLACK = 7;
    enum { Q_FULL = 0, S_FULL = 2, P_LO = 4, P_HI = 6, O_DONE = 8, DRAIN = 10, K_FULL = 11, K_EMPTY = K_FULL + STAGES,
           V_FULL = K_EMPTY + STAGES, V_EMPTY = V_FULL + STAGES, N_BARS = V_EMPTY + STAGES };
    static_assert(N_BARS * 8 <= 256, "barriers");
    // What staging tells the softmax of a tile outlives the tile's K: K's stage is free once its S is made, while the
    // softmax of that S still runs. A slot comes up again only after the S of STAGES tiles later.
    constexpr int INFO = 2 * STAGES;
    extern __shared__ unsigned char smem_raw[];
    // What staging tells the softmax of a stage: K's factors (one per staging warp), V's O factors (if any moved), V's
    // references, the keys that are really there.
    __shared__ __align__(16) float s_kf[INFO][4], s_vf[INFO][4], s_ve[INFO][4];
    __shared__ uint32_t s_there[INFO][4];
    __shared__ int s_flag[INFO];                // 1: V's references moved; 2: keys on a bad page
    __shared__ __align__(16) uint32_t s_vmax[2][4];
    __shared__ int s_stop[2];                     // a staging warp gave up: the four leave at the same tile
    __shared__ int s_abort;
    __shared__ uint32_t s_tmem;

    const View& w = a.w;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    griddep_launch_dependents();
    const int b = blockIdx.x / w.HK, hk = blockIdx.x % w.HK;
    const int qb = gridDim.y - 1 - blockIdx.y, split = blockIdx.z;       // later rows (more keys) first
    int row0, n, kv;
    if (!seq_bounds(w, b, row0, n, kv)) return;
    if (qb * T::ROWS_CTA >= n * a.G) return;
    const ChunkWork cw = chunk_work<BN, T::ROWS_CTA>(a, row0, n, kv, qb);
    if (split > 0 && split >= cw.pieces) return;
    const int t0 = split * a.chunk, t1 = min(cw.span.n, t0 + a.chunk), n_tiles = t1 - t0;
    // Tile A ends with an earlier position than the block: the key tiles it has to see.
    const bool has_b = T::TILES == 2 && cw.r0 + 128 < cw.R;
    const int last_a = cw.pos0 + min(cw.R - 1, cw.r0 + 127) / a.G;
    const int seen_a = last_a < 0 ? 0 : last_a / BN + 1;
    const int n_a = max(0, min(n_tiles, min(cw.span.sunk, seen_a) + max(0, seen_a - cw.span.lo) - t0));
    const int n_b = has_b ? n_tiles : 0, n_all = max(n_a, n_b);

    const uint32_t raw_u32 = smem_u32(smem_raw);
    const uint32_t base_u32 = (raw_u32 + 1023u) & ~1023u;
    unsigned char* base = smem_raw + (base_u32 - raw_u32);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + T::SMEM_BAR);
    if (tid == 0) {
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bars[Q_FULL + x], 4);
            mbar_init(&bars[S_FULL + x], 2);      // the products, and the thread that saw the tile's words
            mbar_init(&bars[P_LO + x], 4);
            mbar_init(&bars[P_HI + x], 4);
            mbar_init(&bars[O_DONE + x], 1);
        }
        mbar_init(&bars[DRAIN], 1);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bars[K_FULL + s], 4);
            mbar_init(&bars[V_FULL + s], 4);
            mbar_init(&bars[K_EMPTY + s], 1);
            mbar_init(&bars[V_EMPTY + s], 1);
        }
        mbar_fence_init();
        s_abort = s_stop[0] = s_stop[1] = 0;
    }
    if (warp == CHUNK_MMA_WARP) tmem_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    auto aborted = [&]() { return *(volatile int*)&s_abort != 0; };
    auto fail = [&](int code) { record_error(w.err, code); *(volatile int*)&s_abort = 1; };

    if (warp >= CHUNK_MMA_WARP) {
        regs_down<48>();
        if (warp == CHUNK_MMA_WARP && lane == 0) {
            // ---------------- MMA issue ----------------
            const uint32_t id_s = chunk_idesc(BF, BN, 0), id_o = chunk_idesc(BF, D, 1);
            auto kv_addr = [&](int j) { return base_u32 + T::SMEM_KV + (j % STAGES) * T::STAGE; };
            auto issue_s = [&](int x, int j) {
                #pragma unroll
                for (int p = 0; p < NP; ++p)
                    #pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        mma_bf16(tmem + x * 128,
                                 smem_desc(base_u32 + (x * NP + p) * T::Q_TILE + (ks / 4) * T::Q_HALF + (ks % 4) * 32, 16, 1024),
                                 smem_desc(kv_addr(j) + (ks / 4) * T::KV_HALF + (ks % 4) * 32, 16, 1024), id_s, p > 0 || ks > 0);
                mma_commit(&bars[S_FULL + x]);
                mbar_arrive(&bars[S_FULL + x]);
                // The last tile of rows that reads this K lets it go.
                if (x == 1 || j >= n_b) mma_commit(&bars[K_EMPTY + j % STAGES]);
            };
            auto issue_o = [&](int x, int j, int ks0) {
                #pragma unroll
                for (int p = 0; p < NP; ++p)
                    #pragma unroll
                    for (int k = 0; k < BN / 32; ++k) {
                        const int ks = ks0 + k;
                        const uint32_t p_tm = tmem + (p < 2 ? x * 128 + p * (BN / 2) : 384 + x * 64);
                        mma_bf16_ts(tmem + 256 + x * D, p_tm + ks * 8,
                                    smem_desc(kv_addr(j) + T::KV_TILE + ks * 16 * 128, T::KV_HALF, 1024), id_o,
                                    j > 0 || ks0 > 0 || p > 0 || k > 0);
                    }
            };
            bool ok = true;
            int k_ready = -1, v_ready = -1;
            auto wait_tile = [&](int bar, int& ready, int j) {
                if (ok && j > ready) {
                    ok = mbar_wait(&bars[bar + j % STAGES], (j / STAGES) & 1);
                    ready = j;
                }
                tc_fence_after();
            };
            for (int x = 0; x < 2 && ok; ++x)
                if (x ? n_b : n_a) {
                    ok = mbar_wait(&bars[Q_FULL + x], 0);
                    wait_tile(K_FULL, k_ready, 0);
                    if (ok) issue_s(x, 0);
                }
            for (int j = 0; ok && j < n_all; ++j) {
                for (int x = 0; x < 2 && ok; ++x) {
                    const int n_x = x ? n_b : n_a;
                    if (j >= n_x) continue;
                    ok = mbar_wait(&bars[P_LO + x], j & 1);
                    wait_tile(V_FULL, v_ready, j);
                    if (!ok) break;
                    issue_o(x, j, 0);
                    ok = mbar_wait(&bars[P_HI + x], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    issue_o(x, j, BN / 32);
                    if (j + 1 == n_x) mma_commit(&bars[O_DONE + x]);
                    if (x == 1 || j >= n_b) mma_commit(&bars[V_EMPTY + j % STAGES]);
                    if (j + 1 < n_x) {
                        wait_tile(K_FULL, k_ready, j + 1);
                        if (ok) issue_s(x, j + 1);
                    }
                }
            }
            if (!ok) fail(PCU_DEVERR_MMA_WAIT);
            mma_commit(&bars[DRAIN]);
            if (!mbar_wait(&bars[DRAIN], 0)) record_error(w.err, PCU_DEVERR_DRAIN_WAIT);
        }
    } else if (warp >= CHUNK_STAGE_WARP) {
        regs_down<112>();
        // ---------------- keys: pages -> operands ----------------
        constexpr int KPW = BN / 4;                                 // keys of a tile that this warp brings
        const int sw = warp - CHUNK_STAGE_WARP;
        const uint32_t cpp = w.page_size / CELL;
        // Lane i looks after key i of the warp's: its cell in the pool, or NONE where no row sees it. A page id is
        // asked for a tile before it is turned into a cell, so that nothing waits for the table.
        constexpr uint32_t NONE = 0xffffffffu;
        struct Ask {
            int id, cell_in_page;            // cell_in_page < 0: no row sees the key
        };
        struct Look {
            uint32_t at;
            bool bad;
        };
        // The pages of the warp's keys: KPW / CELL cells, so only one division a tile and lane.
        auto ask = [&](int j) {
            Ask x{0, -1};
            if (j < n_all && lane < KPW) {
                const int key = cw.span.step(t0 + j) * BN + sw * KPW + lane;
                if (key <= cw.last && (key >= cw.span.lo_key || key < a.sinks)) {
                    const uint32_t cell = (uint32_t)key / CELL, page = cell / cpp;
                    x.id = w.table[(size_t)b * w.table_stride + page];
                    x.cell_in_page = (int)(cell - page * cpp);
                }
            }
            return x;
        };
        auto look = [&](const Ask& q) {
            Look x{NONE, false};
            if (q.cell_in_page >= 0) {
                x.bad = (unsigned)q.id >= (unsigned)w.n_pages;
                if (!x.bad) x.at = ((uint32_t)q.id * w.HK + hk) * cpp + q.cell_in_page;
            }
            return x;
        };
        // Ask for a tile's rows in L2 (a lane its key's): the copies that come two tiles later then find them there
        // instead of waiting for DRAM with only a tile in flight.
        auto prefetch = [&](const Look& x) {
            if (x.at == NONE) return;
            const unsigned char* cell = w.pool + (size_t)x.at * cell_bytes(KV, D);
            const int r = lane % CELL;
            #pragma unroll
            for (int i = 0; i < D * elem_bytes(KV); i += 128) {
                prefetch_l2(cell + k_row(KV, D, r) + i);
                prefetch_l2(cell + v_row(KV, D, r) + i);
            }
            if (!BF && r == 0) prefetch_l2(cell + k_scale(D, 0));
        };
        auto row_ptr = [&](uint32_t at, int row, bool v) {
            return w.pool + (size_t)at * cell_bytes(KV, D) + (v ? v_row(KV, D, row % CELL) : k_row(KV, D, row % CELL));
        };
        bool ok = true;
        // Tell the softmax which keys are missing although some row sees them.
        auto publish = [&](int i, const Look& x, int moved) {
            const uint32_t there = __ballot_sync(0xffffffffu, x.at != NONE);
            const uint32_t bad = __ballot_sync(0xffffffffu, x.bad);
            if (lane == 0) {
                s_there[i][sw] = there;
                if (bad) {
                    atomicOr(&s_flag[i], 2);
                    record_error(w.err, PCU_DEVERR_ARG);
                }
                if (moved) atomicOr(&s_flag[i], 1);
            }
        };
        auto wait_empty = [&](int bar, int j) {
            if (ok && j >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&bars[bar + j % STAGES], ((j / STAGES) - 1) & 1));
        };
        // Wait until tile j's K may be written, clear its words, and meet the other staging warps; false: all four stop.
        auto begin = [&](int j) {
            wait_empty(K_EMPTY, j);
            if (lane == 0) {
                if (!ok || aborted()) *(volatile int*)&s_stop[j & 1] = 1;
                if (sw == 0) *(volatile int*)&s_flag[j % INFO] = 0;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            return *(volatile int*)&s_stop[j & 1] == 0;
        };
        auto full = [&](int bar, int j) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[bar + j % STAGES]);
        };
        if constexpr (BF) {
            constexpr int CPR = D / 8, RPI = 32 / CPR, NI = KPW / RPI;
            Ask far = ask(2);
            Look x = look(ask(0)), nxt = look(ask(1));
            prefetch(nxt);
            // Step 2j copies tile j's K, step 2j + 1 its V; a step is announced LAG steps after its copies went out.
            // V(j) waits for the products of tile j - STAGES, which wait for K(j - STAGES + 1), so LAG is 2 at most.
            constexpr int LAG = 2;
            for (int step = 0; step < 2 * n_all + LAG; ++step) {
                const int j = step >> 1, v = step & 1;
                if (j < n_all) {
                    if (v == 0) {
                        if (!begin(j)) break;
                        publish(j % INFO, x, 0);
                    } else {
                        wait_empty(V_EMPTY, j);
                    }
                    const uint32_t dst = base_u32 + T::SMEM_KV + (j % STAGES) * T::STAGE + v * T::KV_TILE;
                    #pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const int row = i * RPI + lane / CPR, c = lane % CPR, r = sw * KPW + row;
                        const uint32_t at = __shfl_sync(0xffffffffu, x.at, row);
                        const uint32_t to = dst + (c >> 3) * T::KV_HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                        cp_async16_or_zero(to, at == NONE ? w.pool : row_ptr(at, row, v) + c * 16, at == NONE ? 0u : 16u);
                    }
                    if (v) {
                        x = nxt;
                        nxt = look(far);
                        prefetch(nxt);
                        far = ask(j + 3);
                    }
                }
                cp_async_commit();
                if (step >= LAG) {
                    cp_async_wait<LAG>();
                    full((step - LAG) & 1 ? V_FULL : K_FULL, (step - LAG) >> 1);
                }
            }
            cp_async_wait<0>();
        } else {
            constexpr int CPR = D / 16, RPI = 32 / CPR, NI = KPW / RPI;
            uint32_t ev = 0;                       // V's reference exponents, a byte per 32 elements
            Ask far = ask(2);
            Look x0 = look(ask(0)), x1 = look(ask(1));
            prefetch(x1);
            uint32_t ks0 = 0, vs0 = 0, ks1 = 0, vs1 = 0;
            auto scales = [&](const Look& x, uint32_t& ks, uint32_t& vs) {
                ks = vs = 0;
                if (x.at == NONE) return;
                const unsigned char* cell = w.pool + (size_t)x.at * cell_bytes(KV, D);
                const int r = lane % CELL;
                if (D == 128) {
                    ks = *reinterpret_cast<const uint32_t*>(cell + k_scale(D, r));
                    vs = *reinterpret_cast<const uint32_t*>(cell + v_scale(D, r));
                } else {
                    ks = *reinterpret_cast<const uint16_t*>(cell + k_scale(D, r));
                    vs = *reinterpret_cast<const uint16_t*>(cell + v_scale(D, r));
                }
            };
            auto load = [&](const Look& x, bool v, uint4 (&q)[NI]) {
                #pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int row = i * RPI + lane / CPR, c = lane % CPR;
                    const uint32_t at = __shfl_sync(0xffffffffu, x.at, row);
                    q[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (at != NONE) q[i] = *reinterpret_cast<const uint4*>(row_ptr(at, row, v) + c * 16);
                }
            };
            // Chunk c of 16 codes of each row to its two 16-byte places, times 2^(e - ref).
            auto store = [&](uint32_t dst, const uint4 (&q)[NI], uint32_t sc, uint32_t ref) {
                #pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int row = i * RPI + lane / CPR, c = lane % CPR, r = sw * KPW + row;
                    const uint32_t e = (__shfl_sync(0xffffffffu, sc, row) >> (8 * (c >> 1))) & 255u;
                    const float ff = rel_scale((int)e, (int)((ref >> (8 * (c >> 1))) & 255u));
                    const uint32_t f = f16x2(ff, ff);
                    uint32_t cc = 0;
                    if (KV == I8) cc = as_u32(__hmul2(as_half2(f), __floats2half2_rn(-1152.f, -1152.f)));
                    uint4 lo, hi;
                    codes_row<KV>(q[i].x, f, cc, lo.x, lo.y);
                    codes_row<KV>(q[i].y, f, cc, lo.z, lo.w);
                    codes_row<KV>(q[i].z, f, cc, hi.x, hi.y);
                    codes_row<KV>(q[i].w, f, cc, hi.z, hi.w);
                    const uint32_t half = dst + (c >> 2) * T::KV_HALF + r * 128;
                    const int first = ((2 * c) & 7) ^ (c >> 2);
                    sts128(half + ((first ^ (r & 7)) << 4), lo);
                    sts128(half + (((first ^ 1) ^ (r & 7)) << 4), hi);
                }
            };
            uint4 kq[NI], vq[NI];
            scales(x0, ks0, vs0);
            load(x0, false, kq);
            for (int j = 0; j < n_all; ++j) {
                const int i = j % INFO;
                load(x0, true, vq);
                scales(x1, ks1, vs1);
                const Look x2 = look(far);
                prefetch(x2);
                far = ask(j + 3);
                // K: one reference for the warp's keys. V: the tile's maxima, through shared memory.
                uint32_t km = ks0 & 255u;
                #pragma unroll
                for (int k = 1; k < NB; ++k) km = max(km, (ks0 >> (8 * k)) & 255u);
                km = __reduce_max_sync(0xffffffffu, km);
                uint32_t vm = 0;
                #pragma unroll
                for (int k = 0; k < NB; ++k)
                    vm |= __reduce_max_sync(0xffffffffu, (vs0 >> (8 * k)) & 255u) << (8 * k);
                if (lane == 0) s_vmax[j & 1][sw] = vm;
                if (!begin(j)) break;
                // Every thread keeps all of V's references; lane k of warp 0 tells the softmax about block k.
                const uint4 vm4 = *reinterpret_cast<const uint4*>(s_vmax[j & 1]);
                const uint32_t top4 = __vmaxu4(__vmaxu4(vm4.x, vm4.y), __vmaxu4(vm4.z, vm4.w));
                const uint32_t old4 = ev;
                // Saturated bytes: top > old + SLACK.
                const uint32_t past = __vcmpgtu4(top4, __vaddus4(old4, 0x01010101u * SLACK));
                ev = (old4 & ~past) | (top4 & past);
                publish(i, x0, sw == 0 && past != 0);
                if (lane == 0) s_kf[i][sw] = km == 255u ? INFINITY : __uint_as_float(km << 23);
                if (sw == 0 && lane < NB) {
                    const uint32_t e = (ev >> (8 * lane)) & 255u, o = (old4 >> (8 * lane)) & 255u;
                    s_ve[i][lane] = e == 255u ? INFINITY : __uint_as_float(e << 23);
                    s_vf[i][lane] = rel_scale((int)o, (int)e);
                }
                const uint32_t dst = base_u32 + T::SMEM_KV + (j % STAGES) * T::STAGE;
                store(dst, kq, ks0, km * 0x01010101u);
                full(K_FULL, j);
                load(x1, false, kq);
                wait_empty(V_EMPTY, j);
                store(dst + T::KV_TILE, vq, vs0, ev);
                full(V_FULL, j);
                x0 = x1;
                x1 = x2;
                ks0 = ks1;
                vs0 = vs1;
            }
        }
        if (!ok && lane == 0) fail(PCU_DEVERR_EMPTY_WAIT);
    } else {
        regs_up<176>();
        // ---------------- softmax: one thread per row of tile X ----------------
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tm = tmem + x * 128 + lane_off, o_tm = tmem + 256 + x * D + lane_off;
        const int n_x = x ? n_b : n_a;
        const int r = cw.r0 + x * 128 + row;                       // row of the sequence's KV head
        const bool live = r < cw.R && (x == 0 || has_b);
        const int tok = r / a.G, head = hk * a.G + r % a.G;
        const int p = live ? cw.pos0 + tok : -1;
        bool ok = true;
        float rf = a.scale_log2;
        if (n_x > 0) {
            // The warp's 32 q rows into shared memory, in the operand order: D / 8 lanes a row, eight steps in flight.
            constexpr int LPR = D / 8, RPS = 32 / LPR, STEPS = 32 / RPS;
            const int i0 = 8 * (lane % LPR), wr0 = cw.r0 + x * 128 + (warp & 3) * 32;
            float my_qs = 1.f;
            #pragma unroll 1
            for (int s0 = 0; s0 < STEPS; s0 += 8) {
                Row8 v[8];
                #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int q = wr0 + (s0 + k) * RPS + lane / LPR;
                    v[k].a = v[k].b = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (q < cw.R)
                    {
                        const int t = div_group(q, a);
                        v[k] = load_row8<ROWS>(a.q, (size_t)(cw.row0 + t) * a.q_stride + (size_t)(hk * a.G + q - t * a.G) * D + i0);
                    }
                }
                #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int rr = (s0 + k) * RPS + lane / LPR;              // row of the warp
                    float qs = 1.f;
                    if (!BF) {
                        uint32_t m = max(amax_bits(v[k].a), amax_bits(v[k].b));
                        #pragma unroll
                        for (int y = 1; y < LPR; y <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, y));
                        qs = __uint_as_float(min(268u - (m >> 23), 254u) << 23);
                        const float theirs = __shfl_sync(0xffffffffu, qs, (lane % RPS) * LPR);
                        if (lane / RPS == s0 + k) my_qs = theirs;
                    }
                    const float e[8] = {v[k].a.x * qs, v[k].a.y * qs, v[k].a.z * qs, v[k].a.w * qs,
                                        v[k].b.x * qs, v[k].b.y * qs, v[k].b.z * qs, v[k].b.w * qs};
                    constexpr int o1 = KV == I8 ? 2 : 1, o2 = KV == I8 ? 1 : 2;
                    uint32_t q0[NP], q1[NP], q2[NP], q3[NP];
                    split_parts<BF, NP>(e[0], e[o1], q0);
                    split_parts<BF, NP>(e[o2], e[3], q1);
                    split_parts<BF, NP>(e[4], e[4 + o1], q2);
                    split_parts<BF, NP>(e[4 + o2], e[7], q3);
                    const int c = operand_pos<KV, D>(i0) >> 3, r_t = (warp & 3) * 32 + rr;      // 16-byte chunk, row of the tile
                    const uint32_t to = base_u32 + x * NP * T::Q_TILE + (c >> 3) * T::Q_HALF + r_t * 128 + (((c & 7) ^ (r_t & 7)) << 4);
                    #pragma unroll
                    for (int y = 0; y < NP; ++y) sts128(to + y * T::Q_TILE, make_uint4(q0[y], q1[y], q2[y], q3[y]));
                }
            }
            rf = a.scale_log2 / my_qs;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[Q_FULL + x]);
        }
        // Positions of the tile's first and last rows: tiles of keys that all of them see need no mask.
        const int p_first = cw.pos0 + (cw.r0 + x * 128) / a.G;
        const int p_last = cw.pos0 + min(cw.R - 1, cw.r0 + x * 128 + 127) / a.G;
        float m_run = -INFINITY, l_run = 0.f;
        float4 ve = make_float4(1.f, 1.f, 1.f, 1.f);
        for (int j = 0; j < n_x; ++j) {
            const int s = j % INFO;
            ok = __all_sync(0xffffffffu, mbar_wait(&bars[S_FULL + x], j & 1));
            if (!ok) break;
            tc_fence_after();
            float sc[BN];
            if constexpr (BN == 128) tmem_ld2x64(s_tm, sc);
            else tmem_ld64(s_tm, sc);
            const int j0 = cw.span.step(t0 + j) * BN;
            const int flag = *(volatile int*)&s_flag[s];
            if (j0 + BN - 1 > p_first || (a.window > 0 && j0 <= p_last - a.window && j0 + BN - 1 >= a.sinks) || (flag & 2)) {
                // The row's visible columns as bits: at or before its position, inside its window or among the
                // sinks, and really there. Two instructions a column then.
                const int hi = max(p, -1) - j0, sk = a.sinks - j0;
                const int lo = (a.window > 0 ? max(max(p, -1) - a.window, -1) : -1) - j0;
                #pragma unroll
                for (int k = 0; k < BN / 32; ++k) {
                    uint32_t see = bits_below(hi + 1 - 32 * k) & (~bits_below(lo + 1 - 32 * k) | bits_below(sk - 32 * k));
                    if (flag & 2) see &= BN == 128 ? s_there[s][k] : s_there[s][2 * k] | s_there[s][2 * k + 1] << 16;
                    #pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(see & (1u << c))) sc[32 * k + c] = -INFINITY;
                }
            }
            // Factors of the four key groups; never 0, a masked score is -inf times it.
            float f[4];
            #pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = BF ? rf : fmaxf(rf * s_kf[s][k], 1.2e-38f);
            float m_tile = -INFINITY;
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                constexpr int N = BN / 4;
                const float* v = sc + k * N;
                float a0 = v[0], a1 = v[1];
                #pragma unroll
                for (int c = 2; c < N - 2; c += 4) {
                    a0 = fmax3(a0, v[c], v[c + 1]);
                    a1 = fmax3(a1, v[c + 2], v[c + 3]);
                }
                m_tile = fmaxf(m_tile, fmax3(fmaxf(a0, a1), v[N - 2], v[N - 1]) * f[k]);
            }
            const bool grow = m_tile > m_run + GROW;
            float alpha = 1.0f;
            if (grow) {
                alpha = ex2(m_run - m_tile);
                m_run = m_tile;
            }
            const float nm = m_run == -INFINITY ? 0.f : P_SHIFT - m_run;
            if (!BF && j + 1 == n_x) ve = *reinterpret_cast<const float4*>(s_ve[s]);
            float2 sm2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                // keys [h * BN / 2, ...): P parts over columns of S (the third in columns of its own)
                #pragma unroll
                for (int q = 0; q < BN / 64; ++q) {
                    uint32_t pk[NP][16];
                    #pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const int col = h * (BN / 2) + q * 32 + c;
                        const float ff = f[col / (BN / 4)];
                        const float2 e = ffma2(make_float2(sc[col], sc[col + 1]), make_float2(ff, ff), make_float2(nm, nm));
                        const float2 pp = make_float2(ex2(e.x), ex2(e.y));
                        sm2[(c >> 1) & 1] = fadd2(sm2[(c >> 1) & 1], pp);
                        uint32_t parts[NP];
                        split_parts<BF, NP>(pp.x, pp.y, parts);
                        #pragma unroll
                        for (int k = 0; k < NP; ++k) pk[k][c >> 1] = parts[k];
                    }
                    #pragma unroll
                    for (int k = 0; k < NP; ++k)
                        tmem_st16((k < 2 ? s_tm + k * (BN / 2) : tmem + 384 + x * 64 + lane_off) + h * (BN / 4) + q * 16, pk[k]);
                }
                if (h == 0 && j > 0 && __any_sync(0xffffffffu, grow || (flag & 1))) {
                    // S_FULL_X(j) implies PV_X(j - 1) is complete, and PV_X(j) waits for the arrival below.
                    #pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float o[32];
                        tmem_ld32(o_tm + c * 32, o);
                        const float g = alpha * (!BF && (flag & 1) ? s_vf[s][c] : 1.0f);
                        #pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= g;
                        tmem_st32(o_tm + c * 32, o);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[(h ? P_HI : P_LO) + x]);
            }
            const float2 t = fadd2(sm2[0], sm2[1]);
            l_run = l_run * alpha + (t.x + t.y);
        }
        // ---------------- epilogue ----------------
        // The ring becomes the output's staging once both tiles' products are done.
        if (ok && n_a > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[O_DONE + 0], 0));
        if (ok && n_b > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[O_DONE + 1], 0));
        ok = ok && !aborted();
        if (ok && (x == 0 || has_b)) {
            tc_fence_after();
            const bool whole = cw.pieces <= 1;
            const float inv = whole ? 1.0f / (l_run == 0.f ? 1.0f : l_run) : 1.0f;
            const size_t rows = (size_t)w.n_tok * a.H;
            if (!whole && live)
                *reinterpret_cast<float2*>(a.ws_ml + 2 * (split * rows + (size_t)(cw.row0 + tok) * a.H + head)) = make_float2(m_run, l_run);
            const uint32_t stage = base_u32 + T::SMEM_KV + warp * 4096;
            const int wr0 = cw.r0 + x * 128 + (warp & 3) * 32;         // the warp's first row
            // 128 bytes a row at a time: 32 floats, or 64 BF16 numbers (two loads of 32 columns).
            auto store_rows = [&](auto f32, int d0) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rr = 4 * i + (lane >> 3), q = wr0 + rr;
                    const uint4 v = lds128(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                    if (q < cw.R) {
                        const int t = div_group(q, a), tk = cw.row0 + t, hd = hk * a.G + q - t * a.G;
                        if constexpr (decltype(f32)::value) {
                            float* to = whole ? reinterpret_cast<float*>(a.out) + (size_t)tk * a.out_stride + hd * D
                                              : a.ws_o + (split * rows + (size_t)tk * a.H + hd) * D;
                            *reinterpret_cast<uint4*>(to + d0 + 4 * (lane & 7)) = v;
                        } else {
                            __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)tk * a.out_stride + hd * D;
                            *reinterpret_cast<uint4*>(to + d0 + 8 * (lane & 7)) = v;
                        }
                    }
                }
            };
            #pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                if (n_x > 0) {
                    tmem_ld32(o_tm + c * 32, o);
                } else {
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                }
                const float g = inv * (c == 0 ? ve.x : c == 1 ? ve.y : c == 2 ? ve.z : ve.w);
                // Element d0 + i (in order) is operand column operand_pos(d0 + i): the same 32 columns.
                if (ROWS == PICKLE_CUDA_ROW_F32 || !whole) {
                    __syncwarp();
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float e[4];
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) e[k] = o[operand_pos<KV, D>(c * 32 + 4 * i + k) - c * 32] * g;
                        sts128(stage + lane * 128 + ((i ^ (lane & 7)) << 4),
                               make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3])));
                    }
                    __syncwarp();
                    store_rows(std::true_type(), c * 32);
                } else {
                    if (c % 2 == 0) __syncwarp();
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float e[8];
                        #pragma unroll
                        for (int k = 0; k < 8; ++k) e[k] = o[operand_pos<KV, D>(c * 32 + 8 * i + k) - c * 32] * g;
                        sts128(stage + lane * 128 + ((((c % 2) * 4 + i) ^ (lane & 7)) << 4),
                               make_uint4(bf16x2(e[0], e[1]), bf16x2(e[2], e[3]), bf16x2(e[4], e[5]), bf16x2(e[6], e[7])));
                    }
                    if (c % 2 == 1) {
                        __syncwarp();
                        store_rows(std::false_type(), (c - 1) * 32);
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
