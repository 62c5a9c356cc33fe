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
    enum { Q_FULL = 0, S_FULL = 2, P_LO = 4, P_HI = 6, O_DONE = 8, DRAIN = 10, KV_FULL = 11, KV_EMPTY = KV_FULL + STAGES,
           N_BARS = KV_EMPTY + STAGES };
    static_assert(N_BARS * 8 <= 256, "barriers");
    extern __shared__ unsigned char smem_raw[];
    // What staging tells the softmax of a stage: K's factors (one per staging warp), V's O factors (if any moved), V's
    // references, the keys that are really there.
    __shared__ __align__(16) float s_kf[STAGES][4], s_vf[STAGES][4], s_ve[STAGES][4];
    __shared__ uint32_t s_there[STAGES][4];
    __shared__ int s_flag[STAGES];                // 1: V's references moved; 2: keys on a bad page
    __shared__ uint32_t s_vmax[2][4];
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
            mbar_init(&bars[S_FULL + x], 1);
            mbar_init(&bars[P_LO + x], 4);
            mbar_init(&bars[P_HI + x], 4);
            mbar_init(&bars[O_DONE + x], 1);
        }
        mbar_init(&bars[DRAIN], 1);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bars[KV_FULL + s], 4);
            mbar_init(&bars[KV_EMPTY + s], 1);
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
            int kv_ready = -1;
            auto wait_kv = [&](int j) {
                if (ok && j > kv_ready) {
                    ok = mbar_wait(&bars[KV_FULL + j % STAGES], (j / STAGES) & 1);
                    kv_ready = j;
                }
                tc_fence_after();
            };
            for (int x = 0; x < 2 && ok; ++x)
                if (x ? n_b : n_a) {
                    ok = mbar_wait(&bars[Q_FULL + x], 0);
                    wait_kv(0);
                    if (ok) issue_s(x, 0);
                }
            for (int j = 0; ok && j < n_all; ++j) {
                for (int x = 0; x < 2 && ok; ++x) {
                    const int n_x = x ? n_b : n_a;
                    if (j >= n_x) continue;
                    ok = mbar_wait(&bars[P_LO + x], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    issue_o(x, j, 0);
                    ok = mbar_wait(&bars[P_HI + x], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    issue_o(x, j, BN / 32);
                    if (j + 1 == n_x) {
                        mma_commit(&bars[O_DONE + x]);
                    } else {
                        wait_kv(j + 1);
                        if (ok) issue_s(x, j + 1);
                    }
                }
                if (ok) mma_commit(&bars[KV_EMPTY + j % STAGES]);
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
        // Lane i looks after key i of the warp's: its cell in the pool, or NONE where no row sees it.
        constexpr uint32_t NONE = 0xffffffffu;
        struct Look {
            uint32_t at;
            bool bad;
        };
        auto look_up = [&](int j) {
            Look x{NONE, false};
            if (j < n_all && lane < KPW) {
                const int key = cw.span.step(t0 + j) * BN + sw * KPW + lane;
                if (key <= cw.last && (key >= cw.span.lo_key || key < a.sinks)) {
                    const uint32_t cell = (uint32_t)key / CELL, page = cell / cpp;
                    const int id = w.table[(size_t)b * w.table_stride + page];
                    x.bad = (unsigned)id >= (unsigned)w.n_pages;
                    if (!x.bad) x.at = ((uint32_t)id * w.HK + hk) * cpp + (cell - page * cpp);
                }
            }
            return x;
        };
        auto row_ptr = [&](uint32_t at, int row, bool v) {
            return w.pool + (size_t)at * cell_bytes(KV, D) + (v ? v_row(KV, D, row % CELL) : k_row(KV, D, row % CELL));
        };
        bool ok = true;
        // Tell the softmax which keys are missing although some row sees them.
        auto publish = [&](int s, const Look& x, int moved) {
            const uint32_t there = __ballot_sync(0xffffffffu, x.at != NONE);
            const uint32_t bad = __ballot_sync(0xffffffffu, x.bad);
            if (lane == 0) {
                s_there[s][sw] = there;
                if (bad) {
                    atomicOr(&s_flag[s], 2);
                    record_error(w.err, PCU_DEVERR_ARG);
                }
                if (moved) atomicOr(&s_flag[s], 1);
            }
        };
        auto full = [&](int j) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[KV_FULL + j % STAGES]);
        };
        // Wait until tile j's stage is empty, clear its flag, and meet the other staging warps; false: all four stop.
        auto begin = [&](int j) {
            if (j >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&bars[KV_EMPTY + j % STAGES], ((j / STAGES) - 1) & 1));
            if (lane == 0) {
                if (!ok || aborted()) *(volatile int*)&s_stop[j & 1] = 1;
                if (sw == 0) *(volatile int*)&s_flag[j % STAGES] = 0;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            return *(volatile int*)&s_stop[j & 1] == 0;
        };
        if constexpr (BF) {
            constexpr int CPR = D / 8, RPI = 32 / CPR, NI = KPW / RPI;
            Look nxt = look_up(0);
            // A tile is announced LAG tiles after its copies went out. Tile j's stage empties only after tile
            // j - STAGES + 1 has been announced (its S is issued between the products that free the stage).
            constexpr int LAG = STAGES - 2;
            for (int j = 0; j < n_all + LAG; ++j) {
                if (j < n_all) {
                    const Look x = nxt;
                    nxt = look_up(j + 1);
                    if (!begin(j)) break;
                    const int s = j % STAGES;
                    publish(s, x, 0);
                    const uint32_t dst = base_u32 + T::SMEM_KV + s * T::STAGE;
                    #pragma unroll
                    for (int v = 0; v < 2; ++v)
                        #pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            const int row = i * RPI + lane / CPR, c = lane % CPR, r = sw * KPW + row;
                            const uint32_t at = __shfl_sync(0xffffffffu, x.at, row);
                            const uint32_t to = dst + v * T::KV_TILE + (c >> 3) * T::KV_HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                            cp_async16_or_zero(to, at == NONE ? w.pool : row_ptr(at, row, v) + c * 16, at == NONE ? 0u : 16u);
                        }
                }
                cp_async_commit();
                if (j >= LAG) {
                    cp_async_wait<LAG>();
                    full(j - LAG);
                }
            }
            cp_async_wait<0>();
        } else {
            constexpr int CPR = D / 16, RPI = 32 / CPR, NI = KPW / RPI;
            uint32_t ev = 0;                       // V's reference exponents, a byte per 32 elements
            Look x0 = look_up(0), x1 = look_up(1);
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
                const int s = j % STAGES;
                load(x0, true, vq);
                scales(x1, ks1, vs1);
                const Look x2 = look_up(j + 2);
                // K: one reference for the warp's keys. V: the tile's maxima, through shared memory.
                uint32_t km = ks0;
                #pragma unroll
                for (int k = 1; k < NB; ++k) km = max(km & 255u, (ks0 >> (8 * k)) & 255u);
                km = __reduce_max_sync(0xffffffffu, km & 255u);
                uint32_t vm = 0;
                #pragma unroll
                for (int k = 0; k < NB; ++k)
                    vm |= __reduce_max_sync(0xffffffffu, (vs0 >> (8 * k)) & 255u) << (8 * k);
                if (lane == 0) s_vmax[j & 1][sw] = vm;
                if (!begin(j)) break;
                int moved = 0;
                float vf[4] = {1.f, 1.f, 1.f, 1.f};
                #pragma unroll
                for (int k = 0; k < NB; ++k) {
                    const uint32_t old = (ev >> (8 * k)) & 255u;
                    uint32_t top = 0;
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) top = max(top, (s_vmax[j & 1][i] >> (8 * k)) & 255u);
                    if (top > old + SLACK) {
                        moved = 1;
                        vf[k] = rel_scale((int)old, (int)top);
                        ev = (ev & ~(255u << (8 * k))) | (top << (8 * k));
                    }
                }
                publish(s, x0, sw == 0 && moved);
                if (lane == 0) s_kf[s][sw] = km == 255u ? INFINITY : __uint_as_float(km << 23);
                if (sw == 0 && lane < NB) {
                    const uint32_t e = (ev >> (8 * lane)) & 255u;
                    s_ve[s][lane] = e == 255u ? INFINITY : __uint_as_float(e << 23);
                    s_vf[s][lane] = lane == 0 ? vf[0] : lane == 1 ? vf[1] : lane == 2 ? vf[2] : vf[3];
                }
                const uint32_t dst = base_u32 + T::SMEM_KV + s * T::STAGE;
                store(dst, kq, ks0, km * 0x01010101u);
                load(x1, false, kq);
                store(dst + T::KV_TILE, vq, vs0, ev);
                full(j);
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
            // This thread's q row into shared memory, in the operand order.
            const size_t at = live ? (size_t)(cw.row0 + tok) * a.q_stride + (size_t)head * D : 0;
            float qs = 1.f;
            if (!BF) {
                uint32_t m = 0;
                if (live) {
                    #pragma unroll 4
                    for (int i = 0; i < D; i += 8) {
                        const Row8 v = load_row8<ROWS>(a.q, at + i);
                        m = max(m, max(amax_bits(v.a), amax_bits(v.b)));
                    }
                }
                qs = __uint_as_float(min(268u - (m >> 23), 254u) << 23);
                rf = a.scale_log2 / qs;
            }
            #pragma unroll 2
            for (int i = 0; i < D; i += 8) {
                Row8 v;
                v.a = v.b = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live) v = load_row8<ROWS>(a.q, at + i);
                const float e[8] = {v.a.x * qs, v.a.y * qs, v.a.z * qs, v.a.w * qs, v.b.x * qs, v.b.y * qs, v.b.z * qs, v.b.w * qs};
                constexpr int o1 = KV == I8 ? 2 : 1, o2 = KV == I8 ? 1 : 2;
                uint32_t q0[NP], q1[NP], q2[NP], q3[NP];
                split_parts<BF, NP>(e[0], e[o1], q0);
                split_parts<BF, NP>(e[o2], e[3], q1);
                split_parts<BF, NP>(e[4], e[4 + o1], q2);
                split_parts<BF, NP>(e[4 + o2], e[7], q3);
                const int c = operand_pos<KV, D>(i) >> 3;            // 16-byte chunk of the row
                const uint32_t to = base_u32 + x * NP * T::Q_TILE + (c >> 3) * T::Q_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                #pragma unroll
                for (int k = 0; k < NP; ++k) sts128(to + k * T::Q_TILE, make_uint4(q0[k], q1[k], q2[k], q3[k]));
            }
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
            const int s = j % STAGES;
            ok = __all_sync(0xffffffffu, mbar_wait(&bars[S_FULL + x], j & 1) && mbar_wait(&bars[KV_FULL + s], (j / STAGES) & 1));
            if (!ok) break;
            tc_fence_after();
            float sc[BN];
            #pragma unroll
            for (int c = 0; c < BN / 64; ++c) tmem_ld64(s_tm + c * 64, sc + c * 64);
            const int j0 = cw.span.step(t0 + j) * BN;
            const int flag = *(volatile int*)&s_flag[s];
            if (j0 + BN - 1 > p_first || (a.window > 0 && j0 <= p_last - a.window && j0 + BN - 1 >= a.sinks) || (flag & 2)) {
                // Columns past the row's position, and those before its window that are no sinks.
                const int hi = max(p, -1) - j0, sk = a.sinks - j0;
                const int lo = (a.window > 0 ? max(max(p, -1) - a.window, -1) : -1) - j0;
                #pragma unroll
                for (int c = 0; c < BN; ++c)
                    if (c > hi || (c <= lo && c >= sk)) sc[c] = -INFINITY;
                if (flag & 2) {
                    #pragma unroll
                    for (int c = 0; c < BN; ++c)
                        if (!((s_there[s][c / (BN / 4)] >> (c % (BN / 4))) & 1)) sc[c] = -INFINITY;
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
                        const size_t tk = cw.row0 + q / a.G, hd = hk * a.G + q % a.G;
                        if constexpr (decltype(f32)::value) {
                            float* to = whole ? reinterpret_cast<float*>(a.out) + tk * a.out_stride + hd * D
                                              : a.ws_o + (split * rows + tk * a.H + hd) * D;
                            *reinterpret_cast<uint4*>(to + d0 + 4 * (lane & 7)) = v;
                        } else {
                            __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(a.out) + tk * a.out_stride + hd * D;
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
