// pages.cu - the paged KV cache's entry points (include/pickle_cuda.h), its
// writer and its reader.
#include "pages.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "pages_attn.cuh"
#include "pages_chunk.cuh"
#include "pages_decode.cuh"

namespace {

using namespace pages;

// ---- write: rotate, quantise, append --------------------------------------

struct AppendArgs {
    View w;
    const void *q, *k, *v;
    size_t q_stride, k_stride, v_stride;   // elements between tokens
    void* q_out;
    size_t q_out_stride;
    int q_out_bf16;
    const float *sin_tab, *cos_tab;
    int H, half, rope_len;
};

// c * x + s * y rounded once: both products and the sum with their errors
// (Dekker / Knuth), the errors added last, which is off by 2^-46 (|c x| + |s y|)
// at most. A code must not depend on how a sum was rounded on the way.
PCU_DEV float dot2_rn(float c, float x, float s, float y) {
    const float p = __fmul_rn(c, x), q = __fmul_rn(s, y);
    const float ep = __fmaf_rn(c, x, -p), eq = __fmaf_rn(s, y, -q);
    const float d = __fadd_rn(p, q), z = __fsub_rn(d, p);
    const float e = __fadd_rn(__fsub_rn(p, __fsub_rn(d, z)), __fsub_rn(q, z));
    const float r = __fadd_rn(d, __fadd_rn(e, __fadd_rn(ep, eq)));
    return fabsf(d) < INFINITY ? r : d;
}

template <bool ONCE>
PCU_DEV float rot(float c, float x, float s, float y) {
    return ONCE ? dot2_rn(c, x, s, y) : __fmaf_rn(c, x, __fmul_rn(s, y));
}

template <bool ONCE>
PCU_DEV void rotate8(Row8& x, const float4 (&c)[2], const float4 (&s)[2], int partner, bool rotated) {
    Row8 y;
    y.a = make_float4(__shfl_sync(0xffffffffu, x.a.x, partner), __shfl_sync(0xffffffffu, x.a.y, partner),
                      __shfl_sync(0xffffffffu, x.a.z, partner), __shfl_sync(0xffffffffu, x.a.w, partner));
    y.b = make_float4(__shfl_sync(0xffffffffu, x.b.x, partner), __shfl_sync(0xffffffffu, x.b.y, partner),
                      __shfl_sync(0xffffffffu, x.b.z, partner), __shfl_sync(0xffffffffu, x.b.w, partner));
    if (!rotated) return;
    x.a = make_float4(rot<ONCE>(c[0].x, x.a.x, s[0].x, y.a.x), rot<ONCE>(c[0].y, x.a.y, s[0].y, y.a.y),
                      rot<ONCE>(c[0].z, x.a.z, s[0].z, y.a.z), rot<ONCE>(c[0].w, x.a.w, s[0].w, y.a.w));
    x.b = make_float4(rot<ONCE>(c[1].x, x.b.x, s[1].x, y.b.x), rot<ONCE>(c[1].y, x.b.y, s[1].y, y.b.y),
                      rot<ONCE>(c[1].z, x.b.z, s[1].z, y.b.z), rot<ONCE>(c[1].w, x.b.w, s[1].w, y.b.w));
}

// Where token t's rows go: its page position, found by the warp that handles the token.
enum { NOT_OURS = 0, NO_PLACE = 1, PLACED = 2 };   // left alone; zero rows, no page; a page position
struct Place {
    int state, pos, r;       // position in the sequence, row in the cell
    uint32_t cell;           // KV head 0's cell in the pool; head h's is h * (page_size / 16) further
};

PCU_DEV Place place_of(const View& w, int t, int rope_len, int lane) {
    Place x{NOT_OURS, 0, 0, 0u};
    const int b = t < w.n_tok ? seq_of_row(w, t, lane) : w.n_seqs;
    int row0, n, kv;
    // (t - row0 lies outside [0, n) only where q_start does not ascend.)
    if (b >= w.n_seqs || !seq_bounds(w, b, row0, n, kv) || t < row0 || t - row0 >= n) return x;
    x.pos = kv - n + (t - row0);
    x.state = NO_PLACE;
    if (x.pos < 0) return x;
    if (x.pos >= rope_len) {
        record_error(w.err, PCU_DEVERR_ARG);
        return x;
    }
    const uint32_t cpp = w.page_size / CELL, cell = (uint32_t)x.pos / CELL, page = cell / cpp;
    const int id = w.table[(size_t)b * w.table_stride + page];
    if ((unsigned)id >= (unsigned)w.n_pages) {
        record_error(w.err, PCU_DEVERR_ARG);
        return x;
    }
    x.state = PLACED;
    x.r = x.pos % CELL;
    x.cell = (uint32_t)id * w.HK * cpp + (cell - page * cpp);
    return x;
}

constexpr int ROW_WARPS = 4, ROW_AHEAD = 4;        // warps of a CTA; steps whose loads are in flight together

// A warp takes a token; its H + 2 HK rows are spread over gridDim.y warps. D / 8
// lanes hold a row, 8 elements each, so a scale's 32 elements are 4 lanes and
// a rotation partner is half / 8 lanes away. The token's sin / cos stay in
// registers for all its rows. Bound by its instructions, K's exact sums and the codes before all (4 ragged prompts
// of up to 2048 tokens, 32 + 2 x 32 BF16 heads of 128, written as E4M3: 56 us with 68 % of the issue slots and 32 % of
// DRAM's rate used; with the rows read back 73 us, 3.9 TB/s);
// for one token a sequence by its launch (64 sequences, written and read back: 13 us for the two calls).
// Finding a token's page takes four dependent loads, so a warp has many rows
// to go with them (two tokens a warp, looked up together, were slower: 92 us
// against 75, for want of warps).
template <int KV, int D, int ROWS>
__global__ void __launch_bounds__(32 * ROW_WARPS) pages_append_kernel(const AppendArgs a) {
    constexpr int LPR = D / 8, RPW = 32 / LPR;
    const View& w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x * ROW_WARPS + warp;
    const Place p = place_of(w, t, a.half > 0 ? a.rope_len : 0x7fffffff, lane);
    if (p.state == NOT_OURS) return;
    const int sub = lane / LPR, l = lane % LPR, i0 = 8 * l;
    const int hl = a.half / 8;
    const bool turns = l < 2 * hl;
    const int partner = !turns ? lane : l < hl ? lane + hl : lane - hl;
    const int HK = w.HK, nq = a.q ? a.H : 0, units = nq + 2 * HK, cpp = w.page_size / CELL;
    const int step = gridDim.y * RPW;
    const bool live = p.state == PLACED, rotated = live && turns;
    float4 c[2], s[2];
    if (rotated) {
        const size_t o = (size_t)p.pos * a.half + (l < hl ? i0 : i0 - a.half);
        const float4* sp = reinterpret_cast<const float4*>(a.sin_tab + o);
        const float4* cp = reinterpret_cast<const float4*>(a.cos_tab + o);
        const float sg = l < hl ? -1.0f : 1.0f;
        #pragma unroll
        for (int k = 0; k < 2; ++k) {
            c[k] = cp[k];
            s[k] = sp[k];
            s[k] = make_float4(sg * s[k].x, sg * s[k].y, sg * s[k].z, sg * s[k].w);
        }
    }
    for (int u0 = blockIdx.y * RPW; u0 < units; u0 += ROW_AHEAD * step) {
        RawRow8<ROWS> rows[ROW_AHEAD];
        #pragma unroll
        for (int k = 0; k < ROW_AHEAD; ++k) {
            const int u = u0 + k * step + sub;
            const bool is_q = u < nq, is_v = u >= nq + HK;
            const int h = is_q ? u : is_v ? u - nq - HK : u - nq;
            rows[k].clear();
            if (u < units && live)
                rows[k].load(is_q ? a.q : is_v ? a.v : a.k,
                                          (size_t)t * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + (size_t)h * D + i0);
        }
        #pragma unroll
        for (int k = 0; k < ROW_AHEAD; ++k) {
            const int uk = u0 + k * step, u = uk + sub;             // uk: the same for the warp
            if (uk >= units) break;
            const bool mine = u < units, is_q = u < nq, is_v = u >= nq + HK;
            const int h = is_q ? u : is_v ? u - nq - HK : u - nq;
            Row8 x = rows[k].row();
            // K and F32 q are rounded once. In q rows that become BF16 a second F32 rounding is 2^-16 of theirs: 4 prompts
            // of up to 2048 tokens, 32 + 2 x 32 heads, written and read back, take 73.0 us so and 76.4 rounded once.
            if (a.q_out_bf16 && uk + RPW <= nq) rotate8<false>(x, c, s, partner, rotated);
            else if (uk < nq + HK) rotate8<true>(x, c, s, partner, rotated && !is_v);
            if (mine && is_q) {
                const size_t o = (size_t)t * a.q_out_stride + (size_t)h * D + i0;
                if (a.q_out_bf16) store_row8<PICKLE_CUDA_ROW_BF16>(a.q_out, o, x);
                else store_row8<PICKLE_CUDA_ROW_F32>(a.q_out, o, x);
            }
            if (uk + RPW <= nq) continue;
            uint32_t m = 0;
            if (KV != BF16) {
                m = max(amax_bits(x.a), amax_bits(x.b));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            }
            if (mine && !is_q && live) {
                unsigned char* cell = w.pool + (size_t)(p.cell + (uint32_t)(h * cpp)) * cell_bytes(KV, D);
                unsigned char* row = cell + (is_v ? v_row(KV, D, p.r) : k_row(KV, D, p.r));
                if (KV == BF16) {
                    store_row8<PICKLE_CUDA_ROW_BF16>(row, i0, x);
                } else {
                    const uint32_t sc = block_scale<KV>(m);
                    *reinterpret_cast<uint2*>(row + i0) = make_uint2(codes4<KV>(x.a, sc), codes4<KV>(x.b, sc));
                    if (l % 4 == 0) cell[(is_v ? v_scale(D, p.r) : k_scale(D, p.r)) + i0 / BLOCK] = (unsigned char)sc;
                }
            }
        }
    }
}

// ---- read back ---------------------------------------------------------------

struct ReadArgs {
    View w;
    void *k, *v;
    size_t k_stride, v_stride;
};

// As the writer: a token a warp, D / 8 lanes a row, twice as many steps in
// flight (their loads are 8 bytes a lane). 8 x 4096 rows of 2 x 8 int8 heads into BF16: 37 us (5.5 TB/s, most of them
// written).
template <int KV, int D, int ROWS>
__global__ void __launch_bounds__(32 * ROW_WARPS) pages_read_kernel(const ReadArgs a) {
    constexpr int LPR = D / 8, RPW = 32 / LPR, AHEAD = 2 * ROW_AHEAD;
    const View& w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x * ROW_WARPS + warp;
    const Place p = place_of(w, t, 0x7fffffff, lane);
    if (p.state == NOT_OURS) return;
    const int sub = lane / LPR, i0 = 8 * (lane % LPR), units = 2 * w.HK, cpp = w.page_size / CELL;
    const int step = gridDim.y * RPW;
    for (int u0 = blockIdx.y * RPW + sub; u0 < units; u0 += AHEAD * step) {
        uint4 raw[AHEAD];
        uint32_t sc[AHEAD];
        #pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int u = u0 + k * step;
            raw[k] = make_uint4(0u, 0u, 0u, 0u);
            sc[k] = 0;
            if (u < units && p.state == PLACED) {
                const bool is_v = u >= w.HK;
                const unsigned char* cell = w.pool + (size_t)(p.cell + (uint32_t)((is_v ? u - w.HK : u) * cpp)) * cell_bytes(KV, D);
                const unsigned char* row = cell + (is_v ? v_row(KV, D, p.r) : k_row(KV, D, p.r));
                if (KV == BF16) {
                    raw[k] = *reinterpret_cast<const uint4*>(row + 2 * i0);
                } else {
                    const uint2 c = *reinterpret_cast<const uint2*>(row + i0);
                    raw[k].x = c.x;
                    raw[k].y = c.y;
                    sc[k] = cell[(is_v ? v_scale(D, p.r) : k_scale(D, p.r)) + i0 / BLOCK];
                }
            }
        }
        #pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int u = u0 + k * step;
            if (u >= units) break;
            const bool is_v = u >= w.HK;
            const int h = is_v ? u - w.HK : u;
            Row8 x;
            if (KV == BF16) {
                x = bf16_row8(raw[k]);
            } else {
                const float f = scale_f32(sc[k]);
                x = Row8{numbers4<KV>(raw[k].x), numbers4<KV>(raw[k].y)};
                x.a = make_float4(x.a.x * f, x.a.y * f, x.a.z * f, x.a.w * f);
                x.b = make_float4(x.b.x * f, x.b.y * f, x.b.z * f, x.b.w * f);
            }
            store_row8<ROWS>(is_v ? a.v : a.k, (size_t)t * (is_v ? a.v_stride : a.k_stride) + (size_t)h * D + i0, x);
        }
    }
}

// ---- host ----------------------------------------------------------------------

bool dims_ok(int kv_type, int n_pages, int page_size, int n_kv_heads, int head_dim) {
    return kv_type >= BF16 && kv_type <= E4M3 && n_pages > 0 && page_size >= CELL && page_size % CELL == 0 &&
           n_kv_heads > 0 && (head_dim == 64 || head_dim == 128);
}

int check(const pickle_cuda_pages_t* p, const pickle_cuda_batch_t* b, View* w) {
    if (!p || !b || !p->pool || (uintptr_t)p->pool % 16 ||
        !dims_ok(p->kv_type, p->n_pages, p->page_size, p->n_kv_heads, p->head_dim))
        return PICKLE_ERR_ARG;
    // Cells are counted in 32 bits, rows of a BF16 pool in a tensor copy's signed 32.
    if ((double)p->n_pages * p->n_kv_heads * (p->page_size / CELL) >= (p->kv_type == BF16 ? 67108864.0 : 4294967296.0))
        return PICKLE_ERR_RANGE;
    if (b->n_seqs < 1 || b->n_tok < 0 || b->max_q < 1 || b->max_kv < 0 || b->table_stride < 1 || !b->kv_len || !b->table)
        return PICKLE_ERR_ARG;
    if (!b->q_start && (b->max_q != 1 || b->n_tok != b->n_seqs)) return PICKLE_ERR_ARG;
    if ((long long)b->max_kv > (long long)b->table_stride * p->page_size) return PICKLE_ERR_RANGE;
    w->pool = (unsigned char*)p->pool;
    w->n_pages = p->n_pages;
    w->page_size = p->page_size;
    w->HK = p->n_kv_heads;
    w->n_seqs = b->n_seqs;
    w->n_tok = b->n_tok;
    w->max_q = b->max_q;
    w->max_kv = b->max_kv;
    w->q_start = b->q_start;
    w->kv_len = b->kv_len;
    w->table = b->table;
    w->table_stride = b->table_stride;
    w->err = p->err;
    return PICKLE_OK;
}

// A rows argument: 16-byte aligned, `heads * D` elements per token at least.
// *stride 0 becomes dense.
bool rows_ok(const void* ptr, int type, int heads, int D, size_t* stride) {
    if (!ptr || (uintptr_t)ptr % 16 || (type != PICKLE_CUDA_ROW_F32 && type != PICKLE_CUDA_ROW_BF16)) return false;
    const size_t dense = (size_t)heads * D;
    if (*stride == 0) *stride = dense;
    return *stride >= dense && *stride % (type == PICKLE_CUDA_ROW_F32 ? 4 : 8) == 0;
}

int sm_count() {
    static thread_local int dev_of = -1, sms = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev != dev_of) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        dev_of = dev;
    }
    return sms;
}

// T itself, from which no template argument is deduced.
template <class T>
struct same {
    using type = T;
};
template <class T>
using same_t = typename same<T>::type;

// Launch as a programmatic dependent of the kernel before it on the stream
// (each kernel waits before its first global access).
template <class... Args>
int launch(void (*fn)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t st, const same_t<Args>&... a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, a...) == cudaSuccess ? PICKLE_OK : PICKLE_ERR_DEVICE;
}

// f(kv type, D, row type) as compile-time constants.
template <class F>
int dispatch(int kv, int D, int rows, F f) {
    auto by_rows = [&](auto k, auto d) {
        return rows == PICKLE_CUDA_ROW_F32 ? f(k, d, std::integral_constant<int, PICKLE_CUDA_ROW_F32>())
                                           : f(k, d, std::integral_constant<int, PICKLE_CUDA_ROW_BF16>());
    };
    auto by_d = [&](auto k) {
        return D == 64 ? by_rows(k, std::integral_constant<int, 64>()) : by_rows(k, std::integral_constant<int, 128>());
    };
    if (kv == BF16) return by_d(std::integral_constant<int, BF16>());
    if (kv == I8) return by_d(std::integral_constant<int, I8>());
    return by_d(std::integral_constant<int, E4M3>());
}

// One kernel's shared-memory limit; `done` has a bit per device on which it is set.
template <class... Args>
int allow_smem(void (*fn)(Args...), int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return PICKLE_ERR_DEVICE;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return PICKLE_OK;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return PICKLE_ERR_DEVICE;
    done.fetch_or(bit, std::memory_order_release);
    return PICKLE_OK;
}

struct Plan {
    bool few;           // the kernel for few rows
    int blocks;         // else: blocks of rows a sequence may have
    int n_splits, chunk, chunk_min, target;
};

// How many pieces the keys of `groups` independent streams of `steps` steps
// are cut into: waves of CTAs of the same length, per_sm of them on an SM. A
// step takes step_s[k - 1] in a CTA that shares its SM with k - 1 others, or what
// HBM needs for the wave's bytes; a wave adds a ramp, several pieces add the
// join (a launch, and a piece at a time) and its traffic. The host knows the longest
// stream only: where streams may differ, what counts is this time plus that
// of lengths spread evenly from none to `steps`, the work shared out with
// half a piece's time left over (32 sequences of 8192 keys, 8 heads: one piece 130 us, 8 pieces 71 where they are
// ragged, up to 6% lost where they are not).
struct Costs {
    int per_sm;
    bool ragged;
    double step_s[4], step_bytes, ramp_s, join_s, join_piece_s, join_bytes;
};
int plan_pieces(long long groups, long long steps, int sms, const Costs& c) {
    // The same plan is asked for layer after layer, step after step.
    struct Memo {
        long long groups, steps;
        int sms, pick;
        bool ragged;
        double a, b;
    };
    static thread_local Memo memo[16];
    Memo& k = memo[(unsigned long long)(groups * 31 + steps) % 16];
    if (k.pick && k.groups == groups && k.steps == steps && k.sms == sms && k.ragged == c.ragged && k.a == c.step_s[0] &&
        k.b == c.join_bytes)
        return k.pick;
    const double hbm = 6.5e12;
    const long long slots = (long long)sms * c.per_sm;
    const int most = steps < 64 ? (int)steps : 64;
    double best = 1e30;
    int pick = 1;
    for (int s = 1; s <= most; ++s) {
        const long long chunk = (steps + s - 1) / s;
        if ((steps + chunk - 1) / chunk != s) continue;
        auto wave = [&](long long ctas) {
            const double alone = c.step_s[(ctas + sms - 1) / sms - 1] * chunk, bytes = c.step_bytes * chunk * ctas / hbm;
            return (alone > bytes ? alone : bytes) + c.ramp_s;
        };
        const long long n = groups * s, full = n / slots, rem = n % slots;
        double t = full * wave(slots) + (rem ? wave(rem) : 0.0);
        if (c.ragged) {
            const long long some = groups * (s + 1) / 2;
            const double step = c.step_s[c.per_sm - 1], first = wave(some < 1 ? 1 : some < slots ? some : slots);
            const double shared = (0.5 * groups * steps * step + some * c.ramp_s) / slots + 0.5 * chunk * step;
            t += first > shared ? first : shared;
        }
        if (s > 1) t += (c.ragged ? 2 : 1) * (c.join_s + s * (c.join_piece_s + c.join_bytes / hbm));
        if (t < best) {
            best = t;
            pick = s;
        }
    }
    k = Memo{groups, steps, sms, pick, c.ragged, c.step_s[0], c.join_bytes};
    return pick;
}

// Tile sizes of the kernel for many rows, by types.
struct ChunkDims {
    int bn, rows;
};
ChunkDims chunk_dims(int kv_type, int D, int row_type) {
    ChunkDims d = {0, 0};
    dispatch(kv_type, D, row_type, [&](auto kv, auto dd, auto rows) {
        using T = ChunkTile<kv(), dd(), rows()>;
        d = {T::BN, T::ROWS_CTA};
        return 0;
    });
    return d;
}

Plan plan_attn(const View& w, int kv_type, int D, int row_type, int H, int window, int sinks) {
    Plan p;
    const int G = H / w.HK;
    // Up to 8 rows fit the few-rows kernel's one tile of columns. int8, 8 KV heads, the few-rows kernel and the other at 1
    // to 8 rows: one sequence of 4096 keys 17 and 26 us, 16 of them 46 and 78, one of 32768 32 and 50, 16 of them 212 and
    // 510. The other takes the same time up to 128 rows.
    p.few = (long long)w.max_q * G <= 8;
    const ChunkDims cd = p.few ? ChunkDims{CELL, 8} : chunk_dims(kv_type, D, row_type);
    p.blocks = (int)(((long long)w.max_q * G + cd.rows - 1) / cd.rows);
    // The most keys that a block's rows can see.
    long long keys = w.max_kv;
    if (window > 0) {
        const long long tokens = p.few ? w.max_q : cd.rows / G + 2;
        const long long seen = (long long)window + tokens + (sinks < w.max_kv ? sinks : w.max_kv) + 2 * cd.bn;
        if (seen < keys) keys = seen;
    }
    const long long steps = keys < 1 ? 1 : (keys + cd.bn - 1) / cd.bn;
    const long long groups = (long long)w.n_seqs * w.HK * p.blocks;
    const double bytes = (double)cell_bytes(kv_type, D) * (cd.bn / CELL);
    Costs c;
    c.step_bytes = bytes;
    c.join_bytes = 2.0 * w.n_tok * H * D * 4;
    const int sms = sm_count() > 0 ? sm_count() : 1;
    if (p.few) {
        // Fitted to sweeps of the piece count (1 to 128 sequences of 2048 to 32768 keys, ragged or not): a CTA
        // streams 19.5 GB/s (8-bit) or 35 GB/s (BF16) alone on its SM, four 9.7 each, three BF16 ones 17.
        c.per_sm = kv_type == BF16 ? 3 : 4;
        c.ragged = w.n_seqs > 1 && window == 0;
        const double rate[2][4] = {{19.5e9, 16e9, 12.3e9, 9.7e9}, {35e9, 22e9, 17e9, 17e9}};
        for (int k = 0; k < 4; ++k) c.step_s[k] = bytes / rate[kv_type == BF16][k];
        c.ramp_s = 5e-6;
        c.join_s = 2.5e-6;
        c.join_piece_s = 0.1e-6;
    } else {
        c.per_sm = 1;
        c.ragged = false;            // see piece_steps
        // A tile of 128 keys takes this long with 256 rows, and two thirds of it with 128 or fewer.
        const double tile = (row_type != PICKLE_CUDA_ROW_F32 ? 2.5e-6 : D == 64 ? 3.1e-6 : kv_type == BF16 ? 8e-6 : 5e-6) * cd.bn / 128;
        c.step_s[0] = (long long)w.max_q * G <= 128 ? tile * 0.7 : tile;
        c.ramp_s = 10e-6;
        c.join_s = 3e-6;
        c.join_piece_s = 0.1e-6;
    }
    p.n_splits = plan_pieces(groups, steps, sms, c);
    // Knob for sweeps of the piece count: that many, as if all sequences were the longest.
    const char* env = getenv("PICKLE_CUDA_PAGES_SPLITS");
    const int asked = env ? atoi(env) : 0;
    if (asked > 0) p.n_splits = asked < steps ? asked : (int)steps;
    p.chunk = p.chunk_min = (int)((steps + p.n_splits - 1) / p.n_splits);
    p.target = 0;
    // Sequences may be shorter: room for twice the pieces of each, no more in all. Not with a window, under which long ones
    // are alike, nor with several blocks of rows, which end at different keys.
    if (!p.few && asked <= 0 && p.n_splits > 1 && window == 0 && p.blocks == 1 && w.n_seqs <= TARGET_SEQS) {
        p.target = w.n_seqs * p.n_splits;
        p.n_splits = 2 * p.n_splits < steps ? 2 * p.n_splits : (int)steps;
        p.chunk_min = (int)((steps + p.n_splits - 1) / p.n_splits);
    }
    return p;
}

size_t split_bytes(const View& w, const Plan& p, int H, int D) {
    return p.n_splits > 1 ? (size_t)p.n_splits * w.n_tok * H * (D + 2) * sizeof(float) : 0;
}

// The pool's rows as a tensor of [rows][D] BF16 numbers, boxes of 64 columns
// and a cell's 16 rows in the 128-byte swizzle. Zero for 8-bit pages, which
// are not read through it.
int rows_map(CUtensorMap* map, const pickle_cuda_pages_t* p) {
    memset(map, 0, sizeof(*map));
    if (p->kv_type != BF16) return PICKLE_OK;
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> encode{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 fn = encode.load(std::memory_order_acquire);
    if (!fn) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess || !sym)
            return PICKLE_ERR_DEVICE;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym);
        encode.store(fn, std::memory_order_release);
    }
    const cuuint64_t rows = (cuuint64_t)p->n_pages * p->n_kv_heads * (p->page_size / CELL) * 2 * CELL;
    const cuuint64_t dims[2] = {(cuuint64_t)p->head_dim, rows}, strides[1] = {(cuuint64_t)p->head_dim * 2};
    const cuuint32_t box[2] = {64, CELL}, one[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p->pool, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? PICKLE_OK
               : PICKLE_ERR_DEVICE;
}

// CTAs of ROW_WARPS tokens, and over how many of them a token's `steps` warp
// steps are spread: about 16 a warp (4 prompts of 2048 tokens with 96 rows:
// 84, 75, 73 and 82 us at 48, 24, 12 and 6 steps a warp; reading 16 rows back:
// 38 and 48 us at 8 and 4), fewer where that leaves SMs without work.
dim3 row_grid(int n_tok, int steps) {
    const int x = (n_tok + ROW_WARPS - 1) / ROW_WARPS;
    const int fill = (4 * sm_count() + x - 1) / x, most = (steps + 15) / 16;
    const int y = fill > most ? fill : most;
    return dim3(x, y < 1 ? 1 : y < steps ? y : steps);
}

}  // namespace

extern "C" {

size_t pickle_cuda_pages_bytes(int kv_type, int n_pages, int page_size, int n_kv_heads, int head_dim) {
    if (!dims_ok(kv_type, n_pages, page_size, n_kv_heads, head_dim)) return 0;
    return (size_t)n_pages * n_kv_heads * (page_size / CELL) * cell_bytes(kv_type, head_dim);
}

int pickle_cuda_pages_append_dev(const pickle_cuda_pages_t* pages, const pickle_cuda_batch_t* batch, int n_heads,
                                 int row_type, const void* q, size_t q_stride, const void* k, size_t k_stride,
                                 const void* v, size_t v_stride, const float* rope_sin, const float* rope_cos, int half,
                                 int rope_len, int q_out_type, void* q_out, size_t q_out_stride, void* stream) {
    AppendArgs a;
    memset(&a, 0, sizeof(a));
    int rc = check(pages, batch, &a.w);
    if (rc != PICKLE_OK) return rc;
    const int D = pages->head_dim, HK = pages->n_kv_heads;
    if (!rows_ok(k, row_type, HK, D, &k_stride) || !rows_ok(v, row_type, HK, D, &v_stride)) return PICKLE_ERR_ARG;
    if ((q == nullptr) != (q_out == nullptr)) return PICKLE_ERR_ARG;
    if (q && (n_heads < 1 || !rows_ok(q, row_type, n_heads, D, &q_stride) ||
              !rows_ok(q_out, q_out_type, n_heads, D, &q_out_stride)))
        return PICKLE_ERR_ARG;
    if (half < 0 || half % 8 || 2 * half > D || rope_len < 0) return PICKLE_ERR_ARG;
    if (half > 0 && (!rope_sin || !rope_cos || ((uintptr_t)rope_sin | (uintptr_t)rope_cos) % 16)) return PICKLE_ERR_ARG;
    if (half > 0 && batch->max_kv > rope_len) return PICKLE_ERR_RANGE;
    if (batch->n_tok == 0) return PICKLE_OK;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out = q_out;
    a.q_out_stride = q_out_stride;
    a.q_out_bf16 = q_out_type == PICKLE_CUDA_ROW_BF16;
    a.sin_tab = rope_sin;
    a.cos_tab = rope_cos;
    a.H = n_heads;
    a.half = half;
    a.rope_len = rope_len;
    const int units = (q ? n_heads : 0) + 2 * HK, rpw = 256 / D;
    const dim3 grid = row_grid(batch->n_tok, (units + rpw - 1) / rpw);
    return dispatch(pages->kv_type, D, row_type, [&](auto kv, auto d, auto rows) {
        return launch(pages_append_kernel<kv(), d(), rows()>, grid, 32 * ROW_WARPS, 0, (cudaStream_t)stream, a);
    });
}

int pickle_cuda_pages_read_dev(const pickle_cuda_pages_t* pages, const pickle_cuda_batch_t* batch, int row_type,
                               void* k_out, size_t k_stride, void* v_out, size_t v_stride, void* stream) {
    ReadArgs a;
    int rc = check(pages, batch, &a.w);
    if (rc != PICKLE_OK) return rc;
    const int D = pages->head_dim, HK = pages->n_kv_heads;
    if (!rows_ok(k_out, row_type, HK, D, &k_stride) || !rows_ok(v_out, row_type, HK, D, &v_stride)) return PICKLE_ERR_ARG;
    if (batch->n_tok == 0) return PICKLE_OK;
    a.k = k_out;
    a.v = v_out;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    const dim3 grid = row_grid(batch->n_tok, (2 * HK * D + 255) / 256);
    return dispatch(pages->kv_type, D, row_type, [&](auto kv, auto d, auto rows) {
        return launch(pages_read_kernel<kv(), d(), rows()>, grid, 32 * ROW_WARPS, 0, (cudaStream_t)stream, a);
    });
}

size_t pickle_cuda_pages_workspace(const pickle_cuda_pages_t* pages, const pickle_cuda_batch_t* batch, int n_heads,
                                   int row_type, int window, int sinks) {
    View w;
    if (check(pages, batch, &w) != PICKLE_OK || n_heads < 1 || n_heads % w.HK || n_heads / w.HK > 8 || window < 0 ||
        sinks < 0 || batch->n_tok == 0 || (row_type != PICKLE_CUDA_ROW_F32 && row_type != PICKLE_CUDA_ROW_BF16))
        return 0;
    return split_bytes(w, plan_attn(w, pages->kv_type, pages->head_dim, row_type, n_heads, window, sinks), n_heads,
                       pages->head_dim);
}

int pickle_cuda_pages_attn_dev(const pickle_cuda_pages_t* pages, const pickle_cuda_batch_t* batch, int n_heads,
                               int row_type, const void* q, size_t q_stride, void* out, size_t out_stride, int window,
                               int sinks, void* workspace, size_t ws_bytes, void* stream) {
    AttnArgs a;
    memset(&a, 0, sizeof(a));
    int rc = check(pages, batch, &a.w);
    if (rc != PICKLE_OK) return rc;
    const int D = pages->head_dim, HK = pages->n_kv_heads;
    if (n_heads < 1 || n_heads % HK || n_heads / HK > 8 || window < 0 || sinks < 0) return PICKLE_ERR_ARG;
    if (!rows_ok(q, row_type, n_heads, D, &q_stride) || !rows_ok(out, row_type, n_heads, D, &out_stride))
        return PICKLE_ERR_ARG;
    if ((long long)batch->max_q * (n_heads / HK) > (1 << 22)) return PICKLE_ERR_RANGE;
    if (batch->n_tok == 0) return PICKLE_OK;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.H = n_heads;
    a.G = n_heads / HK;
    a.inv_g = a.G == 1 ? 0u : (uint32_t)(((1ull << 32) + a.G - 1) / a.G);
    a.window = window;
    a.sinks = sinks;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)D);
    const cudaStream_t st = (cudaStream_t)stream;
    const Plan p = plan_attn(a.w, pages->kv_type, D, row_type, n_heads, window, sinks);
    const size_t need = split_bytes(a.w, p, n_heads, D);
    if (need && (!workspace || (uintptr_t)workspace % 16 || ws_bytes < need)) return PICKLE_ERR_ARG;
    a.n_splits = p.n_splits;
    a.chunk = p.chunk;
    a.chunk_min = p.chunk_min;
    a.target = p.target;
    a.ws_o = (float*)workspace;
    a.ws_ml = a.ws_o + (size_t)p.n_splits * batch->n_tok * n_heads * D;
    const size_t out_rows = (size_t)batch->n_tok * n_heads;
    const dim3 merge_grid((unsigned)(p.few ? out_rows : (out_rows + MERGE_WARPS - 1) / MERGE_WARPS));
    return dispatch(pages->kv_type, D, row_type, [&](auto kv, auto d, auto rows) {
        static std::atomic<uint64_t> few_set{0}, many_set{0};
        if (p.few) {
            using T = DecodeTile<kv(), d()>;
            const auto fn = pages_decode_kernel<kv(), d(), rows()>;
            int e = allow_smem(fn, T::SMEM, few_set);
            if (e == PICKLE_OK) e = launch(fn, dim3(a.w.n_seqs * HK, p.n_splits), 32 * T::WARPS, T::SMEM, st, a);
            if (e == PICKLE_OK && p.n_splits > 1)
                e = launch(pages_merge_kernel<d(), rows(), CELL, 0>, merge_grid, 32 * MERGE_WARPS, 0, st, a);
            return e;
        }
        using T = ChunkTile<kv(), d(), rows()>;
        const auto fn = pages_chunk_kernel<kv(), d(), rows()>;
        alignas(64) CUtensorMap tm;
        int e = rows_map(&tm, pages);
        if (e == PICKLE_OK) e = allow_smem(fn, T::SMEM, many_set);
        if (e == PICKLE_OK)
            e = launch(fn, dim3(a.w.n_seqs * HK, p.blocks, p.n_splits), CHUNK_THREADS, T::SMEM, st, tm, a);
        if (e == PICKLE_OK && p.n_splits > 1)
            e = launch(pages_merge_kernel<d(), rows(), T::BN, T::ROWS_CTA>, merge_grid, 32 * MERGE_WARPS, 0, st, a);
        return e;
    });
}

}  // extern "C"
