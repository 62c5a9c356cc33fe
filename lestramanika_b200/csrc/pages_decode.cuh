// pages_decode.cuh - attention over the paged cache for calls of few rows:
// up to 8 (token, query head) rows per KV head and sequence, so a decode step
// (one token, H / HK heads) or a few drafted tokens of a small group.
//
// Every cached byte is read once; the work per byte is what has to stay small,
// because an 8-bit row brings 2 x 8 multiply-adds a byte. So the products
// run on the tensor cores with the keys as the long side (mma.sync m16n8k16;
// at 8 rows there is nothing to fill a tcgen05 tile's 64 rows with):
//     S^T [16 keys][8 rows] = K Q^T,   O^T [16 elements][8 rows] += V^T P^T
// A warp takes a cell (16 keys) at a time from a ring of its own that it fills
// with cp.async (no barrier beyond the warp); chunks of a row are swizzled as
// they are copied, so that fragments are read without bank conflicts. The
// order of the elements of K and Q, and of an output tile, is free, and
// chosen so that a lane's elements are contiguous.
//
// 8-bit codes become F16 numbers in registers: a code is exact in F16, and so
// is code * 2^(e - E) for a reference exponent E near the largest one seen, down
// to e - E = -24 (int8) or -15 (E4M3). Smaller blocks are rounded to F16's smallest
// step, 2^-24, and from e - E = -25 on count as 0: off by 2^-24 at most of the largest magnitude
// that is behind E, which shows where a row sees, but gives next to no weight, a key far larger than
// the others. K
// has one E per warp, which the scores' factor undoes; V has one per 32
// elements of the output, and moving it rescales O by a power of two. BF16
// pages are multiplied as they are.
//
// F32 rows keep F32 accuracy: q (scaled to a row maximum near 2^15) and the
// weights p are sums of two F16 numbers (22 bits), each with a product of
// its own; of three BF16 numbers (24 bits) on BF16 pages. BF16 rows: q is exact
// in one number; p is one F16 number (its 2^-12 is an eighth of the output's
// own 2^-8 rounding's root-mean-square) or two BF16 numbers.
//
// The running maximum moves only when some score passes it by 2^8 (a warp
// vote), so most cells need no reduction over the keys; p is held times 2^7
// so that small weights stay above F16's subnormals (one below 2^-21 of the largest
// is off by 2^-32 of it at most).
//
// What bounds it: 8-bit cells, the chain of instructions that turns codes into numbers and products, at 16
// warps an SM (an SM streams 39 GB/s of them at best, 5.7 TB/s in all, against 6.5 that HBM
// gives and 6.3 of BF16 cells; 58 to 60 % of the issue slots are used, so it is latency as much as slots); then how
// evenly the SMs are filled: work comes in CTAs of one
// piece of one sequence's keys, with about 5 us before and after its stream. 64 ragged sequences keep an SM busy for 73 %
// of the time on average.
// Measured (us; with the join): 16 sequences of 32768 keys, 64 / 8 heads, int8: 217 to 231 (5.1 to 4.8 TB/s, by GPU);
// 64 ragged ones up to 4096, 32 / 8 heads, E4M3, F32 rows: 88 (3.2); 16 with a window of
// 4096 of 32768, BF16 pages, F32 rows: 48 (5.0); one of 4096, int8: 11.6 (latency: a launch, page
// ids, keys, the join).
// Registers: 128 a thread (168 with BF16 cells, D = 128, F32 rows), of which 16 to 48 bytes spill with F32 rows and D = 128.
#pragma once
#include <cuda_fp16.h>

#include "pages_attn.cuh"

namespace pages {

template <int KV, int D>
struct DecodeTile {
    static constexpr int ES = elem_bytes(KV);
    static constexpr int ROWB = D * ES;               // bytes of a row
    static constexpr int CH = ROWB / 16;              // 16-byte chunks of a row
    static constexpr int KCH = CH / 4;                // chunks of a K row that a lane takes
    static constexpr int CELLB = cell_bytes(KV, D);
    // 8-bit: 16 warps an SM with 12 KB of ring each (203 KB in all), in four CTAs: in two of eight warps, what a CTA does
    // before its first and after its last cell is hidden less (16 sequences of 32768, 8 heads: 232 us instead of 219; 64
    // ragged ones up to 4096: 89 instead of 85). BF16 cells are twice as large and cheaper to use: 12 warps with 16 KB.
    static constexpr int WARPS = 4;
    static constexpr int CTAS = KV == BF16 ? 3 : 4;
    static constexpr int STAGES = (KV == BF16 ? 2 : 3) * 128 / D;
    static constexpr int OPAD = D + 4;                // floats between output columns of a warp's partial
    static constexpr int RING = WARPS * STAGES * CELLB;
    static constexpr int JOIN = WARPS * 8 * (OPAD + 2) * 4;
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;

    // Where chunk c of row r lies in the row's shared-memory copy.
    PCU_DEV static int at(int r, int c) {
        if (KV == BF16) return c ^ ((r & 6) ^ ((r & 1) << 2));
        return D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
    }
    // The j-th chunk of a K row that lane quad t takes, and the i-th of the D / 8 elements lane group g has of V.
    PCU_DEV static int k_chunk(int t, int j) { return KV == BF16 ? t + 4 * j : KCH * t + j; }
    PCU_DEV static int v_elem(int g, int i) {
        return KV == BF16 ? 8 * g + (i & 7) + 64 * (i >> 3) : (D / 8) * g + i;
    }
};

template <bool BF>
PCU_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

PCU_DEV uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

PCU_DEV uint32_t bf16x2(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
PCU_DEV uint32_t f16x2(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
PCU_DEV __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
PCU_DEV uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// Two numbers as N BF16 (or F16) parts each, largest first: x = part 0 + part 1 + ...
template <bool BF, int N>
PCU_DEV void split_parts(float lo, float hi, uint32_t (&p)[N]) {
    #pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = BF ? bf16x2(lo, hi) : f16x2(lo, hi);
        if (i + 1 < N) {
            if (BF) {
                lo -= __uint_as_float(p[i] << 16);
                hi -= __uint_as_float(p[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(as_half2(p[i]));
                lo -= f.x;
                hi -= f.y;
            }
        }
    }
}

// o += the PP products of a cell. The tensor cores cut their sums off instead of rounding them, always towards 0; F32
// rows add a cell's sum to o in F32 arithmetic, or the bias of hundreds of cells would show (1.4e-6 instead of 5e-7
// after 4096 keys).
template <bool BF, bool APART, int PP>
PCU_DEV void add_products(float (&o)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&lo)[PP], const uint32_t (&hi)[PP]) {
    if (APART) {
        float u[4] = {0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int k = 0; k < PP; ++k) mma16816<BF>(u, a0, a1, a2, a3, lo[k], hi[k]);
        #pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += u[c];
    } else {
        #pragma unroll
        for (int k = 0; k < PP; ++k) mma16816<BF>(o, a0, a1, a2, a3, lo[k], hi[k]);
    }
}

// 2^(e - ref) of scale bytes, as F32; at or below 2^-127 it is 0, infinite for e - ref = 128, no more.
PCU_DEV float rel_scale(int e, int ref) { return __uint_as_float((uint32_t)max(e - ref + 127, 0) << 23); }

// How far a block's exponent may pass the reference that its codes are made F16 numbers under. E4M3: code * 2^SLACK has
// to be an F16 number. I8: so has 1152 * 2^SLACK, which codes_row and codes_pair take off again. And 255, the scale of
// blocks that are not finite, has to pass the largest reference that finite ones make by more (i8: 249, E4M3: 247).
template <int KV>
struct Slack {
    static constexpr int value = KV == I8 ? 5 : 7;
    static_assert((KV == I8 ? 1152 : 448) * (1 << value) <= 65504, "numbers that codes are unpacked through are finite in F16");
    static_assert((KV == I8 ? 249 : 247) + value < 255, "a scale of 255 is noticed");
};

PCU_DEV uint32_t e4m3x2_f16x2(uint32_t pair) {
    uint32_t h;
    asm("{\n\t.reg .b16 p, u;\n\tmov.b32 {p, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, p;\n\t}" : "=r"(h) : "r"(pair));
    return h;
}

// Bytes 0 and 2 of x as F16 numbers 1152 + code (the offset-binary code in the low byte of 1024's mantissa): one
// three-input operation, (x & mask) ^ magic, which the compiler makes two of when both constants are literals.
PCU_DEV uint32_t i8_magic(uint32_t x) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(y) : "r"(x), "r"(0x00ff00ffu), "r"(0x64806480u));
    return y;
}

// Four consecutive codes of a row, times f (both halves, at most 2^SLACK): the pairs of one k-step. I8: elements (0, 2),
// (1, 3); E4M3: (0, 1), (2, 3). c = -1152 f; the fused product is exact.
template <int KV>
PCU_DEV void codes_row(uint32_t w, uint32_t f, uint32_t c, uint32_t& p0, uint32_t& p1) {
    if (KV == I8) {
        p0 = as_u32(__hfma2(as_half2(i8_magic(w)), as_half2(f), as_half2(c)));
        p1 = as_u32(__hfma2(as_half2(i8_magic(w >> 8)), as_half2(f), as_half2(c)));
    } else {
        p0 = as_u32(__hmul2(as_half2(e4m3x2_f16x2(w)), as_half2(f)));
        p1 = as_u32(__hmul2(as_half2(e4m3x2_f16x2(w >> 16)), as_half2(f)));
    }
}

// Four consecutive codes of two rows, times (fa, fb): pairs (row a, row b) of each element.
template <int KV>
PCU_DEV void codes_pair(uint32_t wa, uint32_t wb, uint32_t f, uint32_t c, uint32_t (&p)[4]) {
    if (KV == I8) {
        const uint32_t x = __byte_perm(wa, wb, 0x5410), y = __byte_perm(wa, wb, 0x7632);
        p[0] = i8_magic(x);
        p[1] = i8_magic(x >> 8);
        p[2] = i8_magic(y);
        p[3] = i8_magic(y >> 8);
        #pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = as_u32(__hfma2(as_half2(p[i]), as_half2(f), as_half2(c)));
    } else {
        const uint32_t x = __byte_perm(wa, wb, 0x5140), y = __byte_perm(wa, wb, 0x7362);
        p[0] = e4m3x2_f16x2(x);
        p[1] = e4m3x2_f16x2(x >> 16);
        p[2] = e4m3x2_f16x2(y);
        p[3] = e4m3x2_f16x2(y >> 16);
        #pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = as_u32(__hmul2(as_half2(p[i]), as_half2(f)));
    }
}

PCU_DEV void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
PCU_DEV void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
PCU_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
PCU_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Copy one cell into a ring stage, rows swizzled; rows whose bit of `need`
// is clear become zeros and their bytes are not read. The scale bytes come
// in chunks of several rows, so they are copied if any row is needed (and are
// ignored for the others).
template <int KV, int D>
PCU_DEV void fill_cell(uint32_t dst, const unsigned char* cell, uint32_t need, int lane) {
    using T = DecodeTile<KV, D>;
    constexpr int N = 2 * CELL * T::CH / 32;
    const unsigned char* src = cell + lane * 16;
    if (need == 0xffffu) {
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = i * 32 + lane, row = x / T::CH, c = x % T::CH;
            cp_async16(dst + row * T::ROWB + T::at(row % CELL, c) * 16, src + i * 512);
        }
    } else {
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = i * 32 + lane, row = x / T::CH, c = x % T::CH, r = row % CELL;
            cp_async16_or_zero(dst + row * T::ROWB + T::at(r, c) * 16, src + i * 512, (need >> r) & 1 ? 16u : 0u);
        }
    }
    if (KV != BF16 && lane < D / CELL && need) cp_async16(dst + 2 * CELL * T::ROWB + lane * 16, src + N * 512);
}

template <int KV, int D, int ROWS>
__global__ void __launch_bounds__(32 * DecodeTile<KV, D>::WARPS, DecodeTile<KV, D>::CTAS)
pages_decode_kernel(const AttnArgs a) {
    using T = DecodeTile<KV, D>;
    constexpr bool BF = KV == BF16, F32 = ROWS == PICKLE_CUDA_ROW_F32;
    constexpr int QP = !F32 ? 1 : BF ? 3 : 2, PP = BF ? (F32 ? 3 : 2) : (F32 ? 2 : 1);
    constexpr int W = T::WARPS, STAGES = T::STAGES;
    constexpr int KS = D / 16, MT = D / 16;
    constexpr int SLACK = Slack<KV>::value;
    constexpr float P_SHIFT = BF ? 0.f : 7.f, GROW = 8.f;
    extern __shared__ __align__(128) unsigned char smem[];
    const View& w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    griddep_wait();
    griddep_launch_dependents();
    const int b = blockIdx.x / w.HK, hk = blockIdx.x % w.HK, split = blockIdx.y;
    int row0, n, kv;
    const int chunk = a.chunk;
    if (!seq_bounds(w, b, row0, n, kv) || n == 0) return;
    const int G = a.G, R = n * G, pos0 = kv - n;       // rows of this KV head; position of the first token
    const Span span = span_of<CELL>(max(0, pos0), kv - 1, a.window, a.sinks);
    const int pieces = (span.n + chunk - 1) / chunk;
    if (split > 0 && split >= pieces) return;
    const int e0 = split * chunk, e1 = min(span.n, e0 + chunk);
    const int mine = (e1 - e0 - warp + W - 1) / W;     // cells e0 + warp, e0 + warp + W, ... of the span

    // What the warp has to know of 32 of its cells, one a lane: where the cell lies in the pool and which of
    // its keys some row sees. Looking a page up and dividing is done for all of them at once, far ahead.
    struct Info {
        uint32_t at;
        int need;
    };
    const uint32_t cpp = w.page_size / CELL;
    auto look_up = [&](int first) {
        Info x{0u, 0};
        const int i = first + lane;
        if (i < mine) {
            const uint32_t step = span.step(e0 + warp + i * W);
            const uint32_t page = step / cpp;
            const int id = w.table[(size_t)b * w.table_stride + page];
            if ((unsigned)id < (unsigned)w.n_pages) {
                const int j0 = step * CELL;
                uint32_t need = j0 + CELL <= kv ? 0xffffu : (1u << (kv - j0)) - 1u;
                if (j0 < span.lo_key) {
                    const uint32_t in = span.lo_key - j0 >= CELL ? 0u : 0xffffu << (span.lo_key - j0);
                    const uint32_t sk = a.sinks <= j0 ? 0u : a.sinks - j0 >= CELL ? 0xffffu : (1u << (a.sinks - j0)) - 1u;
                    need &= in | sk;
                }
                x.at = ((uint32_t)id * w.HK + hk) * cpp + (step - page * cpp);
                x.need = (int)need;
            } else {
                record_error(w.err, PCU_DEVERR_ARG);
            }
        }
        return x;
    };
    const uint32_t ring = smem_u32(smem) + warp * STAGES * T::CELLB;
    const unsigned char* ring_ptr = smem + warp * STAGES * T::CELLB;
    auto fill = [&](const Info& x, int i, int slot) {
        const uint32_t at = __shfl_sync(0xffffffffu, x.at, i & 31);
        const uint32_t need = (uint32_t)__shfl_sync(0xffffffffu, x.need, i & 31);
        if (i < mine) fill_cell<KV, D>(ring + slot * T::CELLB, w.pool + (size_t)at * T::CELLB, need, lane);
    };
    Info cur = look_up(0);
    #pragma unroll
    for (int i = 0; i < STAGES; ++i) {
        fill(cur, i, i);
        cp_async_commit();
    }
    Info nxt = look_up(32);

    // Q^T as B fragments: column g is row g = (token g / G, head g % G).
    uint32_t qf[QP][KS][2];
    float qs = 1.0f;                       // F16: what the row was multiplied by
    {
        const bool live = g < R;
        const size_t at = (size_t)(row0 + (live ? g / G : 0)) * a.q_stride + (size_t)(hk * G + (live ? g % G : 0)) * D;
        constexpr int EPC = 16 / T::ES;                // elements of a chunk
        Row8 x[KS / 2];
        #pragma unroll
        for (int k = 0; k < KS / 2; ++k) {
            x[k].a = x[k].b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (live) x[k] = load_row8<ROWS>(a.q, at + T::k_chunk(t, 8 * k / EPC) * EPC + 8 * k % EPC);
        }
        if (!BF) {
            uint32_t m = 0;
            #pragma unroll
            for (int k = 0; k < KS / 2; ++k) m = max(m, max(amax_bits(x[k].a), amax_bits(x[k].b)));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // 2^(14 - floor(log2 max)): the largest element comes to lie in [2^14, 2^15).
            qs = __uint_as_float(min(268u - (m >> 23), 254u) << 23);
        }
        #pragma unroll
        for (int k = 0; k < KS / 2; ++k) {
            const float v[8] = {x[k].a.x * qs, x[k].a.y * qs, x[k].a.z * qs, x[k].a.w * qs,
                                x[k].b.x * qs, x[k].b.y * qs, x[k].b.z * qs, x[k].b.w * qs};
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                constexpr int o1 = KV == I8 ? 2 : 1, o2 = KV == I8 ? 1 : 2;      // the pairs codes_row makes
                uint32_t p[QP];
                split_parts<BF, QP>(v[4 * h], v[4 * h + o1], p);
                #pragma unroll
                for (int i = 0; i < QP; ++i) qf[i][2 * k + h][0] = p[i];
                split_parts<BF, QP>(v[4 * h + o2], v[4 * h + 3], p);
                #pragma unroll
                for (int i = 0; i < QP; ++i) qf[i][2 * k + h][1] = p[i];
            }
        }
    }
    // Scores of the lane's columns (rows 2t, 2t + 1) in log2 units: S * fc. fc0: without K's reference exponent.
    float fc0[2], fc[2];
    #pragma unroll
    for (int i = 0; i < 2; ++i) fc[i] = fc0[i] = a.scale_log2 / __shfl_sync(0xffffffffu, qs, (2 * t + i) * 4);

    float o[MT][4];
    #pragma unroll
    for (int i = 0; i < MT; ++i)
        #pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    // m: the maximum that p is relative to (log2 units); mz: what is subtracted; thr: the score (as S) past which m moves.
    float m[2] = {-INFINITY, -INFINITY}, mz[2] = {0.f, 0.f}, thr[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int ek = 0, ev = 0;                    // reference exponents (scale bytes) of K (warp) and V (lane group)
    const int pc[2] = {2 * t < R ? pos0 + 2 * t / G : -1, 2 * t + 1 < R ? pos0 + (2 * t + 1) / G : -1};

    int slot = 0;
    for (int i = 0; i < mine; ++i) {
        if (i && (i & 31) == 0) {
            cur = nxt;
            nxt = look_up(i + 32);
        }
        uint32_t need = (uint32_t)__shfl_sync(0xffffffffu, cur.need, i & 31);
        const int j0 = span.step(e0 + warp + i * W) * CELL;
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        if (need) {
            const unsigned char* cell = ring_ptr + slot * T::CELLB;
            // S^T: A = K rows g, g + 8.
            float sp[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            {
                uint32_t f0 = 0, f1 = 0, c0 = 0, c1 = 0;
                if (!BF) {
                    const int blk = D == 128 ? t : t >> 1;
                    int x0 = cell[k_scale(D, g) + blk], x1 = cell[k_scale(D, g + 8) + blk];
                    if (need != 0xffffu) {
                        x0 = (need >> g) & 1 ? x0 : 0;
                        x1 = (need >> (g + 8)) & 1 ? x1 : 0;
                    }
                    if (__any_sync(0xffffffffu, max(x0, x1) > ek + SLACK)) {
                        // A key with a block of scale 255 gets infinite factors, so NaN scores, and moves no reference.
                        ek = max(ek, __reduce_max_sync(0xffffffffu, max(x0 == 255 ? 0 : x0, x1 == 255 ? 0 : x1)));
                        x0 = x0 == 255 ? ek + 128 : x0;
                        x1 = x1 == 255 ? ek + 128 : x1;
                        const float f = __uint_as_float((uint32_t)ek << 23);
                        #pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            fc[k] = fmaxf(fc0[k] * f, 1.2e-38f);      // never 0: a masked score is -inf * fc
                            thr[k] = m[k] == -INFINITY ? m[k] : (m[k] + GROW) / fc[k];
                        }
                    }
                    f0 = f16x2(rel_scale(x0, ek), rel_scale(x0, ek));
                    f1 = f16x2(rel_scale(x1, ek), rel_scale(x1, ek));
                    if (KV == I8) {
                        c0 = as_u32(__hmul2(as_half2(f0), __floats2half2_rn(-1152.f, -1152.f)));
                        c1 = as_u32(__hmul2(as_half2(f1), __floats2half2_rn(-1152.f, -1152.f)));
                    }
                }
                #pragma unroll
                for (int j = 0; j < T::KCH; ++j) {
                    const int ch = T::k_chunk(t, j);
                    const uint4 x = *reinterpret_cast<const uint4*>(cell + k_row(KV, D, g) + T::at(g, ch) * 16);
                    const uint4 y = *reinterpret_cast<const uint4*>(cell + k_row(KV, D, g + 8) + T::at(g + 8, ch) * 16);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
                    #pragma unroll
                    for (int e = 0; e < (BF ? 2 : 4); ++e) {
                        const int ks = j * (BF ? 2 : 4) + e;
                        uint32_t a0, a1, a2, a3;
                        if (BF) {
                            a0 = xs[2 * e]; a2 = xs[2 * e + 1];
                            a1 = ys[2 * e]; a3 = ys[2 * e + 1];
                        } else {
                            codes_row<KV>(xs[e], f0, c0, a0, a2);
                            codes_row<KV>(ys[e], f1, c1, a1, a3);
                        }
                        #pragma unroll
                        for (int p = 0; p < QP; ++p)
                            mma16816<BF>(sp[(QP == 1 ? ks : p) & 1], a0, a1, a2, a3, qf[p][ks][0], qf[p][ks][1]);
                    }
                }
            }
            // Scores of keys g (0, 1) and g + 8 (2, 3) for columns 2t, 2t + 1.
            float s[4];
            #pragma unroll
            for (int k = 0; k < 4; ++k) s[k] = sp[0][k] + sp[1][k];
            if (need != 0xffffu || j0 + CELL - 1 > pos0 ||
                (a.window > 0 && j0 <= kv - 1 - a.window && j0 + CELL - 1 >= a.sinks)) {
                // Not all rows see all of the cell: a V row that is not finite must not reach those that do not see it, and
                // 0 times it is no 0. The rows that see it get a NaN score, and it counts as not needed: 0.
                bool bad[2] = {false, false};
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = g + 8 * h;
                    if (BF) {
                        #pragma unroll
                        for (int j = 0; j < T::KCH; ++j)
                            bad[h] |= bf16x8_bad(*reinterpret_cast<const uint4*>(cell + v_row(KV, D, r) + T::at(r, T::k_chunk(t, j)) * 16));
                        bad[h] |= __shfl_xor_sync(0xffffffffu, (int)bad[h], 1) != 0;
                        bad[h] |= __shfl_xor_sync(0xffffffffu, (int)bad[h], 2) != 0;
                    } else {
                        const uint32_t e = D == 128 ? *reinterpret_cast<const uint32_t*>(cell + v_scale(D, r))
                                                    : *reinterpret_cast<const uint16_t*>(cell + v_scale(D, r));
                        bad[h] = __vcmpeq4(e, 0xffffffffu) != 0;
                    }
                    bad[h] = bad[h] && ((need >> r) & 1);
                }
                #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = g + 8 * (k >> 1);
                    if (!((need >> r) & 1) || !sees(pc[k & 1], j0 + r, a.window, a.sinks)) s[k] = -INFINITY;
                    else if (bad[k >> 1]) s[k] = __uint_as_float(0x7fc00000u);
                }
                const uint32_t v0 = __ballot_sync(0xffffffffu, bad[0]), v1 = __ballot_sync(0xffffffffu, bad[1]);     // bit 4 g
                if (v0 | v1) {
                    #pragma unroll
                    for (int k = 0; k < 16; ++k) need &= ~((((k < 8 ? v0 : v1) >> (4 * (k & 7))) & 1u) << k);
                }
            }
            const float top[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
            if (__any_sync(0xffffffffu, top[0] > thr[0] || top[1] > thr[1])) {
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x = fmaxf(top[k] == -INFINITY ? top[k] : top[k] * fc[k], m[k]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float f = x == m[k] ? 1.0f : ex2(m[k] - x);
                    m[k] = x;
                    mz[k] = x == -INFINITY ? 0.f : x - P_SHIFT;
                    thr[k] = x == -INFINITY ? x : (x + GROW) / fc[k];
                    l[k] *= f;
                    #pragma unroll
                    for (int q = 0; q < MT; ++q) {
                        o[q][k] *= f;
                        o[q][k + 2] *= f;
                    }
                }
            }
            float p[4];
            #pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = ex2(fmaf(s[k], fc[k & 1], -mz[k & 1]));
            l[0] += p[0] + p[2];
            l[1] += p[1] + p[3];
            // P^T as B fragments: rows (columns of S^T) by keys.
            uint32_t pf[2][PP];
            split_parts<BF, PP>(p[0], p[1], pf[0]);
            split_parts<BF, PP>(p[2], p[3], pf[1]);
            #pragma unroll
            for (int k = 0; k < PP; ++k) {
                pf[0][k] = movmatrix(pf[0][k]);
                pf[1][k] = movmatrix(pf[1][k]);
            }
            // O^T: A = V^T, keys 2t, 2t + 1, 2t + 8, 2t + 9 of the lane's elements.
            const int rk[4] = {2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9};
            if (BF) {
                #pragma unroll
                for (int half = 0; half < D / 64; ++half) {
                    uint4 x[4];
                    #pragma unroll
                    for (int k = 0; k < 4; ++k)
                        x[k] = *reinterpret_cast<const uint4*>(cell + v_row(KV, D, rk[k]) + T::at(rk[k], g + 8 * half) * 16);
                    if (need != 0xffffu) {
                        #pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (!((need >> rk[k]) & 1)) x[k] = make_uint4(0u, 0u, 0u, 0u);
                    }
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x0 = (&x[0].x)[e], x1 = (&x[1].x)[e], x2 = (&x[2].x)[e], x3 = (&x[3].x)[e];
                        const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
                        const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
                        add_products<BF, F32, PP>(o[4 * half + e], a0, a1, a2, a3, pf[0], pf[1]);
                    }
                }
            } else {
                const int blk = D == 128 ? g >> 1 : g >> 2;
                int x4[4];
                #pragma unroll
                for (int k = 0; k < 4; ++k) x4[k] = cell[v_scale(D, rk[k]) + blk];
                if (need != 0xffffu) {
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) x4[k] = (need >> rk[k]) & 1 ? x4[k] : 0;
                }
                int top_e = max(max(x4[0], x4[1]), max(x4[2], x4[3]));
                if (__any_sync(0xffffffffu, top_e > ev + SLACK)) {
                    // The four lanes of a group share their output rows.
                    top_e = max(top_e, __shfl_xor_sync(0xffffffffu, top_e, 1));
                    top_e = max(top_e, __shfl_xor_sync(0xffffffffu, top_e, 2));
                    top_e = max(top_e, ev);
                    const float f = rel_scale(ev, top_e);
                    ev = top_e;
                    #pragma unroll
                    for (int q = 0; q < MT; ++q)
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) o[q][k] *= f;
                }
                const uint32_t f0 = f16x2(rel_scale(x4[0], ev), rel_scale(x4[1], ev));
                const uint32_t f1 = f16x2(rel_scale(x4[2], ev), rel_scale(x4[3], ev));
                uint32_t c0 = 0, c1 = 0;
                if (KV == I8) {
                    c0 = as_u32(__hmul2(as_half2(f0), __floats2half2_rn(-1152.f, -1152.f)));
                    c1 = as_u32(__hmul2(as_half2(f1), __floats2half2_rn(-1152.f, -1152.f)));
                }
                constexpr int VW = D / 32;                 // words of codes per key
                uint32_t x[4][VW];
                #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (D == 128) {
                        const uint4 y = *reinterpret_cast<const uint4*>(cell + v_row(KV, D, rk[k]) + T::at(rk[k], g) * 16);
                        x[k][0] = y.x; x[k][1] = y.y; x[k][VW - 2] = y.z; x[k][VW - 1] = y.w;
                    } else {
                        const uint2 y = *reinterpret_cast<const uint2*>(cell + v_row(KV, D, rk[k]) +
                                                                        T::at(rk[k], g >> 1) * 16 + (g & 1) * 8);
                        x[k][0] = y.x; x[k][1] = y.y;
                    }
                }
                #pragma unroll
                for (int e = 0; e < VW; ++e) {
                    uint32_t lo[4], hi[4];
                    codes_pair<KV>(x[0][e], x[1][e], f0, c0, lo);
                    codes_pair<KV>(x[2][e], x[3][e], f1, c1, hi);
                    add_products<BF, F32, PP>(o[2 * e], lo[0], lo[1], hi[0], hi[1], pf[0], pf[1]);
                    add_products<BF, F32, PP>(o[2 * e + 1], lo[2], lo[3], hi[2], hi[3], pf[0], pf[1]);
                }
            }
        }
        __syncwarp();
        const int ahead = i + STAGES;
        fill((ahead ^ i) & ~31 ? nxt : cur, ahead, slot);
        cp_async_commit();
        slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
    cp_async_wait<0>();

    // Join the warps: partial (m, l, O) of each through shared memory.
    const float vf = BF ? 1.0f : scale_f32((uint32_t)ev);
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
    }
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(smem);                       // [W][8][OPAD]
    float* s_ml = s_o + W * 8 * T::OPAD;                               // [W][8][2]
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        float* dst = s_o + (warp * 8 + 2 * t + i) * T::OPAD;
        #pragma unroll
        for (int k = 0; k < MT; ++k) {
            // elements 2k, 2k + 1 of the lane's run are adjacent
            *reinterpret_cast<float2*>(dst + T::v_elem(g, 2 * k)) = make_float2(o[k][i] * vf, o[k][i + 2] * vf);
        }
        if (g == 0) {
            s_ml[(warp * 8 + 2 * t + i) * 2] = m[i];
            s_ml[(warp * 8 + 2 * t + i) * 2 + 1] = l[i];
        }
    }
    __syncthreads();
    const size_t rows = (size_t)w.n_tok * a.H;
    for (int x = threadIdx.x; x < R * (D / 8); x += blockDim.x) {
        const int r = x / (D / 8), i0 = 8 * (x % (D / 8));
        float M = -INFINITY;
        #pragma unroll
        for (int k = 0; k < W; ++k) M = fmaxf(M, s_ml[(k * 8 + r) * 2]);
        const float Mz = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        Row8 y;
        y.a = y.b = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = ex2(s_ml[(k * 8 + r) * 2] - Mz);
            const float4* src = reinterpret_cast<const float4*>(s_o + (k * 8 + r) * T::OPAD + i0);
            const float4 u = src[0], v = src[1];
            L = fmaf(f, s_ml[(k * 8 + r) * 2 + 1], L);
            y.a = make_float4(fmaf(f, u.x, y.a.x), fmaf(f, u.y, y.a.y), fmaf(f, u.z, y.a.z), fmaf(f, u.w, y.a.w));
            y.b = make_float4(fmaf(f, v.x, y.b.x), fmaf(f, v.y, y.b.y), fmaf(f, v.z, y.b.z), fmaf(f, v.w, y.b.w));
        }
        const int tok = row0 + r / G, head = hk * G + r % G;
        if (pieces <= 1) {
            const float inv = 1.0f / (L == 0.f ? 1.0f : L);
            y.a = make_float4(y.a.x * inv, y.a.y * inv, y.a.z * inv, y.a.w * inv);
            y.b = make_float4(y.b.x * inv, y.b.y * inv, y.b.z * inv, y.b.w * inv);
            store_row8<ROWS>(a.out, (size_t)tok * a.out_stride + (size_t)head * D + i0, y);
        } else {
            const size_t row = split * rows + (size_t)tok * a.H + head;
            store_row8<PICKLE_CUDA_ROW_F32>(a.ws_o, row * D + i0, y);
            if (i0 == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * row) = make_float2(M, L);
        }
    }
}

// Output row (t, h) from its pieces:
//   M = max m_i,  o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
// The number of pieces follows from the sequence as in the split kernel, so
// pieces that never ran are never read. A row has one warp where there are many rows, and
// all MERGE_WARPS, each with every fourth piece, behind the kernel for few rows: a decode of
// one sequence has 32 rows of 16 pieces, and their loads are then all in flight.
constexpr int MERGE_WARPS = 4;

// ROWS_CTA: rows of the split kernel's blocks (0: it takes a sequence's rows together).
template <int D, int ROWS, int STEP, int ROWS_CTA>
__global__ void __launch_bounds__(32 * MERGE_WARPS) pages_merge_kernel(const AttnArgs a) {
    constexpr int E = D / 32, RW = ROWS_CTA > 0 ? 1 : MERGE_WARPS;           // warps of a row
    const View& w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = RW == 1 ? 0 : warp;
    const size_t rows = (size_t)w.n_tok * a.H, row = RW == 1 ? (size_t)blockIdx.x * MERGE_WARPS + warp : blockIdx.x;
    // The batch is read before the wait: the split kernel, all of whose CTAs run by now, has waited for its writers.
    int tok = 0, head = 0, pieces = 0;
    const int chunk = ROWS_CTA > 0 ? piece_steps<STEP>(a, lane) : a.chunk;
    if (row < rows) {
        tok = (int)(row / a.H);
        head = (int)(row % a.H);
        const int b = seq_of_row(w, tok, lane);
        int row0, n, kv;
        if (b < w.n_seqs && seq_bounds(w, b, row0, n, kv) && tok >= row0 && tok - row0 < n) {
            if constexpr (ROWS_CTA > 0) {
                pieces = chunk_work<STEP, ROWS_CTA>(a, row0, n, kv, ((tok - row0) * a.G + head % a.G) / ROWS_CTA, chunk).pieces;
            } else {
                pieces = (span_of<STEP>(max(0, kv - n), kv - 1, a.window, a.sinks).n + chunk - 1) / chunk;
            }
        }
    }
    griddep_wait();
    griddep_launch_dependents();
    if (pieces <= 1) return;
    float M = -INFINITY;
    for (int i = lane; i < pieces; i += 32) M = fmaxf(M, a.ws_ml[2 * (i * rows + row)]);
    #pragma unroll
    for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float Mz = M == -INFINITY ? 0.f : M;
    float L = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    // 32 of the warp's pieces a time: a lane holds the statistics of one.
    for (int i0 = part; i0 < pieces; i0 += 32 * RW) {
        float2 ml = make_float2(-INFINITY, 0.f);
        const int own = i0 + lane * RW;
        if (own < pieces) ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * ((size_t)own * rows + row));
        const float f = ex2(ml.x - Mz);
        L += f * ml.y;
        const int m = min(32, (pieces - i0 + RW - 1) / RW);
        #pragma unroll 4
        for (int i = 0; i < m; ++i) {
            const float fi = __shfl_sync(0xffffffffu, f, i);
            const float* src = a.ws_o + ((size_t)(i0 + i * RW) * rows + row) * D + E * lane;
            if (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(src);
                y[0] = fmaf(fi, v.x, y[0]); y[1] = fmaf(fi, v.y, y[1]);
                y[2] = fmaf(fi, v.z, y[2]); y[3] = fmaf(fi, v.w, y[3]);
            } else {
                const float2 v = *reinterpret_cast<const float2*>(src);
                y[0] = fmaf(fi, v.x, y[0]); y[1] = fmaf(fi, v.y, y[1]);
            }
        }
    }
    #pragma unroll
    for (int x = 16; x; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
    if constexpr (RW > 1) {
        __shared__ float4 s_y[RW][32];
        __shared__ float s_l[RW];
        s_y[warp][lane] = make_float4(y[0], y[1], y[2], y[3]);
        if (lane == 0) s_l[warp] = L;
        __syncthreads();
        if (warp) return;
        #pragma unroll
        for (int k = 1; k < RW; ++k) {
            const float4 v = s_y[k][lane];
            y[0] += v.x; y[1] += v.y; y[2] += v.z; y[3] += v.w;
            L += s_l[k];
        }
    }
    const float inv = 1.0f / (L == 0.f ? 1.0f : L);
    const size_t at = (size_t)tok * a.out_stride + (size_t)head * D + E * lane;
    if (ROWS == PICKLE_CUDA_ROW_F32) {
        float* dst = reinterpret_cast<float*>(a.out) + at;
        if (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        else *reinterpret_cast<float2*>(dst) = make_float2(y[0] * inv, y[1] * inv);
    } else {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
        if (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(bf16x2(y[0] * inv, y[1] * inv), bf16x2(y[2] * inv, y[3] * inv));
        else *reinterpret_cast<uint32_t*>(dst) = bf16x2(y[0] * inv, y[1] * inv);
    }
}

}  // namespace pages
