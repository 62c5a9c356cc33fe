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
// they are copied, so that fragments are read without bank conflicts. Codes
// become BF16 numbers in registers: an element is code * 2^e exactly, so
// nothing is rounded. The order of the d's (of K and Q) and of the d's of an
// output tile is free, and chosen so that a lane's elements are contiguous.
//
// F32 rows keep F32 accuracy: q and the weights p are sums of three BF16
// numbers (24 bits), each with a product of its own. BF16 rows: q is exact in one,
// p takes two (16 bits, an error of 2^-17 against the output's own 2^-8).
//
// The running maximum moves only when some score passes it by 2^8 (a warp
// vote), so most cells need no reduction over the keys at all.
#pragma once
#include "pages_attn.cuh"

namespace pages {

template <int KV, int D>
struct DecodeTile {
    static constexpr int ES = elem_bytes(KV);
    static constexpr int ROWB = D * ES;               // bytes of a row
    static constexpr int CH = ROWB / 16;              // 16-byte chunks of a row
    static constexpr int KCH = CH / 4;                // chunks of a K row that a lane takes
    static constexpr int CELLB = cell_bytes(KV, D);
    static constexpr int CPS = 128 / D;               // cells of a ring stage
    // 8-bit: 16 warps an SM in two CTAs, three stages each (203 KB in all). BF16 cells are twice as large
    // and cheaper to use: 12 warps in three CTAs, two stages each.
    static constexpr int WARPS = KV == BF16 ? 4 : 8;
    static constexpr int CTAS = KV == BF16 ? 3 : 2;
    static constexpr int STAGES = KV == BF16 ? 2 : 3;
    static constexpr int STAGEB = CPS * CELLB;
    static constexpr int OPAD = D + 4;                // floats between output columns of a warp's partial
    static constexpr int RING = WARPS * STAGES * STAGEB;
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

PCU_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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

// Two numbers as N BF16 parts each, largest first: x = part 0 + part 1 + ...
template <int N>
PCU_DEV void split_bf16(float lo, float hi, uint32_t (&p)[N]) {
    #pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = bf16x2(lo, hi);
        if (i + 1 < N) {
            lo -= __uint_as_float(p[i] << 16);
            hi -= __uint_as_float(p[i] & 0xffff0000u);
        }
    }
}

PCU_DEV void fma2(float& a, float& b, float sa, float sb, float ca, float cb) {
    asm("{\n\t.reg .b64 x, s, c;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\t"
        "fma.rn.f32x2 x, x, s, c;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a), "+f"(b) : "f"(sa), "f"(sb), "f"(ca), "f"(cb));
}

PCU_DEV void mul2(float& a, float& b, float sa, float sb) {
    asm("{\n\t.reg .b64 x, s;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\t"
        "mul.rn.f32x2 x, x, s;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a), "+f"(b) : "f"(sa), "f"(sb));
}

// A scale byte as the factor and (I8) the addend that turn 2^23 + 128 + code
// into code * 2^e, exactly, in one fused multiply-add. 255 (not finite) gives NaN, 0 (a row left out) zero.
struct Scale {
    float f, c;
};
template <int KV>
PCU_DEV Scale scale_of(uint32_t byte) {
    Scale s;
    s.f = __uint_as_float(byte << 23);
    s.c = KV == I8 ? -8388736.0f * s.f : 0.f;
    return s;
}

// Byte i of offset-binary codes as the float 2^23 + 128 + code.
template <int I>
PCU_DEV float magic(uint32_t w) { return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 + I)); }

PCU_DEV void e4m3x2_f32(uint32_t pair, float& lo, float& hi) {
    uint32_t h;
    asm("{\n\t.reg .b16 p, u;\n\tmov.b32 {p, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, p;\n\t}" : "=r"(h) : "r"(pair));
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}"
        : "=f"(lo), "=f"(hi) : "r"(h));
}

// Four consecutive codes of a row under one scale -> BF16 pairs (0, 1), (2, 3).
template <int KV>
PCU_DEV void codes_row(uint32_t w, const Scale& s, uint32_t& p01, uint32_t& p23) {
    float x0, x1, x2, x3;
    if (KV == I8) {
        w ^= 0x80808080u;
        x0 = magic<0>(w); x1 = magic<1>(w); x2 = magic<2>(w); x3 = magic<3>(w);
        fma2(x0, x1, s.f, s.f, s.c, s.c);
        fma2(x2, x3, s.f, s.f, s.c, s.c);
    } else {
        e4m3x2_f32(w, x0, x1);
        e4m3x2_f32(w >> 16, x2, x3);
        mul2(x0, x1, s.f, s.f);
        mul2(x2, x3, s.f, s.f);
    }
    p01 = bf16x2(x0, x1);
    p23 = bf16x2(x2, x3);
}

// Four consecutive codes of two rows -> BF16 pairs (row a, row b) of each element.
template <int KV>
PCU_DEV void codes_pair(uint32_t wa, uint32_t wb, const Scale& sa, const Scale& sb, uint32_t (&p)[4]) {
    float a[4], b[4];
    if (KV == I8) {
        wa ^= 0x80808080u;
        wb ^= 0x80808080u;
        a[0] = magic<0>(wa); a[1] = magic<1>(wa); a[2] = magic<2>(wa); a[3] = magic<3>(wa);
        b[0] = magic<0>(wb); b[1] = magic<1>(wb); b[2] = magic<2>(wb); b[3] = magic<3>(wb);
        #pragma unroll
        for (int i = 0; i < 4; ++i) fma2(a[i], b[i], sa.f, sb.f, sa.c, sb.c);
    } else {
        e4m3x2_f32(wa, a[0], a[1]);
        e4m3x2_f32(wa >> 16, a[2], a[3]);
        e4m3x2_f32(wb, b[0], b[1]);
        e4m3x2_f32(wb >> 16, b[2], b[3]);
        #pragma unroll
        for (int i = 0; i < 4; ++i) mul2(a[i], b[i], sa.f, sb.f);
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = bf16x2(a[i], b[i]);
}

PCU_DEV void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
PCU_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
PCU_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Copy one cell into a ring stage, rows swizzled; rows whose bit of `need`
// is clear become zeros and their bytes are not read.
template <int KV, int D>
PCU_DEV void fill_cell(uint32_t dst, const unsigned char* cell, uint32_t need, int lane) {
    using T = DecodeTile<KV, D>;
    #pragma unroll
    for (int i = 0; i < 2 * CELL * T::CH / 32; ++i) {
        const int x = i * 32 + lane, row = x / T::CH, c = x % T::CH, r = row % CELL;
        cp_async16(dst + row * T::ROWB + T::at(r, c) * 16, cell + x * 16, (need >> r) & 1 ? 16u : 0u);
    }
    if (KV != BF16 && lane < D / CELL) {
        // 16 scale bytes are 16 / (D / 32) rows: they are copied if any of these rows is needed; a row
        // left out has codes 0, and the scale of such a row is replaced where it is used.
        cp_async16(dst + 2 * CELL * T::ROWB + lane * 16, cell + 2 * CELL * D + lane * 16, need ? 16u : 0u);
    }
}

template <int KV, int D, int ROWS>
__global__ void __launch_bounds__(32 * DecodeTile<KV, D>::WARPS, DecodeTile<KV, D>::CTAS)
pages_decode_kernel(const AttnArgs a) {
    using T = DecodeTile<KV, D>;
    constexpr int QP = ROWS == PICKLE_CUDA_ROW_F32 ? 3 : 1, PP = ROWS == PICKLE_CUDA_ROW_F32 ? 3 : 2;
    constexpr int W = T::WARPS, STAGES = T::STAGES, CPS = T::CPS;
    constexpr int KS = D / 16, MT = D / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t s_need[W][STAGES][CPS];
    const View& w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    griddep_wait();
    griddep_launch_dependents();
    const int b = blockIdx.x / w.HK, hk = blockIdx.x % w.HK, split = blockIdx.y;
    int row0, n, kv;
    if (!seq_bounds(w, b, row0, n, kv) || n == 0) return;
    const int G = a.G, R = n * G, pos0 = kv - n;       // rows of this KV head; position of the first token
    const Span span = span_of<CELL>(max(0, pos0), kv - 1, a.window, a.sinks);
    const int pieces = (span.n + a.chunk - 1) / a.chunk;
    if (split > 0 && split >= pieces) return;
    const int e0 = split * a.chunk, e1 = min(span.n, e0 + a.chunk);
    const int units = (e1 - e0 + CPS - 1) / CPS;

    // Q^T as B fragments: column g is row g = (token g / G, head g % G).
    uint32_t qf[QP][KS][2];
    {
        const bool mine = g < R;
        const size_t at = (size_t)(row0 + (mine ? g / G : 0)) * a.q_stride + (size_t)(hk * G + (mine ? g % G : 0)) * D;
        constexpr int EPC = 16 / T::ES;                // elements of a chunk
        #pragma unroll
        for (int j = 0; j < T::KCH; ++j)
            #pragma unroll
            for (int e = 0; e < EPC; e += 8) {
                Row8 x;
                x.a = x.b = make_float4(0.f, 0.f, 0.f, 0.f);
                if (mine) x = load_row8<ROWS>(a.q, at + T::k_chunk(t, j) * EPC + e);
                const int ks = (j * EPC + e) / 4;
                uint32_t p[QP];
                split_bf16<QP>(x.a.x, x.a.y, p);
                #pragma unroll
                for (int i = 0; i < QP; ++i) qf[i][ks][0] = p[i];
                split_bf16<QP>(x.a.z, x.a.w, p);
                #pragma unroll
                for (int i = 0; i < QP; ++i) qf[i][ks][1] = p[i];
                split_bf16<QP>(x.b.x, x.b.y, p);
                #pragma unroll
                for (int i = 0; i < QP; ++i) qf[i][ks + 1][0] = p[i];
                split_bf16<QP>(x.b.z, x.b.w, p);
                #pragma unroll
                for (int i = 0; i < QP; ++i) qf[i][ks + 1][1] = p[i];
            }
    }

    const uint32_t ring = smem_u32(smem) + warp * STAGES * T::STAGEB;
    const unsigned char* ring_ptr = smem + warp * STAGES * T::STAGEB;
    auto cell_of = [&](int u, int c) { return e0 + u * CPS + c; };      // index into the span
    auto page_id = [&](int u, int c) {
        const int e = cell_of(u, c);
        return u < units && e < e1 ? w.table[(size_t)b * w.table_stride + span.step(e) * CELL / w.page_size] : -1;
    };
    auto fill = [&](int u, int slot, const int (&id)[CPS]) {
        if (u >= units) return;
        #pragma unroll
        for (int c = 0; c < CPS; ++c) {
            const int e = cell_of(u, c);
            uint32_t need = 0;
            const unsigned char* src = w.pool;
            if (e < e1) {
                const int j0 = span.step(e) * CELL;
                if ((unsigned)id[c] < (unsigned)w.n_pages) {
                    // Positions below kv that some row sees.
                    need = j0 + CELL <= kv ? 0xffffu : (1u << (kv - j0)) - 1u;
                    if (j0 < span.lo_key) {
                        const uint32_t in = span.lo_key - j0 >= CELL ? 0u : 0xffffu << (span.lo_key - j0);
                        const uint32_t sk = a.sinks <= j0 ? 0u : a.sinks - j0 >= CELL ? 0xffffu : (1u << (a.sinks - j0)) - 1u;
                        need &= in | sk;
                    }
                    src = cell_ptr<KV, D>(w, id[c], hk, j0 % w.page_size);
                } else if (lane == 0) {
                    record_error(w.err, PCU_DEVERR_ARG);
                }
            }
            if (lane == 0) s_need[warp][slot][c] = need;
            fill_cell<KV, D>(ring + slot * T::STAGEB + c * T::CELLB, src, need, lane);
        }
    };

    // The warp's units: warp, warp + W, ...
    int ids[STAGES][CPS];
    #pragma unroll
    for (int s = 0; s < STAGES; ++s)
        #pragma unroll
        for (int c = 0; c < CPS; ++c) ids[s][c] = page_id(warp + s * W, c);
    int next[CPS];
    #pragma unroll
    for (int c = 0; c < CPS; ++c) next[c] = page_id(warp + STAGES * W, c);
    #pragma unroll
    for (int s = 0; s < STAGES; ++s) {
        fill(warp + s * W, s, ids[s]);
        cp_async_commit();
    }

    float o[MT][4];
    #pragma unroll
    for (int i = 0; i < MT; ++i)
        #pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, mz[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
    // Positions of the lane's two columns (rows 2t, 2t + 1 of the call).
    const int pc[2] = {2 * t < R ? pos0 + 2 * t / G : -1, 2 * t + 1 < R ? pos0 + (2 * t + 1) / G : -1};

    int slot = 0;
    for (int u = warp; u < units; u += W) {
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const unsigned char* stage = ring_ptr + slot * T::STAGEB;
        #pragma unroll
        for (int c = 0; c < CPS; ++c) {
            const uint32_t need = s_need[warp][slot][c];
            if (need == 0) continue;
            const unsigned char* cell = stage + c * T::CELLB;
            const int j0 = span.step(cell_of(u, c)) * CELL;
            // S^T: A = K rows g, g + 8.
            float sp[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            {
                Scale s0, s1;
                if (KV != BF16) {
                    const int blk = D == 128 ? t : t >> 1;
                    s0 = scale_of<KV>(cell[k_scale(D, g) + blk]);
                    s1 = scale_of<KV>(cell[k_scale(D, g + 8) + blk]);
                }
                #pragma unroll
                for (int j = 0; j < T::KCH; ++j) {
                    const int ch = T::k_chunk(t, j);
                    const uint4 x = *reinterpret_cast<const uint4*>(cell + k_row(KV, D, g) + T::at(g, ch) * 16);
                    const uint4 y = *reinterpret_cast<const uint4*>(cell + k_row(KV, D, g + 8) + T::at(g + 8, ch) * 16);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
                    #pragma unroll
                    for (int e = 0; e < (KV == BF16 ? 2 : 4); ++e) {
                        const int ks = j * (KV == BF16 ? 2 : 4) + e;
                        uint32_t a0, a1, a2, a3;
                        if (KV == BF16) {
                            a0 = xs[2 * e]; a2 = xs[2 * e + 1];
                            a1 = ys[2 * e]; a3 = ys[2 * e + 1];
                        } else {
                            codes_row<KV>(xs[e], s0, a0, a2);
                            codes_row<KV>(ys[e], s1, a1, a3);
                        }
                        #pragma unroll
                        for (int p = 0; p < QP; ++p)
                            mma16816(sp[(QP == 1 ? ks : p) & 1], a0, a1, a2, a3, qf[p][ks][0], qf[p][ks][1]);
                    }
                }
            }
            // Scores of keys g (0, 1) and g + 8 (2, 3) for columns 2t, 2t + 1.
            float s[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = (sp[0][i] + sp[1][i]) * a.scale_log2;
            if (need != 0xffffu || j0 + CELL - 1 > pos0 ||
                (a.window > 0 && j0 <= kv - 1 - a.window && j0 + CELL - 1 >= a.sinks)) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = g + 8 * (i >> 1);
                    if (!((need >> r) & 1) || !sees(pc[i & 1], j0 + r, a.window, a.sinks)) s[i] = -INFINITY;
                }
            }
            const float top0 = fmaxf(s[0], s[2]), top1 = fmaxf(s[1], s[3]);
            if (__any_sync(0xffffffffu, top0 > m[0] + 8.0f || top1 > m[1] + 8.0f)) {
                float x[2] = {fmaxf(top0, m[0]), fmaxf(top1, m[1])};
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[i] = fmaxf(x[i], __shfl_xor_sync(0xffffffffu, x[i], 4));
                    x[i] = fmaxf(x[i], __shfl_xor_sync(0xffffffffu, x[i], 8));
                    x[i] = fmaxf(x[i], __shfl_xor_sync(0xffffffffu, x[i], 16));
                    const float f = x[i] == m[i] ? 1.0f : ex2(m[i] - x[i]);
                    m[i] = x[i];
                    mz[i] = x[i] == -INFINITY ? 0.f : x[i];
                    l[i] *= f;
                    #pragma unroll
                    for (int k = 0; k < MT; ++k) {
                        o[k][i] *= f;
                        o[k][i + 2] *= f;
                    }
                }
            }
            float p[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = ex2(s[i] - mz[i & 1]);
            l[0] += p[0] + p[2];
            l[1] += p[1] + p[3];
            // P^T as B fragments: rows (columns of S^T) by keys.
            uint32_t pf[2][PP];
            split_bf16<PP>(p[0], p[1], pf[0]);
            split_bf16<PP>(p[2], p[3], pf[1]);
            #pragma unroll
            for (int i = 0; i < PP; ++i) {
                pf[0][i] = movmatrix(pf[0][i]);
                pf[1][i] = movmatrix(pf[1][i]);
            }
            // O^T: A = V^T, keys 2t, 2t + 1, 2t + 8, 2t + 9 of the lane's elements.
            const int rk[4] = {2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9};
            Scale sv[4];
            if (KV != BF16) {
                const int blk = D == 128 ? g >> 1 : g >> 2;
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    sv[i] = scale_of<KV>((need >> rk[i]) & 1 ? cell[v_scale(D, rk[i]) + blk] : 0);
            }
            if (KV == BF16) {
                #pragma unroll
                for (int half = 0; half < D / 64; ++half) {
                    uint4 x[4];
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[i] = *reinterpret_cast<const uint4*>(cell + v_row(KV, D, rk[i]) + T::at(rk[i], g + 8 * half) * 16);
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x0 = (&x[0].x)[e], x1 = (&x[1].x)[e], x2 = (&x[2].x)[e], x3 = (&x[3].x)[e];
                        const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
                        const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
                        #pragma unroll
                        for (int i = 0; i < PP; ++i) mma16816(o[4 * half + e], a0, a1, a2, a3, pf[0][i], pf[1][i]);
                    }
                }
            } else {
                constexpr int VW = D / 32;                 // words of codes per key
                uint32_t x[4][VW];
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (D == 128) {
                        const uint4 y = *reinterpret_cast<const uint4*>(cell + v_row(KV, D, rk[i]) + T::at(rk[i], g) * 16);
                        x[i][0] = y.x; x[i][1] = y.y; x[i][VW - 2] = y.z; x[i][VW - 1] = y.w;
                    } else {
                        const uint2 y = *reinterpret_cast<const uint2*>(cell + v_row(KV, D, rk[i]) +
                                                                        T::at(rk[i], g >> 1) * 16 + (g & 1) * 8);
                        x[i][0] = y.x; x[i][1] = y.y;
                    }
                }
                #pragma unroll
                for (int e = 0; e < VW; ++e) {
                    uint32_t lo[4], hi[4];
                    codes_pair<KV>(x[0][e], x[1][e], sv[0], sv[1], lo);
                    codes_pair<KV>(x[2][e], x[3][e], sv[2], sv[3], hi);
                    #pragma unroll
                    for (int i = 0; i < PP; ++i) {
                        mma16816(o[2 * e], lo[0], lo[1], hi[0], hi[1], pf[0][i], pf[1][i]);
                        mma16816(o[2 * e + 1], lo[2], lo[3], hi[2], hi[3], pf[0][i], pf[1][i]);
                    }
                }
            }
        }
        __syncwarp();
        fill(u + STAGES * W, slot, next);
        cp_async_commit();
        #pragma unroll
        for (int c = 0; c < CPS; ++c) next[c] = page_id(u + (STAGES + 1) * W, c);
        slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
    cp_async_wait<0>();

    // Join the warps: partial (m, l, O) of each through shared memory.
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
            *reinterpret_cast<float2*>(dst + T::v_elem(g, 2 * k)) = make_float2(o[k][i], o[k][i + 2]);
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

// Output row (t, h) from its pieces, one warp a row:
//   M = max m_i,  o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
// The number of pieces follows from the sequence as in the split kernel, so
// pieces that never ran are never read.
constexpr int MERGE_WARPS = 4;

template <int D, int ROWS, int STEP>
__global__ void __launch_bounds__(32 * MERGE_WARPS) pages_merge_kernel(const AttnArgs a) {
    constexpr int E = D / 32;
    const View& w = a.w;
    const int lane = threadIdx.x & 31;
    const size_t rows = (size_t)w.n_tok * a.H, row = (size_t)blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5);
    griddep_wait();
    griddep_launch_dependents();
    if (row >= rows) return;
    const int tok = (int)(row / a.H), head = (int)(row % a.H);
    const int b = seq_of_row(w, tok, lane);
    if (b >= w.n_seqs) return;
    int row0, n, kv;
    if (!seq_bounds(w, b, row0, n, kv)) return;
    const Span span = span_of<STEP>(max(0, kv - n), kv - 1, a.window, a.sinks);
    const int pieces = (span.n + a.chunk - 1) / a.chunk;
    if (pieces <= 1) return;
    // lane i holds piece i's statistics (pieces beyond 32: the loop below takes 32 at a time)
    float M = -INFINITY;
    for (int i = lane; i < pieces; i += 32) M = fmaxf(M, a.ws_ml[2 * (i * rows + row)]);
    #pragma unroll
    for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float Mz = M == -INFINITY ? 0.f : M;
    float L = 0.f, y[E];
    #pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.f;
    for (int i0 = 0; i0 < pieces; i0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (i0 + lane < pieces) ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * ((size_t)(i0 + lane) * rows + row));
        const float f = ex2(ml.x - Mz);
        L += f * ml.y;
        const int m = min(32, pieces - i0);
        #pragma unroll 4
        for (int i = 0; i < m; ++i) {
            const float fi = __shfl_sync(0xffffffffu, f, i);
            const float* src = a.ws_o + ((size_t)(i0 + i) * rows + row) * D + E * lane;
            if (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(src);
                y[0] = fmaf(fi, v.x, y[0]); y[1] = fmaf(fi, v.y, y[1]);
                y[E - 2] = fmaf(fi, v.z, y[E - 2]); y[E - 1] = fmaf(fi, v.w, y[E - 1]);
            } else {
                const float2 v = *reinterpret_cast<const float2*>(src);
                y[0] = fmaf(fi, v.x, y[0]); y[1] = fmaf(fi, v.y, y[1]);
            }
        }
    }
    #pragma unroll
    for (int x = 16; x; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
    const float inv = 1.0f / (L == 0.f ? 1.0f : L);
    const size_t at = (size_t)tok * a.out_stride + (size_t)head * D + E * lane;
    if (ROWS == PICKLE_CUDA_ROW_F32) {
        float* dst = reinterpret_cast<float*>(a.out) + at;
        if (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0] * inv, y[1] * inv, y[E - 2] * inv, y[E - 1] * inv);
        else *reinterpret_cast<float2*>(dst) = make_float2(y[0] * inv, y[1] * inv);
    } else {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
        if (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(bf16x2(y[0] * inv, y[1] * inv), bf16x2(y[E - 2] * inv, y[E - 1] * inv));
        else *reinterpret_cast<uint32_t*>(dst) = bf16x2(y[0] * inv, y[1] * inv);
    }
}

}  // namespace pages
