// pages.cuh - the paged KV cache's layout, its 8-bit blocks, and the
// placement of a call's rows (include/pickle_cuda.h, "Paged KV cache").
#pragma once
#include <cstddef>
#include <cstdint>

#include "pcu_common.cuh"
#include "pickle_cuda.h"

namespace pages {

constexpr int CELL = 16;       // positions of a cell
constexpr int BLOCK = 32;      // elements under one scale byte
enum { BF16 = PICKLE_CUDA_KV_BF16, I8 = PICKLE_CUDA_KV_I8, E4M3 = PICKLE_CUDA_KV_E4M3 };

__host__ __device__ constexpr int elem_bytes(int kv) { return kv == BF16 ? 2 : 1; }
__host__ __device__ constexpr int cell_bytes(int kv, int D) {
    return 2 * CELL * D * elem_bytes(kv) + (kv == BF16 ? 0 : 2 * CELL * D / BLOCK);
}
// Byte offsets inside a cell.
__host__ __device__ constexpr int k_row(int kv, int D, int r) { return r * D * elem_bytes(kv); }
__host__ __device__ constexpr int v_row(int kv, int D, int r) { return (CELL + r) * D * elem_bytes(kv); }
__host__ __device__ constexpr int k_scale(int D, int r) { return 2 * CELL * D + r * (D / BLOCK); }
__host__ __device__ constexpr int v_scale(int D, int r) { return 2 * CELL * D + (CELL + r) * (D / BLOCK); }

// What every kernel needs of the pool and the batch.
struct View {
    unsigned char* pool;
    int n_pages, page_size, HK;
    int n_seqs, n_tok, max_q, max_kv;
    const int* q_start;
    const int* kv_len;
    const int* table;
    int table_stride;
    int* err;
};

// The sequence that row t belongs to, found by a whole warp at once: the
// number of sequences that end at or before t. n_seqs: t is behind the last.
PCU_DEV int seq_of_row(const View& w, int t, int lane) {
    if (!w.q_start) return t < w.n_seqs ? t : w.n_seqs;
    int b = 0;
    for (int i = 0; i < w.n_seqs; i += 32) {
        const bool ended = i + lane < w.n_seqs && w.q_start[i + lane + 1] <= t;
        const int n = __popc(__ballot_sync(0xffffffffu, ended));
        b += n;
        if (n < 32) break;
    }
    return b;
}

// Rows and length of sequence b. False (recorded) where its rows pass the
// call's bounds: they are left alone. A length outside the bounds (recorded)
// counts as 0: no page is touched and the rows lie before position 0.
PCU_DEV bool seq_bounds(const View& w, int b, int& row0, int& n, int& kv) {
    row0 = w.q_start ? w.q_start[b] : b;
    n = w.q_start ? w.q_start[b + 1] - row0 : 1;
    kv = w.kv_len[b];
    const bool rows_ok = n >= 0 && n <= w.max_q && row0 >= 0 && row0 <= w.n_tok - n;
    if (!rows_ok || kv < 0 || kv > w.max_kv) {
        record_error(w.err, PCU_DEVERR_ARG);
        kv = 0;
    }
    return rows_ok;
}

// F32 of a scale byte: 2^(s - 127), NaN for 255.
PCU_DEV float scale_f32(uint32_t s) { return __uint_as_float(s == 255u ? 0x7fc00000u : s << 23); }

// The scale byte of a block from the bits of its largest magnitude: the
// smallest power of two for which that element's code is in range. Adding
// `bump` carries into the exponent exactly where the mantissa would round
// past the largest code (i8: 127.5 / 64 on; E4M3: above 464 / 256).
template <int KV>
PCU_DEV uint32_t block_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int e = (int)((amax_bits + (KV == I8 ? 0x10000u : 0x17FFFFu)) >> 23) - (KV == I8 ? 6 : 8);
    return (uint32_t)(e < 16 ? 16 : e);
}

// Four codes of a block as bytes. The product by a power of two is exact.
template <int KV>
PCU_DEV uint32_t codes4(float4 x, uint32_t scale) {
    if (scale == 255u) return 0u;
    const float f = __uint_as_float((254u - scale) << 23);
    if (KV == I8) {
        // + 1.5 * 2^23 rounds to the nearest integer, ties to even, and
        // leaves it in the low byte.
        const float m = 12582912.0f;
        const uint32_t a = __float_as_uint(__fadd_rn(__fmul_rn(x.x, f), m)), b = __float_as_uint(__fadd_rn(__fmul_rn(x.y, f), m));
        const uint32_t c = __float_as_uint(__fadd_rn(__fmul_rn(x.z, f), m)), d = __float_as_uint(__fadd_rn(__fmul_rn(x.w, f), m));
        return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    }
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x.y * f), "f"(x.x * f));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x.w * f), "f"(x.z * f));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Four code bytes as numbers, before the scale.
template <int KV>
PCU_DEV float4 numbers4(uint32_t c) {
    if (KV == I8) {
        return make_float4((float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)(int8_t)(c >> 24));
    }
    uint32_t h0, h1;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"((uint16_t)c));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"((uint16_t)(c >> 16)));
    float4 x;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(x.x), "=f"(x.y) : "r"(h0));
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(x.z), "=f"(x.w) : "r"(h1));
    return x;
}

PCU_DEV uint32_t amax_bits(const float4& x) {
    const uint32_t m = 0x7fffffffu;
    return max(max(__float_as_uint(x.x) & m, __float_as_uint(x.y) & m), max(__float_as_uint(x.z) & m, __float_as_uint(x.w) & m));
}

// Eight consecutive elements of a row.
struct Row8 {
    float4 a, b;
};

PCU_DEV Row8 bf16_row8(const uint4& u) {
    Row8 r;
    r.a = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                      __uint_as_float(u.y & 0xffff0000u));
    r.b = make_float4(__uint_as_float(u.z << 16), __uint_as_float(u.z & 0xffff0000u), __uint_as_float(u.w << 16),
                      __uint_as_float(u.w & 0xffff0000u));
    return r;
}

template <int ROWS>
PCU_DEV Row8 load_row8(const void* base, size_t i) {
    Row8 r;
    if (ROWS == PICKLE_CUDA_ROW_F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + i);
        r.a = p[0];
        r.b = p[1];
    } else {
        r = bf16_row8(*reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + i));
    }
    return r;
}

// The same as loaded, not yet turned into F32 (BF16 rows: half the registers).
template <int ROWS>
struct RawRow8 {
    uint4 u[ROWS == PICKLE_CUDA_ROW_F32 ? 2 : 1];
    PCU_DEV void clear() {
        #pragma unroll
        for (auto& x : u) x = make_uint4(0u, 0u, 0u, 0u);
    }
    PCU_DEV void load(const void* base, size_t i) {
        if (ROWS == PICKLE_CUDA_ROW_F32) {
            const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + i);
            #pragma unroll
            for (int k = 0; k < (int)(sizeof(u) / sizeof(u[0])); ++k) u[k] = p[k];
        } else {
            u[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + i);
        }
    }
    PCU_DEV Row8 row() const {
        if (ROWS == PICKLE_CUDA_ROW_BF16) return bf16_row8(u[0]);
        const uint4 &x = u[0], &y = u[ROWS == PICKLE_CUDA_ROW_F32 ? 1 : 0];
        return Row8{make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w)),
                    make_float4(__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w))};
    }
};

template <int ROWS>
PCU_DEV void store_row8(void* base, size_t i, const Row8& r) {
    if (ROWS == PICKLE_CUDA_ROW_F32) {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i);
        p[0] = r.a;
        p[1] = r.b;
    } else {
        const uint2 lo = pack_bf16x4(r.a, 1.0f), hi = pack_bf16x4(r.b, 1.0f);
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(base) + i) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
}

}  // namespace pages
