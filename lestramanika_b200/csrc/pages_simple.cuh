// pages_simple.cuh - attention over the paged cache, the plain way.
#pragma once
#include "pages_attn.cuh"

namespace pages {

constexpr int SIMPLE_WARPS = 4;

// One CTA per (row, query head). D / 8 lanes take a key each, with a running
// maximum, sum and weighted V of their own; they are joined at the end.
template <int KV, int D, int ROWS>
__global__ void __launch_bounds__(32 * SIMPLE_WARPS) pages_attn_simple_kernel(const AttnArgs a) {
    constexpr int LPR = D / 8, KPW = 32 / LPR, NG = SIMPLE_WARPS * KPW;
    __shared__ float s_m[NG], s_l[NG], s_o[NG][D];
    const View& w = a.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x, h = blockIdx.y;
    const int b = seq_of_row(w, t, lane);
    if (b >= w.n_seqs) return;
    int row0, n, kv;
    if (!seq_bounds(w, b, row0, n, kv)) return;
    const int pos = max(-1, kv - n + (t - row0));
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int sunk = min(a.sinks, lo), n_keys = pos < 0 ? 0 : sunk + pos + 1 - lo;
    const int sub = lane / LPR, l = lane % LPR, grp = warp * KPW + sub;
    const Row8 q = load_row8<ROWS>(a.q, (size_t)t * a.q_stride + (size_t)h * D + 8 * l);
    float m = -INFINITY, sum = 0.f;
    Row8 o;
    o.a = o.b = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n_keys; i0 += NG) {
        const int i = i0 + grp;
        const int j = i < sunk ? i : lo + i - sunk;
        const int page = i < n_keys ? page_of(w, b, j) : -1;
        const int p = j % w.page_size;
        const unsigned char* cell = cell_ptr<KV, D>(w, max(page, 0), h / a.G, p);
        float s = 0.f;
        if (page >= 0) {
            const Row8 k = load_cached8<KV, D>(cell, p % CELL, 8 * l, false);
            s = q.a.x * k.a.x + q.a.y * k.a.y + q.a.z * k.a.z + q.a.w * k.a.w + q.b.x * k.b.x + q.b.y * k.b.y +
                q.b.z * k.b.z + q.b.w * k.b.w;
        }
        #pragma unroll
        for (int x = 1; x < LPR; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (page < 0) continue;
        s *= a.scale_log2;
        const float m2 = fmaxf(m, s), f = m == m2 ? 1.0f : ex2(m - m2), e = ex2(s - m2);
        m = m2;
        sum = sum * f + e;
        const Row8 v = load_cached8<KV, D>(cell, p % CELL, 8 * l, true);
        o.a = make_float4(o.a.x * f + e * v.a.x, o.a.y * f + e * v.a.y, o.a.z * f + e * v.a.z, o.a.w * f + e * v.a.w);
        o.b = make_float4(o.b.x * f + e * v.b.x, o.b.y * f + e * v.b.y, o.b.z * f + e * v.b.z, o.b.w * f + e * v.b.w);
    }
    if (l == 0) {
        s_m[grp] = m;
        s_l[grp] = sum;
    }
    *reinterpret_cast<float4*>(&s_o[grp][8 * l]) = o.a;
    *reinterpret_cast<float4*>(&s_o[grp][8 * l + 4]) = o.b;
    __syncthreads();
    if (threadIdx.x < LPR) {
        float M = -INFINITY, L = 0.f;
        for (int g = 0; g < NG; ++g) M = fmaxf(M, s_m[g]);
        Row8 r;
        r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int g = 0; g < NG; ++g) {
            if (s_m[g] == -INFINITY) continue;
            const float f = ex2(s_m[g] - M);
            const float* x = &s_o[g][8 * threadIdx.x];
            L += f * s_l[g];
            r.a = make_float4(r.a.x + f * x[0], r.a.y + f * x[1], r.a.z + f * x[2], r.a.w + f * x[3]);
            r.b = make_float4(r.b.x + f * x[4], r.b.y + f * x[5], r.b.z + f * x[6], r.b.w + f * x[7]);
        }
        const float inv = 1.0f / (L == 0.f ? 1.0f : L);
        r.a = make_float4(r.a.x * inv, r.a.y * inv, r.a.z * inv, r.a.w * inv);
        r.b = make_float4(r.b.x * inv, r.b.y * inv, r.b.z * inv, r.b.w * inv);
        store_row8<ROWS>(a.out, (size_t)t * a.out_stride + (size_t)h * D + 8 * threadIdx.x, r);
    }
}

}  // namespace pages
