// pages_attn.cuh - what the attention kernels over the paged KV cache share:
// their arguments, the keys a sequence's rows can see, and the join of split
// partials.
#pragma once
#include <type_traits>

#include "pages.cuh"

namespace pages {

struct AttnArgs {
    View w;
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    int H, G;
    uint32_t inv_g;       // ceil(2^32 / G), 0 for G = 1
    int window, sinks;
    float scale_log2;     // log2(e) / sqrtf(D)
    int n_splits;         // most pieces a sequence's keys are cut into
    int chunk;            // steps of keys a piece holds (cells, or tiles), if all sequences are the longest
    int chunk_min, target;   // it may be as short as this, as long as there are no more than `target` pieces of a KV head
    float* ws_ml;         // [n_splits][n_tok * H][2]: running maximum (log2 units), sum
    float* ws_o;          // [n_splits][n_tok * H][D]: unnormalised output
};

PCU_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// row / G for rows below 2^29: the multiply's error, row * (G - 1) / 2^32, stays below 1 / G.
PCU_DEV int div_group(int row, const AttnArgs& a) { return a.inv_g ? (int)__umulhi((uint32_t)row, a.inv_g) : row; }

// The keys that the rows at positions first..last can see, in steps of STEP
// keys: steps [0, sunk) and [lo, end) of the sequence, `n` in all. Without a
// gap between them sunk = lo = 0.
struct Span {
    int lo_key;           // first position inside some row's window
    int sunk, lo, n;
    PCU_DEV int step(int i) const { return i < sunk ? i : lo + i - sunk; }
};

template <int STEP>
PCU_DEV Span span_of(int first, int last, int window, int sinks) {
    Span s;
    const int end = last < 0 ? 0 : last / STEP + 1;
    // first - window + 1 cannot overflow: window >= 1 here.
    s.lo_key = window > 0 ? max(0, first - window + 1) : 0;
    s.sunk = (min(sinks, s.lo_key) + STEP - 1) / STEP;
    s.lo = s.lo_key / STEP;
    if (s.sunk >= s.lo) s.sunk = s.lo = 0;
    s.n = s.sunk + max(0, end - s.lo);
    return s;
}

// The steps of a piece, for the kernel that takes rows in blocks. The host plans for sequences that are all as long as
// they may be; where they are shorter, pieces are cut shorter too, to as many in
// all as were planned for (within a sixteenth), so that a long sequence among short
// ones does not keep the others' SMs waiting. Asked by whole warps, the same
// answer for all. 8 x 16 tokens on ragged contexts up to 4096: 43 us planned for the longest, 35 so. The kernel for few
// rows has several CTAs an SM and many waves; there the host's guess at raggedness did better (64 sequences up to 4096:
// 85 us against 90, 32 up to 8192: 71 against 79).
constexpr int TARGET_SEQS = 128;

template <int STEP>
PCU_DEV int piece_steps(const AttnArgs& a, int lane) {
    if (!a.target) return a.chunk;
    const View& w = a.w;
    int steps[TARGET_SEQS / 32], total = 0;
    #pragma unroll
    for (int k = 0; k < TARGET_SEQS / 32; ++k) {
        const int b = 32 * k + lane;
        steps[k] = 0;
        if (b < w.n_seqs) {
            const int kv = w.kv_len[b], n = w.q_start ? w.q_start[b + 1] - w.q_start[b] : 1;
            if (n > 0 && kv > 0 && kv <= w.max_kv) steps[k] = (kv - 1) / STEP + 1;       // no window: see the host
        }
        total += steps[k];
    }
    total = __reduce_add_sync(0xffffffffu, total);
    int lo = max(a.chunk_min, (total + a.target - 1) / a.target), hi = a.chunk;
    while (hi - lo > hi >> 4) {
        const uint32_t mid = (uint32_t)(lo + hi) >> 1, inv = 0xffffffffu / mid + 1u;     // x / mid, or one more for huge x
        uint32_t n = 0;
        #pragma unroll
        for (int k = 0; k < TARGET_SEQS / 32; ++k) n += __umulhi((uint32_t)steps[k] + mid - 1, inv);
        if (__reduce_add_sync(0xffffffffu, n) <= (uint32_t)a.target) hi = (int)mid;
        else lo = (int)mid + 1;
    }
    return hi;
}

// Whether the row at position p sees key j.
PCU_DEV bool sees(int p, int j, int window, int sinks) {
    return j <= p && (window <= 0 || j > p - window || j < sinks);
}

// Whether one of two BF16 numbers is not finite.
PCU_DEV bool bf16x2_bad(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
PCU_DEV bool bf16x8_bad(const uint4& x) { return bf16x2_bad(x.x) || bf16x2_bad(x.y) || bf16x2_bad(x.z) || bf16x2_bad(x.w); }

// The rows and keys of one block of ROWS_CTA rows (a row: a token and a query
// head of its KV head's group), for the kernel that takes them in blocks.
struct ChunkWork {
    int row0, R, pos0;        // the sequence's first row in the buffers, its rows of a KV head, first position
    int r0;                   // first row of the block
    Span span;
    int last;                 // position of the block's last row
    int pieces;
};

template <int BN, int ROWS_CTA>
PCU_DEV ChunkWork chunk_work(const AttnArgs& a, int row0, int n, int kv, int qb, int chunk) {
    ChunkWork c;
    c.row0 = row0;
    c.R = n * a.G;
    c.pos0 = kv - n;
    c.r0 = qb * ROWS_CTA;
    c.last = c.pos0 + min(c.R - 1, c.r0 + ROWS_CTA - 1) / a.G;
    c.span = span_of<BN>(max(0, c.pos0 + c.r0 / a.G), c.last, a.window, a.sinks);
    c.pieces = (c.span.n + chunk - 1) / chunk;
    return c;
}

}  // namespace pages
