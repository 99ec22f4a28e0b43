// xkv_decode.cuh -- rebuilding BF16 words from the sections of an XKV block in shared memory: how a lane
// reads its 8-element chunk of a row (Lay) and turns its words into four BF16 pairs (build_chunk).
#pragma once

#include "common.cuh"

namespace kvx {

__host__ __device__ constexpr uint32_t rep2(uint32_t b) {  // bytes b, b, b+1, b+1
    return b | (b << 4) | ((b + 1) << 8) | ((b + 1) << 12);
}
__host__ __device__ constexpr uint32_t shift4(uint32_t o) {  // bytes o .. o+3
    return o | ((o + 1) << 4) | ((o + 2) << 8) | ((o + 3) << 12);
}
__host__ __device__ constexpr uint32_t sel_code(int j) {  // byte j of A -> bytes 0, 1; of B -> 2, 3
    return uint32_t(j) | (uint32_t(j) << 4) | (uint32_t(4 + j) << 8) | (uint32_t(4 + j) << 12);
}

// Two BF16 values from sign/mantissa bytes (bytes 0 and 1 of each half hold the element's byte:
// bits 0-6 give the mantissa, bit 15 the sign) and exponent residuals in bytes 0 and 2 of cw.
// Exponent = base + residual modulo 256 like bf16_from_delta's uint8 sum (reference
// include/kvexp/bf16.hpp:35-37).  Bytes 1 and 3 of cw may hold other residuals (< 16): times 128
// they land in bits 15-18 of each half, which the select drops, and no carry reaches bit 23.
// The select is written as one LOP3 (mask 0x807F807F picks sg, its complement the sum).
__device__ __forceinline__ uint32_t merge(uint32_t sg, uint32_t cw, uint32_t b7) {
    uint32_t t, w;
    asm("mad.lo.u32 %0, %1, 128, %2;" : "=r"(t) : "r"(cw), "r"(b7));
    asm("lop3.b32 %0, %1, %2, 0x807F807F, 0xE4;" : "=r"(w) : "r"(sg), "r"(t));
    return w;
}

// How this lane reads one tensor of the current block from a ring stage: the 8-element chunk c8
// (head dims 8 c8 .. 8 c8 + 7) of rows t0 + RPI k.  The residual codes start in the 16-byte line at
// code_base (the codes' own copy, or right behind the rows when rows and codes came as one).  Row
// sections start m = 0 or 2 bytes past a 4-byte boundary of the ring; the chunk adds a multiple of
// 4 to the sign/mantissa and raw rows, and 4 (4-bit), 3 (3-bit) or 2 (2-bit) bytes per chunk to
// the residual rows.
struct Lay {
    uint32_t p0, p1;  // sign/mantissa bytes of element pairs 2q and 2q+1 from words q, q+1
    uint32_t w;       // one realigned word from two loaded ones (raw rows)
    uint32_t cs;      // one realigned word of residual codes
    uint32_t rows;    // byte offset of the lane's row window in the stage (4-aligned)
    uint32_t codes;   // byte offset of the lane's residual window in the stage (4-aligned)
};
// rd / cd: data offsets of the block's row and code pieces.
template <int D>
__device__ __forceinline__ Lay make_lay(uint32_t rd, uint32_t cd, int mode, int c8, bool bf16,
                                       uint32_t code_base) {
    // Every offset in a blob is even, so a section starts 0 or 2 bytes past a 4-byte boundary and
    // each selector is one of two constants.
    Lay l;
    const bool m2 = (rd & 2u) != 0u;
    l.p0 = m2 ? rep2(2) : rep2(0);
    l.p1 = m2 ? rep2(4) : rep2(2);
    l.w = m2 ? shift4(2) : shift4(0);
    l.rows = (rd & ~3u) + uint32_t((bf16 || mode == 0) ? 16 * c8 : 8 * c8);
    const uint32_t cb = (cd & 3u) + uint32_t(c8 * (mode == 0 ? 0 : mode));
    l.cs = shift4(0) + (cb & 3u) * 0x1111u;  // bytes o .. o + 3, o = cb mod 4 (odd only for 3-bit)
    l.codes = code_base + (cd & ~3u) + (cb & ~3u);
    return l;
}

// Loads of chunk steps [K0, K0 + G) of one tensor's stage: row words W, residual code words X.
template <int D, int MODE, int G, int K0>
__device__ __forceinline__ void load_chunks(uint32_t qr, uint32_t qc, uint32_t (&W)[G][MODE == 0 ? 5 : 3],
                                            uint32_t (&X)[G][2]) {
    constexpr int RPI = 32 / (D / 8);  // rows a warp step covers
    constexpr int RB = MODE == 0 ? 2 * D : D;  // row bytes
    constexpr int CB = D * MODE / 8;           // residual bytes per row
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const uint32_t q = qr + uint32_t((K0 + g) * RPI * RB);
#pragma unroll
        for (int i = 0; i < (MODE == 0 ? 5 : 3); ++i) W[g][i] = lds_u32(q + 4u * i);
        if constexpr (MODE != 0) {
            const uint32_t c = qc + uint32_t((K0 + g) * RPI * CB);
            X[g][0] = lds_u32(c);
            if constexpr (MODE >= 3) X[g][1] = lds_u32(c + 4u);
        }
    }
}

// The four BF16 pair words of one chunk from its loaded words.
template <int MODE>
__device__ __forceinline__ void build_chunk(const Lay &ly, const uint32_t (&b7)[4],
                                            const uint32_t (&W)[MODE == 0 ? 5 : 3], const uint32_t (&X)[2],
                                            uint32_t (&w)[4]) {
    if constexpr (MODE == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = prmt(W[i], W[i + 1], ly.w);
    } else {
        uint32_t c0, c1, c2, c3;
        if constexpr (MODE == 4) {
            const uint32_t x = prmt(X[0], X[1], ly.cs);
            const uint32_t lo = x & 0x0F0F0F0Fu, hi = (x >> 4) & 0x0F0F0F0Fu;
            c0 = prmt(lo, hi, sel_code(0));
            c1 = prmt(lo, hi, sel_code(1));
            c2 = prmt(lo, hi, sel_code(2));
            c3 = prmt(lo, hi, sel_code(3));
        } else if constexpr (MODE == 3) {
            // 8 residuals of 3 bits in bits 0-23 of x (the library's 3-bit extension): pair j is
            // the 6 bits at 6 j; times 0x2001 puts its first residual at bit 0 and its second at
            // bit 16, and the mask keeps those
            const uint32_t x = prmt(X[0], X[1], ly.cs);
            c0 = ((x & 0x3Fu) * 0x2001u) & 0x70007u;
            c1 = (((x >> 6) & 0x3Fu) * 0x2001u) & 0x70007u;
            c2 = (((x >> 12) & 0x3Fu) * 0x2001u) & 0x70007u;
            c3 = (((x >> 18) & 0x3Fu) * 0x2001u) & 0x70007u;
        } else {  // 8 residuals of 2 bits in the low 16 bits of x
            const uint32_t x = prmt(X[0], 0u, ly.cs);
            const uint32_t ev = x & 0x3333u, od = (x >> 2) & 0x3333u;
            const uint32_t el = ev & 0x0F0Fu, eh = (ev >> 4) & 0x0F0Fu;
            const uint32_t ol = od & 0x0F0Fu, oh = (od >> 4) & 0x0F0Fu;
            c0 = prmt(el, ol, sel_code(0));
            c1 = prmt(eh, oh, sel_code(0));
            c2 = prmt(el, ol, sel_code(1));
            c3 = prmt(eh, oh, sel_code(1));
        }
        w[0] = merge(prmt(W[0], W[1], ly.p0), c0, b7[0]);
        w[1] = merge(prmt(W[0], W[1], ly.p1), c1, b7[1]);
        w[2] = merge(prmt(W[1], W[2], ly.p0), c2, b7[2]);
        w[3] = merge(prmt(W[1], W[2], ly.p1), c3, b7[3]);
    }
}

}  // namespace kvx
