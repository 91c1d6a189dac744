// q8_slice.h -- a 16-key slice of an 8-bit (block_q8_0) cache: its geometry, the conversion of its values to f16
// and Q.K^T straight from it (kqkv_decode_q8.hip describes the design).
#pragma once

#include "decode_common.h"

namespace mla {
namespace decode {

template <int DK>
struct Q8Geom {
    static constexpr int ROWB = DK / 32 * 34;                    // bytes per cache row
    static constexpr int ROWS_BYTES = WK * ROWB;                  // one slice: 16 rows
    static_assert(ROWS_BYTES % 16 == 0 && ROWB % 4 == 0, "16-byte DMA of whole slices");
    static constexpr int SLOT = ROWS_BYTES + 256;                 // rows, then the mask slot
    static constexpr int DMA_FULL = ROWS_BYTES / 1024;            // 64-lane 16-byte instructions
    static constexpr int DMA_TAIL = (ROWS_BYTES % 1024) / 16;     // lanes of the partial last one
    static constexpr int DMA_N = DMA_FULL + (DMA_TAIL ? 1 : 0) + 1;   // + the mask
    static constexpr int HB = DK / 16;                            // 16-value half-blocks per row
    static_assert((WK * HB) % 64 == 0, "whole half-blocks per lane");
    static constexpr int ITEMS = WK * HB / 64;                    // half-blocks per lane
};

// Eight int8 values and their block scale d -> f16(q * d).  w0..w2: the aligned dwords that hold
// the values from byte SH of w0 on (SH = 0: w0, w1 alone).  Each byte enters f16 exactly as
// (1024 + (q + 128)) - 1152 (the byte biased by 128 under the f16 bit pattern of 1024), then one
// multiplication by d rounds once: the value a conversion of the exact f32 product q * d gives.
template <int SH>
__device__ __forceinline__ half8 q8x8_to_f16(uint32_t w0, uint32_t w1, uint32_t w2, half_t d) {
    const half2 bias = {1152.0f16, 1152.0f16};
    const half2 dd = {d, d};
    uint32_t x[2];
    if constexpr (SH == 0) {
        x[0] = w0;
        x[1] = w1;
    } else {
        x[0] = __builtin_amdgcn_alignbyte(w1, w0, SH);
        x[1] = __builtin_amdgcn_alignbyte(w2, w1, SH);
    }
    half8 r;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t y = x[k] ^ 0x80808080u;                                   // q + 128 per byte
        const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u);  // bytes 0, 1 under 0x64
        const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u);  // bytes 2, 3 under 0x64
        const half2 a = (__builtin_bit_cast(half2, lo) - bias) * dd;
        const half2 b = (__builtin_bit_cast(half2, hi) - bias) * dd;
        r[4 * k] = a[0];
        r[4 * k + 1] = a[1];
        r[4 * k + 2] = b[0];
        r[4 * k + 3] = b[1];
    }
    return r;
}

// S^T = K . Q^T for the wave's 16 keys, straight from its int8 slice at src (C rows = keys 4 g + r,
// C cols = heads j16 (s0) and 16 + j16 (s1)), dequantising each A fragment in registers: step s is
// Q8_0 block s of every row (D_k / 32 blocks = the K-steps of the 16x16x32 MFMA), lane (j16, g)
// taking values 8 g .. 8 g + 7 of block s of row j16 -- 8 bytes at 34 s + 2 + 8 g of the row, 4-byte
// aligned for odd s, 2 bytes past it for even s (rows are 612 bytes, a multiple of 4) -- and the
// block's scale.  Each converted fragment is also stored to its place in the f16 slot at dst (the
// layout of decode_common.h, slot_byte: chunk 4 s + g of row j16) when P.V reads it (the first D_v
// values of a row: steps s < D_v / 32), after the maxima barrier, so the dequantisation's VALU work
// runs under the Q.K^T MFMAs instead of in a pass of its own.  Operand reads run PF steps ahead of
// their conversion.  Every DMA of the slice has landed.
template <int DK, int DV>
__device__ __forceinline__ void qk_slice_q8(const char * src, char * dst, int lane,
                                            const half8 (&qreg)[2][SliceGeom<DK>::QSTEPS], f32x4 & s0, f32x4 & s1) {
    using G = SliceGeom<DK>;
    using G8 = Q8Geom<DK>;
    static_assert(G::QSTEPS == DK / 32 && G8::ROWB % 4 == 0, "one Q8_0 block per K-step, dword-aligned rows");
    constexpr int PF = 4;
    const int g = lane >> 4, j16 = lane & 15;
    const char * row = src + j16 * G8::ROWB;
    const int a0 = slot_byte(j16, g);
    uint32_t raw[PF][3];
    half_t dsc[PF];
    auto rd = [&](int s) {
        const int b = 34 * s + 2 + 8 * g;                  // = 2 (mod 4) for even s, 0 for odd s
        const uint32_t * p = reinterpret_cast<const uint32_t *>(row + (b & ~3));
        raw[s % PF][0] = p[0];
        raw[s % PF][1] = p[1];
        if ((s & 1) == 0) raw[s % PF][2] = p[2];
        dsc[s % PF] = *reinterpret_cast<const half_t *>(row + 34 * s);
    };
#pragma unroll
    for (int s = 0; s < PF; ++s) rd(s);
    f32x4 acc0, acc1, acc2, acc3;
#pragma unroll
    for (int s = 0; s < G::QSTEPS; ++s) {
        const uint32_t * r = raw[s % PF];
        const half8 av = (s & 1) ? q8x8_to_f16<0>(r[0], r[1], 0u, dsc[s % PF]) : q8x8_to_f16<2>(r[0], r[1], r[2], dsc[s % PF]);
        if (s + PF < G::QSTEPS) rd(s + PF);
        if (32 * s < DV) *reinterpret_cast<half8 *>(dst + (a0 ^ (64 * (s & 1))) + 2048 * (s >> 1)) = av;
        if (s & 1) {
            mfma16(acc2, av, qreg[0][s], s == 1);
            mfma16(acc3, av, qreg[1][s], s == 1);
        } else {
            mfma16(acc0, av, qreg[0][s], s == 0);
            mfma16(acc1, av, qreg[1][s], s == 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    s0 = acc0 + acc2;
    s1 = acc1 + acc3;
}

}  // namespace decode
}  // namespace mla
