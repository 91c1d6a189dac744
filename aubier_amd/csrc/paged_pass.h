// paged_pass.h -- one piece of the attention over pages (kqkv_paged.hip): up to 128 rows against a run of 64-key
// tiles whose cells are found through a block table.  Two forms, on the decode and the prefill kernels' products:
// up to 32 rows (the four waves share the keys of Q.K^T and the columns of P.V) and up to 128 (a wave per 32 rows).
//
// A row is a (token, head) pair of the piece's rows, numbered token * H + head, so any head count and any number of
// tokens fill the matrix instructions' 32 columns.  Pages are multiples of 16 cells, so a wave's 16-key slice of a
// tile lies in one page: its address is one scalar load of the table and a buffer resource at the page's own 64-bit
// base, whose record count ends with the last cell that is seen.  Cells past it read as zeros, whatever they hold.
#pragma once

#include "paged_common.h"
#include "q8_slice.h"

namespace mla {
namespace paged {

using namespace decode;

// LDS DMA as mla_common.h's dma16, with the five wait states that a vector-memory instruction needs behind a vector
// instruction that writes one of its scalar registers (a v_readlane that brings back a spilled resource, a
// v_readfirstlane): the compiler does not see that this text holds one, and without them the load has gone to the
// address that the registers held before.
template <bool NT>
__device__ __forceinline__ void page_dma16(i32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds_base) {
    if constexpr (NT)
        asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen nt lds" :: "v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds_base) : "memory");
    else
        asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" :: "v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds_base) : "memory");
}

constexpr int BLOCK_ROWS = 128;             // rows of the wide form

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Where the keys of a piece are and which of its rows sees which (uniform over the workgroup)
struct Piece {
    int row0, rows;         // its rows: flat rows row0 .. row0 + rows - 1 of the tokens from tok0 on
    int tok0;               // batch row of that first token
    int past;               // flat row r sees the keys before min(past + r / H + 1, key1)
    int key0, key1;         // the keys: tile k holds key0 + 64 k .. + 63, those before key1
    int ta, tb;             // its tiles
    int lim_min;            // the fewest keys that a row sees
    const int32_t * table;  // the block table
    int slot;               // the record that takes the result, or -1: it is complete and goes to dst
};

// Records: (m, l) of the block's 128 rows, m in log2 units (a reference for the scores, at most 15 below their
// maximum; M_NONE: keys were seen, but no score is above -inf; -inf: no key was seen, and o need not be there), then
// o / l in f16 as the accumulators' lanes hold it, so that neither side needs LDS: for every 32 rows D_v / 16 slabs of 1 KB,
// slab s holding columns 16 s .. + 15, lane l's 8 of them (of row l & 31, the upper 8 in the upper half) at 16 l.
// Why f16: |o / l| <= max |V| cannot overflow, and records are half the bytes; in f32 the calls whose groups are cut took 7
// to 15% longer.  The rounding moves a result by 2.0e-4 (relative 2-norm), as much as storing the result in f16 does; a
// group in one piece has none.
template <int DV>
constexpr size_t record_bytes() { return BLOCK_ROWS * 8 + (size_t)BLOCK_ROWS * DV * 2; }

template <int DK, int DV, bool Q8>
struct PieceLds {
    using G = SliceGeom<DK>;
    static constexpr int SLOT8 = Q8 ? Q8Geom<DK>::ROWS_BYTES : 0;       // an int8 slice
    static constexpr int TILE = 2 * NWAVE * SLOT8;                      // the f16 tile behind the int8 ring
    static constexpr int RING = Q8 ? TILE + NWAVE * G::STAGE : G::RING;
    __attribute__((aligned(16))) char ring[RING];
    __attribute__((aligned(16))) half_t px[Q8 ? 1 : 2][HG * DecodeCfg<DK, DV>::PROW];
    __attribute__((aligned(16))) float red[2][HG][NWAVE];
    uint32_t qoff[BLOCK_ROWS];                                          // byte offset of a row's q from its block's first token's
    int drow[BLOCK_ROWS];                                               // its row of dst (head * nt + token), -1: none
    int lim[BLOCK_ROWS];                                                // keys it sees
    // cells of a slice that are seen (by tile modulo 4: tile k + 2's are written while others read tile k's), and
    // the rows of a slice that hold a NaN or an infinity (by tile parity)
    __attribute__((aligned(16))) int vc[4][NWAVE];
    uint64_t bad[2][NWAVE][2];
    Piece piece;                                                        // for what hardly ever runs behind the tiles: saw_any and
    int odd;                                                            // seen_nonfinite, and whether the latter has to
};

// the thread index by way of an opaque move, so that what follows from it is computed where it is used, rather than
// before the loop over pieces and kept (or spilled) through it
__device__ __forceinline__ int opaque_tid() {
    int t;
    asm volatile("v_mov_b32 %0, %1" : "=v"(t) : "v"(threadIdx.x));
    return t;
}

// zero likewise (sixteen registers of it were kept in scratch memory between pieces, and their reload waited for the
// first tile)
__device__ __forceinline__ float opaque_zero() {
    float z;
    asm volatile("v_mov_b32 %0, 0" : "=v"(z));
    return z;
}

template <typename L>
__device__ __forceinline__ void piece_rows(const AttnArgs & a, const Piece & p, L & sh) {
    const int tid = threadIdx.x;
    if (tid == 0) {
        sh.piece = p;
        sh.odd = 0;
    }
    if (tid >= BLOCK_ROWS) return;
    const int r = p.row0 + tid;
    const int t = r / a.n_head, h = r - t * a.n_head;
    const bool live = tid < p.rows;
    // (a row that is not there brings in the first token's first head; nothing of it is used)
    sh.qoff[tid] = live ? (uint32_t)(t - p.row0 / a.n_head) * (uint32_t)a.q_nb2 + (uint32_t)h * (uint32_t)a.q_nb1 : 0u;
    sh.drow[tid] = live ? h * a.nt + p.tok0 + t : -1;
    sh.lim[tid] = live ? min(p.past + t + 1, p.key1) : 0;
}

// A wave's view of a piece's keys
template <int DK>
struct PageStream {
    using G = SliceGeom<DK>;
    struct Dma { i32x4 krs; uint32_t sb; int n; };      // n: cells of the slice that are seen
    static constexpr int MASK = 0;
    const char * kc;
    int64_t kc_nb1;
    const int32_t * table;
    int n_pages, shift, key0, key1, w;
    uint32_t ring_lds, kvoff0, kvoff1;

    __device__ __forceinline__ PageStream(const AttnArgs & a, const Piece & p, int w_, uint32_t ring_lds_, int lane) {
        kc = a.kc;
        kc_nb1 = a.kc_nb1;
        table = p.table;
        n_pages = a.n_pages;
        shift = a.page_shift;
        key0 = p.key0;
        key1 = p.key1;
        w = w_;
        ring_lds = ring_lds_;
        const int r0 = 2 * (lane >> 4) + ((lane >> 3) & 1);
        kvoff0 = (uint32_t)(r0 * (uint32_t)kc_nb1) + 16u * (uint32_t)((lane & 7) ^ row_sw(r0));
        kvoff1 = (uint32_t)((r0 + 8) * (uint32_t)kc_nb1) + 16u * (uint32_t)((lane & 7) ^ row_sw(r0 + 8));
    }
    // the wave's slice of tile k: its first cell and how many cells of it are seen
    __device__ __forceinline__ int slice(int k, int64_t & cell) const {
        const int key = key0 + k * TK + WK * w;
        cell = 0;
        if (key >= key1) return 0;
        const int id = __builtin_amdgcn_readfirstlane(*(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(table + (key >> shift)));
        if (id < 0 || id >= n_pages) return 0;
        cell = ((int64_t)id << shift) + (key & ((1 << shift) - 1));
        return min(WK, key1 - key);
    }
    __device__ __forceinline__ Dma plan(int s, int k, bool there = true) const {
        Dma d;
        int64_t cell = 0;
        d.n = there ? slice(k, cell) : 0;
        d.krs = make_rsrc(kc + cell * kc_nb1, d.n > 0 ? (uint32_t)((int64_t)(d.n - 1) * kc_nb1 + DK * 2) : 0u);
        d.sb = ring_lds + (uint32_t)((s * NWAVE + w) * G::STAGE);
        return d;
    }
    template <bool NT = true>
    __device__ __forceinline__ void put(const Dma & d, int i) const {
        const uint32_t vo = (i & 1) ? kvoff1 : kvoff0, so = 128u * (uint32_t)(i >> 1);
        page_dma16<NT>(d.krs, vo, so, d.sb + (uint32_t)(1024 * i));
    }
    // the same over an 8-bit cache: the slice as linear 16-byte chunks into its int8 slot of stage s, N8 instructions
    static constexpr int ROWB = DK / 32 * 34, SLOT8 = WK * ROWB, FULL8 = SLOT8 / 1024, TAIL8 = SLOT8 % 1024 / 16, N8 = FULL8 + 1;
    static_assert(TAIL8 > 0, "a partial last instruction");
    template <bool NT = true>
    __device__ __forceinline__ int put8(int s, int k, int lane) const {
        int64_t cell;
        const int n = slice(k, cell);
        const i32x4 krs = make_rsrc(kc + cell * ROWB, (uint32_t)(n * ROWB));
        const uint32_t sb = ring_lds + (uint32_t)((s * NWAVE + w) * SLOT8), vo = 16u * (uint32_t)lane;
#pragma unroll
        for (int i = 0; i < FULL8; ++i) page_dma16<NT>(krs, vo, 1024u * (uint32_t)i, sb + 1024u * (uint32_t)i);
        if (lane < TAIL8) page_dma16<NT>(krs, vo, 1024u * (uint32_t)FULL8, sb + 1024u * (uint32_t)FULL8);
        return n;
    }
};

// Of a row whose piece found no score above -inf: whether it sees a key at all, one whose page is there.  By the definition
// the first has weights 0 / 0, NaN, if the other pieces find none either, and an infinity that it sees is NaN times weight
// 0 in the others; the second adds nothing.  Both hardly ever run, so the table is asked again, 64 pages at a time (the
// whole wavefront; lim: keys that the lane's row sees; none: rows without a score).
__device__ __forceinline__ bool saw_any(const AttnArgs & a, const Piece & in_lds, bool none, int lim, int lane) {
    if (__builtin_amdgcn_ballot_w64(none && lim > 0) == 0) return false;        // (0: a row that is not there)
    const Piece p = in_lds;
    const int ka = p.key0 + TK * p.ta, kb = min(p.key1, p.key0 + TK * p.tb);
    if (__builtin_amdgcn_ballot_w64(none && lim > ka) == 0) return false;
    for (int at = ka >> a.page_shift; at <= (kb - 1) >> a.page_shift; at += 64) {
        const bool in = at + lane <= (kb - 1) >> a.page_shift;
        const int id = in ? p.table[at + lane] : -1;
        const uint64_t there = __builtin_amdgcn_ballot_w64(id >= 0 && id < a.n_pages);
        if (there != 0) return lim > max(ka, (at + __builtin_ctzll(there)) << a.page_shift);
    }
    return false;
}

// Non-finite values of the first COLS columns of an f16 slice set to zero (the whole wavefront, its own slice); b0, b1:
// which of rows 0 .. 7 and 8 .. 15 held one (a byte per row).  Only for the tiles that some rows of a piece see and others
// do not: a cell that a row does not see has weight 0 there, and 0 times a NaN or an infinity would reach its sums.  What
// they mean for the rows that do see them is put in by seen_nonfinite.
template <int COLS>
__device__ __forceinline__ void clear_nonfinite(char * sb, int lane, uint64_t & b0, uint64_t & b1) {
    b0 = b1 = 0;
    for (int i = 0; i < COLS / 32; ++i) {                   // 1 KB block i: rows 8 (i & 1) .. + 7, eight lanes a row, 64 columns
        u32x4 * at = reinterpret_cast<u32x4 *>(sb + 1024 * i + 16 * lane);
        u32x4 v = *at;
        bool any = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t x = ((v[c] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;      // exponent all ones
            any |= x != 0;
            v[c] &= ~((x >> 15) * 0xffffu);
        }
        const uint64_t b = __builtin_amdgcn_ballot_w64(any);
        if (b != 0) *at = v;
        if (i & 1) b1 |= b;
        else b0 |= b;
    }
}

// A piece whose tiles held NaN or infinities that clear_nonfinite has taken out: their effect on the rows that see them, after
// the piece's results have been stored (all waves).  By the definition, of a seen cell whose score is NaN or +inf the
// whole row is NaN (inf - inf); one of score -inf has weight 0, and the columns in which it is not finite are NaN (0
// times infinity).  The score's class comes from the cell's non-finite values alone.  The cells are read again, a wavefront
// per cell, as this hardly ever runs; a row that is NaN is not looked at any more, so that a cache full of them takes
// little longer.
template <int DK, int DV, bool Q8, bool QF16>
__device__ __forceinline__ void seen_nonfinite(const AttnArgs & a, const PieceLds<DK, DV, Q8> & sh, char * rec) {
    static_assert(DK % 64 == 0 && DV % 64 == 0, "64 columns at a time");
    const int tid = opaque_tid(), lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Piece p = sh.piece;
    const char * q = a.q + (int64_t)(p.tok0 + p.row0 / a.n_head) * a.q_nb2;
    auto put_nan = [&](int r, int c) {
        if (p.slot >= 0) {
            char * o = rec + BLOCK_ROWS * 8 + (size_t)((r >> 5) * (DV / 16) + (c >> 4)) * 1024 + 16 * ((r & 31) + 4 * (c & 8)) + 2 * (c & 7);
            *reinterpret_cast<half_t *>(o) = (half_t)__builtin_nanf("");
        } else {
            const size_t at = (size_t)sh.drow[r] * DV + c;
            if (a.dst_f16) reinterpret_cast<half_t *>(a.dst)[at] = (half_t)__builtin_nanf("");
            else reinterpret_cast<float *>(a.dst)[at] = __builtin_nanf("");
        }
    };
    const int ka = p.key0 + TK * p.ta, kb = min(p.key1, p.key0 + TK * p.tb);
    // two halves of the rows one after the other, row r0 + lane a lane
#pragma unroll 1
    for (int r0 = 0; r0 < p.rows; r0 += 64) {
        const int r = r0 + lane, lim = sh.lim[r];           // (0 for a row that is not there)
        bool nan = false;
        // from the first tile that not all rows see
        for (int j = max(ka, p.key0 + max(p.lim_min - p.key0, 0) / TK * TK) + w; j < kb; j += NWAVE) {
            bool open = j < lim && !nan;                    // sees the cell, and is not NaN yet
            if (__builtin_amdgcn_ballot_w64(open) == 0) continue;
            const int id = __builtin_amdgcn_readfirstlane(p.table[j >> a.page_shift]);
            if (id < 0 || id >= a.n_pages) continue;
            const char * cell = a.kc + (((int64_t)id << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * a.kc_nb1;
            float score = 0.0f;
#pragma unroll 1
            for (int d0 = 0; d0 < DK; d0 += 64) {
                half_t v;
                if constexpr (Q8) {
                    const char * blk = cell + (d0 + lane) / 32 * 34;
                    v = to_half((float)*reinterpret_cast<const half_t *>(blk) * (float)*reinterpret_cast<const int8_t *>(blk + 2 + (lane & 31)));
                } else {
                    v = *reinterpret_cast<const half_t *>(cell + 2 * (d0 + lane));
                }
                const int bits = __builtin_bit_cast(uint16_t, v);
                for (uint64_t bad = __builtin_amdgcn_ballot_w64((bits & 0x7c00) == 0x7c00);
                     bad != 0 && __builtin_amdgcn_ballot_w64(open) != 0; bad &= bad - 1) {
                    const int at = __builtin_ctzll(bad), d = d0 + at;
                    const float x = (float)__builtin_bit_cast(half_t, (uint16_t)__builtin_amdgcn_readlane(bits, at));
                    if (!open) continue;
                    const half_t qv = QF16 ? reinterpret_cast<const half_t *>(q + sh.qoff[r])[d] : to_half(reinterpret_cast<const float *>(q + sh.qoff[r])[d]);
                    score += (float)qv * x;
                    open = score == score;
                    nan |= !open;
                    if (d < DV) put_nan(r, d);
                }
            }
            const float s = score * a.scale_log2;
            nan |= open && score != 0.0f && !(s < INFINITY);        // (0: the cell holds none)
        }
        // (the narrow form took the scores before it cleared the cells)
        if (p.rows > HG && nan) {
            if (p.slot >= 0) reinterpret_cast<f32x2 *>(rec)[r][1] = __builtin_nanf("");
#pragma unroll 1
            for (int c = 0; c < DV; ++c) put_nan(r, c);
        }
    }
}

// o / l of 32 rows (rg-th of the block), columns c0 .. c0 + 32 N - 1, in f16 to the record, or, complete, to dst: the
// halves swap four columns, so that every lane has eight in a row
template <int DV, int N>
__device__ __forceinline__ void rows_out_f16(const AttnArgs & a, const Piece & p, const f32x16 (&o)[N], float inv, char * rec, int rg, int c0,
                                             int dr, int lane) {
    auto chunk = [&](int i, int qp) {
        u32x2 x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int e = 8 * qp + 4 * j;
            x[j] = __builtin_bit_cast(u32x2, half4{to_half(o[i][e] * inv), to_half(o[i][e + 1] * inv), to_half(o[i][e + 2] * inv),
                                                   to_half(o[i][e + 3] * inv)});
        }
        const auto s0 = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
        return u32x4{s0[0], s1[0], s0[1], s1[1]};
    };
    if (p.slot >= 0) {
        char * to = rec + BLOCK_ROWS * 8 + (size_t)(rg * (DV / 16) + c0 / 16) * 1024 + 16 * lane;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int qp = 0; qp < 2; ++qp) __builtin_nontemporal_store(chunk(i, qp), reinterpret_cast<u32x4 *>(to + 1024 * (2 * i + qp)));
    } else {
        char * to = a.dst + ((size_t)max(dr, 0) * DV + c0 + 8 * (lane >> 5)) * 2;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int qp = 0; qp < 2; ++qp) {
                const u32x4 v = chunk(i, qp);
                if (dr >= 0) *reinterpret_cast<u32x4 *>(to + 32 * (2 * i + qp)) = v;
            }
    }
}

// a lane's four columns of one row, f32, complete, to dst
__device__ __forceinline__ void out_f32(const AttnArgs & a, int dr, int dv, int col, f32x4 v) {
    if (dr >= 0) *reinterpret_cast<f32x4 *>(a.dst + ((size_t)dr * dv + col) * 4) = v;
}

template <int N>
__device__ __forceinline__ void scale_acc(f32x16 (&o)[N], float f) {
    // in place on the accumulator registers (kept in AGPRs); the s_nops cover the MFMA -> VALU read distance
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float tmp;
            asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
                         : "+a"(o[i][r]), "=&v"(tmp) : "v"(f));
        }
    asm volatile("s_nop 7" ::: "memory");
}

// ---------------------------------------------------------------- up to 32 rows
// Over an f16 cache bound by the memory: 480 MB of four long contexts in 76 us, 6.3 TB/s (counters: 1.002 of the bytes read,
// matrix pipes busy in 14% of the cycles), a tile of 72 KB per workgroup in 2.75 us; the next tile's DMA is spread through
// this one's Q.K^T.  Over an 8-bit cache by the conversion's instructions and the waits at four phases' barriers: 48 requests
// of 300 to 9,000 cells at (320, 256) run at 1.9 TB/s, 53 MB in 28 us, where reading alone takes 10.  A tile's latency, 2 us
// where a workgroup has the card to itself, is why small batches are cut into single tiles.
// Rows of q are reached by 32-bit offsets from the first token's (Q_SPAN, which the host checks); a 64-bit address per
// lane (global_load_lds) takes 1 to 2 us more a piece.
// q enters Q.K^T as f16, the weights P.V as f16: the matrix instructions for f32 operands have an eighth of their rate.  The
// weights' rounding moves a result by 1.0e-4 (relative 2-norm; 200 cells, 32 heads), an f32 q's by 3.4e-4.
// Eight rows of f32 q into LDS by a wavefront: DMA instruction i brings chunks 8 i .. 8 i + 7 (16 bytes) of every row, lane
// l's to 1 KB block i at 16 l.  squeeze() then turns them into f16 in place, row r's 16-byte chunk c at
// 1024 (c >> 3) + 128 r + 16 ((c & 7) ^ r) of the first half: the fragments' reads find no bank twice.
__device__ __forceinline__ uint32_t f32_rows_offset(const uint32_t * qoff, int lane) {
    return qoff[lane >> 3] + 16u * (uint32_t)(lane & 7);
}
template <int DK, typename AT>
__device__ __forceinline__ void squeeze(char * ring, AT && at, char * to, int lane) {
    using G = SliceGeom<DK>;
    const int l7 = lane & 7, r = lane >> 3;
    f32x4 x[G::DMA_N];
#pragma unroll
    for (int i = 0; i < G::DMA_N; ++i) x[i] = *reinterpret_cast<const f32x4 *>(ring + at(i) + 16 * lane);
    char * t = to + 128 * r + 16 * ((l7 >> 1) ^ r) + 8 * (l7 & 1);
    char * t1 = to + 128 * r + 16 * (((l7 >> 1) + 4) ^ r) + 8 * (l7 & 1);
#pragma unroll
    for (int i = 0; i < G::DMA_N; ++i)
        *reinterpret_cast<half4 *>(((i & 1) ? t1 : t) + 1024 * (i >> 1)) = half4{to_half(x[i][0]), to_half(x[i][1]), to_half(x[i][2]), to_half(x[i][3])};
}

// q of the 32 rows into LDS at qs, this wave's share: its 8 rows, as f32 (squeezed later), or as f16 half a slice of 16
// rows, as K rows lie
template <int DK, bool F16>
__device__ __forceinline__ void q_rows_dma(const AttnArgs & a, const Piece & p, const uint32_t * qoff, uint32_t qs, int w, int lane) {
    using G = SliceGeom<DK>;
    const i32x4 rs = make_rsrc(a.q + (int64_t)(p.tok0 + p.row0 / a.n_head) * a.q_nb2, (uint32_t)Q_SPAN);
    if constexpr (F16) {
        const int r0 = 2 * (lane >> 4) + ((lane >> 3) & 1);
        const uint32_t at = qoff[8 * w + r0] + 16u * (uint32_t)((lane & 7) ^ row_sw(r0));
#pragma unroll
        for (int i = 0; i < G::DMA_N / 2; ++i)
            page_dma16<false>(rs, at, 128u * (uint32_t)i, qs + (uint32_t)((w >> 1) * G::STAGE + 1024 * (2 * i + (w & 1))));
    } else {
        const uint32_t at = f32_rows_offset(qoff + 8 * w, lane);
#pragma unroll
        for (int i = 0; i < G::DMA_N; ++i) page_dma16<false>(rs, at, 128u * (uint32_t)i, qs + (uint32_t)(w * G::STAGE + 1024 * i));
    }
}

template <int DK, int DV, bool Q8, bool QF16>
__device__ __forceinline__ void narrow_piece(const AttnArgs & a, const Piece & p, PieceLds<DK, DV, Q8> & sh, char * rec) {
    using G = SliceGeom<DK>;
    using C = DecodeCfg<DK, DV>;
    using S = PageStream<DK>;
    using L = PieceLds<DK, DV, Q8>;
    const int tid = opaque_tid(), lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, j16 = lane & 15;
    const S ss(a, p, w, lds_addr(sh.ring), lane);
    const int n_my = p.tb - p.ta;

    // ---- q by way of LDS the stream does not use yet, the first tile (8 bits: two tiles) behind it ----
    half8 qreg[2][G::QSTEPS];
    char * qs = Q8 ? sh.ring + L::TILE : sh.ring + NWAVE * G::STAGE;
    q_rows_dma<DK, QF16>(a, p, sh.qoff, lds_addr(qs), w, lane);
    int n_cur, n_nxt = 0;                    // cells that are seen, of this wave's slice of the tile and of the next
    if constexpr (Q8) {
        n_cur = ss.put8(0, p.ta, lane);
        if (n_my > 1) {
            n_nxt = ss.put8(1, p.ta + 1, lane);
            wait_vm<2 * S::N8>();
        } else {
            wait_vm<S::N8>();
        }
    } else {
        const typename S::Dma d0 = ss.plan(0, p.ta);
#pragma unroll
        for (int i = 0; i < G::DMA_N; ++i) ss.put(d0, i);
        n_cur = d0.n;
        wait_vm<G::DMA_N>();
    }
    if constexpr (!QF16) squeeze<DK>(qs + w * G::STAGE, [](int i) { return 1024 * i; }, qs + w * G::STAGE, lane);
    __syncthreads();
    {
        // chunk 4 s + g of row 16 n + j16
        const int a0 = QF16 ? slot_byte(j16, g) : (j16 >> 3) * G::STAGE + 128 * (j16 & 7) + 16 * (g ^ (j16 & 7));
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int s = 0; s < G::QSTEPS; ++s)
                qreg[n][s] = *reinterpret_cast<const half8 *>(qs + (QF16 ? n : 2 * n) * G::STAGE + (a0 ^ (64 * (s & 1))) +
                                                              (QF16 ? 2048 : 1024) * (s >> 1));
    }
    const int lim[2] = {sh.lim[j16], sh.lim[16 + j16]};
    __syncthreads();

    float m_ref[2] = {M_NONE, M_NONE};       // rows 16 n + j16, log2 units
    float l_acc = 0.0f;                      // row lane & 31, keys 8 (lane >> 5) .. + 7 of each slice
    f32x16 o[C::NTQ];                        // o^T tiles, as kqkv_decode.hip
    const float zero = opaque_zero();
#pragma unroll
    for (int i = 0; i < C::NTQ; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = zero;
    const PvAddr pv(lane);

    for (int k = 0; k < n_my; ++k) {
        const int par = k & 1;
        const int key = p.key0 + (p.ta + k) * TK + WK * w;       // this wave's first key
        f32x4 s0, s1;
        char * sb;
        int n_new = 0;
        if constexpr (Q8) {
            if (k + 1 < n_my) wait_vm<S::N8>();
            else wait_vm<0>();
            if (k > 0) __syncthreads();      // every wave is past the P.V of tile k - 1
            sb = sh.ring + L::TILE + w * G::STAGE;
            qk_slice_q8<DK, DV>(sh.ring + (par * NWAVE + w) * L::SLOT8, sb, lane, qreg, s0, s1);
            if (k + 2 < n_my) {              // the slot has been read: tile k + 2 takes it
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                n_new = ss.put8(par, p.ta + k + 2, lane);
            }
        } else {
            if (k > 0) __syncthreads();
            sb = sh.ring + (par * NWAVE + w) * G::STAGE;
            const typename S::Dma dn = ss.plan(par ^ 1, p.ta + k + 1, k + 1 < n_my);
            if (k + 1 < n_my) qk_slice<DK, true, S>(ss, dn, sb, lane, qreg, s0, s1);
            else qk_slice<DK, false, S>(ss, dn, sb, lane, qreg, s0, s1);
            n_nxt = dn.n;
        }
        if (key + WK > p.lim_min && key < p.key1 && p.lim_min < p.key1) {     // some rows see these keys, others do not
            uint64_t b0, b1;                 // (the scores have been taken)
            clear_nonfinite<DV>(sb, lane, b0, b1);
            if ((b0 | b1) != 0 && lane == 0) sh.odd = 1;
        }
        float sc[2][4], mx[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int e = min(n_cur, lim[n] - key) - 4 * g;      // keys of this lane's four that the row sees
            const f32x4 & s = n ? s1 : s0;
            mx[n] = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sc[n][r] = r < e ? s[r] * a.scale_log2 : -INFINITY;
                mx[n] = fmaxf(mx[n], sc[n][r]);
            }
            mx[n] = rows4_max(mx[n]);
        }
        half_t * pxv = sh.px[Q8 ? 0 : par];
        auto put_p = [&]() {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                half4 ph;
#pragma unroll
                for (int r = 0; r < 4; ++r) ph[r] = to_half(exp2_fast(sc[n][r] - m_ref[n]));
                *reinterpret_cast<half4 *>(&pxv[(16 * n + j16) * C::PROW + WK * w + 4 * g]) = ph;
            }
        };
        put_p();
        if (lane < 16) {
            sh.red[par][lane][w] = mx[0];
            sh.red[par][16 + lane][w] = mx[1];
        }
        __syncthreads();
        bool move = false;
        float tm[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const f32x4 r4 = *reinterpret_cast<const f32x4 *>(&sh.red[par][16 * n + j16][0]);
            tm[n] = fmaxf(fmaxf(r4[0], r4[1]), fmaxf(r4[2], r4[3]));
            move |= ref_moves(m_ref[n], tm[n]);
        }
        if (__builtin_amdgcn_ballot_w64(move) != 0) {     // rare: move the reference, rescale, redo P
            float al[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const bool mv = ref_moves(m_ref[n], tm[n]);
                al[n] = !mv ? 1.0f : exp2_fast(m_ref[n] - (tm[n] - REF_DROP));      // 0 from M_NONE
                m_ref[n] = mv ? tm[n] - REF_DROP : m_ref[n];
            }
            const float own = al[(lane >> 4) & 1];
            l_acc *= own;
            if (k > 0) scale_acc(o, own);
            put_p();
            __syncthreads();
        }
        pv_tile<DK, DV>(Q8 ? sh.ring + L::TILE : sh.ring, pxv, Q8 ? 0 : par, w, lane, pv, o, l_acc);
        n_cur = n_nxt;
        if constexpr (Q8) n_nxt = n_new;
    }
    wait_vm<0>();                            // nothing of this wave may still target the ring

    // ---- the end: every wave holds its rows' l and its columns of o ----
    const int lane_e = opaque_tid() & 63, hl = lane_e & 31, hi4 = 4 * (lane_e >> 5);
    const float l = halves_sum(l_acc), mr = m_ref[(lane_e >> 4) & 1];
    const bool none = mr == M_NONE, saw = saw_any(a, sh.piece, none, lim[(lane_e >> 4) & 1], lane_e);
    const float inv = l > 0.0f ? 1.0f / l : none && saw && p.slot < 0 ? __builtin_nanf("") : 0.0f;
    if (p.slot < 0 && !a.dst_f16) {
        const int dr = sh.drow[hl];
#pragma unroll
        for (int i = 0; i < C::NTQ; ++i)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                out_f32(a, dr, DV, C::DVQ * w + 32 * i + 8 * q4 + hi4,
                        f32x4{o[i][4 * q4] * inv, o[i][4 * q4 + 1] * inv, o[i][4 * q4 + 2] * inv, o[i][4 * q4 + 3] * inv});
        return;
    }
    if (p.slot >= 0 && w == 0 && lane_e < HG) reinterpret_cast<f32x2 *>(rec)[lane_e] = f32x2{none && !saw ? -INFINITY : mr, l};
    rows_out_f16<DV, C::NTQ>(a, p, o, inv, rec, 0, C::DVQ * w, sh.drow[hl], lane_e);
}

// ---------------------------------------------------------------- up to 128 rows
// 4.24 us a tile on all CUs, 1.08 PFLOP/s, at (576, 512), 2.46 at (320, 256); over an 8-bit cache 4.71 and 2.72, as the
// slices' conversion stands between two barriers.  Counters at (576, 512): the matrix pipes are busy in 44% of the cycles,
// the LDS pipe in 45% (each wave reads the whole tile, 0.55 MB a tile and CU; half of it bank conflicts of the transpose
// reads), at 2.0 GHz of the card's 2.4.  No unit is full: with every register taken there is one wave per SIMD, and its
// chain of operand reads, products and exponentials takes the time.
// A wave's int8 slice at src -> its f16 slot at dst: per lane, half-blocks (16 values) of one row
template <int DK>
__device__ __forceinline__ void slice_to_f16(const char * src, char * dst, int lane) {
    using G8 = Q8Geom<DK>;
    // half-block h + 4 i of a row, h = lane >> 4: block (h >> 1) + 2 i, so everything moves by constants with i
    const int row = lane & 15, h = lane >> 4;
    const int o = 34 * (h >> 1) + 2 + 16 * (h & 1);                      // its first byte of the row; 68 i further on
    const uint32_t sh = (uint32_t)(o & 2);
    const char * q = src + row * G8::ROWB + (o & ~3), * d = src + row * G8::ROWB + 34 * (h >> 1);
    char * t0 = dst + slot_byte(row, 2 * h), * t1 = dst + slot_byte(row, 2 * h + 1);
#pragma unroll
    for (int i = 0; i < G8::ITEMS; ++i) {
        uint32_t x[5], y[4];
        // (the fifth word of an aligned run is the next block's, or lies behind the slice's last row: not used then)
#pragma unroll
        for (int k = 0; k < 5; ++k) x[k] = *reinterpret_cast<const uint32_t *>(q + 68 * i + 4 * k);
        const half_t ds = *reinterpret_cast<const half_t *>(d + 68 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = __builtin_amdgcn_alignbyte(x[k + 1], x[k], sh);
        *reinterpret_cast<half8 *>(t0 + 2048 * i) = q8x8_to_f16<0>(y[0], y[1], 0u, ds);
        *reinterpret_cast<half8 *>(t1 + 2048 * i) = q8x8_to_f16<0>(y[2], y[3], 0u, ds);
        if (i % 3 == 2) __builtin_amdgcn_sched_barrier(0);               // three half-blocks' loads in flight
    }
}

// q of a wave's 32 rows as fragments, qf[st] = row lane & 31, d = 16 st + 8 (lane >> 5) .. + 7, by way of LDS of the
// wave's own, so that the rows are read in whole lines: lane by lane a fragment is 16 bytes of a row, and 128 rows'
// lines do not stay in the L1 from one fragment to the next (4 us a piece).  In units of 16 rows of f16 or 8 of f32, as
// large as an f16 slice: even ones through buffer A, odd ones through B, two in flight, and the piece's first tiles
// behind the last even one.  A buffer lies in two halves (the 8-bit ring's slots are half a slice): 1 KB block i at
// lo + 1024 i below G::DMA_N / 2, at hi + 1024 i from there on.
struct QBuffer { int lo, hi; };
template <int DK, bool F16>
struct QWide {
    using G = SliceGeom<DK>;
    static constexpr int RPU = F16 ? 16 : 8, UNITS = 32 / RPU, HALF = G::DMA_N / 2;
    // unit u's DMA_N instructions
    static __device__ __forceinline__ void put(const i32x4 rs, const uint32_t * qoff, uint32_t ring, const QBuffer to, int u, int lane) {
        auto at = [&](int i) { return ring + (uint32_t)(i < HALF ? to.lo : to.hi) + 1024u * (uint32_t)i; };
        if constexpr (F16) {
            const int r0 = 2 * (lane >> 4) + ((lane >> 3) & 1);
            const uint32_t c0 = 16u * (uint32_t)((lane & 7) ^ row_sw(r0));
            const uint32_t a0 = qoff[RPU * u + r0] + c0, a1 = qoff[RPU * u + r0 + 8] + c0;
#pragma unroll
            for (int i = 0; i < G::DMA_N; ++i) page_dma16<false>(rs, (i & 1) ? a1 : a0, 128u * (uint32_t)(i >> 1), at(i));
        } else {
            const uint32_t a0 = f32_rows_offset(qoff + RPU * u, lane);
#pragma unroll
            for (int i = 0; i < G::DMA_N; ++i) page_dma16<false>(rs, a0, 128u * (uint32_t)i, at(i));
        }
    }
    static __device__ __forceinline__ void get(char * ring, const QBuffer from, int u, int lane, half8 (&qf)[DK / 16]) {
        const int hl = lane & 31, hi = lane >> 5, r = hl - RPU * u;
        const int lo = from.lo, step = from.hi - from.lo;
        if constexpr (!F16) squeeze<DK>(ring, [&](int i) { return lo + (i < HALF ? 0 : step) + 1024 * i; }, ring + lo, lane);
        if (r >= 0 && r < RPU) read(ring, lo, step, r, hi, qf);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the buffer has been read
    }
    static __device__ __forceinline__ void read(const char * ring, int lo, int step, int r, int hi, half8 (&qf)[DK / 16]) {
        if constexpr (F16) {
            const int c0 = slot_byte(r, hi);
#pragma unroll
            for (int st = 0; st < DK / 16; ++st) {
                const int blk = 2 * (st >> 2);                           // of rows 0 .. 7; rows 8 .. 15: the next
                const int o = blk + 1 < HALF ? 0 : blk < HALF ? step * (r >> 3) : step;
                qf[st] = *reinterpret_cast<const half8 *>(ring + lo + o + (c0 ^ (32 * (st & 3))) + 2048 * (st >> 2));
            }
        } else {
            const int c0 = 128 * r + 16 * (hi ^ r);
#pragma unroll
            for (int st = 0; st < DK / 16; ++st)
                qf[st] = *reinterpret_cast<const half8 *>(ring + lo + (c0 ^ (32 * (st & 3))) + 1024 * (st >> 2));
        }
    }
};

template <int DK, int DV, bool Q8, bool QF16>
__device__ __forceinline__ void wide_piece(const AttnArgs & a, const Piece & p, PieceLds<DK, DV, Q8> & sh, char * rec) {
    using G = SliceGeom<DK>;
    using S = PageStream<DK>;
    using L = PieceLds<DK, DV, Q8>;
    constexpr int NB = DV / 32;                         // 32-column o^T tiles per wave
    const int tid = opaque_tid(), lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hl = lane & 31, hi = lane >> 5;
    const S ss(a, p, w, lds_addr(sh.ring), lane);
    const bool live_w = HG * w < p.rows;                // a wave without rows only brings in its slices
    const int n_my = p.tb - p.ta;

    // ---- the rows' q and the first tile (8 bits: two), o ----
    using QW = QWide<DK, QF16>;
    half8 qf[DK / 16];
#pragma unroll
    for (int st = 0; st < DK / 16; ++st) qf[st] = half8{0, 0, 0, 0, 0, 0, 0, 0};
    f32x16 o[NB];                                       // o^T tile i: C row = column 32 i + 8 (r / 4) + 4 hi + (r & 3), C col = row hl
    const int lim = sh.lim[HG * w + hl];
    {
        const i32x4 qrs = make_rsrc(a.q + (int64_t)(p.tok0 + p.row0 / a.n_head) * a.q_nb2, (uint32_t)Q_SPAN);
        const uint32_t * qoff = sh.qoff + HG * w;
        const uint32_t ring = lds_addr(sh.ring);
        // buffer A is where the first tiles go: the slot of stage 0, or the int8 slots of both stages
        constexpr int HALF_BYTES = 1024 * QW::HALF;
        static_assert(!Q8 || HALF_BYTES <= L::SLOT8, "half a unit fits an int8 slot");
        const QBuffer A = Q8 ? QBuffer{w * L::SLOT8, (NWAVE + w) * L::SLOT8 - HALF_BYTES} : QBuffer{w * G::STAGE, w * G::STAGE};
        const int b_at = Q8 ? L::TILE + w * G::STAGE : (NWAVE + w) * G::STAGE;
        const QBuffer B = {b_at, b_at};
        QW::put(qrs, qoff, ring, A, 0, lane);
        QW::put(qrs, qoff, ring, B, 1, lane);
        const float zero = opaque_zero();
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = zero;
#pragma unroll 1
        for (int u = 2; u < QW::UNITS; u += 2) {
            wait_vm<G::DMA_N>();
            QW::get(sh.ring, A, u - 2, lane, qf);
            QW::put(qrs, qoff, ring, A, u, lane);
            wait_vm<G::DMA_N>();
            QW::get(sh.ring, B, u - 1, lane, qf);
            QW::put(qrs, qoff, ring, B, u + 1, lane);
        }
        wait_vm<G::DMA_N>();
        QW::get(sh.ring, A, QW::UNITS - 2, lane, qf);
        if constexpr (Q8) {
            const int n0 = ss.template put8<false>(0, p.ta, lane);
            int n1 = 0;
            if (n_my > 1) {
                n1 = ss.template put8<false>(1, p.ta + 1, lane);
                wait_vm<2 * S::N8>();
            } else {
                wait_vm<S::N8>();
            }
            if (lane == 0) {
                sh.vc[0][w] = n0;
                sh.vc[1][w] = n1;
            }
        } else {
            const typename S::Dma d0 = ss.plan(0, p.ta);
#pragma unroll
            for (int i = 0; i < G::DMA_N; ++i) ss.template put<false>(d0, i);
            if (lane == 0) sh.vc[0][w] = d0.n;
            wait_vm<G::DMA_N>();
        }
        QW::get(sh.ring, B, QW::UNITS - 1, lane, qf);
    }

    float m_run = M_NONE;                               // row hl, log2 units
    float l_acc = 0.0f;                                 // row hl, this lane's half of the keys
    const PairPvAddr pv(lane);

    for (int k = 0; k < n_my; ++k) {
        const int par = k & 1;
        const int key_t = p.key0 + (p.ta + k) * TK;
        char * tile;
        typename S::Dma dn = {};
        const bool pf = k + 1 < n_my;
        if constexpr (Q8) {
            if (pf) wait_vm<S::N8>();                   // this wave's int8 slice of the tile has landed
            else wait_vm<0>();
            if (k > 0) __syncthreads();                 // every wave is past the P.V of tile k - 1
            tile = sh.ring + L::TILE;
            slice_to_f16<DK>(sh.ring + (par * NWAVE + w) * L::SLOT8, tile + w * G::STAGE, lane);
        } else {
            wait_vm<0>();                               // this wave's slice of the tile has landed
            tile = sh.ring + par * NWAVE * G::STAGE;
        }
        // all keys seen by all rows: no masks; else the rows that do not see a cell take no part of what it holds, and a cell
        // that holds a NaN or an infinity has no finite score: weight 0 here, the rest is seen_nonfinite's
        const bool split = key_t + TK > p.lim_min && p.lim_min < p.key1;
        if (split) {
            uint64_t b0, b1;
            clear_nonfinite<DK>(tile + w * G::STAGE, lane, b0, b1);
            if (lane == 0) {
                sh.bad[par][w][0] = b0;
                sh.bad[par][w][1] = b1;
                if ((b0 | b1) != 0) sh.odd = 1;
            }
        }
        __syncthreads();                                // the whole tile is in place; every wave is done with tile k - 1
        const int4 vc = *reinterpret_cast<const int4 *>(sh.vc[k & 3]);
        const bool masked = split || key_t + TK > p.key1 || min(min(vc.x, vc.y), min(vc.z, vc.w)) < WK;
        if constexpr (Q8) {
            if (k + 2 < n_my) {                         // its int8 slot is free: tile k + 2 takes it
                const int n = ss.template put8<false>(par, p.ta + k + 2, lane);
                if (lane == 0) sh.vc[(k + 2) & 3][w] = n;
            }
        } else {
            // (behind the last tile: a slice without cells, whose zeros land in the stage that is free)
            dn = ss.plan(par ^ 1, p.ta + k + 1, pf);
            if (lane == 0) sh.vc[(k + 1) & 3][w] = dn.n;
        }
        if (!live_w) {
            if constexpr (!Q8) {
#pragma unroll
                for (int i = 0; i < G::DMA_N; ++i) ss.template put<false>(dn, i);
            }
            continue;
        }
        half8 abuf[QPF_LANDED];
        qk_operands<DK>(tile, lane, abuf);
#pragma unroll 1
        for (int kp = 0; kp < NWAVE / 2; ++kp) {
            const char * sb = tile + 2 * kp * G::STAGE;
            f32x16 s;
            qk_pair_landed<DK>(sb, lane, qf, abuf, s, [&](int st) {
                constexpr int HALF = G::DMA_N / 2;
                static_assert(G::DMA_N % 2 == 0 && DK / 16 == 2 * G::DMA_N, "two pairs of slices of row blocks");
                if constexpr (!Q8)
                    if ((st & 3) == 0) ss.template put<false>(dn, HALF * kp + st / 4);
            });
            constexpr int VPF = 3;
            half8 vb[VPF];
#pragma unroll
            for (int i = 0; i < VPF; ++i) vb[i] = pv.load(sb, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= a.scale_log2;
            if (masked) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int sl = 2 * kp + j;
                    const int n = sl == 0 ? vc.x : sl == 1 ? vc.y : sl == 2 ? vc.z : vc.w;
                    const int e = min(n, lim - key_t - WK * sl) - 4 * hi;
                    if (split) {
                        const uint64_t b0 = sh.bad[par][sl][0], b1 = sh.bad[par][sl][1];
                        if (__builtin_amdgcn_ballot_w64((b0 | b1) != 0) != 0) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (((((i >> 2) ? b1 : b0) >> (8 * ((i & 3) + 4 * hi))) & 0xff) != 0) s[8 * j + i] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)                          // key 8 (i >> 2) + (i & 3) + 4 hi of the slice
                        s[8 * j + i] = 8 * (i >> 2) + (i & 3) < e ? s[8 * j + i] : -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
            if (__builtin_amdgcn_ballot_w64(ref_moves(m_run, mx)) != 0) {
                // rare: move the reference to the row's max over the pair, rescale
                float lo, up;
                halves_pair(mx, lo, up);
                mx = fmaxf(lo, up);
                const bool mv = ref_moves(m_run, mx);
                const bool scale = mv && m_run != M_NONE;
                const float al = scale ? exp2_fast(m_run - (mx - REF_DROP)) : 1.0f;
                m_run = mv ? mx - REF_DROP : m_run;
                if (__builtin_amdgcn_ballot_w64(scale) != 0) {
                    l_acc *= al;
                    scale_acc(o, al);
                }
            }
            half8 pt[2];
            auto put_p = [&](int j, int e0) __attribute__((always_inline)) {
#pragma unroll
                for (int e = e0; e < e0 + 4; ++e) pt[j][e] = to_half(exp2_fast(s[8 * j + e] - m_run));
            };
            put_p(0, 0);
            put_p(0, 4);
#pragma unroll
            for (int u = 0; u < 2 * NB; ++u) {
                const half8 va = vb[u % VPF];
                if (u + VPF < 2 * NB) vb[u % VPF] = pv.load(sb + G::STAGE * ((u + VPF) / NB), (u + VPF) % NB);
                o[u % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pt[u / NB], o[u % NB], 0, 0, 0);
                if (u == 1) put_p(1, 0);
                if (u == 3) put_p(1, 4);
                if (u % NB < 4)
                    l_acc = __builtin_amdgcn_fdot2(half2{pt[u / NB][2 * (u % NB)], pt[u / NB][2 * (u % NB) + 1]}, ONE2, l_acc, false);
                if (u == NB + NB / 2 && kp + 1 < NWAVE / 2) qk_operands<DK>(tile + 2 * (kp + 1) * G::STAGE, lane, abuf);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    wait_vm<0>();                                       // nothing of this wave may still target the ring
    if (!live_w) return;
    const int lane_e = opaque_tid() & 63, hle = lane_e & 31, hi4 = 4 * (lane_e >> 5);
    const float l = halves_sum(l_acc);
    const bool none = m_run == M_NONE, saw = saw_any(a, sh.piece, none, lim, lane_e);
    const float inv = l > 0.0f ? 1.0f / l : none && saw && p.slot < 0 ? __builtin_nanf("") : 0.0f;
    if (p.slot < 0 && !a.dst_f16) {
        const int dr = sh.drow[HG * w + hle];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                out_f32(a, dr, DV, 32 * i + 8 * q4 + hi4,
                        f32x4{o[i][4 * q4] * inv, o[i][4 * q4 + 1] * inv, o[i][4 * q4 + 2] * inv, o[i][4 * q4 + 3] * inv});
        return;
    }
    if (p.slot >= 0 && lane_e < HG)
        reinterpret_cast<f32x2 *>(rec)[HG * w + lane_e] = f32x2{none && !saw ? -INFINITY : m_run, l};
    rows_out_f16<DV, NB>(a, p, o, inv, rec, w, 0, sh.drow[HG * w + hle], lane_e);
}

}  // namespace paged
}  // namespace mla
