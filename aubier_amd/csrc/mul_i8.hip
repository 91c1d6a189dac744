// mul_i8.hip -- the product of int8 rows and int8 weights with a scale for each row and each channel
// (mla_m4_mul_i8): y[t][c] = xs[t] ws[c] sum_k w[c][k] x[t][k], the sum exact in 32 bits (k <= 131,056), rounded to f32 (exactly
// up to 2^24), then two f32 products and, for an f16 result, one rounding more.  Integer sums have no order, so however a form cuts k the
// result is the same bit for bit.
//
// Three kernels, as three things bound it.  Few rows (48 at most, fewer of more weights: up to 32 with 2112 x 4096, 8 with 7168 x 7168, 1
// with 24,576 x 7168): reading the weights once, and latency (direct_kernel).  From there to hundreds: what a CU can fetch and how many
// CUs the shape keeps busy (split_kernel, and sum_kernel where k is cut).  More: the matrix instructions (tile_kernel).  choose()
// (mul_i8_forms.h) estimates each form's time.
#include "mla_common.h"
#include "mul_i8_forms.h"
#include "rows.h"
#include <type_traits>

namespace mla {
namespace rows {

namespace {

// N neighbouring channels of a row of the result: one store where they are all there and aligned (whole; three need no more than a
// value's alignment), else the first `left`
template <int N, typename T>
__device__ __forceinline__ void put_as(char * p, bool whole, int left, const float (&y)[N]) {
    T v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if constexpr (sizeof(T) == 2) v[k] = to_half(y[k]);
        else v[k] = y[k];
    }
    if (whole) {
        if constexpr (N == 3) {         // (a vector of three would be stored as four)
            __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), v, 3 * sizeof(T));
        } else {
            typedef T vec __attribute__((ext_vector_type(N)));
            vec q;
#pragma unroll
            for (int k = 0; k < N; ++k) q[k] = v[k];
            *reinterpret_cast<vec *>(p) = q;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < left) reinterpret_cast<T *>(p)[k] = v[k];
    }
}
template <int N>
__device__ __forceinline__ void put(char * p, bool f16, bool whole, int left, const float (&y)[N]) {
    if (f16) put_as<N, _Float16>(p, whole, left, y);
    else put_as<N, float>(p, whole, left, y);
}

// direct_kernel: few rows.  A workgroup of NW waves takes 16 TN channels and 16 rows; wave w takes the 256-byte runs
// w, w + NW, ... of k, its operands straight from memory (lane l: row l % 16, 16 bytes at 16 (l / 16), as
// v_mfma_i32_16x16x64_i8 takes both; a run is 4 of its steps), and the waves' integers are added in LDS.  Integer sums have
// no order, so the result is the same however k is cut.  Bound by memory latency (a wave has one run's loads on their way, and sends
// the next run's when they are here) and by what a CU fetches (40 KB/us): 1 row x 576 x 7168 5.9 us, x 7168 x 4096 8.1 us (3.6 TB/s), x 24576 x 1536 8.3 us (4.6 TB/s).
template <int NW, int TN>
__global__ __launch_bounds__(64 * NW) void direct_kernel(MulArgs a) {
    constexpr int U = 4, RUN = 64 * U;
    __shared__ i32x4 part[NW][TN][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.x * 16 * TN, t = blockIdx.y * 16 + r;
    // rows past the last one read it again; what they give is not stored
    const char * wr[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) wr[j] = a.w + (int64_t)min(c0 + 16 * j + r, a.n - 1) * a.w_nb1 + 16 * g;
    const char * xr = a.x + (int64_t)min(t, a.n_rows - 1) * a.x_nb1 + 16 * g;
    // the scales of what the wave will put together, on their way with the operands
    const int c = c0 + 16 * (w % TN) + 4 * g;
    const float xs = a.x_scale[min(t, a.n_rows - 1)];
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = a.w_scale[min(c + i, a.n - 1)];
    i32x4 acc[TN] = {};
    auto run = [&](int k, auto whole) {
        i32x4 wv[U][TN], xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = whole || k + 64 * u + 16 * g < a.k;         // (k is a multiple of 16: a lane's bytes are there or not)
            const int at = in ? k + 64 * u : -16 * g;
#pragma unroll
            for (int j = 0; j < TN; ++j) wv[u][j] = *reinterpret_cast<const i32x4 *>(wr[j] + at);
            xv[u] = *reinterpret_cast<const i32x4 *>(xr + at);
            if (!in) xv[u] = i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < TN; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][i], xv[u], acc[i], 0, 0, 0);
    };
    for (int k = RUN * w; k < a.k; k += RUN * NW) {
        if (k + RUN <= a.k) run(k, std::true_type{});
        else run(k, std::false_type{});
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) part[w][i][lane] = acc[i];
    __syncthreads();
    // lane l's four: channels c0 + 16 w + 4 (l / 16) .. + 3 of row l % 16
    if (w >= TN || t >= a.n_rows || c >= a.n) return;
    i32x4 s = part[0][w][lane];
#pragma unroll
    for (int i = 1; i < NW; ++i) s += part[i][w][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (float)s[i] * xs * y[i];
    const int es = a.dst_f16 ? 2 : 4;
    const bool aligned = a.dst_nb1 % (4 * es) == 0 && (reinterpret_cast<uintptr_t>(a.dst) & (4 * es - 1)) == 0;
    put<4>(a.dst + (int64_t)t * a.dst_nb1 + (int64_t)c * es, a.dst_f16, aligned && c + 4 <= a.n, a.n - c, y);
}

// tile_kernel: WN x WM waves take a tile of 32 TN WN channels and 32 TM WM rows, a wave 32 TN x 32 TM of it on
// v_mfma_i32_32x32x32_i8.  k goes in steps of 128 bytes through two LDS stages, filled by DMA a step ahead.
//
// LDS rows are 128 bytes, eight 16-byte chunks, chunk c of row r at place c ^ (r / 2 & 7) (the order in which lanes fetch it), so
// that the operand reads, one chunk of 32 rows by 32 lanes, meet no bank twice (c ^ (r & 7): twice the cycles).  A DMA instruction
// takes 8 rows' whole lines.  Row 32 t + j of a wave's channels is channel TN j + t, so that a lane's accumulators
// of the TN products hold neighbouring channels, and a store takes whole lines of the result.
//
// One barrier a step, ahead of the last quarter's products, whose operands are in registers by then: behind it the next
// step's first operands are read and the DMA of the step after the next is sent into the stage that all have read.
//
// Bound by power where the card is full: 8,000 rows x 7168 x 16,384 798 us on the best card (2.36 POP/s at 1.7 GHz, matrix instructions
// busy 64% of the cycles; the library's int8 product alone 781).  8192 x 8192 x 4096: 291 us; without the DMA 257, without the operand
// reads 263, without both 219, 212 without the barrier too.  300 x 24,576 x 1536 in 192 x 256: 22 us, a step 0.9, start and end 5.5.
typedef int i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void tile_dma16(i32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds_base) {
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" :: "v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds_base) : "memory");
}

constexpr uint32_t PAST = 0xfffffff0u;      // an offset past any resource's end: reads as zeros

template <int WN, int WM, int TN, int TM, int LATE>
struct Tile {
    static constexpr int NW = WN * WM, NT = 64 * NW, BN = 32 * TN * WN, BM = 32 * TM * WM, BK = 128;
    static constexpr int STAGE = (BN + BM) * BK;
    static constexpr int DW = BN / 8 / NW, DX = BM / 8 / NW;           // DMA instructions of a wave and step
    static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0, "whole DMA instructions a wave");
};

template <int WN, int WM, int TN, int TM, int LATE>
__global__ __launch_bounds__(64 * WN * WM) void tile_kernel(MulArgs a, int n_ct, int n_tt) {
    using G = Tile<WN, WM, TN, TM, LATE>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * G::STAGE];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // A compute die's workgroups (every eighth) take a run of neighbouring tiles, groups of eight rows of tiles, the rows
    // inside, so that what runs there at a time is a compact block and its operands are shared in the die's L2.
    int ct, tt;
    {
        const int all = n_ct * n_tt, x = blockIdx.x & 7, i = blockIdx.x >> 3;
        const int tile = x * (all >> 3) + min(x, all & 7) + i;
        const int per = 8 * n_ct, grp = tile / per, in = tile - grp * per;
        const int high = min(8, n_tt - 8 * grp);
        ct = __builtin_amdgcn_readfirstlane(in / high);        // (an integer division is vector work)
        tt = __builtin_amdgcn_readfirstlane(8 * grp + in - ct * high);
    }
    const int c0 = ct * G::BN, t0 = tt * G::BM;
    // Resources that end with the last row's last byte: rows past it read as zeros.  Both move 128 bytes a step.
    const char * wb = a.w + (int64_t)c0 * a.w_nb1;
    const char * xb = a.x + (int64_t)t0 * a.x_nb1;
    const uint32_t wn = (uint32_t)((int64_t)(min(G::BN, a.n - c0) - 1) * a.w_nb1 + a.k);
    const uint32_t xn = (uint32_t)((int64_t)(min(G::BM, a.n_rows - t0) - 1) * a.x_nb1 + a.k);
    const int steps = (a.k + G::BK - 1) / G::BK, tail = (a.k & (G::BK - 1)) >> 4;      // tail: chunks of the last step, 0: all
    const uint32_t base = lds_addr(lds);
    // lane l of a DMA instruction: row l / 8 of its eight, chunk (l & 7) ^ (row >> 1) & 7, of odd eights ^ 4 more
    const int chunk = (lane & 7) ^ (lane >> 4);
    constexpr int DMAS = G::DW + G::DX;
    uint32_t vo[DMAS];
#pragma unroll
    for (int i = 0; i < G::DW; ++i) {
        const int b = w * G::DW + i, wave = b / (4 * TN), t = b / 4 % TN, j = 8 * (b & 3) + (lane >> 3);       // row 32 t + j of a wave's channels
        vo[i] = (uint32_t)((32 * TN * wave + TN * j + t) * a.w_nb1) + 16u * (b & 1 ? chunk ^ 4 : chunk);
    }
#pragma unroll
    for (int i = 0; i < G::DX; ++i) {
        const int b = w * G::DX + i;
        vo[G::DW + i] = (uint32_t)((8 * b + (lane >> 3)) * a.x_nb1) + 16u * (b & 1 ? chunk ^ 4 : chunk);
    }
    i32x4 wr, xr;
    bool cut;
    auto prepare = [&](int s) {                             // of step s; one past the last reads zeros, so that the loop needs no branch
        wr = make_rsrc(wb + 128u * s, s < steps ? wn - 128u * s : 0u);
        xr = make_rsrc(xb + 128u * s, s < steps ? xn - 128u * s : 0u);
        cut = s == steps - 1 && tail != 0;
    };
    auto send = [&](int s, int i) {                         // DMA instruction i of the wave
        const uint32_t to = base + (uint32_t)(s & 1) * G::STAGE;
        if (i < G::DW) {
            // past k a row's bytes are another's: zeros in their place (of one operand: it is enough)
            const int b = w * G::DW + i;
            const bool past = cut && (b & 1 ? chunk ^ 4 : chunk) >= tail;
            tile_dma16(wr, past ? PAST : vo[i], 0u, to + 1024u * b);
        } else {
            tile_dma16(xr, vo[i], 0u, to + G::BN * G::BK + 1024u * (w * G::DX + i - G::DW));
        }
    };
    const int wi = w % WN, xi = w / WN;
    const int r = lane & 31, h = lane >> 5;
    const int c = c0 + 32 * TN * wi + TN * r;           // the lane's channels
    float ws[TN], mine = 0.0f;                          // their scales, and the scale of row t0 + thread
#pragma unroll
    for (int t = 0; t < TN; ++t) ws[t] = c + t < a.n ? a.w_scale[c + t] : 0.0f;
    static_assert(G::BM <= G::NT, "a row's scale a thread");
    if (threadIdx.x < G::BM && t0 + (int)threadIdx.x < a.n_rows) mine = a.x_scale[t0 + threadIdx.x];
    prepare(0);
#pragma unroll
    for (int i = 0; i < DMAS; ++i) send(0, i);
    const char * wl = lds + 128 * (32 * TN * wi + r);
    const char * xl = lds + G::BN * G::BK + 128 * (32 * TM * xi + r);
    i32x16 acc[TN][TM] = {};
    i32x4 fw[2][TN], fx[2][TM];
    auto fetch = [&](int to, int stage, int kk) {
        const int at = stage * G::STAGE + 16 * ((2 * kk + h) ^ ((r >> 1) & 7));
#pragma unroll
        for (int t = 0; t < TN; ++t) fw[to][t] = *reinterpret_cast<const i32x4 *>(wl + at + 4096 * t);
#pragma unroll
        for (int t = 0; t < TM; ++t) fx[to][t] = *reinterpret_cast<const i32x4 *>(xl + at + 4096 * t);
    };
    // the products of a quarter, and DMA instructions i0 .. i0 + n - 1 of step s between them: sent at once they would hold the
    // wave until they are taken
    auto products = [&](int of, int s, int i0, int n) {
        int i = 0;
#pragma unroll
        for (int m = 0; m < TN * TM; ++m) {
            const int t = m / TM, u = m % TM;
            acc[t][u] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[of][u], fw[of][t], acc[t][u], 0, 0, 0);
            if (i < n && (m + 1) * n >= (i + 1) * TN * TM) {
                __builtin_amdgcn_sched_barrier(0);
                send(s, i0 + i++);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    fetch(0, 0, 0);
    prepare(1);
#pragma unroll
    for (int i = 0; i < LATE; ++i) send(1, i);
    for (int s = 0; s < steps; ++s) {
        const int st = s & 1;
        fetch(1, st, 1);
        products(0, s + 1, LATE, DMAS - LATE);
        fetch(0, st, 2);
        products(1, 0, 0, 0);
        fetch(1, st, 3);
        products(0, 0, 0, 0);
        // the last quarter's operands are here, the next step's bytes too; nobody reads this stage any more
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        fetch(0, st ^ 1, 0);
        prepare(s + 2);
        products(1, s + 2, 0, LATE);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // acc[t][u][i] of lane l: channel TN r + t of the wave's, row 32 u + 8 (i / 4) + 4 h + i % 4 of the wave's
    float * xs = reinterpret_cast<float *>(lds);
    if (threadIdx.x < G::BM) xs[threadIdx.x] = mine;
    __syncthreads();
    const int es = a.dst_f16 ? 2 : 4;
    // whole groups of TN channels at aligned places go out in one store
    const bool whole = c + TN <= a.n && (TN == 3 || (a.dst_nb1 % (TN * es) == 0 && (reinterpret_cast<uintptr_t>(a.dst) & (TN * es - 1)) == 0));
#pragma unroll
    for (int u = 0; u < TM; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int tl = 32 * (TM * xi + u) + 8 * q + 4 * h;
            const f32x4 s4 = *reinterpret_cast<const f32x4 *>(xs + tl);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + tl + i;
                if (t >= a.n_rows) continue;
                float y[TN];
#pragma unroll
                for (int k = 0; k < TN; ++k) y[k] = (float)acc[k][u][4 * q + i] * s4[i] * ws[k];
                put<TN>(a.dst + (int64_t)t * a.dst_nb1 + (int64_t)c * es, a.dst_f16, whole, a.n - c, y);
            }
        }
}

template <int WN, int WM, int TN, int TM, int LATE = 4>
hipError_t tile(const MulArgs & a, hipStream_t stream) {
    using G = Tile<WN, WM, TN, TM, LATE>;
    const int n_ct = (a.n + G::BN - 1) / G::BN, n_tt = (a.n_rows + G::BM - 1) / G::BM;
    if ((int64_t)n_ct * n_tt * G::NT >= (1ll << 32)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((tile_kernel<WN, WM, TN, TM, LATE>), dim3(n_ct * n_tt), dim3(G::NT), 0, stream, a, n_ct, n_tt);
    return hipGetLastError();
}

// split_kernel: what lies between.  WN x WM x WK waves take 32 TN WN channels and 32 TM WM rows of a part of k (one of n_split); of
// every 128-byte step the WK waves of one place take 128 / WK bytes of each row, so operand bytes are read from LDS less often than by
// waves that share k, and their integers are added in LDS at the end.  ST stages, filled by DMA ST - 1 steps ahead.  Where k is cut,
// the sums of the parts go to the workspace as they lie in the lanes, and sum_kernel puts them together (2.3 us of the launch and its
// reads).  Bound by the start of the stream and by what a CU fetches: 64 rows x 7168 x 4096 9.2 us (3.3 TB/s), 64 x 7168 x 16,384 33 us
// (3.6 TB/s), 300 x 4096 x 4096 14.5 us.
template <int WN_, int WM_, int WK_, int TN_, int TM_>
struct Split {
    static constexpr int WN = WN_, WM = WM_, WK = WK_, TN = TN_, TM = TM_;
    static constexpr int NW = WN * WM * WK, NT = 64 * NW, BN = 32 * TN * WN, BM = 32 * TM * WM, STAGE = (BN + BM) * 128;
    static constexpr int ROOM = (NW > 4 ? 160 : 80) * 1024;             // four waves: two workgroups share a CU
    static constexpr int ST = ROOM / STAGE > 6 ? 6 : ROOM / STAGE;
    static constexpr int DW = BN / 8 / NW, DX = BM / 8 / NW;            // DMA instructions of a wave and step
    static constexpr int F = TN * TM, KK = 4 / WK;
    static constexpr int AT_ONCE = F <= 4 ? F : F % 4 == 0 ? 4 : F % 3 == 0 ? 3 : 2;       // products of a wave added at a time, 4 KB each
    static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0 && NW % 2 == 0, "whole DMA instructions a wave");
    static_assert(ST >= 3 && F % AT_ONCE == 0 && AT_ONCE * NW * 4096 <= ST * STAGE, "stages, and room to add in");
};

template <typename G>
__global__ __launch_bounds__(G::NT, 2) void split_kernel(MulArgs a, int n_ct, int n_tt, int n_split, i32x4 * work) {
    constexpr int TN = G::TN, TM = G::TM;
    __shared__ __attribute__((aligned(1024))) char lds[G::ST * G::STAGE];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // A compute die's workgroups (every eighth) take a run of neighbouring tiles, the rows inside, so that the rows' tiles that read the
    // same weights share them in the die's L2
    int tt, ct, part;
    {
        const int x = blockIdx.x & 7, groups = gridDim.x;
        const int i = x * (groups >> 3) + min(x, groups & 7) + (blockIdx.x >> 3);
        const int at = __builtin_amdgcn_readfirstlane(i / n_tt);
        tt = i - at * n_tt;
        part = __builtin_amdgcn_readfirstlane(at / n_ct);
        ct = at - part * n_ct;
    }
    const int c0 = ct * G::BN, t0 = tt * G::BM;
    const int all = (a.k + 127) >> 7;
    const int base = __builtin_amdgcn_readfirstlane(all / n_split), rem = all - base * n_split;
    const int s0 = part * base + min(part, rem), steps = base + (part < rem ? 1 : 0);
    const int tail = (a.k & 127) >> 4, last = all - 1;                   // tail: chunks of k's last step, 0: all
    const uint32_t wn = (uint32_t)((int64_t)(min(G::BN, a.n - c0) - 1) * a.w_nb1 + a.k);
    const uint32_t xn = (uint32_t)((int64_t)(min(G::BM, a.n_rows - t0) - 1) * a.x_nb1 + a.k);
    const char * wb = a.w + (int64_t)c0 * a.w_nb1;
    const char * xb = a.x + (int64_t)t0 * a.x_nb1;
    const uint32_t to0 = lds_addr(lds);
    const int chunk = (lane & 7) ^ (lane >> 4);
    // wave w sends the eights of rows w, w + NW, ... of a step's channels, then of its rows (all of one parity)
    const uint32_t at = 16u * (w & 1 ? chunk ^ 4 : chunk);
    const uint32_t wvo = (uint32_t)((8 * w + (lane >> 3)) * a.w_nb1) + at, xvo = (uint32_t)((8 * w + (lane >> 3)) * a.x_nb1) + at;
    auto send = [&](int s) {
        // (past the last step zeros, so that the loop needs no branch)
        const uint32_t k = 128u * (uint32_t)(s0 + s);
        const i32x4 wr = make_rsrc(wb + k, s < steps ? wn - k : 0u), xr = make_rsrc(xb + k, s < steps ? xn - k : 0u);
        const uint32_t to = to0 + (uint32_t)(s % G::ST) * G::STAGE + 1024u * w;
        // past k a row's bytes are another's: zeros in their place (of one operand: it is enough)
        const bool past = s0 + s == last && tail != 0 && (int)(at >> 4) >= tail;
#pragma unroll
        for (int i = 0; i < G::DW; ++i) tile_dma16(wr, past ? PAST : wvo + (uint32_t)(8 * G::NW * i * a.w_nb1), 0u, to + 1024u * G::NW * i);
#pragma unroll
        for (int i = 0; i < G::DX; ++i) tile_dma16(xr, xvo + (uint32_t)(8 * G::NW * i * a.x_nb1), 0u, to + G::BN * 128 + 1024u * G::NW * i);
    };
    const int r = lane & 31, h = lane >> 5;
    const int kq = w % G::WK, pos = w / G::WK, wn_ = pos % G::WN, wm_ = pos / G::WN;
    for (int s = 0; s < G::ST; ++s) send(s);
    i32x16 acc[TN][TM] = {};
    const char * wl = lds + 128 * (32 * TN * wn_ + r), * xl = lds + G::BN * 128 + 128 * (32 * TM * wm_ + r);
    i32x4 fw[2][G::KK][TN], fx[2][G::KK][TM];
    auto fetch = [&](int to, int s) {
#pragma unroll
        for (int k = 0; k < G::KK; ++k) {
            const int from = (s % G::ST) * G::STAGE + 16 * ((2 * (G::KK * kq + k) + h) ^ ((r >> 1) & 7));
#pragma unroll
            for (int t = 0; t < TN; ++t) fw[to][k][t] = *reinterpret_cast<const i32x4 *>(wl + from + 4096 * t);
#pragma unroll
            for (int t = 0; t < TM; ++t) fx[to][k][t] = *reinterpret_cast<const i32x4 *>(xl + from + 4096 * t);
        }
    };
    auto step = [&](int s, auto odd) {
        constexpr int me = decltype(odd)::value;
        // the next step's bytes are here, and this step's have been read by everyone: its stage is free
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((G::ST - 2) * (G::DW + G::DX)) : "memory");
        fetch(me ^ 1, s + 1);
        send(s + G::ST);
#pragma unroll
        for (int k = 0; k < G::KK; ++k)
#pragma unroll
            for (int t = 0; t < TN; ++t)
#pragma unroll
                for (int u = 0; u < TM; ++u) acc[t][u] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[me][k][t], fx[me][k][u], acc[t][u], 0, 0, 0);
    };
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"((G::ST - 1) * (G::DW + G::DX)) : "memory");
    fetch(0, 0);
    for (int s = 0; s < steps; s += 2) {        // (an odd count: one more, of zeros)
        step(s, std::integral_constant<int, 0>{});
        step(s + 1, std::integral_constant<int, 1>{});
    }
    // quad q of product f of place pos, lane l: channels 32 (TN wn + f / TM) + 8 q + 4 (l / 32) .. + 3 of row 32 (TM wm + f % TM) + l % 32;
    // the place's wave kq adds quads kq, kq + WK, ...
    i32x4 * add = reinterpret_cast<i32x4 *>(lds);
    const int es = a.dst_f16 ? 2 : 4;
    const bool aligned = a.dst_nb1 % (4 * es) == 0 && (reinterpret_cast<uintptr_t>(a.dst) & (4 * es - 1)) == 0;
#pragma unroll
    for (int f0 = 0; f0 < G::F; f0 += G::AT_ONCE) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int f = 0; f < G::AT_ONCE; ++f)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const i32x16 & v = acc[(f0 + f) / TM][(f0 + f) % TM];
                add[(((pos * G::AT_ONCE + f) * 4 + q) * G::WK + kq) * 64 + lane] = i32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            }
        __syncthreads();
#pragma unroll
        for (int f = 0; f < G::AT_ONCE; ++f)
#pragma unroll
            for (int qi = 0; qi < 4 / G::WK; ++qi) {
                const int q = kq + G::WK * qi;
                const i32x4 * from = add + ((pos * G::AT_ONCE + f) * 4 + q) * G::WK * 64 + lane;
                i32x4 s = from[0];
#pragma unroll
                for (int i = 1; i < G::WK; ++i) s += from[64 * i];
                if (n_split > 1) {
                    const int64_t quad = ((int64_t)(part * n_tt + tt) * n_ct + ct) * (G::WN * G::WM * G::F * 4) + (pos * G::F + f0 + f) * 4 + q;
                    work[quad * 64 + lane] = s;
                    continue;
                }
                const int t = t0 + 32 * (TM * wm_ + (f0 + f) % TM) + r, c = c0 + 32 * (TN * wn_ + (f0 + f) / TM) + 8 * q + 4 * h;
                if (t >= a.n_rows || c >= a.n) continue;
                const float xs = a.x_scale[t];
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (float)s[i] * xs * a.w_scale[min(c + i, a.n - 1)];
                put<4>(a.dst + (int64_t)t * a.dst_nb1 + (int64_t)c * es, a.dst_f16, aligned && c + 4 <= a.n, a.n - c, y);
            }
    }
}

// The parts' sums, and the scales: a wavefront a quad of split_kernel's
template <typename G>
__global__ __launch_bounds__(256) void sum_kernel(MulArgs a, int n_ct, int n_tiles, int n_split, const i32x4 * work) {
    constexpr int PER = G::WN * G::WM * G::F * 4;
    const int64_t quads = (int64_t)n_tiles * PER, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= quads) return;
    const int lane = threadIdx.x & 63;
    const int tile = (int)(at / PER), in = (int)(at - (int64_t)tile * PER), pos = in / (4 * G::F), f = in / 4 % G::F, q = in & 3;
    const int tt = tile / n_ct, ct = tile - tt * n_ct;
    const int t = tt * G::BM + 32 * (G::TM * (pos / G::WN) + f % G::TM) + (lane & 31);
    const int c = ct * G::BN + 32 * (G::TN * (pos % G::WN) + f / G::TM) + 8 * q + 4 * (lane >> 5);
    if (t >= a.n_rows || c >= a.n) return;
    const float xs = a.x_scale[t];
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = a.w_scale[min(c + i, a.n - 1)];
    i32x4 s = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < n_split; ++i) s += work[((int64_t)i * quads + at) * 64 + lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (float)s[i] * xs * y[i];
    const int es = a.dst_f16 ? 2 : 4;
    const bool aligned = a.dst_nb1 % (4 * es) == 0 && (reinterpret_cast<uintptr_t>(a.dst) & (4 * es - 1)) == 0;
    put<4>(a.dst + (int64_t)t * a.dst_nb1 + (int64_t)c * es, a.dst_f16, aligned && c + 4 <= a.n, a.n - c, y);
}

template <typename G>
hipError_t split(const MulArgs & a, int n_split, hipStream_t stream) {
    const int n_ct = (a.n + G::BN - 1) / G::BN, n_tt = (a.n_rows + G::BM - 1) / G::BM;
    if ((int64_t)n_ct * n_tt * n_split * G::NT >= (1ll << 32)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((split_kernel<G>), dim3(n_ct * n_tt * n_split), dim3(G::NT), 0, stream, a, n_ct, n_tt, n_split, reinterpret_cast<i32x4 *>(a.work));
    if (n_split > 1)
        hipLaunchKernelGGL((sum_kernel<G>), dim3(n_ct * n_tt * G::WN * G::WM * G::F), dim3(256), 0, stream, a, n_ct, n_ct * n_tt, n_split,
                           reinterpret_cast<const i32x4 *>(a.work));
    return hipGetLastError();
}

template <int NW, int TN>
hipError_t direct(const MulArgs & a, hipStream_t stream) {
    const dim3 grid((a.n + 16 * TN - 1) / (16 * TN), (a.n_rows + 15) / 16);
    hipLaunchKernelGGL((direct_kernel<NW, TN>), grid, dim3(64 * NW), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

size_t mul_workspace_bytes(int n, int k, int n_rows) { return (size_t)choose(n, k, n_rows, true).work; }

hipError_t launch_mul_i8(const MulArgs & a, hipStream_t stream) {
    const Choice c = choose(a.n, a.k, a.n_rows, a.work != nullptr);
    switch (c.kind) {
        case DIRECT8: return direct<8, 1>(a, stream);
        case DIRECT8_2: return direct<8, 2>(a, stream);
        case SPLIT11: return split<Split<1, 1, 4, 1, 1>>(a, c.n_split, stream);
        case SPLIT12: return split<Split<1, 1, 4, 1, 2>>(a, c.n_split, stream);
        case SPLIT22: return split<Split<1, 1, 4, 2, 2>>(a, c.n_split, stream);
        case SPLIT32: return split<Split<1, 1, 4, 3, 2>>(a, c.n_split, stream);
        case SPLIT128: return split<Split<2, 2, 2, 2, 2>>(a, c.n_split, stream);
        case TILE128: return tile<2, 2, 2, 2, 4>(a, stream);
        case TILE192: return tile<2, 4, 3, 2, 5>(a, stream);
        default: return tile<2, 4, 4, 2, 6>(a, stream);
    }
}

}  // namespace rows
}  // namespace mla
