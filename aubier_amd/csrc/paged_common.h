// paged_common.h -- device helpers of the paged-batch kernels (paged.h describes the batch).
#pragma once

#include "mla_common.h"
#include "paged.h"

namespace mla {
namespace paged {

// v of lane l from lane l - k of its row of 16 (k = 1, 2, 4, 8), or from the last lane of the row(s) before (15: odd rows
// from the row before, 31: the upper half from the lower); `none` where there is no such lane
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_from(int none, int v) { return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ int step_sum(int v) { return v + dpp_from<CTRL, ROWS>(0, v); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double step_sum(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp_from<CTRL, ROWS>(0, (int)(uint32_t)u), hi = (uint32_t)dpp_from<CTRL, ROWS>(0, (int)(uint32_t)(u >> 32));
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// the sum over lanes 0 .. l of the wavefront, at lane l
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v = step_sum<0x111, 0xf>(v);        // row_shr:1, 2, 4, 8
    v = step_sum<0x112, 0xf>(v);
    v = step_sum<0x114, 0xf>(v);
    v = step_sum<0x118, 0xf>(v);
    v = step_sum<0x142, 0xa>(v);        // row_bcast:15 into rows 1 and 3
    return step_sum<0x143, 0xc>(v);     // row_bcast:31 into rows 2 and 3
}
// the least over the wavefront, at its last lane
__device__ __forceinline__ int wave_min(int v) {
    constexpr int MOST = 0x7fffffff;
    v = min(v, dpp_from<0x111, 0xf>(MOST, v));
    v = min(v, dpp_from<0x112, 0xf>(MOST, v));
    v = min(v, dpp_from<0x114, 0xf>(MOST, v));
    v = min(v, dpp_from<0x118, 0xf>(MOST, v));
    v = min(v, dpp_from<0x142, 0xa>(MOST, v));
    return min(v, dpp_from<0x143, 0xc>(MOST, v));
}

// out[i] = the sum of f(0 .. i - 1) for i < n, in LDS, by the whole workgroup of NT threads; returns the total.
// A thread sums a run of consecutive values, so f is evaluated twice per value.  wsum: NT / 64 words of LDS.
// Ends with a barrier.
template <int NT, typename T, typename F>
__device__ __forceinline__ T block_scan(int n, F && f, T * out, T * wsum) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int per = (n + NT - 1) / NT;
    const int i0 = tid * per, i1 = min(i0 + per, n);
    T own = 0;
    for (int i = i0; i < i1; ++i) own += f(i);
    const T incl = wave_scan(own);
    if (lane == 63) wsum[w] = incl;
    __syncthreads();
    T base = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        base += i < w ? wsum[i] : 0;
        total += wsum[i];
    }
    T run = base + incl - own;
    for (int i = i0; i < i1; ++i) {
        const T v = f(i);
        out[i] = run;
        run += v;
    }
    __syncthreads();
    return total;
}

// The last i in [0, n) with start[i] <= x (start ascending, start[0] <= x)
template <typename T>
__device__ __forceinline__ int last_at_most(const T * start, int n, T x) {
    int lo = 0, len = n;
    while (len > 1) {
        const int half = len >> 1;
        if (start[lo + half] <= x) {
            lo += half;
            len -= half;
        } else {
            len = half;
        }
    }
    return lo;
}

__device__ __forceinline__ int clamp_past(int32_t p) { return min(max(p, 0), MAX_PAST); }

}  // namespace paged
}  // namespace mla
