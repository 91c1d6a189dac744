// paged_common.h -- device helpers of the paged-batch kernels (paged.h describes the batch).
#pragma once

#include "mla_common.h"
#include "paged.h"

namespace mla {
namespace paged {

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
    T incl = own;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const T up = __shfl_up(incl, k);
        if (lane >= k) incl += up;
    }
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
