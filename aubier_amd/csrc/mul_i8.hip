// mul_i8.hip -- the product of int8 rows and int8 weights with a scale for each row and each channel
// (mla_m4_mul_i8): y[t][c] = xs[t] ws[c] sum_k w[c][k] x[t][k], the sum exact in 32 bits.
//
// direct_kernel: a workgroup of NW waves takes 16 channels and 16 T rows; wave w takes the 64-byte steps w, w + NW, ... of k,
// its operands straight from memory (lane l: row l % 16, 16 bytes at 16 (l / 16), as v_mfma_i32_16x16x64_i8 takes both),
// and the waves' integers are added in LDS.  Integer sums have no order, so the result is the same however k is cut.
#include "mla_common.h"
#include "rows.h"

namespace mla {
namespace rows {

namespace {

template <int NW, int T>
__global__ __launch_bounds__(64 * NW) void direct_kernel(MulArgs a) {
    __shared__ i32x4 part[NW][T][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * T;
    // rows past the last one read it again; what they give is not stored
    const char * wr = a.w + (int64_t)min(c0 + r, a.n - 1) * a.w_nb1;
    const char * xr[T];
#pragma unroll
    for (int j = 0; j < T; ++j) xr[j] = a.x + (int64_t)min(t0 + 16 * j + r, a.n_rows - 1) * a.x_nb1;
    i32x4 acc[T] = {};
    for (int k = 64 * w; k < a.k; k += 64 * NW) {
        const int at = k + 16 * g;
        const bool in = at < a.k;                       // k is a multiple of 16: a lane's bytes are there or not
        i32x4 wv = *reinterpret_cast<const i32x4 *>(wr + (in ? at : 0));
        if (!in) wv = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < T; ++j) {
            const i32x4 xv = *reinterpret_cast<const i32x4 *>(xr[j] + (in ? at : 0));
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xv, acc[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < T; ++j) part[w][j][lane] = acc[j];
    __syncthreads();
    // lane l's four: channels c0 + 4 (l / 16) .. + 3 of row t0 + 16 j + l % 16
    for (int j = w; j < T; j += NW) {
        i32x4 s = part[0][j][lane];
#pragma unroll
        for (int i = 1; i < NW; ++i) s += part[i][j][lane];
        const int t = t0 + 16 * j + r;
        if (t >= a.n_rows) continue;
        const float xs = a.x_scale[t];
        char * row = a.dst + (int64_t)t * a.dst_nb1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + 4 * g + i;
            if (c >= a.n) continue;
            const float y = (float)s[i] * xs * a.w_scale[c];
            if (a.dst_f16) *reinterpret_cast<half_t *>(row + 2 * (int64_t)c) = to_half(y);
            else *reinterpret_cast<float *>(row + 4 * (int64_t)c) = y;
        }
    }
}

}  // namespace

hipError_t launch_mul_i8(const MulArgs & a, hipStream_t stream) {
    constexpr int T = 4;
    const dim3 grid((a.n + 15) / 16, (a.n_rows + 16 * T - 1) / (16 * T));
    hipLaunchKernelGGL((direct_kernel<4, T>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace rows
}  // namespace mla
