// row_ops.hip -- rows around a batch's attention: the norms with gate and residual and the int8 rows (norm_kernel), the
// rope parts of q (qrope_kernel).
//
// norm_kernel: a workgroup per row, the row in registers, so x and the residual are read once and r and h written once.
// Everything is taken in 64 bits and rounded where it is stored.  That makes the int8 rows what their definition says
// (a value next to a border between two integers falls on its side) and costs little, as the card's rate for 64-bit
// vector instructions is that of 32-bit ones and the kernel waits for memory.
//
// qrope_kernel: a wavefront per token; a lane turns the same pairs of several heads, so an angle is taken once for them.
#include "mla_common.h"
#include "rows.h"

namespace mla {
namespace rows {

namespace {

// v of another lane, 64 bits wide, by DPP
template <int CTRL>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)v, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
struct Sum {
    __device__ __forceinline__ uint64_t operator()(uint64_t a, uint64_t b) const {
        return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b));
    }
};
struct Max {
    __device__ __forceinline__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
// v of all lanes of the wavefront combined, at every lane
template <typename Op>
__device__ __forceinline__ uint64_t wave_all(uint64_t v, Op op) {
    v = op(v, dpp64<0xB1>(v));                  // lane ^ 1, ^ 2
    v = op(v, dpp64<0x4E>(v));
    v = op(v, dpp64<0x1B>(dpp64<0x141>(v)));    // ^ 4
    v = op(v, dpp64<0x128>(v));                 // ^ 8
    auto pair = [&](bool rows16) {
        const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
        if (rows16) {
            const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
            const auto b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            return op((uint64_t)b[0] << 32 | a[0], (uint64_t)b[1] << 32 | a[1]);
        }
        const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
        return op((uint64_t)b[0] << 32 | a[0], (uint64_t)b[1] << 32 | a[1]);
    };
    v = pair(true);
    return pair(false);
}

// the workgroup's sum and largest of a value each per thread; red: NT / 64 pairs of LDS that no other reduction uses
template <int NT>
__device__ __forceinline__ void block_all(double & sum, uint64_t & top, uint64_t * red) {
    constexpr int NW = NT / 64;
    uint64_t s = wave_all(__builtin_bit_cast(uint64_t, sum), Sum{}), t = wave_all(top, Max{});
    if constexpr (NW > 1) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            red[2 * w] = s;
            red[2 * w + 1] = t;
        }
        __syncthreads();
        s = red[0];
        t = red[1];
#pragma unroll
        for (int i = 1; i < NW; ++i) {
            s = Sum{}(s, red[2 * i]);
            t = Max{}(t, red[2 * i + 1]);
        }
    }
    sum = __builtin_bit_cast(double, s);
    top = t;
}

__device__ __forceinline__ uint64_t magnitude(double v) { return __builtin_bit_cast(uint64_t, v) & 0x7fffffffffffffffull; }
constexpr uint64_t INF64 = 0x7ff0000000000000ull;

template <bool F16>
__device__ __forceinline__ f32x4 load4(const char * row, int c) {
    if constexpr (F16) {
        const half4 h = *reinterpret_cast<const half4 *>(row + 2 * c);
        return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
    } else {
        return *reinterpret_cast<const f32x4 *>(row + 4 * c);
    }
}
__device__ __forceinline__ void store4(char * row, int type, int c, f32x4 v) {
    if (type == OUT_F32) {
        *reinterpret_cast<f32x4 *>(row + 4 * c) = v;
    } else {
        half4 h;
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = to_half(v[k]);
        *reinterpret_cast<half4 *>(row + 2 * c) = h;
    }
}

// The integer of v = |value| in a row whose largest magnitude is top: 127 v / top, half away from zero.  `per` is
// 127 / top in 64 bits, so the quotient is off by 2^-51 of itself at most; within 2^-40 of a border it is taken by division.
__device__ __forceinline__ int steps_of(double v, double top, double per) {
    double u = v * per + 0.5, k = floor(u);
    const double past = u - k;
    if (past < 0x1p-40 || past > 1.0 - 0x1p-40) k = floor(v * 127.0 / top + 0.5);
    return (int)k;
}

// NT threads, C groups of four values a thread.  RES: 0 none, 1 f32, 2 f16.
template <int NT, int C, bool XH, int RES>
__global__ __launch_bounds__(NT) void norm_kernel(NormArgs a) {
    // by turns, so that a row's reductions need not wait for the row before to have read its own
    __shared__ uint64_t reds[2][2][2 * (NT / 64)];
    const int tid = threadIdx.x;
    int turn = 0;
    for (int row = blockIdx.x; row < a.n_rows; row += gridDim.x, turn ^= 1) {
        auto & red = reds[turn];
        const char * xr = a.x + (int64_t)row * a.x_nb1;
        f32x4 v[C], rs[RES ? C : 1];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = 4 * (NT * i + tid);
            v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (c < a.n) {
                const int piece = c / a.d;
                v[i] = load4<XH>(xr + (int64_t)piece * a.x_nbh, c - piece * a.d);
                if constexpr (RES != 0) rs[i] = load4<RES == 2>(a.res + (int64_t)row * a.res_nb1, c);
            }
        }
        double factor = 1.0;
        if (a.post != nullptr) {
            double s = 0.0;
            uint64_t none = 0;
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) s += (double)v[i][k] * (double)v[i][k];
            block_all<NT>(s, none, red[0]);
            factor = 1.0 / sqrt(s / (double)a.n + (double)a.eps);
        }
        const char * gate = a.gate != nullptr ? a.gate + (int64_t)row * a.gate_nb1 : nullptr;
        if (gate != nullptr && !a.gate_wide) factor *= (double)*reinterpret_cast<const float *>(gate);
        if constexpr (RES != 0) factor *= (double)a.scale;
        // r, as it is stored
        double sum = 0.0;
        uint64_t top = 0;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = 4 * (NT * i + tid);
            if (c >= a.n) continue;
            f32x4 pw = {1.f, 1.f, 1.f, 1.f}, gw = pw, hw = pw;
            if (a.post != nullptr) pw = *reinterpret_cast<const f32x4 *>(a.post + c);
            if (gate != nullptr && a.gate_wide) gw = *reinterpret_cast<const f32x4 *>(gate + 4 * (int64_t)c);
            if (a.pre != nullptr) hw = *reinterpret_cast<const f32x4 *>(a.pre + c);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                double y = (double)v[i][k] * factor * (double)pw[k] * (double)gw[k];
                if constexpr (RES != 0) y += (double)rs[i][k];
                v[i][k] = (float)y;
                if (a.res_out_type == OUT_F16) v[i][k] = (float)to_half(v[i][k]);
                sum += (double)v[i][k] * (double)v[i][k];
                const uint64_t m = magnitude((double)v[i][k] * (double)hw[k]);
                top = m > top ? m : top;
            }
            if (a.res_out_type != OUT_NONE) store4(a.res_out + (int64_t)row * a.res_out_nb1, a.res_out_type, c, v[i]);
        }
        if (a.dst_type == OUT_NONE) continue;
        double inv = 1.0;
        if (a.rms || a.dst_type == OUT_I8) {
            block_all<NT>(sum, top, red[1]);
            if (a.rms) inv = 1.0 / sqrt(sum / (double)a.n + (double)a.eps);
        }
        const double most = __builtin_bit_cast(double, top);
        const bool finite = top < INF64;
        const double per = finite && top != 0 ? 127.0 / most : 0.0;
        char * out = a.dst + (int64_t)row * a.dst_nb1;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = 4 * (NT * i + tid);
            if (c >= a.n) continue;
            f32x4 hw = {1.f, 1.f, 1.f, 1.f};
            if (a.pre != nullptr) hw = *reinterpret_cast<const f32x4 *>(a.pre + c);
            if (a.dst_type == OUT_I8) {
                uint32_t q = 0;
                if (per != 0.0) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const double h = (double)v[i][k] * (double)hw[k];
                        const int steps = steps_of(fabs(h), most, per);
                        q |= (uint32_t)((h < 0.0 ? -steps : steps) & 0xff) << (8 * k);
                    }
                }
                *reinterpret_cast<uint32_t *>(out + c) = q;
            } else {
                f32x4 h;
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = (float)((double)v[i][k] * inv * (double)hw[k]);
                store4(out, a.dst_type, c, h);
            }
        }
        if (a.dst_type == OUT_I8 && tid == 0) a.dst_scale[row] = finite ? (float)(most * inv / 127.0) : __builtin_nanf("");
    }
}

// H heads' pieces of n_dims values: lane l has the 4 values (two pairs) at 4 (l % G) of heads l / G, l / G + 64 / G, ...
// with G = n_dims / 4 groups (8 to 64)
template <bool QH>
__global__ __launch_bounds__(256) void qrope_kernel(QropeArgs a) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n_rows) return;
    const int groups = a.n_dims >> 2, per = 64 / groups;
    const int g = lane % groups, h0 = lane / groups;
    if (h0 >= per) return;
    const double pos = (double)a.pos[row];
    float co[2], si[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const double t = pos * a.turns[2 * g + k];
        sincospif(2.0f * (float)(t - rint(t)), &si[k], &co[k]);
        si[k] *= a.mscale;
        co[k] *= a.mscale;
    }
    for (int h = h0; h < a.n_head; h += per) {
        f32x4 v = load4<QH>(a.q + (int64_t)row * a.q_nb2 + (int64_t)h * a.q_nb1, 4 * g);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const float x0 = v[k], x1 = v[k + 1];
            v[k] = x0 * co[k >> 1] - x1 * si[k >> 1];
            v[k + 1] = x0 * si[k >> 1] + x1 * co[k >> 1];
        }
        store4(a.dst + (int64_t)row * a.dst_nb2 + (int64_t)h * a.dst_nb1, a.dst_f16 ? OUT_F16 : OUT_F32, 4 * g, v);
    }
}

constexpr int MAX_GRID = 1 << 20;       // the grid's threads stay below 2^32

template <int NT, int C>
hipError_t norm(const NormArgs & a, hipStream_t stream) {
    const dim3 grid(a.n_rows < MAX_GRID ? a.n_rows : MAX_GRID), block(NT);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, block, 0, stream, a);
        return hipGetLastError();
    };
    const int res = a.res == nullptr ? 0 : a.res_f16 ? 2 : 1;
    if (a.x_f16) return res == 0 ? go(norm_kernel<NT, C, true, 0>) : res == 1 ? go(norm_kernel<NT, C, true, 1>) : go(norm_kernel<NT, C, true, 2>);
    return res == 0 ? go(norm_kernel<NT, C, false, 0>) : res == 1 ? go(norm_kernel<NT, C, false, 1>) : go(norm_kernel<NT, C, false, 2>);
}

}  // namespace

hipError_t launch_norm(const NormArgs & a, hipStream_t stream) {
    if (a.n <= 1024) return norm<256, 1>(a, stream);
    if (a.n <= 4096) return norm<256, 4>(a, stream);
    if (a.n <= 8192) return norm<256, 8>(a, stream);
    if (a.n <= MAX_N) return norm<1024, 8>(a, stream);
    return hipErrorInvalidValue;
}

hipError_t launch_qrope(const QropeArgs & a, hipStream_t stream) {
    const dim3 grid((a.n_rows + 3) / 4), block(256);
    if (a.q_f16) hipLaunchKernelGGL(qrope_kernel<true>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(qrope_kernel<false>, grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace rows
}  // namespace mla
