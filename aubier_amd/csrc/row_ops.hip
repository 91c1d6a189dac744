// row_ops.hip -- rows around a batch's attention: the norms with gate and residual and the int8 rows (norm_kernel), the
// rope parts of q (qrope_kernel).
//
// norm_kernel: a workgroup per row, the row in registers, so x and the residual are read once and r and h written once; of many rows
// the next one's values are on their way meanwhile.  Bound by memory where there are many rows (8,000 of 4096, f16 to int8 over an f32
// residual: 80 us, 4.5 TB/s; of 7168, f32: 163 us, 4.6; int8 rows of 5,000 x 40 x 128: 25 us, 5.1, where a large copy makes 5.0), by
// the launch and a row's latency where there are few (64 of 7168 6.2 us, 48 int8 rows of 4096 2.7).
// Everything is taken in 64 bits and rounded where it is stored, or as if it were (int8).  That makes the int8 rows what their
// definition says (a value next to a border between two integers falls on its side) and costs little, as the card's rate for
// 64-bit vector instructions is that of 32-bit ones and the kernel waits for memory.
//
// qrope_kernel: a wavefront per token; a lane turns the same pairs of several heads, so an angle is taken once for them.  5,000 x 40
// heads of f16: 16.3 us (4.7 TB/s); 64 x 32: 3.7 us, of which the launch takes 2.2, the position, the angle in 64 bits and the heads the
// rest: a lane's heads come one behind the other, as a load waits for the store before it (dst may be q).
#include "mla_common.h"
#include "rows.h"

#include <type_traits>

namespace mla {
namespace rows {

namespace {

// v of another lane, 64 bits wide, by DPP
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
struct Sum {
    __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};
// v of a row of 16 lanes combined, at each of them
template <typename Op>
__device__ __forceinline__ double row_all(double v, Op op) {
    v = op(v, dpp64<0xB1>(v));                  // lane ^ 1, ^ 2
    v = op(v, dpp64<0x4E>(v));
    v = op(v, dpp64<0x1B>(dpp64<0x141>(v)));    // ^ 4
    return op(v, dpp64<0x128>(v));              // ^ 8
}
// v of all lanes of the wavefront combined, at every lane
template <typename Op>
__device__ __forceinline__ double wave_all(double v, Op op) {
    v = row_all(v, op);
    auto pair = [&](auto swap) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto a = swap((uint32_t)u), b = swap((uint32_t)(u >> 32));
        return op(__builtin_bit_cast(double, (uint64_t)b[0] << 32 | a[0]), __builtin_bit_cast(double, (uint64_t)b[1] << 32 | a[1]));
    };
    v = pair([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
    return pair([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
}

// the workgroup's sum and largest of a value each per thread (either may be left out); red: NT / 64 pairs of LDS that no other
// reduction uses.  A lane takes one wave's, and a row of 16 lanes puts them together.
template <int NT, bool SUM, bool MAX>
__device__ __forceinline__ void block_all(double & sum, double & top, double (&red)[NT / 64][2]) {
    constexpr int NW = NT / 64;
    if constexpr (SUM) sum = wave_all(sum, Sum{});
    if constexpr (MAX) top = wave_all(top, Max{});
    if constexpr (NW == 1) return;
    if ((threadIdx.x & 63) == 0) {
        if constexpr (SUM) red[threadIdx.x >> 6][0] = sum;
        if constexpr (MAX) red[threadIdx.x >> 6][1] = top;
    }
    __syncthreads();
    const int l = threadIdx.x & 15;
    if constexpr (SUM) sum = row_all(l < NW ? red[l % NW][0] : 0.0, Sum{});
    if constexpr (MAX) top = row_all(l < NW ? red[l % NW][1] : 0.0, Max{});
}

// 1 / sqrt(x): the hardware's estimate and two steps of Newton's method (to 2^-52 or so)
__device__ __forceinline__ double inverse_root(double x) {
    const double r = __builtin_amdgcn_rsq(x);
    double y = r * fma(-0.5 * x * r, r, 1.5);
    y = y * fma(-0.5 * x * y, y, 1.5);
    return x > 0.0 && x < __builtin_inf() ? y : r;
}

// four neighbouring values as they lie in memory: turned into f32 where they are used, so that loads do not wait for one another
template <bool F16>
struct Four {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typename std::conditional<F16, h4, f32x4>::type v;
    __device__ __forceinline__ void load(const char * row, int c) { v = __builtin_nontemporal_load(reinterpret_cast<const decltype(v) *>(row + (F16 ? 2 : 4) * (int64_t)c)); }
    __device__ __forceinline__ f32x4 get() const { return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }
};
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

__device__ __forceinline__ uint32_t pack4(int q0, int q1, int q2, int q3) {
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)q1, (uint32_t)q0, 0x0c0c0400u), hi = __builtin_amdgcn_perm((uint32_t)q3, (uint32_t)q2, 0x0c0c0400u);
    return hi << 16 | lo;
}
// the values, as far as the compiler knows others: so that it does not keep their 64-bit forms from one pass for the next (a row
// would not fit in the registers with them: spills, or half as many rows on a CU at a time)
template <int N>
__device__ __forceinline__ void again(f32x4 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

constexpr int PIECES = 3;

// NT threads, C groups of four values a thread.  ONE: a row a workgroup, and no row behind it to load.  RES: no residual, one of f32 (1) or f16 (2), or PIECES: int8 rows of x as it is, in
// pieces, without any norm.
//
// int8.  The row's largest |r pre| is found in 64 bits, where such products are exact.  127 |r pre| / top is then taken in f32, off
// by less than 4 * 2^-24 * 127 < 2^-15 (from a quotient in 64 bits where the row is near the ends of f32's range), and compared with
// the border exactly where it lies within 2^-14 of one between two integers (a value in 8,000).
template <int NT, int C, bool XH, int RES, bool ONE>
__global__ __launch_bounds__(NT, C > 3 && NT <= 512 ? 2 : 4) void norm_kernel(NormArgs a) {
    // by turns, so that a row's reductions need not wait for the row before to have read its own
    __shared__ double reds[2][2][NT / 64][2];
    const int tid = threadIdx.x;
    constexpr bool PLAIN = RES == PIECES;
    const bool i8 = PLAIN || a.dst_type == OUT_I8;
    // Weights are loaded ahead of the reductions, and the next row's values ahead of this one's end, but not of rows over 12,288 values
    // (of which those up to 16,384 use 44 to 92 of 128 registers without, and wider ones all)
    constexpr bool EARLY = C <= (NT > 512 ? 3 : 6), AHEAD = EARLY && !ONE;
    int turn = 0;
    auto me = [&]() {                                       // (a wide row's places are worked out anew, not held from use to use)
        int t = tid;
        if constexpr (!EARLY) asm volatile("" : "+v"(t));
        return t;
    };
    // A row's values are on their way while the row before is worked on.  (Places past the row's end read its first values;
    // what is made of them is not stored, and adds nothing.)
    Four<XH> raw[C];
    Four<RES == 2> rs[RES == 1 || RES == 2 ? C : 1];
    auto load_x = [&](int row) {
        const char * xr = a.x + (int64_t)row * a.x_nb1;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = 4 * (NT * i + me()), at = c < a.n ? c : 0;
            if constexpr (RES == PIECES) {
                const int piece = a.d_shift >= 0 ? at >> a.d_shift : at / a.d;      // (one piece: a shift that leaves 0)
                raw[i].load(xr + (int64_t)piece * a.x_nbh, at - piece * a.d);
            } else {
                raw[i].load(xr, at);
            }
        }
    };
    auto load_res = [&](int row) {
        if constexpr (RES == 1 || RES == 2) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = 4 * (NT * i + me());
                rs[i].load(a.res + (int64_t)row * a.res_nb1, c < a.n ? c : 0);
            }
        }
    };
    // weights of the thread's channels, or ones
    auto weight = [&](int i, const void * from) {
        const int c = 4 * (NT * i + me());
        if (PLAIN || from == nullptr) return f32x4{1.f, 1.f, 1.f, 1.f};
        return *reinterpret_cast<const f32x4 *>(static_cast<const char *>(from) + 4 * (int64_t)(c < a.n ? c : 0));
    };
    auto weights = [&](f32x4 (&w)[C], const void * from) {
#pragma unroll
        for (int i = 0; i < C; ++i) w[i] = weight(i, from);
    };
    // A wide row's groups are taken two after two, as the 64-bit forms of all of them at once, and the places that me() hides, do not fit
    // in the registers (64 rows of 16,384: 10.9 us; 18.0 where they spill, and of 24,576 20 and 55).  With a residual rows over 16,384 values
    // still spill 6 to 25 registers.
    auto two = [&](int i) {
        if constexpr (!EARLY) {
            if (i & 1) __builtin_amdgcn_sched_barrier(0);
        }
    };
    if constexpr (EARLY) {
        load_x(blockIdx.x);
        load_res(blockIdx.x);
    }
    for (int row = blockIdx.x; row < a.n_rows; row += gridDim.x, turn ^= 1) {
        const int next = AHEAD ? min(row + (int)gridDim.x, a.n_rows - 1) : 0;
        if constexpr (!EARLY) {
            load_x(row);
            load_res(row);
        }
        f32x4 v[C], pw[C], gw[C], hw[C];
#pragma unroll
        for (int i = 0; i < C; ++i) v[i] = 4 * (NT * i + me()) < a.n ? raw[i].get() : f32x4{0.f, 0.f, 0.f, 0.f};
        const char * gate = a.gate != nullptr ? a.gate + (int64_t)row * a.gate_nb1 : nullptr;
        const char * wide = a.gate_wide ? gate : nullptr;
        if constexpr (EARLY) {
            weights(pw, a.post);
            weights(gw, wide);
        }
        if constexpr (C <= 2) weights(hw, a.pre);
        if constexpr (AHEAD) load_x(next);
        double factor = 1.0;
        if (gate != nullptr && !a.gate_wide) factor = (double)*reinterpret_cast<const float *>(gate);
        if constexpr (RES == 1 || RES == 2) factor *= (double)a.scale;
        double sum = 0.0, top = 0.0;
        if (!PLAIN && a.post != nullptr) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) sum = fma((double)v[i][k], (double)v[i][k], sum);
                two(i);
            }
            again(v);
            block_all<NT, true, false>(sum, top, reds[turn][0]);
            factor *= inverse_root(fma(sum, a.per_n, (double)a.eps));
        }
        if constexpr (!EARLY) weights(pw, a.post);
        // r, as it is stored
        if (!PLAIN && (RES == 1 || RES == 2 || a.post != nullptr || gate != nullptr)) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = 4 * (NT * i + me());
                const f32x4 before = RES == 1 || RES == 2 ? rs[i].get() : f32x4{0.f, 0.f, 0.f, 0.f};
                const f32x4 p = pw[i], g = EARLY ? gw[i] : weight(i, wide);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    double y = (double)v[i][k] * factor;
                    const double w = (double)p[k] * (double)g[k];
                    if constexpr (RES == 1 || RES == 2) y = fma(y, w, (double)before[k]);
                    else y *= w;
                    v[i][k] = c < a.n ? (float)y : 0.0f;
                }
                two(i);
            }
        }
        if constexpr (AHEAD) load_res(next);
        if (!PLAIN && a.res_out_type != OUT_NONE) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = 4 * (NT * i + me());
                if (c >= a.n) continue;
                if (a.res_out_type == OUT_F16) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[i][k] = (float)to_half(v[i][k]);
                }
                store4(a.res_out + (int64_t)row * a.res_out_nb1, a.res_out_type, c, v[i]);
            }
        }
        if (!PLAIN && a.dst_type == OUT_NONE) continue;
        char * out = a.dst + (int64_t)row * a.dst_nb1;
        if constexpr (C > 2) weights(hw, a.pre);
        sum = 0.0;
        if (!i8) {
            double inv = 1.0;
            if (a.rms) {
#pragma unroll
                for (int i = 0; i < C; ++i) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) sum = fma((double)v[i][k], (double)v[i][k], sum);
                    two(i);
                }
                again(v);
                block_all<NT, true, false>(sum, top, reds[turn][1]);
                inv = inverse_root(fma(sum, a.per_n, (double)a.eps));
            }
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = 4 * (NT * i + me());
                if (c >= a.n) continue;
                const f32x4 w = hw[i];
                f32x4 h;
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = (float)((double)v[i][k] * inv * (double)w[k]);
                store4(out, a.dst_type, c, h);
                two(i);
            }
            continue;
        }
        if constexpr (PLAIN) {
            // of the bits, which order magnitudes and put infinities and NaN above them all
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) u = max(u, __float_as_uint(v[i][k]) & 0x7fffffffu);
            top = u < 0x7f800000u ? (double)__uint_as_float(u) : __builtin_inf();
            block_all<NT, false, true>(sum, top, reds[turn][1]);
        } else {
            float finite = 0.0f;                        // NaN where a value is none or an infinity
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const f32x4 w = hw[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const double r = (double)v[i][k];
                    sum = fma(r, r, sum);
                    top = fmax(top, fabs(r * (double)w[k]));
                    finite = fmaf(v[i][k], 0.0f, fmaf(w[k], 0.0f, finite));
                }
                two(i);
            }
            if (finite != 0.0f) top = __builtin_inf();
            again(v);
            again(hw);
            block_all<NT, true, true>(sum, top, reds[turn][1]);
        }
        const bool there = top > 0.0 && top < __builtin_inf();
        const double per64 = there ? 127.0 / top : 0.0;
        const bool mid = top >= 0x1p-90 && top < 0x1p120;       // products and quotients are normal f32
        const float per = mid ? (float)per64 : 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = 4 * (NT * i + me());
            if (c >= a.n) continue;
            const f32x4 w = hw[i];
            int q[4];
            float t[4], off = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (mid) t[k] = v[i][k] * w[k] * per;
                else t[k] = there ? (float)((double)v[i][k] * (double)w[k] * per64) : 0.0f;
                const float n = rintf(t[k]);
                q[k] = (int)n;
                off = fmaxf(off, fabsf(t[k] - n));
            }
            if (off > 0.5f - 0x1p-14f) {
                // 127 |r pre| against (the integer below + 1 / 2) top, which take 55 and 56 bits.  Next to the border the latter's distance
                // from 128 |r pre|, a multiple of 2^-48 of top's leading bit and less than twice top, is a double: compared with |r pre|.
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float below = floorf(fabsf(t[k]));
                    const double h = fabs((double)v[i][k] * (double)w[k]);
                    const int n = (int)below + (fma(-((double)below + 0.5), top, 128.0 * h) >= h ? 1 : 0);
                    q[k] = t[k] < 0.0f ? -n : n;
                }
            }
            *reinterpret_cast<uint32_t *>(out + c) = pack4(q[0], q[1], q[2], q[3]);
            two(i);
        }
        if (tid == 0) {
            const double inv = !PLAIN && a.rms ? inverse_root(fma(sum, a.per_n, (double)a.eps)) : 1.0;
            a.dst_scale[row] = there ? (float)(top * inv / 127.0) : top == 0.0 ? 0.0f : __builtin_nanf("");
        }
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
        Four<QH> q;
        q.load(a.q + (int64_t)row * a.q_nb2 + (int64_t)h * a.q_nb1, 4 * g);
        f32x4 v = q.get();
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const float x0 = v[k], x1 = v[k + 1];
            v[k] = x0 * co[k >> 1] - x1 * si[k >> 1];
            v[k + 1] = x0 * si[k >> 1] + x1 * co[k >> 1];
        }
        store4(a.dst + (int64_t)row * a.dst_nb2 + (int64_t)h * a.dst_nb1, a.dst_f16 ? OUT_F16 : OUT_F32, 4 * g, v);
    }
}

constexpr int FEW = 256;                // rows, one a CU

template <int NT, int C, bool ONE>
hipError_t norm(const NormArgs & a, hipStream_t stream) {
    auto go = [&](auto kernel, int waves) {
        const int at_once = ONE ? FEW : 256 * (64 * waves / NT);        // workgroups that the card holds
        hipLaunchKernelGGL(kernel, dim3(a.n_rows < at_once ? a.n_rows : at_once), dim3(NT), 0, stream, a);
        return hipGetLastError();
    };
    const int res = a.d != 0 ? PIECES : a.res == nullptr ? 0 : a.res_f16 ? 2 : 1;
    switch (res + (a.x_f16 ? 4 : 0)) {
        case 0: return go(norm_kernel<NT, C, false, 0, ONE>, 16);
        case 1: return go(norm_kernel<NT, C, false, 1, ONE>, 16);
        case 2: return go(norm_kernel<NT, C, false, 2, ONE>, 16);
        case 3: return go(norm_kernel<NT, C, false, PIECES, ONE>, C <= 3 ? 32 : 16);
        case 4: return go(norm_kernel<NT, C, true, 0, ONE>, 16);
        case 5: return go(norm_kernel<NT, C, true, 1, ONE>, 16);
        case 6: return go(norm_kernel<NT, C, true, 2, ONE>, 16);
        default: return go(norm_kernel<NT, C, true, PIECES, ONE>, C <= 3 ? 32 : 16);
    }
}

}  // namespace

hipError_t launch_norm(const NormArgs & a, hipStream_t stream) {
    if (a.n > MAX_N) return hipErrorInvalidValue;
    const int fours = (a.n + 255) / 256;                // groups of a thread, of a wavefront
    if (a.n_rows <= FEW) {
        // A CU has one of them: threads that share its work, but not so many that starting and joining them costs more (one of 4,096: 4.0
        // us by 512, 4.4 by 1,024, 4.8 by 256; 64 of 7168: 6.2 by 1,024 and by 512; 64 of 12,288: 9.0 by 512, 9.6 by 1,024)
        if (fours <= 4) return norm<256, 1, true>(a, stream);
        if (fours <= 8) return norm<512, 1, true>(a, stream);
        if (fours <= 16) return norm<512, 2, true>(a, stream);
        if (fours <= 24) return norm<512, 3, true>(a, stream);
        if (fours <= 32) return norm<1024, 2, true>(a, stream);
        if (fours <= 48) return norm<512, 6, true>(a, stream);
        // (wider ones load no row ahead in any case: the kernels of many rows below)
    }
    // As few threads a row as keep its values in registers, so that a CU has several rows at different places of their way (8,000 rows
    // of 1,536: 25 us by 256 threads, 35 by 512; 6,000 of 2,560: 53 by 256, 63 by 512)
    if (fours == 1) return norm<64, 1, false>(a, stream);
    if (fours == 2) return norm<64, 2, false>(a, stream);
    if (fours <= 4) return norm<256, 1, false>(a, stream);
    if (fours <= 8) return norm<256, 2, false>(a, stream);
    if (fours <= 12) return norm<256, 3, false>(a, stream);
    if (fours <= 16) return norm<512, 2, false>(a, stream);
    if (fours <= 24) return norm<512, 3, false>(a, stream);
    if (fours <= 32) return norm<1024, 2, false>(a, stream);
    if (fours <= 48) return norm<1024, 3, false>(a, stream);
    if (fours <= 64) return norm<1024, 4, false>(a, stream);
    return norm<1024, 8, false>(a, stream);
}

hipError_t launch_qrope(const QropeArgs & a, hipStream_t stream) {
    const dim3 grid((a.n_rows + 3) / 4), block(256);
    if (a.q_f16) hipLaunchKernelGGL(qrope_kernel<true>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(qrope_kernel<false>, grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace rows
}  // namespace mla
