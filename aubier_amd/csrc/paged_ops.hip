// paged_ops.hip -- the bookkeeping of a paged batch and its KV rows.
//
// pages_kernel: block tables and slot maps from request lengths.  With have_b = ceil(past_b / page) and
// take_b = ceil((past_b + new_b) / page) - have_b, request b starts take_b pages, which come off the free list
// behind those of the requests before it; row r, the (r - start_b)-th token of request b at position p, lies in
// page p / page of the request: one it held (read from its table) or one it starts (off the free list, entered
// in its table by the row at the page's first cell).  The rows are independent once the two prefix sums over
// the requests are known, and these are cheap: every workgroup takes them for itself, so there is one launch
// and nothing crosses workgroups.  No row reads a table entry that another writes.  Latency: 64 requests 3.3 us, 500 with
// 7,800 rows 4.2, of which the launch is 2.2.
//
// kvrows_kernel: a wave per row; RMS norm over the latent part, YaRN rope over the rest, the row stored at its
// slot.  The angle of pair i at position p is p times a frequency that the host takes in 64 bits; the product is
// reduced to a part of a turn in 64 bits as well, because at p = 100,000 a product in 32 bits is off by some
// hundredths of a radian.  A pass over x and its two copies: 8,000 rows of 576 (46 MB) in 10.2 us, launch included,
// the rate of a large copy; x and Kcur go past the caches (10.6 us with the default policy).
#include "paged_common.h"

namespace mla {
namespace paged {

namespace {

constexpr int NTHR = 256;
constexpr int ROWS_PER_WG = 256;

__global__ __launch_bounds__(NTHR) void pages_kernel(PagesArgs a) {
    __shared__ int start[MAX_SEQS];      // first row of a request
    __shared__ int first[MAX_SEQS];      // its first page on the free list
    __shared__ int wsum[NTHR / 64];
    const int tid = threadIdx.x, sh = a.page_shift;
    const int all = block_scan<NTHR>(a.n_seq, [&](int b) { return min(max(a.n_new[b], 0), a.n_rows); }, start, wsum);
    const int rows = min(all, a.n_rows);
    auto held = [&](int cells) { return min((cells + (1 << sh) - 1) >> sh, a.max_pages); };
    const int taken = block_scan<NTHR>(a.n_seq, [&](int b) {
        const int p = clamp_past(a.past[b]);
        const int s0 = min(start[b], a.n_rows), s1 = b + 1 < a.n_seq ? min(start[b + 1], a.n_rows) : rows;
        return held(p + s1 - s0) - held(p);
    }, first, wsum);
    if (blockIdx.x == 0 && tid == 0) {
        a.used[0] = min(taken, a.n_free);
        a.used[1] = rows;
    }
    const int r = blockIdx.x * ROWS_PER_WG + tid;
    if (r >= a.n_rows) return;
    int64_t slot = -1;
    int p = 0;
    if (r < rows) {
        const int b = last_at_most(start, a.n_seq, r);
        const int past = clamp_past(a.past[b]);
        p = past + r - start[b];
        const int j = p >> sh, have = held(past);
        int32_t * entry = reinterpret_cast<int32_t *>(reinterpret_cast<char *>(a.table) + (size_t)b * a.t_nb1) + j;
        int page = -1;
        if (j < have) {
            page = *entry;
        } else if (j < a.max_pages) {
            const int nth = first[b] + j - have;
            if (nth < a.n_free) page = a.free_ids[nth];
            if ((p & ((1 << sh) - 1)) == 0) *entry = page;
        }
        if (page >= 0) slot = ((int64_t)page << sh) + (p & ((1 << sh) - 1));
    }
    a.slot[r] = slot;
    a.pos[r] = p;
}

// NC: 16-byte groups of four values per lane (n_out <= 256 NC).  A group lies in the latent or in the rope part
// whole, as both are multiples of 32 wide; eight neighbouring lanes hold one block_q8_0 block.
template <int NC, bool XH>
__global__ __launch_bounds__(NTHR) void kvrows_kernel(KvRowsArgs a) {
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.x * (NTHR / 64) + (threadIdx.x >> 6);
    if (r >= a.n_rows) return;
    const int n_out = a.d_lat + a.n_rope;
    const char * xr = static_cast<const char *>(a.x) + (size_t)r * a.x_nb1;
    f32x4 v[NC];
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = 4 * (64 * i + lane);
        v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (c < n_out) {
            if constexpr (XH) {
                const half4 h = *reinterpret_cast<const half4 *>(xr + 2 * c);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = (float)h[k];
            } else {
                v[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(xr + 4 * c));
            }
        }
        if (c < a.d_lat) {
#pragma unroll
            for (int k = 0; k < 4; ++k) sq += v[i][k] * v[i][k];
        }
    }
    const int64_t slot = a.slot[r];
    const double pos = (double)a.pos[r];
    const float scale = 1.0f / sqrtf(wave_sum(sq) / (float)a.d_lat + a.eps);
    const bool store = slot >= 0 && slot < a.n_cells;
    char * row = a.kc + (store ? slot : 0) * a.kc_nb1;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = 4 * (64 * i + lane);
        if (c < a.d_lat) {
            const f32x4 w = *reinterpret_cast<const f32x4 *>(a.nw + c);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = scale * v[i][k] * w[k];
        } else if (c < n_out) {
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const double t = pos * a.turns[(c - a.d_lat + k) >> 1];
                float si, co;
                sincospif(2.0f * (float)(t - rint(t)), &si, &co);
                si *= a.mscale;
                co *= a.mscale;
                const float x0 = v[i][k], x1 = v[i][k + 1];
                v[i][k] = x0 * co - x1 * si;
                v[i][k + 1] = x0 * si + x1 * co;
            }
        }
        if (c < n_out && a.dst != nullptr) __builtin_nontemporal_store(v[i], reinterpret_cast<f32x4 *>(a.dst + (size_t)r * a.dst_nb1 + 4 * c));
        if (!a.kc_q8) {
            if (c < n_out && store) {
                half4 h;
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = to_half(v[i][k]);
                *reinterpret_cast<half4 *>(row + 2 * c) = h;
            }
        } else {
            // ggml's f32 -> q8_0 rounding: d = max / 127, q = roundf(x * (1 / d)), d stored as f16.  The maximum is taken of the
            // bit patterns, which order magnitudes and put a NaN above them all: its block's d is NaN
            auto size = [](float x) { return __float_as_uint(fabsf(x)); };
            uint32_t top = max(max(size(v[i][0]), size(v[i][1])), max(size(v[i][2]), size(v[i][3])));
            top = max(top, __float_as_uint(dpp_xor<1>(__uint_as_float(top))));
            top = max(top, __float_as_uint(dpp_xor<2>(__uint_as_float(top))));
            top = max(top, __float_as_uint(dpp_xor<4>(__uint_as_float(top))));
            const float m = __uint_as_float(top);
            const float d = m / 127.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
            uint32_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = (uint32_t)(int)roundf(v[i][k] * id) & 0xffu;
            if (c < n_out && store) {
                char * blk = row + (c >> 5) * 34;
                if ((lane & 7) == 0) *reinterpret_cast<half_t *>(blk) = to_half(d);
                uint16_t * qs = reinterpret_cast<uint16_t *>(blk + 2 + (c & 31));
                qs[0] = (uint16_t)(q[0] | q[1] << 8);
                qs[1] = (uint16_t)(q[2] | q[3] << 8);
            }
        }
    }
}

}  // namespace

hipError_t launch_pages(const PagesArgs & a, hipStream_t stream) {
    hipLaunchKernelGGL(pages_kernel, dim3((a.n_rows + ROWS_PER_WG - 1) / ROWS_PER_WG), dim3(NTHR), 0, stream, a);
    return hipGetLastError();
}

template <bool XH>
static hipError_t kvrows(const KvRowsArgs & a, hipStream_t stream) {
    const dim3 grid((a.n_rows + NTHR / 64 - 1) / (NTHR / 64));
    const int n_out = a.d_lat + a.n_rope;
    if (n_out <= 512) hipLaunchKernelGGL((kvrows_kernel<2, XH>), grid, dim3(NTHR), 0, stream, a);
    else if (n_out <= 768) hipLaunchKernelGGL((kvrows_kernel<3, XH>), grid, dim3(NTHR), 0, stream, a);
    else if (n_out <= 1024) hipLaunchKernelGGL((kvrows_kernel<4, XH>), grid, dim3(NTHR), 0, stream, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_kvrows(const KvRowsArgs & a, hipStream_t stream) {
    return a.x_f16 ? kvrows<true>(a, stream) : kvrows<false>(a, stream);
}

}  // namespace paged
}  // namespace mla
