// kqkv_paged.hip -- KQKV over the pages of a batch (paged.h): token i of request b, whose q has H heads, sees the
// first past_b + i + 1 cells of the request's table:
//   dst[h][t][:] = softmax_j(kq_scale q[t][h] . K[cell(j)]) . V[cell(j)],  V = the first D_v columns of a row.
// One workgroup per (head, token), one pass over the keys in tiles of 64 with the running maximum and sum of the
// softmax in f32.
#include "paged_common.h"

namespace mla {
namespace paged {

namespace {

constexpr int NTHR = 256;
constexpr int TK = 64;

template <bool Q8>
__device__ __forceinline__ float cell_value(const char * row, int d) {
    if constexpr (!Q8) return (float)reinterpret_cast<const half_t *>(row)[d];
    const char * blk = row + (d >> 5) * 34;
    return (float)*reinterpret_cast<const half_t *>(blk) * (float)reinterpret_cast<const int8_t *>(blk + 2)[d & 31];
}

template <int DK, int DV, bool Q8>
__global__ __launch_bounds__(NTHR) void kqkv_paged_kernel(AttnArgs a) {
    __shared__ int start[MAX_SEQS];
    __shared__ int wsum[NTHR / 64];
    __shared__ float qs[DK];
    __shared__ float p[TK];
    __shared__ const char * rows[TK];
    const int tid = threadIdx.x, h = blockIdx.x, t = blockIdx.y;
    const int all = block_scan<NTHR>(a.n_seq, [&](int b) { return min(max(a.n_new[b], 0), a.nt); }, start, wsum);
    if (t >= all) return;
    const int b = last_at_most(start, a.n_seq, t);
    const int64_t most = (int64_t)a.max_pages << a.page_shift;
    const int n = (int)min((int64_t)clamp_past(a.past[b]) + (t - start[b]) + 1, most);
    const int32_t * table = reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(a.table) + (size_t)b * a.t_nb1);
    const char * qr = a.q + (size_t)t * a.q_nb2 + (size_t)h * a.q_nb1;
    for (int d = tid; d < DK; d += NTHR)
        qs[d] = a.q_f16 ? (float)reinterpret_cast<const half_t *>(qr)[d] : reinterpret_cast<const float *>(qr)[d];
    float m = -INFINITY, l = 0.0f, o[DV / NTHR] = {};
    for (int k0 = 0; k0 < n; k0 += TK) {
        __syncthreads();
        if (tid < TK) {
            const int k = k0 + tid;
            const char * row = nullptr;
            if (k < n) {
                const int page = table[k >> a.page_shift];
                if (page >= 0 && page < a.n_pages) row = a.kc + (((int64_t)page << a.page_shift) + (k & ((1 << a.page_shift) - 1))) * a.kc_nb1;
            }
            rows[tid] = row;
        }
        __syncthreads();
        const char * row = rows[tid >> 2];
        float s = 0.0f;
        if (row != nullptr)
            for (int d = tid & 3; d < DK; d += 4) s += qs[d] * cell_value<Q8>(row, d);
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        if ((tid & 3) == 0) p[tid >> 2] = row != nullptr ? s * a.scale_log2 : -INFINITY;
        __syncthreads();
        float mt = m;
        for (int k = 0; k < TK; ++k) mt = fmaxf(mt, p[k]);
        const float f = exp2_unless(m == -INFINITY, m - mt);
        l *= f;
        for (int i = 0; i < DV / NTHR; ++i) o[i] *= f;
        for (int k = 0; k < TK; ++k) {
            if (rows[k] == nullptr) continue;
            const float e = exp2_fast(p[k] - mt);
            l += e;
            for (int i = 0; i < DV / NTHR; ++i) o[i] += e * cell_value<Q8>(rows[k], tid + NTHR * i);
        }
        m = mt;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int i = 0; i < DV / NTHR; ++i) {
        const size_t at = ((size_t)h * a.nt + t) * DV + tid + NTHR * i;
        if (a.dst_f16) reinterpret_cast<half_t *>(a.dst)[at] = to_half(o[i] * inv);
        else reinterpret_cast<float *>(a.dst)[at] = o[i] * inv;
    }
}

}  // namespace

bool attn_supported(int dk, int dv) { return (dk == 576 && dv == 512) || (dk == 320 && dv == 256); }

size_t attn_workspace_bytes(int, int, int, int, int) { return 0; }

template <int DK, int DV>
static hipError_t launch(bool q8, const AttnArgs & a, hipStream_t stream) {
    const dim3 grid(a.n_head, a.nt);
    if (q8) hipLaunchKernelGGL((kqkv_paged_kernel<DK, DV, true>), grid, dim3(NTHR), 0, stream, a);
    else hipLaunchKernelGGL((kqkv_paged_kernel<DK, DV, false>), grid, dim3(NTHR), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_attn(int dk, int dv, bool q8, const AttnArgs & a, hipStream_t stream) {
    if (dk == 576 && dv == 512) return launch<576, 512>(q8, a, stream);
    if (dk == 320 && dv == 256) return launch<320, 256>(q8, a, stream);
    return hipErrorInvalidValue;
}

}  // namespace paged
}  // namespace mla
