// kqkv_paged.hip -- KQKV over the pages of a batch (paged.h): token i of request b, whose q has H heads, sees the
// first past_b + i + 1 cells of the request's table,
//   dst[h][t][:] = softmax_j(kq_scale q[t][h] . K[cell(j)]) . V[cell(j)],  V = the first D_v columns of a row,
// and the cells that the first requests share are taken once for all of them.
//
// The rows (token, head) of a request are cut into blocks of 128, those of all sharing requests together into blocks
// of 128 against the shared cells: these are the groups, each with its run of 64-key tiles.  A request with at most 32
// rows (a decode step) streams its cells at the memory's rate with four waves on the same 32 rows; the others reuse
// each tile for up to 128 rows, where the matrix cores and the memory are about even (128 rows x 2 x (D_k + D_v)
// operations per 2 D_k bytes of a key), and the shared cells, read once per 128 rows of the whole batch, are a dense
// product.
//
// Work split.  The lengths are on the device and very different, a CU holds one workgroup (150 KB of LDS), and a
// second round of workgroups that is mostly empty costs a whole one.  So the groups' costs (tiles, and OVERHEAD tiles
// for a group's start and end) are laid end to end, and workgroup i of N takes the i-th N-th of the line: pieces of one
// or several groups.  Every workgroup finds its place by itself from the lengths (two prefix sums over the requests),
// so nothing is planned on the host and nothing waits for a planning launch.  A group that ends up in one piece, with
// nothing shared, goes straight to dst; the other pieces leave records, which the second launch merges.  Piece of
// group g in workgroup i has record i + g: along the line one of the two grows from piece to piece.
//
// All positions on the line are computed by the same expressions in every workgroup (in 64-bit floating point, exact
// for whole numbers below 2^53), so the workgroups agree where one ends and the next begins.
#include "paged_pass.h"

namespace mla {
namespace paged {

namespace {

constexpr int N_WG = 256;                   // one workgroup per CU
constexpr double OVERHEAD = 1.0;            // a group's start and end, in tiles
constexpr int MIN_SHARED_TILES = 1;         // fewer shared tiles than this are left to the requests

// Workspace: a header, the pieces of every shared block and of every row, the records
struct Head { int rows, shared_rows; };
struct Pieces { int slot; unsigned n_row; };                    // first record, pieces (low 16 bits) and row of the block
__host__ __device__ inline size_t shared_blocks(int n_head, int nt) { return ((size_t)n_head * nt + BLOCK_ROWS - 1) / BLOCK_ROWS; }
__host__ __device__ inline size_t shared_off() { return 256; }
__host__ __device__ inline size_t own_off(int n_head, int nt) { return shared_off() + (shared_blocks(n_head, nt) * 8 + 255) / 256 * 256; }
__host__ __device__ inline size_t records_off(int n_head, int nt) { return own_off(n_head, nt) + ((size_t)n_head * nt * 8 + 255) / 256 * 256; }

// ---------------------------------------------------------------- the line of work
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The batch and a place on its line; in LDS while a piece is computed, whose registers are all in use
struct Walk {
    double x0, x1, all;                     // this workgroup's stretch, the line's length
    double base;                            // where the requests (b = -1) or request b begin
    int n_wg;
    int total;                              // rows (tokens) of the batch
    int cap;                                // cells that a table lists
    int n_share, shared_keys, shared_rows;  // sharing requests, their cells, their rows (token, head)
    int shared_by;                          // the first of them that has tokens
    int b, j, tok0, g;                      // the next group: block j of request b (-1: of the shared rows), its first
                                            // token, its number
    __device__ __forceinline__ double edge(int i) const { return i >= n_wg ? all : all * (double)i / (double)n_wg; }
    __device__ __forceinline__ int shared_blocks() const { return (shared_rows + BLOCK_ROWS - 1) / BLOCK_ROWS; }
    __device__ __forceinline__ double shared_a(int n_head) const { return (double)n_head * ((double)(shared_keys / TK) + OVERHEAD); }
};

// request b's place: its tokens, what they see, its blocks and their costs in tiles / H (the j-th: a + 2 (j + 1), as
// 128 rows on are 128 / H tokens, 2 / H tiles)
struct Request {
    int n, past, key0, blocks;
    double a;
    __device__ __forceinline__ Request(const AttnArgs & ar, const Walk & wk, int b, int start) {
        n = min(min(max(ar.n_new[b], 0), ar.nt), ar.nt - start);
        past = min(clamp_past(ar.past[b]), wk.cap);
        key0 = b < wk.n_share ? wk.shared_keys : 0;
        blocks = (n * ar.n_head + BLOCK_ROWS - 1) / BLOCK_ROWS;
        const int first = (min(past + 1, wk.cap) - key0 + TK - 1) / TK;
        a = (double)ar.n_head * ((double)max(first, 1) + OVERHEAD);
    }
    __device__ __forceinline__ double upto(int j) const { return (double)j * a + (double)j * ((double)j + 1.0); }
    __device__ __forceinline__ double cost() const { return upto(blocks); }
};

// This workgroup's stretch and its first group, from the lengths.  `mem`: MAX_SEQS * 16 bytes of LDS; red: 64 bytes.
__device__ __forceinline__ Walk find_place(const AttnArgs & a, char * mem, int * red) {
    double * cum = reinterpret_cast<double *>(mem);                     // cost before request b
    int * start = reinterpret_cast<int *>(mem) + 2 * MAX_SEQS;          // its first row
    int * grp = start + MAX_SEQS;                                       // blocks before it
    double * red_d = reinterpret_cast<double *>(red) + 4;
    const int tid = threadIdx.x, lane = tid & 63, H = a.n_head, wg = blockIdx.x;
    Walk k;
    k.cap = a.max_pages << a.page_shift;
    k.total = uni(min(block_scan<NTHR>(a.n_seq, [&](int b) { return min(max(a.n_new[b], 0), a.nt); }, start, red), a.nt));
    k.n_share = k.shared_keys = k.shared_rows = k.shared_by = 0;
    if (a.prefix != nullptr) {
        // as many whole tiles of shared cells as all sharing requests with tokens held before them
        const int n = min(max(a.prefix[1], 0), a.n_seq);
        int keys = min(max(a.prefix[0], 0), k.cap), active = 0, by = MAX_SEQS;
        for (int b = tid; b < n; b += NTHR)
            if (a.n_new[b] > 0) {
                keys = min(keys, clamp_past(a.past[b]));
                by = min(by, b);
                ++active;
            }
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) {
            keys = min(keys, __shfl_xor(keys, i));
            by = min(by, __shfl_xor(by, i));
            active += __shfl_xor(active, i);
        }
        if (lane == 0) {
            red[tid >> 6] = keys;
            red[4 + (tid >> 6)] = active;
            red[8 + (tid >> 6)] = by;
        }
        __syncthreads();
        keys = uni(min(min(red[0], red[1]), min(red[2], red[3])) / TK * TK);
        active = uni(red[4] + red[5] + red[6] + red[7]);
        k.shared_by = uni(min(min(red[8], red[9]), min(red[10], red[11])));
        __syncthreads();
        if (active > 1 && keys >= MIN_SHARED_TILES * TK) {
            k.n_share = uni(n);
            k.shared_keys = keys;
            k.shared_rows = uni((n < a.n_seq ? min(start[n], a.nt) : k.total) * H);
        }
    }
    const double shared_a = k.shared_a(H), shared_cost = (double)k.shared_blocks() * shared_a;
    const int n_own = block_scan<NTHR>(a.n_seq, [&](int b) { return Request(a, k, b, min(start[b], a.nt)).blocks; }, grp, red);
    k.all = shared_cost + block_scan<NTHR>(a.n_seq, [&](int b) { return Request(a, k, b, min(start[b], a.nt)).cost(); }, cum, red_d);
    // at most one workgroup per tile
    const double tiles = k.all / (double)H - OVERHEAD * (double)(k.shared_blocks() + n_own);
    k.n_wg = uni(min(max((int)min(tiles, 65535.0), 1), (int)gridDim.x));
    k.x0 = k.edge(wg);
    k.x1 = k.edge(wg + 1);
    if (wg >= k.n_wg || k.total == 0) return k;

    if (uni(k.x0 < shared_cost)) {
        int j = min((int)(k.x0 / shared_a), k.shared_blocks() - 1);
        while (j > 0 && (double)j * shared_a > k.x0) --j;
        while (j + 1 < k.shared_blocks() && (double)(j + 1) * shared_a <= k.x0) ++j;
        k.b = -1;
        k.base = 0.0;
        k.tok0 = 0;
        k.j = k.g = j;
    } else {
        int b = last_at_most(cum, a.n_seq, k.x0 - shared_cost);
        // requests without tokens take no place: the last request that begins here is one with tokens, unless only
        // such ones follow
        while (b > 0 && Request(a, k, b, min(start[b], a.nt)).blocks == 0) --b;
        k.b = b;
        k.base = shared_cost + cum[b];
        k.tok0 = min(start[b], a.nt);
        const Request rq(a, k, b, k.tok0);
        int lo = 0, len = rq.blocks;
        while (len > 1) {
            const int half = len >> 1;
            if (k.base + rq.upto(lo + half) <= k.x0) {
                lo += half;
                len -= half;
            } else {
                len = half;
            }
        }
        k.j = lo;
        k.g = k.shared_blocks() + grp[b] + lo;
    }
    return k;
}

template <int DK, int DV, bool Q8>
struct KernelLds {
    PieceLds<DK, DV, Q8> piece;
    Walk walk;
};

template <int DK, int DV, bool Q8>
__global__ __launch_bounds__(NTHR, 1) void kqkv_paged_kernel(AttnArgs a) {
    using L = PieceLds<DK, DV, Q8>;
    __shared__ KernelLds<DK, DV, Q8> lds;
    static_assert(MAX_SEQS * 16 <= L::RING, "the prefix sums fit the ring");
    L & sh = lds.piece;
    const int tid = threadIdx.x, wg = blockIdx.x;
    {
        const Walk k = find_place(a, sh.ring, reinterpret_cast<int *>(sh.qoff));
        if (wg == 0 && tid == 0) *reinterpret_cast<Head *>(a.work) = Head{k.total * a.n_head, k.shared_rows};
        if (wg >= k.n_wg || k.total == 0) return;
        if (tid == 0) lds.walk = k;
        __syncthreads();
    }
    for (;;) {
        // ---- the group: its rows, keys, tiles and stretch of the line; the place of the next one ----
        Piece p;
        bool last, first;
        int pieces = 0, j, b;
        Walk next;
        {
            const Walk k = lds.walk;
            const int H = a.n_head;
            b = uni(k.b);
            j = uni(k.j);
            p.tok0 = uni(k.tok0);
            p.row0 = j * BLOCK_ROWS;
            double g0, g1;
            int n_tiles, blocks, n = 0;
            double cost = 0.0;
            bool direct = false;
            if (b < 0) {
                p.rows = uni(min(BLOCK_ROWS, k.shared_rows - p.row0));
                p.past = p.key1 = p.lim_min = uni(k.shared_keys);
                p.key0 = 0;
                p.table = reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(a.table) + (int64_t)uni(k.shared_by) * a.t_nb1);
                n_tiles = p.key1 / TK;
                blocks = k.shared_blocks();
                const double sa = k.shared_a(H);
                g0 = (double)j * sa;
                g1 = (double)(j + 1) * sa;
                cost = (double)blocks * sa;
            } else {
                const Request rq(a, k, b, p.tok0);
                n = rq.n;
                cost = rq.cost();
                blocks = rq.blocks;
                p.rows = uni(min(BLOCK_ROWS, n * H - p.row0));
                p.past = uni(rq.past);
                p.key0 = uni(rq.key0);
                p.key1 = uni(min(rq.past + (p.row0 + p.rows - 1) / H + 1, k.cap));
                p.lim_min = uni(min(rq.past + p.row0 / H + 1, k.cap));
                p.table = reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(a.table) + (int64_t)b * a.t_nb1);
                n_tiles = max(1, (p.key1 - p.key0 + TK - 1) / TK);
                g0 = k.base + rq.upto(j);
                g1 = k.base + rq.upto(j + 1);
                direct = uni(b >= k.n_share && g0 >= k.x0 && g1 <= k.x1);
            }
            auto tile_at = [&](double x) {
                return x <= g0 ? 0 : x >= g1 ? n_tiles : min(n_tiles, (int)((x - g0) / (g1 - g0) * (double)n_tiles + 0.5));
            };
            p.ta = uni(tile_at(k.x0));
            p.tb = uni(tile_at(k.x1));
            p.slot = direct ? -1 : uni(wg + k.g);
            first = uni(g0 >= k.x0);                     // the group's first piece says how many there are
            if (first && !direct) {
                int e = min(max((int)(g1 / k.all * (double)k.n_wg), wg + 1), k.n_wg);
                while (e > wg + 1 && k.edge(e - 1) >= g1) --e;
                while (e < k.n_wg && k.edge(e) < g1) ++e;
                pieces = uni(e - wg);
            }
            last = uni(k.x1 <= g1);
            next = k;
            next.j = j + 1;
            next.g = k.g + 1;
            if (uni(next.j >= blocks)) {                 // the next request with tokens
                next.base = k.base + cost;
                next.tok0 = p.tok0 + n;
                next.j = 0;
                next.b = b + 1;
                while (next.b < a.n_seq && Request(a, k, next.b, next.tok0).blocks == 0) ++next.b;
                last = last || uni(next.b >= a.n_seq);
            }
        }
        __syncthreads();                     // the last piece's rows and ring, and the place, have been read
        if (tid == 0) lds.walk = next;
        piece_rows(a, p, sh.qoff, sh.drow, sh.lim);
        if (first) {
            if (b < 0) {
                if (tid == 0) reinterpret_cast<Pieces *>(a.work + shared_off())[j] = Pieces{p.slot, (unsigned)pieces};
            } else if (tid < p.rows) {
                reinterpret_cast<Pieces *>(a.work + own_off(a.n_head, a.nt))[(size_t)p.tok0 * a.n_head + p.row0 + tid] =
                    Pieces{p.slot, (unsigned)pieces | (unsigned)tid << 16};
            }
        }
        char * rec = a.work + records_off(a.n_head, a.nt) + (size_t)max(p.slot, 0) * record_bytes<DV>();
        __syncthreads();
        if (p.ta >= p.tb) {                  // no tile of the group falls to this workgroup (never where direct)
            if (tid < BLOCK_ROWS) reinterpret_cast<f32x2 *>(rec)[tid] = f32x2{-INFINITY, 0.0f};
        } else if (p.rows <= HG && p.row0 == 0) {
            narrow_piece<DK, DV, Q8>(a, p, sh, rec);
        } else {
            wide_piece<DK, DV, Q8>(a, p, sh, rec);
        }
        if (last) return;
    }
}

// ---------------------------------------------------------------- the merge
// A workgroup per row (and per DV / CB columns of it): its pieces, those of the row's own group and of its shared
// block.  LP lanes hold a piece's columns, eight each; 256 / LP pieces at a time.
template <int DV, int CB>
__global__ __launch_bounds__(NTHR) void kqkv_paged_merge_kernel(AttnArgs a) {
    constexpr int LP = DV / CB / 8, PP = NTHR / LP, U = 4;
    __shared__ float sm[PP], sl[PP];
    __shared__ f32x4 so[2][NTHR];
    const int tid = threadIdx.x, c = tid % LP, pi = tid / LP;
    const int col = (int)blockIdx.y * (DV / CB) + 8 * c;
    const Head head = *reinterpret_cast<const Head *>(a.work);
    const Pieces * shared_at = reinterpret_cast<const Pieces *>(a.work + shared_off());
    const Pieces * own_at = reinterpret_cast<const Pieces *>(a.work + own_off(a.n_head, a.nt));
    const char * records = a.work + records_off(a.n_head, a.nt);
    for (int row = blockIdx.x; row < head.rows; row += gridDim.x) {
        const Pieces own = own_at[row];
        const int n_own = (int)(own.n_row & 0xffffu), r_own = (int)(own.n_row >> 16);
        if (n_own == 0) continue;                        // complete already
        Pieces shd = {0, 0};
        if (row < head.shared_rows) shd = shared_at[row / BLOCK_ROWS];
        const int n = n_own + (int)shd.n_row, r_shd = row % BLOCK_ROWS;
        float m = -INFINITY, l = 0.0f, o[8] = {};
        for (int q0 = pi; q0 < n; q0 += PP * U) {
            float ms[U], ls[U];
            half8 os[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int q = min(q0 + PP * u, n - 1);
                const bool mine = q < n_own;
                const char * rec = records + (size_t)(mine ? own.slot + q : shd.slot + q - n_own) * record_bytes<DV>();
                const int r = mine ? r_own : r_shd;
                const f32x2 ml = reinterpret_cast<const f32x2 *>(rec)[r];
                ms[u] = q0 + PP * u < n ? ml[0] : -INFINITY;
                ls[u] = q0 + PP * u < n ? ml[1] : 0.0f;
                os[u] = *reinterpret_cast<const half8 *>(rec + BLOCK_ROWS * 8 + ((size_t)r * DV + col) * 2);
            }
            float mx = m;
#pragma unroll
            for (int u = 0; u < U; ++u) mx = fmaxf(mx, ms[u]);
            const float f0 = exp2_unless(m == -INFINITY, m - mx);
            l *= f0;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] *= f0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float f = ls[u] * exp2_unless(ms[u] == -INFINITY, ms[u] - mx);     // a NaN l (no finite score) stays one
                l += f;
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] += ms[u] == -INFINITY ? f : f * (float)os[u][k];   // an empty piece has no o
            }
            m = mx;
        }
        __syncthreads();                                 // the row before has been read
        if (c == 0) {
            sm[pi] = m;
            sl[pi] = l;
        }
        so[0][tid] = f32x4{o[0], o[1], o[2], o[3]};
        so[1][tid] = f32x4{o[4], o[5], o[6], o[7]};
        __syncthreads();
        if (pi == 0) {
            float M = -INFINITY, Ls = 0.0f;
            f32x4 r0 = {0.f, 0.f, 0.f, 0.f}, r1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < PP; ++i) M = fmaxf(M, sm[i]);
#pragma unroll
            for (int i = 0; i < PP; ++i) {
                const float f = exp2_unless(sm[i] == -INFINITY, sm[i] - M);
                const float e = sm[i] == -INFINITY ? sl[i] : 0.0f;       // 0, or NaN
                Ls += sl[i] * f + e;
                r0 += so[0][i * LP + c] * f + e;
                r1 += so[1][i * LP + c] * f + e;
            }
            const float inv = Ls == 0.0f ? 0.0f : 1.0f / Ls;
            r0 *= inv;
            r1 *= inv;
            const int t = row / a.n_head, h = row - t * a.n_head;
            const size_t at = ((size_t)h * a.nt + t) * DV + col;
            if (a.dst_f16) {
                half8 v;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[k] = to_half(r0[k]);
                    v[4 + k] = to_half(r1[k]);
                }
                *reinterpret_cast<half8 *>(a.dst + at * 2) = v;
            } else {
                *reinterpret_cast<f32x4 *>(a.dst + at * 4) = r0;
                *reinterpret_cast<f32x4 *>(a.dst + at * 4 + 16) = r1;
            }
        }
    }
}

}  // namespace

bool attn_supported(int dk, int dv) { return (dk == 576 && dv == 512) || (dk == 320 && dv == 256); }

size_t attn_workspace_bytes(int, int dv, int n_seq, int n_head, int nt) {
    // records: one per workgroup and group (own blocks: at most one partly filled per request with tokens)
    const size_t groups = 2 * shared_blocks(n_head, nt) + (size_t)(n_seq < nt ? n_seq : nt);
    return records_off(n_head, nt) + (N_WG + groups) * (dv == 512 ? record_bytes<512>() : record_bytes<256>());
}

template <int DK, int DV>
static hipError_t launch(bool q8, const AttnArgs & a, hipStream_t stream) {
    if (q8) hipLaunchKernelGGL((kqkv_paged_kernel<DK, DV, true>), dim3(N_WG), dim3(NTHR), 0, stream, a);
    else hipLaunchKernelGGL((kqkv_paged_kernel<DK, DV, false>), dim3(N_WG), dim3(NTHR), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int rows = a.n_head * a.nt;
    if (rows <= 512) hipLaunchKernelGGL((kqkv_paged_merge_kernel<DV, DV / 64>), dim3(rows, DV / 64), dim3(NTHR), 0, stream, a);
    else hipLaunchKernelGGL((kqkv_paged_merge_kernel<DV, 1>), dim3(rows < 4096 ? rows : 4096), dim3(NTHR), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_attn(int dk, int dv, bool q8, const AttnArgs & a, hipStream_t stream) {
    if (dk == 576 && dv == 512) return launch<576, 512>(q8, a, stream);
    if (dk == 320 && dv == 256) return launch<320, 256>(q8, a, stream);
    return hipErrorInvalidValue;
}

}  // namespace paged
}  // namespace mla
