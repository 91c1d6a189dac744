// kqkv_paged.hip -- KQKV over the pages of a batch (paged.h): token i of request b, whose q has H heads, sees the
// first past_b + i + 1 cells of the request's table,
//   dst[h][t][:] = softmax_j(kq_scale q[t][h] . K[cell(j)]) . V[cell(j)],  V = the first D_v columns of a row,
// and the cells that the first requests share are taken once for all of them.
//
// The rows (token, head) of a request are cut into blocks of 128 (of 32 where there is little to do: FEW_TILES), those
// of all sharing requests together into blocks of 128 against the shared cells: these are the groups, each with its run
// of 64-key tiles.  Up to 32 rows (a decode step) stream their cells at the memory's rate with four waves on the same
// rows; more reuse each tile for up to 128, where the matrix cores and the memory are about even (128 rows x 2 x
// (D_k + D_v) operations per 2 D_k bytes of a key), and the shared cells, read once per 128 rows of the whole batch, are
// a dense product.
//
// Work split.  The lengths are on the device and very different, a CU holds one workgroup (150 KB of LDS), and a
// second round of workgroups that is mostly empty costs a whole one.  So the groups' costs (of their tiles
// and of a group's start and end) are laid end to end, and workgroup i of N takes the i-th N-th of the line: pieces of one
// or several groups.  Every workgroup finds its place by itself from the lengths (two prefix sums over the requests),
// so nothing is planned on the host and nothing waits for a planning launch.  A group that ends up in one piece, with
// nothing shared, goes straight to dst; the other pieces leave records, which the second launch merges.  Groups of
// rows that share cells come first on the line and always leave records: piece of group g in workgroup i has record
// i + g, as along the line one of the two grows from piece to piece.  Of the other groups a workgroup holds at most two
// in part: one that goes on behind it has record i, one that began before it record N + i.
//
// What it comes to (device times in a graph, both launches; narrow pieces read at 6.3 TB/s, wide ones run at 1.08
// PFLOP/s, where a large copy moves 5.2 and a large f16 matrix product 1.18): 4 requests of 90,000 to 131,000 cells, 16
// heads, 82 us; 48 of 300 to 9,000, 32 heads, 44.1; 64 of 150 to 250 15.9; 64 behind 32,768 shared cells 166; 9 requests
// and a chunk of 700 tokens, 40 heads, 127; one of 200 cells 11.9.  Around the tiles a call spends 2.5 us on the places,
// 0.8 on a piece's setup, 2 (narrow) to 4 (wide, f16) or 7 (wide, f32) on its q, 1 to 2 on its results, and 4 to 22 on the
// second launch, whose bytes are the records'.  Requests without tokens cost a workgroup that passes them between two
// groups 0.09 us each: 5 live ones of 9,000 cells among 5, 256, 1,024 and 4,096 slots 22, 26, 44 and 119 us.
//
// All positions on the line are computed by the same expressions in every workgroup (in 64-bit floating point, exact
// for multiples of a quarter below 2^51, which MAX_LINE keeps them), so the workgroups agree where one ends and the next
// begins.
#include "paged_pass.h"

namespace mla {
namespace paged {

namespace {

constexpr int N_WG = 256;                   // one workgroup per CU
// Costs, in tenths of a wide tile (all of them times H, so that they are whole numbers): a tile for up to 128 rows and
// for up to 32, and a piece's start and end (its rows in, its results out).  Times of tiles and pieces per geometry and
// cache; one set for all of them took 50.5 us instead of 48 for 40 8-bit requests behind 12,000 cells, starts of 8 less 88.7
// instead of 78.2 for 1,000 tokens of one prompt, of 4 more 40.2 instead of 38.2 for four tokens of 24 requests.
template <int DK, bool Q8>
struct Cost {
    static constexpr bool BIG = DK == 576;
    static constexpr int WIDE_TILE = 10, NARROW_TILE = Q8 ? (BIG ? 5 : 6) : BIG ? 6 : 7;
    static constexpr int WIDE_START = Q8 ? (BIG ? 22 : 20) : BIG ? 21 : 28, NARROW_START = Q8 ? (BIG ? 9 : 11) : BIG ? 11 : 16;
};

// Shared cells are taken once where that pays: where it saves every workgroup SHARE_GAIN, as it costs a wide piece more
// with its records (7 us of the larger geometry).  A request that takes them by itself pays for a tile, which it then
// finds in the caches: 5 with up to 32 rows, else 6 and one for every 32 rows of a block, so a block of 128 gains
// nothing.  Device times, shared and not, 32 heads of one token, the larger geometry: 32 requests behind 1,024 cells
// 26.7 and 21.1 us, behind 4,096 32.5 and 32.0, behind 16,384 60.2 and 75.7; 64 behind 4,096 44.1 and 49.3; 4 behind 16,384
// 30.8 and 25.6.
constexpr int SHARE_GAIN = 16;
__device__ __forceinline__ int repeat_cost(int rows) {
    const int part = rows % BLOCK_ROWS;
    return rows <= HG ? (rows > 0 ? 5 : 0) : rows / BLOCK_ROWS * 10 + (part > 0 ? 6 + (part + 31) / 32 : 0);
}

// Of few tiles in all (counted for 32 rows each; nothing shared) every group is of 32 rows: its q, its results and its
// records are a quarter, and the card is not full. Device times with groups of 32 and of 128 rows: 2 requests of 7,500 cells,
// 128 heads (944 tiles) 24.0 and 32.0 us, one of 20,000 (1,252) 25.0 and 31.7, one of 29,000 (1,816) 30.4 and 33.2, of 50,000
// (3,128) 39.2 and 38.8; 4 tokens of 50 requests of 84 to 283 cells (800) 27.0 and 31.6, of 16 of 1,700 (1,728) 36.9 and
// 33.8; over (320, 256) one of 40,000 (2,504) 25.6 and 23.9.
constexpr int FEW_TILES = 1600;

// Workspace: a header, the pieces of every shared block and of every row, the records (those of whole groups, two per
// workgroup, then those of the sharing rows' groups)
struct Head { int rows, shared_rows; };
struct Pieces { int slot; unsigned n_row; };                    // first record, pieces (low 16 bits) and row of the block
constexpr int SHARED_RECORDS = 2 * N_WG;                        // where the latter begin
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
    int block;                              // rows of a request's group: 128, or 32 (few tiles in all)
    int single;                             // 1: a workgroup per tile
    int n_share, shared_keys, shared_rows;  // sharing requests, their cells, their rows (token, head)
    int shared_by;                          // the first of them that has tokens
    int b, j, tok0, g;                      // the next group: block j of request b (-1: of the shared rows), its first
                                            // token, its number
    int n_new, past;                        // request b's, as given
    double per;                             // all / n_wg
    __device__ __forceinline__ double edge(int i) const { return i >= n_wg ? all : per * (double)i; }
    __device__ __forceinline__ int shared_blocks() const { return (shared_rows + BLOCK_ROWS - 1) / BLOCK_ROWS; }
    template <typename C>
    __device__ __forceinline__ double shared_a(int n_head) const { return (double)n_head * (double)(C::WIDE_START + C::WIDE_TILE * (shared_keys / TK)); }
};

// request b's place: its tokens, what they see, its blocks and their costs (the j-th of 128 rows: a + 2 WIDE_TILE (j + 1),
// as 128 rows on are 128 / H tokens, 2 / H tiles; of 32 rows: a + NARROW_TILE (j + 1) / 2)
template <typename C>
struct Request {
    int n, past, key0, blocks;
    bool wide, free_start;
    double a, more;
    __device__ __forceinline__ Request(const AttnArgs & ar, const Walk & wk, int H, int n_new, int past_, int b, int start) {
        n = min(min(max(n_new, 0), ar.nt), ar.nt - start);
        past = min(clamp_past(past_), wk.cap);
        key0 = b < wk.n_share ? wk.shared_keys : 0;
        const bool narrow = wk.block == HG;
        blocks = (n * H + wk.block - 1) >> (narrow ? 5 : 7);
        wide = n * H > HG && !narrow;
        more = wk.single != 0 ? 0.0 : narrow ? 0.25 * (double)C::NARROW_TILE : (double)C::WIDE_TILE;
        free_start = wk.single != 0;
        const int first = max((min(past + 1, wk.cap) - key0 + TK - 1) / TK, 1);
        a = (double)H * (double)(start_cost() + (wide ? C::WIDE_TILE : C::NARROW_TILE) * first);
    }
    __device__ __forceinline__ Request(const AttnArgs & ar, const Walk & wk, int H, int b, int start)
        : Request<C>(ar, wk, H, wk.n_new, wk.past, b, start) {}
    __device__ __forceinline__ int start_cost() const { return free_start ? 0 : wide ? C::WIDE_START : C::NARROW_START; }
    __device__ __forceinline__ double upto(int j) const { return (double)j * a + more * ((double)j * ((double)j + 1.0)); }
    __device__ __forceinline__ double cost() const { return upto(blocks); }
};

// This workgroup's stretch and its first group (b = n_seq: none), from the lengths: two sums over the requests by the
// whole workgroup, then the thread whose request holds the stretch's start says so.
struct PlaceLds {
    int rows[4], tiles[4], shared[4][3];    // per wavefront: rows; narrow tiles; sharing requests' cells, rows, first
    double repeat[4], cost[4];
    int groups[4];
    double base;
    int b, tok0, g, n_new, past;
};
template <typename C>
__device__ __forceinline__ Walk find_place(const AttnArgs & a, PlaceLds & sh) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, H = a.n_head, wg = blockIdx.x;
    const int per = (a.n_seq + NTHR - 1) / NTHR, b0 = min(tid * per, a.n_seq), b1 = min(b0 + per, a.n_seq);
    const int n_pre = a.prefix != nullptr ? min(max(a.prefix[1], 0), a.n_seq) : 0;
    const int k_pre = a.prefix != nullptr ? a.prefix[0] : 0;
    Walk k = {};
    k.cap = a.max_pages << a.page_shift;
    // the first of this thread's requests stays in registers: up to 256 requests it is the only one
    const int n0 = b0 < b1 ? a.n_new[b0] : 0, past0 = b0 < b1 ? a.past[b0] : 0;
    auto n_of = [=](int b) {
        int v = n0;
        if (b != b0) v = a.n_new[b];
        return v;
    };
    auto past_of = [=](int b) {
        int v = past0;
        if (b != b0) v = a.past[b];
        return v;
    };

    int own = 0, tiles32 = 0, keys = min(max(k_pre, 0), k.cap), srows = 0, by = MAX_SEQS;
    double repeat = 0.0;
    for (int b = b0; b < b1; ++b) {
        const int n = min(max(n_of(b), 0), a.nt);
        own += n;
        // (no more than FEW_TILES of either factor, nor more than one past it of a request, count)
        const int tiles = min((n * H + HG - 1) / HG, FEW_TILES) * min((min(clamp_past(past_of(b)), k.cap) + n / 2) / TK + 1, FEW_TILES);
        tiles32 += min(tiles, FEW_TILES + 1);
        if (b < n_pre && n > 0) {
            keys = min(keys, clamp_past(past_of(b)));
            by = min(by, b);
            srows += n;
            repeat += (double)repeat_cost(n * H);
        }
    }
    const int incl = wave_scan(own);
    tiles32 = wave_scan(tiles32);
    if (lane == 63) {
        sh.rows[w] = incl;
        sh.tiles[w] = tiles32;
    }
    if (a.prefix != nullptr) {
        keys = wave_min(keys);
        by = wave_min(by);
        repeat = wave_scan(repeat);
        srows = wave_scan(srows);
        if (lane == 63) {
            sh.shared[w][0] = keys;
            sh.shared[w][1] = srows;
            sh.shared[w][2] = by;
            sh.repeat[w] = repeat;
        }
    }
    if (tid == 0) sh.b = a.n_seq;
    __syncthreads();
    int start = incl - own, total = 0;      // rows before this thread's requests
#pragma unroll
    for (int i = 0; i < NTHR / 64; ++i) {
        start += i < w ? sh.rows[i] : 0;
        total += sh.rows[i];
    }
    k.total = uni(min(total, a.nt));
    if (a.prefix != nullptr) {
        // as many whole tiles of shared cells as all sharing requests with tokens held before them
        keys = uni(min(min(sh.shared[0][0], sh.shared[1][0]), min(sh.shared[2][0], sh.shared[3][0])) / TK * TK);
        k.shared_keys = keys;
        k.shared_rows = uni(min(sh.shared[0][1] + sh.shared[1][1] + sh.shared[2][1] + sh.shared[3][1], a.nt) * H);
        const double saved = (sh.repeat[0] + sh.repeat[1] + sh.repeat[2] + sh.repeat[3]) * (double)(keys / TK) * (double)H -
                             (double)k.shared_blocks() * k.template shared_a<C>(H);
        if (uni(saved > (double)(SHARE_GAIN * N_WG) * (double)H)) {
            k.n_share = n_pre;
            k.shared_by = uni(min(min(sh.shared[0][2], sh.shared[1][2]), min(sh.shared[2][2], sh.shared[3][2])));
        } else {
            k.shared_keys = k.shared_rows = 0;
        }
    }
    tiles32 = sh.tiles[0] + sh.tiles[1] + sh.tiles[2] + sh.tiles[3];
    k.block = uni(k.n_share == 0 && tiles32 <= FEW_TILES ? HG : BLOCK_ROWS);
    k.single = uni(k.n_share == 0 && tiles32 <= N_WG ? 1 : 0);
    const double shared_a = k.template shared_a<C>(H), shared_cost = (double)k.shared_blocks() * shared_a;

    double cost = 0.0;
    int groups = 0;
    {
        int at = min(start, a.nt);
        for (int b = b0; b < b1; ++b) {
            const Request<C> rq(a, k, H, n_of(b), past_of(b), b, at);
            cost += rq.cost();
            groups += rq.blocks;
            at += rq.n;
        }
    }
    const double cost_incl = wave_scan(cost);
    const int groups_incl = wave_scan(groups);
    if (lane == 63) {
        sh.cost[w] = cost_incl;
        sh.groups[w] = groups_incl;
    }
    __syncthreads();
    double base = cost_incl - cost;
    int grp = groups_incl - groups;
    k.all = 0.0;
#pragma unroll
    for (int i = 0; i < NTHR / 64; ++i) {
        base += i < w ? sh.cost[i] : 0.0;
        grp += i < w ? sh.groups[i] : 0;
        k.all += sh.cost[i];
    }
    base += shared_cost;
    k.all += shared_cost;
    // Where there are fewer tiles than workgroups, one workgroup each: tiles alone make up the line then, as every piece
    // starts anew. With starts on it and all workgroups: 64 requests of 150 to 250 cells 17.9 instead of 16.0 us, 100 tokens of a
    // prompt 17.1 instead of 12.8, 8 requests of 500 to 700 15.2 instead of 14.1; but of more tiles (290) 18.0 instead of 21.5.
    k.n_wg = k.single != 0 ? uni(max(tiles32, 1)) : (int)gridDim.x;
    k.per = k.all / (double)k.n_wg;
    k.x0 = k.edge(wg);
    k.x1 = k.edge(wg + 1);

    const bool any = wg < k.n_wg && k.total > 0, at_shared = uni(k.x0 < shared_cost);
    if (any && !at_shared && base <= k.x0 && k.x0 < base + cost) {
        int at = min(start, a.nt), g = grp;
        for (int b = b0; b < b1; ++b) {
            const Request<C> rq(a, k, H, n_of(b), past_of(b), b, at);
            const double c = rq.cost();
            if (rq.blocks > 0 && (k.x0 < base + c || b + 1 == b1)) {
                sh.b = b;
                sh.n_new = n_of(b);
                sh.past = past_of(b);
                sh.tok0 = at;
                sh.g = g;
                sh.base = base;
                break;
            }
            base += c;
            g += rq.blocks;
            at += rq.n;
        }
    }
    __syncthreads();
    k.b = any ? (at_shared ? -1 : uni(sh.b)) : a.n_seq;
    k.tok0 = at_shared ? 0 : uni(sh.tok0);
    k.base = at_shared ? 0.0 : sh.base;
    int j = 0;
    if (at_shared) {
        j = min((int)(k.x0 / shared_a), k.shared_blocks() - 1);
        while (j > 0 && (double)j * shared_a > k.x0) --j;
        while (j + 1 < k.shared_blocks() && (double)(j + 1) * shared_a <= k.x0) ++j;
    } else if (k.b < a.n_seq) {
        k.n_new = uni(sh.n_new);
        k.past = uni(sh.past);
        const Request<C> rq(a, k, H, k.b, k.tok0);
        int len = rq.blocks;
        while (len > 1) {
            const int half = len >> 1;
            if (k.base + rq.upto(j + half) <= k.x0) {
                j += half;
                len -= half;
            } else {
                len = half;
            }
        }
    }
    k.j = uni(j);
    k.g = at_shared ? k.j : uni(k.shared_blocks() + sh.g + j);
    return k;
}

template <int DK, int DV, bool Q8>
struct KernelLds {
    PieceLds<DK, DV, Q8> piece;
    Walk walk;
    PlaceLds place;
};

template <int DK, int DV, bool Q8, bool QF16>
__global__ __launch_bounds__(NTHR, 1) void kqkv_paged_kernel(AttnArgs a) {
    using L = PieceLds<DK, DV, Q8>;
    __shared__ KernelLds<DK, DV, Q8> lds;
    L & sh = lds.piece;
    const int tid = threadIdx.x, wg = blockIdx.x;
    using C = Cost<DK, Q8>;
    Walk k = find_place<C>(a, lds.place);
    if (wg == 0 && tid == 0) *reinterpret_cast<Head *>(a.work) = Head{k.total * a.n_head, k.shared_rows};
    if (k.b >= a.n_seq) return;              // no part of the line
    for (;;) {
        // ---- the group: its rows, keys, tiles and stretch of the line; the place of the next one ----
        Piece p;
        bool last, first;
        int pieces = 0, j, b;
        Walk next;
        {
            int H = a.n_head;
            asm volatile("" : "+s"(H));      // its 64-bit form is taken anew for each piece, not kept through them
            b = uni(k.b);
            j = uni(k.j);
            p.tok0 = uni(k.tok0);
            p.row0 = j * (b < 0 ? BLOCK_ROWS : k.block);
            double g0, g1, body;             // its stretch, and where its tiles begin on it
            int n_tiles, blocks, n = 0;
            double cost;
            bool direct = false;
            if (b < 0) {
                p.rows = uni(min(BLOCK_ROWS, k.shared_rows - p.row0));
                p.past = p.key1 = p.lim_min = uni(k.shared_keys);
                p.key0 = 0;
                p.table = reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(a.table) + (int64_t)uni(k.shared_by) * a.t_nb1);
                n_tiles = p.key1 / TK;
                blocks = k.shared_blocks();
                const double sa = k.template shared_a<C>(H);
                g0 = (double)j * sa;
                g1 = (double)(j + 1) * sa;
                body = g0 + (double)(H * C::WIDE_START);
                cost = (double)blocks * sa;
            } else {
                const Request<C> rq(a, k, H, b, p.tok0);
                n = rq.n;
                cost = rq.cost();
                blocks = rq.blocks;
                p.rows = uni(min(k.block, n * H - p.row0));
                p.past = uni(rq.past);
                p.key0 = uni(rq.key0);
                p.key1 = uni(min(rq.past + (p.row0 + p.rows - 1) / H + 1, k.cap));
                p.lim_min = uni(min(rq.past + p.row0 / H + 1, k.cap));
                p.table = reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(a.table) + (int64_t)b * a.t_nb1);
                n_tiles = max(1, (p.key1 - p.key0 + TK - 1) / TK);
                g0 = k.base + rq.upto(j);
                g1 = k.base + rq.upto(j + 1);
                body = g0 + (double)(H * rq.start_cost());
                direct = uni(b >= k.n_share && g0 >= k.x0 && g1 <= k.x1);
            }
            const double rate = (double)n_tiles / (g1 - body);
            auto tile_at = [&](double x) { return x <= body ? 0 : x >= g1 ? n_tiles : min(n_tiles, (int)((x - body) * rate + 0.5)); };
            p.ta = uni(tile_at(k.x0));
            p.tb = uni(tile_at(k.x1));
            first = uni(g0 >= k.x0);                     // the group's first piece says how many there are
            // (in range whatever the lengths: something that writes them during a call must not turn into an address)
            p.slot = direct ? -1 : uni(min((b < k.n_share ? SHARED_RECORDS + k.g : first ? 0 : N_WG) + wg, a.n_records - 1));
            if (first && !direct) {
                int e = min(max((int)(g1 / k.per), wg + 1), k.n_wg);
                while (e > wg + 1 && k.edge(e - 1) >= g1) --e;
                while (e < k.n_wg && k.edge(e) < g1) ++e;
                pieces = uni(e - wg);
            }
            last = uni(k.x1 <= g1);
            next = k;
            next.j = j + 1;
            next.g = k.g + 1;
            if (!last && uni(next.j >= blocks)) {        // the next request with tokens
                next.base = k.base + cost;
                next.tok0 = p.tok0 + n;
                next.j = 0;
                next.b = b + 1;
                for (; next.b < a.n_seq; ++next.b) {
                    next.n_new = uni(a.n_new[next.b]);
                    if (next.n_new > 0 && next.tok0 < a.nt) break;
                }
                last = uni(next.b >= a.n_seq);
                if (!last) next.past = uni(a.past[next.b]);
            }
        }
        if (!last && tid == 0) lds.walk = next;
        piece_rows(a, p, sh);
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
        } else if (p.rows <= HG) {
            narrow_piece<DK, DV, Q8, QF16>(a, p, sh, rec);
        } else {
            wide_piece<DK, DV, Q8, QF16>(a, p, sh, rec);
        }
        if (p.lim_min < p.key1 && sh.odd != 0) {     // (the same for all: written ahead of a barrier of the piece's)
            wait_vm<0>();
            __syncthreads();                 // the results are in place
            seen_nonfinite<DK, DV, Q8, QF16>(a, sh, rec);
        }
        if (last) return;
        k = lds.walk;
        __syncthreads();                     // the piece's rows and ring, and the place, have been read
    }
}

// ---------------------------------------------------------------- the merge
// The pieces of a row: those of its own group, then those of its shared block.  What the workspace says is brought into range
// (rows, counts, records): another call that writes it between the two launches spoils results, not memory.
struct RowPieces {
    int n, n_own, own, shared, r_own, r_shared, last;
    bool shares;
    __device__ __forceinline__ RowPieces(const AttnArgs & a, const Head & head, int row) {
        // (both read at once, whatever the row: the entries lie in the workspace also where there is no such row)
        const int at = min(row, a.n_head * a.nt - 1);
        const Pieces o = reinterpret_cast<const Pieces *>(a.work + own_off(a.n_head, a.nt))[at];
        const Pieces s = reinterpret_cast<const Pieces *>(a.work + shared_off())[at / BLOCK_ROWS];
        const int live = row <= at ? row : 0x7fffffff;
        n_own = live < head.rows ? min((int)(o.n_row & 0xffffu), N_WG) : 0;
        r_own = (int)(o.n_row >> 16) % BLOCK_ROWS;
        own = o.slot;
        shared = s.slot;
        r_shared = at % BLOCK_ROWS;
        shares = live < head.shared_rows;
        n = n_own + (shares ? (int)min(s.n_row, (unsigned)N_WG) : 0);
        last = a.n_records - 1;
    }
    // piece q's record, and the row's place in it
    template <int DV>
    __device__ __forceinline__ const char * at(const char * records, int q, int & r) const {
        const bool mine = q < n_own;
        r = mine ? r_own : r_shared;
        const unsigned of_own = (unsigned)own + (unsigned)(q + (q > 0 && !shares ? N_WG : 0));
        return records + (size_t)min(mine ? of_own : (unsigned)shared + (unsigned)(q - n_own), (unsigned)last) * record_bytes<DV>();
    }
};

// (m, l, o) of some pieces of a lane's row: eight columns of each of S slabs
template <int DV, int S>
struct Part {
    float m = -INFINITY, l = 0.0f, o[S][8] = {};
    // pieces q0, q0 + step, .. below n, slabs s0 ..
    template <int U>
    __device__ __forceinline__ void add(const RowPieces & rp, const char * records, int q0, int step, int s0, int hi) {
        for (; q0 < rp.n; q0 += step * U) {
            float ms[U], ls[U];
            half8 os[U][S];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int q = q0 + step * u;
                int r;
                const char * rec = rp.at<DV>(records, min(q, rp.n - 1), r);
                const f32x2 ml = reinterpret_cast<const f32x2 *>(rec)[r];
                ms[u] = q < rp.n ? ml[0] : -INFINITY;
                ls[u] = q < rp.n ? ml[1] : 0.0f;
                const char * at = rec + BLOCK_ROWS * 8 + (size_t)((r >> 5) * (DV / 16) + s0) * 1024 + 512 * hi + 16 * (r & 31);
#pragma unroll
                for (int s = 0; s < S; ++s) os[u][s] = *reinterpret_cast<const half8 *>(at + 1024 * s);
            }
            float mx = m;
#pragma unroll
            for (int u = 0; u < U; ++u) mx = fmaxf(mx, ms[u]);
            scale(exp2_unless(m == -INFINITY, m - mx));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // without a key l is 0, or NaN where every score was; o then holds nothing (an empty piece's was never
                // written).  (M_NONE, where no score was above -inf, is as any other: l is 0, o is 0 or NaN.)
                const bool none = ms[u] == -INFINITY;
                const float f = none ? ls[u] : ls[u] * exp2_fast(ms[u] - mx);
                l += f;
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int k = 0; k < 8; ++k) o[s][k] += none ? f : f * (float)os[u][s][k];
            }
            m = mx;
        }
    }
    __device__ __forceinline__ void scale(float f) {
        l *= f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[s][k] *= f;
    }
    __device__ __forceinline__ void out(const AttnArgs & a, int row, int s0, int hi) const {
        // (no key: zeros; keys, but no score above -inf: 0 / 0)
        const float inv = l != 0.0f ? 1.0f / l : m == -INFINITY ? 0.0f : __builtin_nanf("");
        const int t = row / a.n_head, h = row - t * a.n_head;
        const size_t at = ((size_t)h * a.nt + t) * DV + 16 * s0 + 8 * hi;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (a.dst_f16) {
                half8 v;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = to_half(o[s][k] * inv);
                *reinterpret_cast<half8 *>(a.dst + (at + 16 * s) * 2) = v;
            } else {
                f32x4 v[2];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k >> 2][k & 3] = o[s][k] * inv;
                *reinterpret_cast<f32x4 *>(a.dst + (at + 16 * s) * 4) = v[0];
                *reinterpret_cast<f32x4 *>(a.dst + (at + 16 * s) * 4 + 16) = v[1];
            }
        }
    }
};

// RW rows and one slab by a workgroup of NT: 2 RW lanes a part, the pieces dealt to the parts
template <int NT>
struct MergeLds {
    float m[NT], l[NT];
    f32x4 o[2][NT];
};
template <int DV, int NT, int RW>
__device__ __forceinline__ void merge_together(const AttnArgs & a, const RowPieces & rp, const char * records, int row, int slab, MergeLds<NT> & sh) {
    constexpr int LP = 2 * RW;
    const int tid = threadIdx.x, hi = tid / RW & 1, part = tid / LP;
    Part<DV, 1> p;
    p.template add<4>(rp, records, part, NT / LP, slab, hi);
    auto put = [&]() {
        sh.m[tid] = p.m;
        sh.l[tid] = p.l;
        sh.o[0][tid] = f32x4{p.o[0][0], p.o[0][1], p.o[0][2], p.o[0][3]};
        sh.o[1][tid] = f32x4{p.o[0][4], p.o[0][5], p.o[0][6], p.o[0][7]};
    };
    auto get = [&](int at) {
        const float m2 = sh.m[at], l2 = sh.l[at], mx = fmaxf(p.m, m2);
        const f32x4 x = sh.o[0][at], y = sh.o[1][at];
        // (without a finite score: l and o are 0 or NaN)
        p.scale(p.m == -INFINITY ? 1.0f : exp2_fast(p.m - mx));
        const float f2 = m2 == -INFINITY ? 1.0f : exp2_fast(m2 - mx);
        p.l += l2 * f2;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            p.o[0][k] += x[k] * f2;
            p.o[0][4 + k] += y[k] * f2;
        }
        p.m = mx;
    };
    // four parts into one, until one is left
#pragma unroll
    for (int n = NT / LP; n > 1;) {
        const int f = n % 4 == 0 ? 4 : 2;
        if (part < n) put();
        __syncthreads();
        n /= f;
        if (part < n) {
#pragma unroll
            for (int i = 1; i < f; ++i) get(tid + i * n * LP);
        }
        if (n > 1) __syncthreads();
    }
    if (part == 0 && rp.n > 0) p.out(a, row, slab, hi);
}

// Few rows: a workgroup per RW rows and slab
template <int DV, int NT, int RW>
__global__ __launch_bounds__(NT) void kqkv_paged_merge_few_kernel(AttnArgs a) {
    __shared__ MergeLds<NT> sh;
    const Head head = *reinterpret_cast<const Head *>(a.work);
    const int row = RW * (int)blockIdx.x + (int)(threadIdx.x % RW);
    const RowPieces rp(a, head, row);
    if (__builtin_amdgcn_ballot_w64(rp.n > 0) == 0) return;      // (the same rows in every wavefront)
    merge_together<DV, NT, RW>(a, rp, a.work + records_off(a.n_head, a.nt), row, blockIdx.y, sh);
}

// Many rows: a wavefront per 32 rows and S slabs (also rows of many pieces, a long request among short ones: 100,000 cells
// beside 63 requests of 50 88.6 us, and 93.9 with such rows' pieces dealt to four wavefronts)
template <int DV, int S>
__global__ __launch_bounds__(NTHR) void kqkv_paged_merge_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63, hi = lane >> 5;
    const Head head = *reinterpret_cast<const Head *>(a.work);
    const char * records = a.work + records_off(a.n_head, a.nt);
    const int row = 32 * (int)blockIdx.x + (lane & 31), s0 = S * (4 * (int)blockIdx.y + (int)(threadIdx.x >> 6));
    const RowPieces rp(a, head, row);
    Part<DV, S> p;
    if (__builtin_amdgcn_ballot_w64(rp.n > 2) == 0) p.template add<2>(rp, records, 0, 1, s0, hi);     // a chunk's rows
    else p.template add<4>(rp, records, 0, 1, s0, hi);
    if (rp.n > 0) p.out(a, row, s0, hi);
}

}  // namespace

bool attn_supported(int dk, int dv) { return (dk == 576 && dv == 512) || (dk == 320 && dv == 256); }

int attn_records(int n_seq, int n_head, int nt, bool prefix) {
    // the sharing rows' records: one per workgroup and group, shared blocks and own ones, of which each request with
    // tokens has at most one that is not full
    size_t n = SHARED_RECORDS;
    if (prefix) n += N_WG + 2 * shared_blocks(n_head, nt) + (size_t)(n_seq < nt ? n_seq : nt);
    return (int)n;
}

size_t attn_workspace_bytes(int dv, int n_seq, int n_head, int nt, bool prefix) {
    return records_off(n_head, nt) + (size_t)attn_records(n_seq, n_head, nt, prefix) * (dv == 512 ? record_bytes<512>() : record_bytes<256>());
}

template <int DK, int DV>
static hipError_t launch(bool q8, const AttnArgs & a, hipStream_t stream) {
    auto run = [&](void (*kernel)(AttnArgs)) { hipLaunchKernelGGL(kernel, dim3(N_WG), dim3(NTHR), 0, stream, a); };
    if (q8) run(a.q_f16 ? kqkv_paged_kernel<DK, DV, true, true> : kqkv_paged_kernel<DK, DV, true, false>);
    else run(a.q_f16 ? kqkv_paged_kernel<DK, DV, false, true> : kqkv_paged_kernel<DK, DV, false, false>);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int rows = a.n_head * a.nt;
    // The card starts some 400 workgroups per us, so as many as take part at once, no more; the fewer rows, the more
    // pieces each has.  Device times of whole calls either side of a limit, the smaller form first: 96 rows 19.2, 21.9 us
    // and 192 rows 38.7, 41.1; 384 rows 25.0, 29.6 and 1,536 44.7, 45.6, but 2,048 70.8, 68.6; 2,048 rows 69.5, 79.4,
    // 6,400 28.8, 28.9, 32,000 78.4, 77.2.  The rows that count are those there is room for, as the lengths are on the device:
    // few live rows of many pieces in a call with much room take the last form: 2 requests of 60,000 cells, 32 heads, 34.6
    // us in a call of 2 rows, 139 in one of 256; 256 requests of 200 cells 20.8.
    const auto wgs = [=](int r) { return dim3((rows + r - 1) / r, DV / 16); };
    if (rows <= 256) hipLaunchKernelGGL((kqkv_paged_merge_few_kernel<DV, 512, 8>), wgs(8), dim3(512), 0, stream, a);
    else if (rows <= 1536) hipLaunchKernelGGL((kqkv_paged_merge_few_kernel<DV, NTHR, 32>), wgs(32), dim3(NTHR), 0, stream, a);
    else if (rows <= 4096) hipLaunchKernelGGL((kqkv_paged_merge_kernel<DV, 1>), dim3(wgs(32).x, DV / 64), dim3(NTHR), 0, stream, a);
    else hipLaunchKernelGGL((kqkv_paged_merge_kernel<DV, 4>), dim3(wgs(32).x, DV / 256), dim3(NTHR), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_attn(int dk, int dv, bool q8, const AttnArgs & a, hipStream_t stream) {
    if (dk == 576 && dv == 512) return launch<576, 512>(q8, a, stream);
    if (dk == 320 && dv == 256) return launch<320, 256>(q8, a, stream);
    return hipErrorInvalidValue;
}

}  // namespace paged
}  // namespace mla
