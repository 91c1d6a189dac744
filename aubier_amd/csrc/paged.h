// paged.h -- launch interface of the paged-batch kernels (internal to the library): the page bookkeeping and
// the batched KV rows of paged_ops.hip, the attention over pages of kqkv_paged.hip.
//
// A batch is n_seq requests; request b holds past[b] cells and adds n_new[b] tokens, whose rows (tokens) follow
// one another: request b's first row is sum_{a < b} n_new[a].  Cell j of request b is cell
// table[b][j / page] * page + j % page of the pool.  Every length and index lives on the device, so the kernels
// bring it into range themselves before use: negative lengths count as 0, rows past the batch's are not there,
// and an id that is no page of the pool has no cells.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mla {
namespace paged {

constexpr int MAX_SEQS = 4096;      // requests per call: their prefix sums are held in LDS
constexpr int MAX_ROWS = 65535;     // tokens per call (sums over all requests stay far inside 32 bits)
constexpr int MAX_PAST = 1 << 30;

struct PagesArgs {
    const int32_t * past;
    const int32_t * n_new;
    const int32_t * free_ids;
    int32_t * table;
    int64_t t_nb1;          // bytes between the tables of two requests
    int64_t * slot;         // [n_rows]
    int32_t * pos;          // [n_rows]
    int32_t * used;         // [2]: pages taken, rows of the batch
    int n_seq, n_free, max_pages, page_shift, n_rows;
};
hipError_t launch_pages(const PagesArgs & a, hipStream_t stream);

constexpr int MAX_ROPE = 256;       // rope columns of a row
constexpr int MAX_KV_ROWS = 1 << 24;  // a wavefront each: the grid's threads stay below 2^32
struct KvRowsArgs {
    const void * x;         // rows of n_out values, f32 or f16
    int64_t x_nb1;
    int x_f16;
    const float * nw;       // [d_lat]
    char * kc;              // f16 rows, or block_q8_0 rows (kc_q8), kc_nb1 bytes apart
    int64_t kc_nb1;
    int kc_q8;
    int64_t n_cells;
    const int64_t * slot;
    const int32_t * pos;
    char * dst;             // f32 rows dst_nb1 bytes apart, or null
    int64_t dst_nb1;
    int n_rows, d_lat, n_rope;
    float eps, mscale;
    double turns[MAX_ROPE / 2];     // turns (of 2 pi) per position of every rope pair
};
hipError_t launch_kvrows(const KvRowsArgs & a, hipStream_t stream);

struct AttnArgs {
    const char * kc;
    int64_t kc_nb1;
    const char * q;         // rows' heads: q + token * q_nb2 + head * q_nb1
    int64_t q_nb1, q_nb2;
    const int32_t * past;
    const int32_t * n_new;
    const int32_t * table;
    int64_t t_nb1;
    const int32_t * prefix; // [2]: cells, requests; or null
    char * dst;             // [H][nt][D_v]
    char * work;
    float scale_log2;
    int n_seq, max_pages, n_pages, page_shift, n_head, nt;
    int q_f16, dst_f16;
    int n_records;          // what the workspace holds
};
bool attn_supported(int dk, int dv);
int attn_records(int n_seq, int n_head, int nt, bool prefix);
size_t attn_workspace_bytes(int dv, int n_seq, int n_head, int nt, bool prefix);
// n_head^2 nt and the cells that a table lists: the line of work (kqkv_paged.hip), in units of a tenth of a tile's cost by
// n_head, is at most 10 / 8192 of it long and 2^49 for the requests' last blocks, so it stays below 2^51
constexpr double MAX_LINE = 1152921504606846976.0;      // 2^60
constexpr int64_t MAX_STRIDE = 1 << 25;   // bytes between rows of the cache: 32-bit offsets inside a tile
constexpr int64_t Q_SPAN = 1u << 31;      // 128 rows of q span at most this: 127 q_nb2 + n_head q_nb1
hipError_t launch_attn(int dk, int dv, bool q8, const AttnArgs & a, hipStream_t stream);

}  // namespace paged
}  // namespace mla
