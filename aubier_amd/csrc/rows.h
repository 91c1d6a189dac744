// rows.h -- launch interface of the row operators around a batch's attention (internal to the library): norms with
// gate and residual and int8 rows (row_ops.hip), the rope of q (row_ops.hip), the product of int8 rows and weights
// (mul_i8.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mla {
namespace rows {

constexpr int MAX_N = 32768;            // values of a row: a workgroup of 1,024 threads holds it in registers
constexpr int MAX_ROWS = 1 << 24;
constexpr int MAX_K = 131056;           // 128 * 128 * MAX_K < 2^31
constexpr int MAX_MUL = 1 << 22;        // rows and channels of a product
constexpr int64_t MAX_STRIDE = 1 << 22; // bytes between rows of a product's operands: 32-bit offsets inside a tile
constexpr int MAX_ROPE = 256;

enum { OUT_NONE = 0, OUT_F32 = 1, OUT_F16 = 2, OUT_I8 = 3 };

struct NormArgs {
    const char * x;         // row r's value c: x + r x_nb1 + (c / d) x_nbh + (c % d) elements
    int64_t x_nb1, x_nbh;
    int d, d_shift;         // values in a piece, and its binary logarithm or -1; d 0: rows of norm, in one piece
    int x_f16;
    const float * post;     // [n] or null
    const char * gate;      // one value for every channel (gate_wide), or one; rows gate_nb1 bytes apart (0: the same); or null
    int64_t gate_nb1;
    int gate_wide;
    const char * res;       // or null
    int64_t res_nb1;
    int res_f16;
    const float * pre;      // [n] or null
    int rms;                // the second norm (0: h = r, as rows_i8)
    float scale, eps;
    double per_n;           // 1 / n
    char * res_out;
    int64_t res_out_nb1;
    int res_out_type;       // OUT_*
    char * dst;
    int64_t dst_nb1;
    int dst_type;           // OUT_*
    float * dst_scale;
    int n, n_rows;
};
hipError_t launch_norm(const NormArgs & a, hipStream_t stream);

struct MulArgs {
    const char * w;
    int64_t w_nb1;
    const float * w_scale;
    const char * x;
    int64_t x_nb1;
    const float * x_scale;
    char * dst;
    int64_t dst_nb1;
    int dst_f16;
    int n, k, n_rows;
    char * work;            // mul_workspace_bytes, or null: k is not cut
};
size_t mul_workspace_bytes(int n, int k, int n_rows);
hipError_t launch_mul_i8(const MulArgs & a, hipStream_t stream);

struct QropeArgs {
    const char * q;         // row r, head h: q + r q_nb2 + h q_nb1
    int64_t q_nb1, q_nb2;
    int q_f16;
    const int32_t * pos;
    char * dst;
    int64_t dst_nb1, dst_nb2;
    int dst_f16;
    int n_rows, n_head, n_dims;
    float mscale;
    double turns[MAX_ROPE / 2];     // turns (of 2 pi) per position of every rope pair
};
hipError_t launch_qrope(const QropeArgs & a, hipStream_t stream);

}  // namespace rows
}  // namespace mla
