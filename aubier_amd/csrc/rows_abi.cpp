// rows_abi.cpp -- the C ABI of the row operators around a batch's attention (include/mla_m4.h): host-side contract
// checks and launches.  As in mla_m4_abi.cpp nothing here allocates, synchronises or reads device memory, so every
// entry point is legal inside hipGraph capture.
#include <hip/hip_runtime.h>

#include "abi_common.h"
#include "rows.h"

namespace {

using namespace mla::abi;
namespace rw = mla::rows;

bool is_float(const mla_m4_tensor * t) { return t->type == MLA_M4_TYPE_F32 || t->type == MLA_M4_TYPE_F16; }

// a matrix of n_rows rows of n values, packed inside a row, rows and base aligned to `align` bytes
int check_rows(const mla_m4_tensor * t, int64_t n, int64_t n_rows, size_t align) {
    if (t->ne[0] != n || t->ne[1] != n_rows || t->ne[2] != 1 || t->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    const size_t es = elsize(t->type);
    if ((n > 1 && t->nb[0] != es) || (reinterpret_cast<uintptr_t>(t->data) & (align - 1)) != 0) return MLA_M4_ERR_STRIDE;
    if (n_rows > 1 && ((t->nb[1] & (align - 1)) != 0 || t->nb[1] < (size_t)n * es || t->nb[1] > (size_t)INT64_MAX / (size_t)n_rows)) return MLA_M4_ERR_STRIDE;
    return MLA_M4_OK;
}

// rows of pieces, ne [d, H, rows], packed inside a piece, pieces and rows aligned to 4 elements; out: written to, so no
// two values lie in one place (one of the two orders of pieces and rows)
int check_pieces(const mla_m4_tensor * t, bool out) {
    if (t->ne[0] < 1 || t->ne[1] < 1 || t->ne[2] < 1 || t->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    const size_t es = elsize(t->type), align = 4 * es;
    const int64_t h = t->ne[1], r = t->ne[2];
    if ((t->ne[0] > 1 && t->nb[0] != es) || (reinterpret_cast<uintptr_t>(t->data) & (align - 1)) != 0) return MLA_M4_ERR_STRIDE;
    if ((h > 1 && ((t->nb[1] & (align - 1)) != 0 || t->nb[1] > (size_t)INT64_MAX / 2 / (size_t)h)) ||
        (r > 1 && ((t->nb[2] & (align - 1)) != 0 || t->nb[2] > (size_t)INT64_MAX / 2 / (size_t)r)))
        return MLA_M4_ERR_STRIDE;
    if (out) {
        const size_t piece = (size_t)t->ne[0] * es;
        const bool rows_outside = (h == 1 || t->nb[1] >= piece) && (r == 1 || t->nb[2] >= (h == 1 ? piece : (size_t)(h - 1) * t->nb[1] + piece));
        const bool pieces_outside = (r == 1 || t->nb[2] >= piece) && (h == 1 || t->nb[1] >= (r == 1 ? piece : (size_t)(r - 1) * t->nb[2] + piece));
        if (!rows_outside && !pieces_outside) return MLA_M4_ERR_STRIDE;
    }
    return MLA_M4_OK;
}

int check_weight(const mla_m4_tensor * t, int64_t n, bool plan) {
    const int rc = check_vec(t, MLA_M4_TYPE_F32, 4, n, plan);
    return rc == MLA_M4_OK && !al16(t->data, plan) ? MLA_M4_ERR_STRIDE : rc;
}

// ---------------------------------------------------------------- norms, gate and residual
int check_norm(const mla_m4_tensor * x, const mla_m4_tensor * post, const mla_m4_tensor * gate, const mla_m4_tensor * res,
               const mla_m4_tensor * pre, float eps, const mla_m4_tensor * res_out, const mla_m4_tensor * dst,
               const mla_m4_tensor * dst_scale, bool plan = false) {
    if (!has_data(x, plan) || (!res_out && !dst)) return MLA_M4_ERR_NULL;
    for (const mla_m4_tensor * t : {post, gate, res, pre, res_out, dst})
        if (t && !has_data(t, plan)) return MLA_M4_ERR_NULL;
    if (!is_float(x) || (res && !is_float(res)) || (res_out && !is_float(res_out)) ||
        (dst && !is_float(dst) && dst->type != MLA_M4_TYPE_I8) || (gate && gate->type != MLA_M4_TYPE_F32))
        return MLA_M4_ERR_TYPE;
    const int64_t n = x->ne[0], rows = x->ne[1];
    if (n < 4 || n % 4 || rows < 1) return MLA_M4_ERR_SHAPE;
    for (const mla_m4_tensor * t : {x, res, res_out, dst}) {
        if (!t) continue;
        const int rc = check_rows(t, n, rows, 4 * elsize(t->type));
        if (rc != MLA_M4_OK) return rc;
    }
    for (const mla_m4_tensor * t : {post, pre}) {
        if (!t) continue;
        const int rc = check_weight(t, n, plan);
        if (rc != MLA_M4_OK) return rc;
    }
    if (gate) {
        if ((gate->ne[0] != n && gate->ne[0] != 1) || (gate->ne[1] != rows && gate->ne[1] != 1) || gate->ne[2] != 1 || gate->ne[3] != 1)
            return MLA_M4_ERR_SHAPE;
        const int rc = check_rows(gate, gate->ne[0], gate->ne[1], gate->ne[0] == 1 ? 4 : 16);
        if (rc != MLA_M4_OK) return rc;
    }
    if (dst && dst->type == MLA_M4_TYPE_I8) {
        const int rc = check_vec(dst_scale, MLA_M4_TYPE_F32, 4, rows, plan);
        if (rc != MLA_M4_OK) return rc;
    } else if (dst_scale) {
        return MLA_M4_ERR_TYPE;                 // a scale that nothing is scaled by
    }
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return MLA_M4_ERR_ARG;
    if (n > rw::MAX_N || rows > rw::MAX_ROWS) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

int out_type(const mla_m4_tensor * t) {
    return !t ? rw::OUT_NONE : t->type == MLA_M4_TYPE_F32 ? rw::OUT_F32 : t->type == MLA_M4_TYPE_F16 ? rw::OUT_F16 : rw::OUT_I8;
}

// ---------------------------------------------------------------- int8 rows
// a matrix ne [d, rows] stands for ne [d, 1, rows]
mla_m4_tensor pieces(const mla_m4_tensor * t, int64_t n_rows) {
    mla_m4_tensor v = *t;
    if (t->ne[2] == 1 && t->ne[1] == n_rows) {
        v.ne[1] = 1;
        v.ne[2] = t->ne[1];
        v.nb[2] = t->nb[1];
        v.nb[1] = (size_t)t->ne[0] * elsize(t->type);
    }
    return v;
}

int check_rows_i8(const mla_m4_tensor * x, const mla_m4_tensor * dst, const mla_m4_tensor * scale, bool plan = false) {
    if (!has_data(x, plan) || !has_data(dst, plan)) return MLA_M4_ERR_NULL;
    if (!is_float(x) || dst->type != MLA_M4_TYPE_I8) return MLA_M4_ERR_TYPE;
    const mla_m4_tensor p = pieces(x, dst->ne[1]);
    if (p.ne[0] % 4) return MLA_M4_ERR_SHAPE;
    int rc = check_pieces(&p, false);
    if (rc != MLA_M4_OK) return rc;
    if (p.ne[0] > rw::MAX_N || p.ne[1] > rw::MAX_N || p.ne[0] * p.ne[1] > rw::MAX_N || p.ne[2] > rw::MAX_ROWS) return MLA_M4_ERR_UNSUPPORTED;
    rc = check_rows(dst, p.ne[0] * p.ne[1], p.ne[2], 4);
    return rc != MLA_M4_OK ? rc : check_vec(scale, MLA_M4_TYPE_F32, 4, p.ne[2], plan);
}

// ---------------------------------------------------------------- product
int check_mul(const mla_m4_tensor * w, const mla_m4_tensor * w_scale, const mla_m4_tensor * x, const mla_m4_tensor * x_scale,
              const mla_m4_tensor * dst, bool plan = false) {
    if (!has_data(w, plan) || !has_data(x, plan) || !has_data(dst, plan)) return MLA_M4_ERR_NULL;
    if (w->type != MLA_M4_TYPE_I8 || x->type != MLA_M4_TYPE_I8 || !is_float(dst)) return MLA_M4_ERR_TYPE;
    const int64_t k = w->ne[0], n = w->ne[1], rows = x->ne[1];
    if (k < 16 || k % 16 || n < 1 || rows < 1) return MLA_M4_ERR_SHAPE;
    int rc = check_rows(w, k, n, 16);
    if (rc == MLA_M4_OK) rc = check_rows(x, k, rows, 16);
    if (rc == MLA_M4_OK) rc = check_rows(dst, n, rows, elsize(dst->type));
    if (rc == MLA_M4_OK) rc = check_vec(w_scale, MLA_M4_TYPE_F32, 4, n, plan);
    if (rc == MLA_M4_OK) rc = check_vec(x_scale, MLA_M4_TYPE_F32, 4, rows, plan);
    if (rc != MLA_M4_OK) return rc;
    if (k > rw::MAX_K || n > rw::MAX_MUL || rows > rw::MAX_MUL) return MLA_M4_ERR_UNSUPPORTED;
    if ((n > 1 && w->nb[1] > (size_t)rw::MAX_STRIDE) || (rows > 1 && x->nb[1] > (size_t)rw::MAX_STRIDE)) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

// ---------------------------------------------------------------- rope of q
int check_qrope(const mla_m4_tensor * q, const mla_m4_tensor * pos, const mla_m4_rope_params * rp, const mla_m4_tensor * dst,
                bool plan = false) {
    if (!has_data(q, plan) || !has_data(dst, plan) || !rp) return MLA_M4_ERR_NULL;
    if (!is_float(q) || !is_float(dst)) return MLA_M4_ERR_TYPE;
    if (rp->n_dims < 32 || rp->n_dims % 32 || q->ne[0] != rp->n_dims) return MLA_M4_ERR_SHAPE;
    for (int i = 0; i < 4; ++i)
        if (dst->ne[i] != q->ne[i]) return MLA_M4_ERR_SHAPE;
    int rc = check_pieces(q, false);
    if (rc == MLA_M4_OK) rc = check_pieces(dst, true);
    if (rc == MLA_M4_OK) rc = check_vec(pos, MLA_M4_TYPE_I32, 4, q->ne[2], plan);
    if (rc != MLA_M4_OK) return rc;
    if (!rope_in_range(rp)) return MLA_M4_ERR_ARG;
    if (rp->n_dims > rw::MAX_ROPE || q->ne[1] > 1024 || q->ne[2] > rw::MAX_MUL) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

int launched(hipError_t e) { return e == hipSuccess ? MLA_M4_OK : MLA_M4_ERR_LAUNCH; }

}  // namespace

extern "C" {

int mla_m4_norm(const mla_m4_tensor * x, const mla_m4_tensor * post, const mla_m4_tensor * gate, const mla_m4_tensor * res,
                float scale, const mla_m4_tensor * pre, float eps, const mla_m4_tensor * res_out, const mla_m4_tensor * dst,
                const mla_m4_tensor * dst_scale, void * stream) {
    const int rc = check_norm(x, post, gate, res, pre, eps, res_out, dst, dst_scale);
    if (rc != MLA_M4_OK) return rc;
    rw::NormArgs a{};
    a.x = static_cast<const char *>(x->data);
    a.x_nb1 = (int64_t)x->nb[1];
    a.x_f16 = x->type == MLA_M4_TYPE_F16;
    a.post = post ? static_cast<const float *>(post->data) : nullptr;
    if (gate) {
        a.gate = static_cast<const char *>(gate->data);
        a.gate_nb1 = gate->ne[1] > 1 ? (int64_t)gate->nb[1] : 0;
        a.gate_wide = gate->ne[0] > 1;
    }
    if (res) {
        a.res = static_cast<const char *>(res->data);
        a.res_nb1 = (int64_t)res->nb[1];
        a.res_f16 = res->type == MLA_M4_TYPE_F16;
    }
    a.scale = scale;
    a.pre = pre ? static_cast<const float *>(pre->data) : nullptr;
    a.rms = pre != nullptr;
    a.eps = eps;
    if (res_out) {
        a.res_out = static_cast<char *>(res_out->data);
        a.res_out_nb1 = (int64_t)res_out->nb[1];
    }
    a.res_out_type = out_type(res_out);
    if (dst) {
        a.dst = static_cast<char *>(dst->data);
        a.dst_nb1 = (int64_t)dst->nb[1];
    }
    a.dst_type = out_type(dst);
    a.dst_scale = dst_scale ? static_cast<float *>(dst_scale->data) : nullptr;
    a.n = (int)x->ne[0];
    a.per_n = 1.0 / (double)a.n;
    a.n_rows = (int)x->ne[1];
    return launched(rw::launch_norm(a, static_cast<hipStream_t>(stream)));
}

int mla_m4_supports_norm(const mla_m4_tensor * x, const mla_m4_tensor * post, const mla_m4_tensor * gate,
                         const mla_m4_tensor * res, const mla_m4_tensor * pre, float eps, const mla_m4_tensor * res_out,
                         const mla_m4_tensor * dst, const mla_m4_tensor * dst_scale) {
    return check_norm(x, post, gate, res, pre, eps, res_out, dst, dst_scale, true) == MLA_M4_OK;
}

int mla_m4_rows_i8(const mla_m4_tensor * x, const mla_m4_tensor * dst, const mla_m4_tensor * scale, void * stream) {
    const int rc = check_rows_i8(x, dst, scale);
    if (rc != MLA_M4_OK) return rc;
    const mla_m4_tensor p = pieces(x, dst->ne[1]);
    rw::NormArgs a{};
    a.x = static_cast<const char *>(p.data);
    a.x_nb1 = (int64_t)p.nb[2];
    a.x_nbh = p.ne[1] > 1 ? (int64_t)p.nb[1] : 0;
    a.d = (int)p.ne[0];
    a.d_shift = -1;
    for (int i = 2; i < 16; ++i)
        if (p.ne[0] == (int64_t)1 << i) a.d_shift = i;
    if (p.ne[1] == 1) a.d_shift = 31;                   // one piece
    a.x_f16 = p.type == MLA_M4_TYPE_F16;
    a.dst = static_cast<char *>(dst->data);
    a.dst_nb1 = (int64_t)dst->nb[1];
    a.dst_type = rw::OUT_I8;
    a.dst_scale = static_cast<float *>(scale->data);
    a.n = (int)(p.ne[0] * p.ne[1]);
    a.n_rows = (int)p.ne[2];
    return launched(rw::launch_norm(a, static_cast<hipStream_t>(stream)));
}

int mla_m4_supports_rows_i8(const mla_m4_tensor * x, const mla_m4_tensor * dst, const mla_m4_tensor * scale) {
    return check_rows_i8(x, dst, scale, true) == MLA_M4_OK;
}

size_t mla_m4_mul_i8_workspace_bytes(const mla_m4_tensor * w, const mla_m4_tensor * x) {
    if (!w || !x || w->ne[0] < 16 || w->ne[0] > rw::MAX_K || w->ne[1] < 1 || w->ne[1] > rw::MAX_MUL || x->ne[1] < 1 || x->ne[1] > rw::MAX_MUL) return 0;
    return rw::mul_workspace_bytes((int)w->ne[1], (int)w->ne[0], (int)x->ne[1]);
}

int mla_m4_mul_i8(const mla_m4_tensor * w, const mla_m4_tensor * w_scale, const mla_m4_tensor * x, const mla_m4_tensor * x_scale,
                  const mla_m4_tensor * dst, void * workspace, size_t workspace_bytes, void * stream) {
    const int rc = check_mul(w, w_scale, x, x_scale, dst);
    if (rc != MLA_M4_OK) return rc;
    if (workspace && (!aligned16(workspace) || workspace_bytes < mla_m4_mul_i8_workspace_bytes(w, x))) return MLA_M4_ERR_WORKSPACE;
    rw::MulArgs a{};
    a.work = static_cast<char *>(workspace);
    a.w = static_cast<const char *>(w->data);
    a.w_nb1 = w->ne[1] > 1 ? (int64_t)w->nb[1] : 0;
    a.w_scale = static_cast<const float *>(w_scale->data);
    a.x = static_cast<const char *>(x->data);
    a.x_nb1 = x->ne[1] > 1 ? (int64_t)x->nb[1] : 0;
    a.x_scale = static_cast<const float *>(x_scale->data);
    a.dst = static_cast<char *>(dst->data);
    a.dst_nb1 = (int64_t)dst->nb[1];
    a.dst_f16 = dst->type == MLA_M4_TYPE_F16;
    a.n = (int)w->ne[1];
    a.k = (int)w->ne[0];
    a.n_rows = (int)x->ne[1];
    return launched(rw::launch_mul_i8(a, static_cast<hipStream_t>(stream)));
}

int mla_m4_supports_mul_i8(const mla_m4_tensor * w, const mla_m4_tensor * w_scale, const mla_m4_tensor * x,
                           const mla_m4_tensor * x_scale, const mla_m4_tensor * dst) {
    return check_mul(w, w_scale, x, x_scale, dst, true) == MLA_M4_OK;
}

int mla_m4_qrope(const mla_m4_tensor * q, const mla_m4_tensor * pos, const mla_m4_rope_params * rope, const mla_m4_tensor * dst,
                 void * stream) {
    const int rc = check_qrope(q, pos, rope, dst);
    if (rc != MLA_M4_OK) return rc;
    rw::QropeArgs a{};
    a.q = static_cast<const char *>(q->data);
    a.q_nb1 = (int64_t)q->nb[1];
    a.q_nb2 = (int64_t)q->nb[2];
    a.q_f16 = q->type == MLA_M4_TYPE_F16;
    a.pos = static_cast<const int32_t *>(pos->data);
    a.dst = static_cast<char *>(dst->data);
    a.dst_nb1 = (int64_t)dst->nb[1];
    a.dst_nb2 = (int64_t)dst->nb[2];
    a.dst_f16 = dst->type == MLA_M4_TYPE_F16;
    a.n_rows = (int)q->ne[2];
    a.n_head = (int)q->ne[1];
    a.n_dims = (int)q->ne[0];
    a.mscale = rope_mscale(rope);
    rope_turns(rope, a.turns);
    return launched(rw::launch_qrope(a, static_cast<hipStream_t>(stream)));
}

int mla_m4_supports_qrope(const mla_m4_tensor * q, const mla_m4_tensor * pos, const mla_m4_rope_params * rope,
                          const mla_m4_tensor * dst) {
    return check_qrope(q, pos, rope, dst, true) == MLA_M4_OK;
}

}  // extern "C"
