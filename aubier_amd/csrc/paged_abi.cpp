// paged_abi.cpp -- the C ABI of the paged-batch operators (include/mla_m4.h, "Paged batches"): host-side
// contract checks and launches.  As in mla_m4_abi.cpp nothing here allocates, synchronises or reads device
// memory, so every entry point is legal inside hipGraph capture.
#include <hip/hip_runtime.h>

#include "abi_common.h"
#include "paged.h"

namespace {

using namespace mla::abi;
namespace pg = mla::paged;

// a vector: ne [n], packed
int check_vec(const mla_m4_tensor * t, int32_t type, size_t es, int64_t n, bool plan) {
    if (!has_data(t, plan)) return MLA_M4_ERR_NULL;
    if (t->type != type) return MLA_M4_ERR_TYPE;
    if (t->ne[0] != n || t->ne[1] != 1 || t->ne[2] != 1 || t->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    if ((n != 1 && t->nb[0] != es) || (reinterpret_cast<uintptr_t>(t->data) & (es - 1))) return MLA_M4_ERR_STRIDE;
    return MLA_M4_OK;
}

// the lengths of a batch, its block tables and page size
int check_batch(const mla_m4_tensor * past, const mla_m4_tensor * n_new, const mla_m4_tensor * table, int32_t page_size,
                bool plan) {
    if (!has_data(past, plan) || !has_data(table, plan)) return MLA_M4_ERR_NULL;
    const int64_t n_seq = past->ne[0];
    if (n_seq < 1) return MLA_M4_ERR_SHAPE;
    int rc = check_vec(past, MLA_M4_TYPE_I32, 4, n_seq, plan);
    if (rc == MLA_M4_OK) rc = check_vec(n_new, MLA_M4_TYPE_I32, 4, n_seq, plan);
    if (rc != MLA_M4_OK) return rc;
    if (table->type != MLA_M4_TYPE_I32) return MLA_M4_ERR_TYPE;
    if (table->ne[0] < 1 || table->ne[1] != n_seq || table->ne[2] != 1 || table->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    if ((table->ne[0] != 1 && table->nb[0] != 4) || (table->nb[1] & 3u) ||
        (n_seq > 1 && table->nb[1] < (size_t)table->ne[0] * 4) || !al4(table->data, plan))
        return MLA_M4_ERR_STRIDE;
    if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)) != 0) return MLA_M4_ERR_ARG;
    if (n_seq > pg::MAX_SEQS || table->ne[0] > pg::MAX_PAST / page_size) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

int shift_of(int32_t page_size) { return __builtin_ctz((unsigned)page_size); }

// ---------------------------------------------------------------- pages
int check_pages(const mla_m4_tensor * past, const mla_m4_tensor * n_new, const mla_m4_tensor * free_ids,
                const mla_m4_tensor * table, int32_t page_size, const mla_m4_tensor * slot, const mla_m4_tensor * pos,
                const mla_m4_tensor * used, bool plan = false) {
    if (!free_ids || !slot || !pos || !used) return MLA_M4_ERR_NULL;
    int rc = check_batch(past, n_new, table, page_size, plan);
    if (rc != MLA_M4_OK) return rc;
    if (free_ids->ne[0] < 0 || slot->ne[0] < 1) return MLA_M4_ERR_SHAPE;
    // an empty free list needs no data
    if (free_ids->ne[0] > 0) rc = check_vec(free_ids, MLA_M4_TYPE_I32, 4, free_ids->ne[0], plan);
    else if (free_ids->type != MLA_M4_TYPE_I32) rc = MLA_M4_ERR_TYPE;
    if (rc == MLA_M4_OK) rc = check_vec(slot, MLA_M4_TYPE_I64, 8, slot->ne[0], plan);
    if (rc == MLA_M4_OK) rc = check_vec(pos, MLA_M4_TYPE_I32, 4, slot->ne[0], plan);
    if (rc == MLA_M4_OK) rc = check_vec(used, MLA_M4_TYPE_I32, 4, 2, plan);
    if (rc != MLA_M4_OK) return rc;
    if (slot->ne[0] > pg::MAX_ROWS || free_ids->ne[0] > INT32_MAX) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

// ---------------------------------------------------------------- batched KV rows
int check_kvrows(const mla_m4_tensor * x, const mla_m4_tensor * nw, const mla_m4_tensor * kc, const mla_m4_tensor * slot,
                 const mla_m4_tensor * pos, const mla_m4_rope_params * rp, const mla_m4_tensor * dst, bool plan = false) {
    if (!has_data(x, plan) || !has_data(nw, plan) || !has_data(kc, plan) || !rp) return MLA_M4_ERR_NULL;
    if ((x->type != MLA_M4_TYPE_F32 && x->type != MLA_M4_TYPE_F16) || nw->type != MLA_M4_TYPE_F32 ||
        (kc->type != MLA_M4_TYPE_F16 && kc->type != MLA_M4_TYPE_Q8_0))
        return MLA_M4_ERR_TYPE;
    const int64_t n_out = x->ne[0], n_rows = x->ne[1], n_dims = rp->n_dims, d_lat = n_out - n_dims;
    if (n_rows < 1 || x->ne[2] != 1 || x->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    if (n_dims < 32 || n_dims % 32 || d_lat < 32 || d_lat % 32) return MLA_M4_ERR_SHAPE;
    if (kc->ne[0] != n_out || kc->ne[1] < 1 || kc->ne[2] != 1 || kc->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    const size_t es = elsize(x->type);
    if (x->nb[0] != es || (x->nb[1] & (4 * es - 1)) || (n_rows > 1 && x->nb[1] < (size_t)n_out * es) ||
        (reinterpret_cast<uintptr_t>(x->data) & (4 * es - 1)))
        return MLA_M4_ERR_STRIDE;
    int rc = check_vec(nw, MLA_M4_TYPE_F32, 4, d_lat, plan);
    if (rc == MLA_M4_OK && !al16(nw->data, plan)) rc = MLA_M4_ERR_STRIDE;
    if (rc == MLA_M4_OK) rc = check_vec(slot, MLA_M4_TYPE_I64, 8, n_rows, plan);
    if (rc == MLA_M4_OK) rc = check_vec(pos, MLA_M4_TYPE_I32, 4, n_rows, plan);
    if (rc != MLA_M4_OK) return rc;
    if (kc->type == MLA_M4_TYPE_F16) {
        if (kc->nb[0] != 2 || (kc->nb[1] & 7u) || (kc->ne[1] > 1 && kc->nb[1] < (size_t)n_out * 2) ||
            (reinterpret_cast<uintptr_t>(kc->data) & 7u))
            return MLA_M4_ERR_STRIDE;
    } else if (kc->nb[0] != Q8_BLOCK || (kc->nb[1] & 1u) || (kc->ne[1] > 1 && kc->nb[1] < (size_t)(n_out / 32) * Q8_BLOCK) ||
               (reinterpret_cast<uintptr_t>(kc->data) & 1u)) {
        return MLA_M4_ERR_STRIDE;
    }
    if (dst) {
        if (!has_data(dst, plan)) return MLA_M4_ERR_NULL;
        if (dst->type != MLA_M4_TYPE_F32) return MLA_M4_ERR_TYPE;
        if (dst->ne[0] != n_out || dst->ne[1] != n_rows || dst->ne[2] != 1 || dst->ne[3] != 1) return MLA_M4_ERR_SHAPE;
        if (dst->nb[0] != 4 || (dst->nb[1] & 15u) || (n_rows > 1 && dst->nb[1] < (size_t)n_out * 4) || !al16(dst->data, plan))
            return MLA_M4_ERR_STRIDE;
    }
    if (!(rp->freq_base > 0.0f) || !(rp->freq_scale > 0.0f) || !(rp->eps >= 0.0f) || rp->n_ctx_orig < 1 ||
        !std::isfinite(rp->freq_base) || !std::isfinite(rp->freq_scale) || !std::isfinite(rp->eps) ||
        !std::isfinite(rp->ext_factor) || !std::isfinite(rp->attn_factor) || !(rp->beta_fast > 0.0f) || !(rp->beta_slow > 0.0f))
        return MLA_M4_ERR_ARG;
    if (n_out > 1024 || n_dims > pg::MAX_ROPE || n_rows > pg::MAX_KV_ROWS) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

// Turns (of 2 pi) per position of every rope pair, taken in 64 bits: the frequency
// freq_base^(-2 p / n_dims) times freq_scale (1 - mix) + mix (YaRN's ramp, which is linear in the angle).
void rope_turns(const mla_m4_rope_params * rp, double * turns) {
    float corr[2] = {0.0f, 0.0f};
    if (rp->ext_factor != 0.0f) rope_yarn_corr_dims(rp->n_dims, rp->n_ctx_orig, rp->freq_base, rp->beta_fast, rp->beta_slow, corr);
    const double width = (double)corr[1] - (double)corr[0];
    const double step = -2.0 / (double)rp->n_dims * std::log((double)rp->freq_base);
    for (int p = 0; 2 * p < rp->n_dims; ++p) {
        double y = ((double)p - (double)corr[0]) / (width > 0.001 ? width : 0.001);
        y = y < 0.0 ? 0.0 : y > 1.0 ? 1.0 : y;
        const double mix = (1.0 - y) * (double)rp->ext_factor;
        turns[p] = std::exp(step * p) * ((double)rp->freq_scale * (1.0 - mix) + mix) / 6.283185307179586476925;
    }
}

// ---------------------------------------------------------------- attention over pages
int check_attn(const mla_m4_tensor * kc, const mla_m4_tensor * q, const mla_m4_tensor * past, const mla_m4_tensor * n_new,
               const mla_m4_tensor * table, int32_t page_size, const mla_m4_tensor * prefix, const mla_m4_tensor * dst,
               bool plan = false) {
    if (!has_data(kc, plan) || !has_data(q, plan) || !has_data(dst, plan)) return MLA_M4_ERR_NULL;
    const bool q8 = kc->type == MLA_M4_TYPE_Q8_0;
    if ((kc->type != MLA_M4_TYPE_F16 && !q8) || (q->type != MLA_M4_TYPE_F32 && q->type != MLA_M4_TYPE_F16) ||
        (dst->type != MLA_M4_TYPE_F32 && dst->type != MLA_M4_TYPE_F16))
        return MLA_M4_ERR_TYPE;
    if (kc->ne[0] < 1 || kc->ne[1] < 1 || kc->ne[2] != 1 || kc->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    if (q8) {
        if (kc->ne[0] % 32) return MLA_M4_ERR_SHAPE;
        if (!is_q8_rows(kc) || !al16(kc->data, plan)) return MLA_M4_ERR_STRIDE;
    } else if (kc->nb[0] != 2 || (kc->nb[1] & 15u) || (kc->ne[1] > 1 && kc->nb[1] < (size_t)kc->ne[0] * 2) || !al16(kc->data, plan)) {
        return MLA_M4_ERR_STRIDE;
    }
    if (q->ne[0] != kc->ne[0] || q->ne[1] < 1 || q->ne[2] < 1 || q->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    const size_t es = elsize(q->type);
    if (q->nb[0] != es || (q->nb[1] & 15u) || (q->nb[2] & 15u) || !al16(q->data, plan) ||
        (q->ne[1] > 1 && q->nb[1] < (size_t)q->ne[0] * es))
        return MLA_M4_ERR_STRIDE;
    if (dst->ne[0] < 1 || dst->ne[0] > kc->ne[0] || dst->ne[1] != q->ne[2] || dst->ne[2] != q->ne[1] || dst->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    if (!is_contiguous(dst) || !al16(dst->data, plan)) return MLA_M4_ERR_STRIDE;
    int rc = check_batch(past, n_new, table, page_size, plan);
    if (rc == MLA_M4_OK && prefix && (prefix->data || plan)) rc = check_vec(prefix, MLA_M4_TYPE_I32, 4, 2, plan);
    if (rc != MLA_M4_OK) return rc;
    if (kc->ne[1] < page_size) return MLA_M4_ERR_SHAPE;         // not one page
    if (!pg::attn_supported((int)(kc->ne[0] > 4096 ? 0 : kc->ne[0]), (int)(dst->ne[0] > 4096 ? 0 : dst->ne[0]))) return MLA_M4_ERR_UNSUPPORTED;
    if (q->ne[1] > 1024 || q->ne[2] > pg::MAX_ROWS || kc->ne[1] / page_size > INT32_MAX) return MLA_M4_ERR_UNSUPPORTED;
    if (kc->nb[1] > pg::MAX_STRIDE || q->nb[1] > pg::Q_SPAN || q->nb[2] > pg::Q_SPAN) return MLA_M4_ERR_UNSUPPORTED;
    // 128 rows, to the end of the last one (of a single head nb[1] says nothing about a row's length)
    const int64_t row_end = q->ne[1] > 1 ? q->ne[1] * (int64_t)q->nb[1] : q->ne[0] * (int64_t)es;
    if (127 * (int64_t)q->nb[2] + row_end > pg::Q_SPAN) return MLA_M4_ERR_UNSUPPORTED;
    if ((double)(q->ne[1] * q->ne[1] * q->ne[2]) * ((double)table->ne[0] * page_size) > pg::MAX_LINE) return MLA_M4_ERR_UNSUPPORTED;
    return MLA_M4_OK;
}

}  // namespace

extern "C" {

int mla_m4_pages(const mla_m4_tensor * past, const mla_m4_tensor * n_new, const mla_m4_tensor * free_ids,
                 const mla_m4_tensor * table, int32_t page_size, const mla_m4_tensor * slot, const mla_m4_tensor * pos,
                 const mla_m4_tensor * used, void * stream) {
    const int rc = check_pages(past, n_new, free_ids, table, page_size, slot, pos, used);
    if (rc != MLA_M4_OK) return rc;
    pg::PagesArgs a{};
    a.past = static_cast<const int32_t *>(past->data);
    a.n_new = static_cast<const int32_t *>(n_new->data);
    a.free_ids = static_cast<const int32_t *>(free_ids->data);
    a.table = static_cast<int32_t *>(table->data);
    a.t_nb1 = (int64_t)table->nb[1];
    a.slot = static_cast<int64_t *>(slot->data);
    a.pos = static_cast<int32_t *>(pos->data);
    a.used = static_cast<int32_t *>(used->data);
    a.n_seq = (int)past->ne[0];
    a.n_free = (int)free_ids->ne[0];
    a.max_pages = (int)table->ne[0];
    a.page_shift = shift_of(page_size);
    a.n_rows = (int)slot->ne[0];
    return pg::launch_pages(a, static_cast<hipStream_t>(stream)) == hipSuccess ? MLA_M4_OK : MLA_M4_ERR_LAUNCH;
}

int mla_m4_supports_pages(const mla_m4_tensor * past, const mla_m4_tensor * n_new, const mla_m4_tensor * free_ids,
                          const mla_m4_tensor * table, int32_t page_size, const mla_m4_tensor * slot,
                          const mla_m4_tensor * pos, const mla_m4_tensor * used) {
    return check_pages(past, n_new, free_ids, table, page_size, slot, pos, used, true) == MLA_M4_OK;
}

int mla_m4_kvrows(const mla_m4_tensor * x, const mla_m4_tensor * kv_norm, const mla_m4_tensor * kcache,
                  const mla_m4_tensor * slot, const mla_m4_tensor * pos, const mla_m4_rope_params * rope,
                  const mla_m4_tensor * dst, void * stream) {
    const int rc = check_kvrows(x, kv_norm, kcache, slot, pos, rope, dst);
    if (rc != MLA_M4_OK) return rc;
    pg::KvRowsArgs a{};
    a.x = x->data;
    a.x_nb1 = (int64_t)x->nb[1];
    a.x_f16 = x->type == MLA_M4_TYPE_F16;
    a.nw = static_cast<const float *>(kv_norm->data);
    a.kc = static_cast<char *>(kcache->data);
    a.kc_nb1 = (int64_t)kcache->nb[1];
    a.kc_q8 = kcache->type == MLA_M4_TYPE_Q8_0;
    a.n_cells = kcache->ne[1];
    a.slot = static_cast<const int64_t *>(slot->data);
    a.pos = static_cast<const int32_t *>(pos->data);
    a.dst = dst ? static_cast<char *>(dst->data) : nullptr;
    a.dst_nb1 = dst ? (int64_t)dst->nb[1] : 0;
    a.n_rows = (int)x->ne[1];
    a.n_rope = rope->n_dims;
    a.d_lat = (int)x->ne[0] - rope->n_dims;
    a.eps = rope->eps;
    a.mscale = rope->attn_factor;
    if (rope->ext_factor != 0.0f) a.mscale *= 1.0f + 0.1f * logf(1.0f / rope->freq_scale);
    rope_turns(rope, a.turns);
    return pg::launch_kvrows(a, static_cast<hipStream_t>(stream)) == hipSuccess ? MLA_M4_OK : MLA_M4_ERR_LAUNCH;
}

int mla_m4_supports_kvrows(const mla_m4_tensor * x, const mla_m4_tensor * kv_norm, const mla_m4_tensor * kcache,
                           const mla_m4_tensor * slot, const mla_m4_tensor * pos, const mla_m4_rope_params * rope,
                           const mla_m4_tensor * dst) {
    return check_kvrows(x, kv_norm, kcache, slot, pos, rope, dst, true) == MLA_M4_OK;
}

size_t mla_m4_kqkv_paged_workspace_bytes(const mla_m4_tensor * kcache, const mla_m4_tensor * q, const mla_m4_tensor * past,
                                         const mla_m4_tensor * prefix, const mla_m4_tensor * dst) {
    if (!kcache || !q || !past || !dst || q->ne[1] < 1 || q->ne[1] > 1024 || q->ne[2] < 1 || q->ne[2] > pg::MAX_ROWS ||
        past->ne[0] < 1 || past->ne[0] > pg::MAX_SEQS || kcache->ne[0] > 4096 || dst->ne[0] > 4096 ||
        !pg::attn_supported((int)kcache->ne[0], (int)dst->ne[0]))
        return 0;
    // (a prefix that is not allocated yet counts: a planner asks before it allocates)
    return pg::attn_workspace_bytes((int)dst->ne[0], (int)past->ne[0], (int)q->ne[1], (int)q->ne[2], prefix != nullptr);
}

int mla_m4_kqkv_paged(const mla_m4_tensor * kcache, const mla_m4_tensor * q, const mla_m4_tensor * past,
                      const mla_m4_tensor * n_new, const mla_m4_tensor * table, int32_t page_size,
                      const mla_m4_tensor * prefix, float kq_scale, const mla_m4_tensor * dst, void * workspace,
                      size_t workspace_bytes, void * stream) {
    const int rc = check_attn(kcache, q, past, n_new, table, page_size, prefix, dst);
    if (rc != MLA_M4_OK) return rc;
    if (!std::isfinite(kq_scale)) return MLA_M4_ERR_ARG;
    if (prefix && !prefix->data) prefix = nullptr;
    const size_t need = mla_m4_kqkv_paged_workspace_bytes(kcache, q, past, prefix, dst);
    if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return MLA_M4_ERR_WORKSPACE;
    pg::AttnArgs a{};
    a.kc = static_cast<const char *>(kcache->data);
    a.kc_nb1 = (int64_t)kcache->nb[1];
    a.n_pages = (int)(kcache->ne[1] / page_size);
    a.q = static_cast<const char *>(q->data);
    a.q_nb1 = (int64_t)q->nb[1];
    a.q_nb2 = (int64_t)q->nb[2];
    a.past = static_cast<const int32_t *>(past->data);
    a.n_new = static_cast<const int32_t *>(n_new->data);
    a.table = static_cast<const int32_t *>(table->data);
    a.t_nb1 = (int64_t)table->nb[1];
    a.prefix = prefix ? static_cast<const int32_t *>(prefix->data) : nullptr;
    a.dst = static_cast<char *>(dst->data);
    a.work = static_cast<char *>(workspace);
    a.scale_log2 = kq_scale * 1.4426950408889634f;
    a.n_seq = (int)past->ne[0];
    a.max_pages = (int)table->ne[0];
    a.page_shift = shift_of(page_size);
    a.n_head = (int)q->ne[1];
    a.nt = (int)q->ne[2];
    a.q_f16 = q->type == MLA_M4_TYPE_F16;
    a.dst_f16 = dst->type == MLA_M4_TYPE_F16;
    a.n_records = pg::attn_records(a.n_seq, a.n_head, a.nt, a.prefix != nullptr);
    return pg::launch_attn((int)kcache->ne[0], (int)dst->ne[0], kcache->type == MLA_M4_TYPE_Q8_0, a,
                           static_cast<hipStream_t>(stream)) == hipSuccess ? MLA_M4_OK : MLA_M4_ERR_LAUNCH;
}

int mla_m4_supports_kqkv_paged(const mla_m4_tensor * kcache, const mla_m4_tensor * q, const mla_m4_tensor * past,
                               const mla_m4_tensor * n_new, const mla_m4_tensor * table, int32_t page_size,
                               const mla_m4_tensor * prefix, const mla_m4_tensor * dst) {
    return check_attn(kcache, q, past, n_new, table, page_size, prefix, dst, true) == MLA_M4_OK;
}

}  // extern "C"
