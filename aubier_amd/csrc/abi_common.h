// abi_common.h -- host-side helpers shared by the C ABI's contract checks.
#pragma once

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "../../include/mla_m4.h"

namespace mla {
namespace abi {

inline bool aligned16(const void * p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline size_t elsize(int32_t type) {
    switch (type) {
        case MLA_M4_TYPE_F32: return 4;
        case MLA_M4_TYPE_F16: return 2;
        case MLA_M4_TYPE_I8: return 1;
        default: return 0;
    }
}

inline bool is_contiguous(const mla_m4_tensor * t) {
    const size_t es = elsize(t->type);
    if (es == 0) return false;
    size_t expect = es;
    for (int i = 0; i < 4; ++i) {
        if (t->ne[i] != 1 && t->nb[i] != expect) return false;
        expect *= (size_t)t->ne[i];
    }
    return true;
}

// Q8_0 (ggml block_q8_0: f16 scale + 32 int8, 34 bytes): ne[0] a multiple of 32, nb[0] = the block
// size, rows of ne[0] / 32 blocks packed, higher axes packed.
constexpr size_t Q8_BLOCK = 34;
inline bool is_q8_rows(const mla_m4_tensor * t) {
    if (t->type != MLA_M4_TYPE_Q8_0 || t->ne[0] % 32 != 0 || t->nb[0] != Q8_BLOCK) return false;
    size_t expect = Q8_BLOCK * (size_t)(t->ne[0] / 32);
    for (int i = 1; i < 4; ++i) {
        if (t->ne[i] != 1 && t->nb[i] != expect) return false;
        expect *= (size_t)t->ne[i];
    }
    return true;
}

// plan = true: the supports_op mirrors, called on descriptors whose data may not be allocated yet
// (graph planning); only type/ne/nb are checked, and a data pointer only when it is set.
inline bool has_data(const mla_m4_tensor * t, bool plan) { return t && (plan || t->data); }
inline bool al16(const void * p, bool plan) { return (plan && !p) || aligned16(p); }
inline bool al4(const void * p, bool plan) { return (plan && !p) || (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// YaRN correction dims (the host-side ggml_rope_yarn_corr_dims, vendor/llama.cpp/ggml/src/ggml.c:4632-4643)
inline void rope_yarn_corr_dims(int n_dims, int n_ctx_orig, float freq_base, float beta_fast, float beta_slow, float dims[2]) {
    const float pi = 3.14159265358979323846f;
    auto corr_dim = [&](float n_rot) {
        return (float)n_dims * logf((float)n_ctx_orig / (n_rot * 2.0f * pi)) / (2.0f * logf(freq_base));
    };
    const float start = floorf(corr_dim(beta_fast));
    const float end = ceilf(corr_dim(beta_slow));
    dims[0] = start > 0.0f ? start : 0.0f;
    dims[1] = end < (float)(n_dims - 1) ? end : (float)(n_dims - 1);
}

// a vector: ne [n], packed
inline int check_vec(const mla_m4_tensor * t, int32_t type, size_t es, int64_t n, bool plan) {
    if (!has_data(t, plan)) return MLA_M4_ERR_NULL;
    if (t->type != type) return MLA_M4_ERR_TYPE;
    if (t->ne[0] != n || t->ne[1] != 1 || t->ne[2] != 1 || t->ne[3] != 1) return MLA_M4_ERR_SHAPE;
    if ((n != 1 && t->nb[0] != es) || (reinterpret_cast<uintptr_t>(t->data) & (es - 1))) return MLA_M4_ERR_STRIDE;
    return MLA_M4_OK;
}

inline bool rope_in_range(const mla_m4_rope_params * rp) {
    return rp->freq_base > 0.0f && rp->freq_scale > 0.0f && rp->eps >= 0.0f && rp->n_ctx_orig >= 1 &&
        std::isfinite(rp->freq_base) && std::isfinite(rp->freq_scale) && std::isfinite(rp->eps) &&
        std::isfinite(rp->ext_factor) && std::isfinite(rp->attn_factor) && rp->beta_fast > 0.0f && rp->beta_slow > 0.0f;
}

// The magnitude of a rope pair's cosine and sine (YaRN)
inline float rope_mscale(const mla_m4_rope_params * rp) {
    return rp->ext_factor != 0.0f ? rp->attn_factor * (1.0f + 0.1f * logf(1.0f / rp->freq_scale)) : rp->attn_factor;
}

// Turns (of 2 pi) per position of every rope pair, taken in 64 bits: the frequency
// freq_base^(-2 p / n_dims) times freq_scale (1 - mix) + mix (YaRN's ramp, which is linear in the angle).
inline void rope_turns(const mla_m4_rope_params * rp, double * turns) {
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

}  // namespace abi
}  // namespace mla
