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

}  // namespace abi
}  // namespace mla
