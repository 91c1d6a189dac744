// mul_i8_forms.h -- which form of the int8 product's kernels (mul_i8.hip) takes a shape.  Host code alone, without HIP.
#pragma once

#include <cstdint>

namespace mla {
namespace rows {

// Which kernel takes a product, and in how many parts of k.  Each form's time (us) is estimated as
//   fixed + step * (steps of 128 bytes a CU runs) + group * (workgroups a CU runs) + mb * (operands and result, MB)
// and, where k is cut, the sums' launch and their traffic; of direct_kernel as fixed + mb * MB + what a CU fetches.  The constants
// are fitted to 3,000 times of 225 shapes (1 to 8,000 rows, 576 to 24,576 channels, k 512 to 16,384; six copies of the operands in turn,
// the smaller ones in the card's 256 MB cache); the form they choose takes 1.01 times the best form's time in the mean, 1.19 at most
// (150 rows x 24,576 x 1536), and with operands out of memory (1,500 times of 96 shapes) 1.02 and 1.22 (1 x 7168 x 16,384).  What they weigh:
// 64 rows x 7168 x 4096 takes 9.7 us in tiles of 32 x 64 and 11.5 in 64 x 64 (112 workgroups leave half of the CUs idle), 64 x 576 x
// 7168 takes 7.7 us with k in 7 parts and 10.9 in one, 32 x 2112 x 7168 9.0 in 3 and 15.1, 4,001 x 4096 x 4096 71 us in tiles of 256 and 86 in tiles of 128, 200 x
// 24,576 x 1536 32 and 23, and 1,500 x 7168 x 4096 takes 54 us in 192 x 256 (228 workgroups, one round), 64 in 256 x 256 and 76 in 128.
struct Form {
    int kind, bn, bm;
    float fixed, step, group, mb, pair, cut, cut_mb;   // pair: per step of two workgroups at once on a CU; direct_kernel: us per 100 KB
};
enum { DIRECT8, DIRECT8_2, SPLIT11, SPLIT12, SPLIT22, SPLIT32, SPLIT128, TILE128, TILE192, TILE256 };
constexpr Form FORMS[] = {
    {DIRECT8, 16, 16, 2.2f, 0.f, 0.f, 0.095f, 2.6f, 0.f, 0.f},
    {DIRECT8_2, 32, 16, 2.1f, 0.f, 0.f, 0.062f, 2.8f, 0.f, 0.f},
    {SPLIT11, 32, 32, 2.5f, 0.058f, 0.73f, 0.066f, 0.063f, 2.3f, 0.19f},
    {SPLIT12, 32, 64, 2.2f, 0.11f, 1.3f, 0.042f, 0.044f, 2.2f, 0.17f},
    {SPLIT22, 64, 64, 2.4f, 0.16f, 1.9f, 0.075f, 0.027f, 2.0f, 0.16f},
    {SPLIT32, 96, 64, 3.0f, 0.20f, 2.2f, 0.098f, 0.011f, 1.7f, 0.14f},
    {SPLIT128, 128, 128, 6.7f, 0.33f, 0.f, 0.11f, 0.f, 0.8f, 0.25f},
    {TILE128, 128, 128, 2.9f, 0.20f, 1.8f, 0.15f, 0.44f, 0.f, 0.f},
    {TILE192, 192, 256, 0.f, 0.91f, 5.5f, 0.18f, 0.f, 0.f, 0.f},
    {TILE256, 256, 256, 0.f, 1.1f, 8.2f, 0.19f, 0.f, 0.f, 0.f},
};
constexpr int CUS = 256, MOST_PARTS = 12, FEW_ROWS = 48, MANY_ROWS = 100, MOST_CUT = 512;

struct Choice {
    int kind, n_split;
    int64_t work;       // bytes of the workspace
};
inline Choice choose(int n, int k, int n_rows, bool may_cut) {
    Choice best{TILE256, 1, 0};
    float least = 3.0e38f;
    const float mb = ((float)n * k + (float)n_rows * k + 4.0f * n * (float)n_rows) * 1e-6f;
    const int all = (k + 127) / 128;
    for (const Form & f : FORMS) {
        const int64_t tiles = (int64_t)((n + f.bn - 1) / f.bn) * ((n_rows + f.bm - 1) / f.bm);
        if (f.kind <= DIRECT8_2) {
            if (n_rows > FEW_ROWS) continue;
            const float fetched = (float)tiles * (f.bn + (n_rows < f.bm ? n_rows : f.bm)) * (float)k * 1e-5f / (tiles < CUS ? (float)tiles : (float)CUS);
            const float t = f.fixed + f.mb * mb + f.pair * fetched;
            if (t < least) {
                least = t;
                best = {f.kind, 1, 0};
            }
            continue;
        }
        if (f.kind >= TILE128 && n_rows < MANY_ROWS) continue;
        for (int parts = 1; parts <= MOST_PARTS; ++parts) {
            if (parts > 1 && (!may_cut || f.cut == 0.f || tiles * parts > MOST_CUT || all < 4 * parts)) break;
            const int64_t groups = tiles * parts;
            if (f.kind == SPLIT128 && groups > CUS) break;          // one workgroup a CU: the ends of a second round are not hidden
            const float per = (float)((groups + CUS - 1) / CUS);
            const float steps = (float)((all + parts - 1) / parts);
            float t = f.fixed + f.step * per * steps + f.group * per + f.mb * mb;
            if (f.pair != 0.f) t += f.pair * steps * (float)((groups + 2 * CUS - 1) / (2 * CUS));
            if (parts > 1) t += f.cut + f.cut_mb * 8e-6f * (float)parts * (float)n_rows * (float)n;
            if (t < least) {
                least = t;
                best = {f.kind, parts, parts > 1 ? groups * f.bn * f.bm * 4 : 0};
            }
        }
    }
    return best;
}

}  // namespace rows
}  // namespace mla
