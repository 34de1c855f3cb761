// The forms of nb_linear8's product and the choice among them.  Host arithmetic only:
// the tests compile it by itself.
#pragma once

#include <cmath>
#include <cstdint>

namespace nb {
namespace linear8 {

// A form, and what it costs in microseconds: `launch` once, `start` for the
// workgroups that a CU holds at once, `step[c - 1]` for a block of K (of `split`) with c of
// them.  Fitted to 413 shapes (1 to 2500 rows, 64 to 16000 outputs, K of 128 to 8192)
// times 10 forms on MI355X; the form of least estimated time is 2 % slower than
// the fastest one on the mean, half as long again at worst (long K, few outputs,
// hundreds of rows).  What the other forms lose where each is taken: 9 rows of 7680 x 2560
// 4.4 us by 32 x 32 (rows), 5.2 by 16 x 16, 6.4 by 64 x 32; 129 of 2560 x 6912 13.0 by 64 x
// 32, 14.4 by 64 x 64, 18.3 by rows; 512 of 2560 x 6912 20.2 by 128 x 64 of two
// groups, 27.3 of one, 27.9 by 64 x 64; 1500 of it 30.7 by 128 x 128 of two groups, 36.0 by
// 128 x 64, 36.8 of one; 2048 of 13824 x 2560 80 by 256 x 256, 88 by 128 x 128 of one.  Where
// whole rounds of the CUs meet the estimate is the other way round by a little: 1500 rows
// of 13824 x 2560 take 76 by 256 x 256, estimated at 72, and would take 73 by 128 x 128 of
// one, estimated at 76 (1200 to 1400 and 1700 rows are the same by both).
struct Form {
    int outputs, rows;   // of a workgroup
    int split;           // groups of waves that share K
    int resident;        // workgroups of a CU
    bool tiles;          // tiles through LDS (else few rows)
    float launch, start, step[2];
};
constexpr Form kForms[] = {
    {16, 16, 8, 1, false, 3.11f, 0.f, {0.276f}},
    {32, 32, 8, 2, false, 3.0f, 0.f, {0.58f, 1.21f}},
    {64, 32, 2, 2, true, 1.65f, 1.98f, {0.287f, 0.516f}},
    {64, 64, 2, 1, true, 1.03f, 2.46f, {0.397f}},
    {128, 64, 2, 1, true, 0.38f, 3.25f, {0.603f}},
    {128, 64, 1, 2, true, 1.25f, 2.36f, {0.392f, 0.546f}},
    {128, 128, 2, 1, true, 0.f, 4.53f, {0.919f}},
    {128, 128, 1, 1, true, 2.12f, 2.32f, {0.497f}},
    {256, 256, 1, 1, true, 0.f, 6.93f, {1.446f}},
};
constexpr int kFormCount = sizeof(kForms) / sizeof(kForms[0]);

// Workgroups of a launch: of outputs and of rows.
inline int64_t output_groups(const Form& f, int N) { return ((int64_t)N + f.outputs - 1) / f.outputs; }
inline int64_t row_groups(const Form& f, int M) { return ((int64_t)M + f.rows - 1) / f.rows; }

// Whether its launch is one that the runtime takes: under 2^32 threads, and the rows'
// workgroups of a form for few rows, a grid's second dimension, at most 65535.  (256 x 256
// always fits: M N is under 2^36, M at most 2^20 and N at most 2^24.)
inline bool form_fits(const Form& f, int M, int N) {
    return output_groups(f, N) * row_groups(f, M) < 1 << 22 && (f.tiles || row_groups(f, M) <= 65535);
}

inline int form_of(int M, int N, int K, int64_t cus) {
    int best = kFormCount - 1;
    float least = INFINITY;
    for (int i = 0; i < kFormCount; ++i) {
        const Form& f = kForms[i];
        if (!form_fits(f, M, N)) continue;
        const int64_t each = (output_groups(f, N) * row_groups(f, M) + cus - 1) / cus, rest = each % f.resident;
        const float steps = (float)((K / 128 + f.split - 1) / f.split);
        float t = f.launch + (float)(each / f.resident) * (f.start + steps * f.step[f.resident - 1]);
        if (rest) t += f.start + steps * f.step[rest - 1];
        if (t < least) least = t, best = i;
    }
    return best;
}

}  // namespace linear8
}  // namespace nb
