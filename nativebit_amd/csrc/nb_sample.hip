// Tokens drawn from a batch of logits (gfx950): nb_sample.
//
// For a row x of V logits with its maximum m, temperature T, and order "larger
// first, of equal ones the lower index first":
//     w(v) = exp((x(v) - m) / T)                       0 for -inf and NaN
//     kept = the first top_k of the order,
//            of those the shortest beginning whose weights reach top_p of theirs,
//            of those the ones with w >= min_p
//     token = the first v whose running sum of kept weights, by index, is over
//             u times their total;  logprob = log(w(token) / total)
// Sums decide which token it is, so they are exact: weights are whole numbers of
// 2^-S (S = 45 for V up to 2^17), exp in 64 bits rounded once, and every sum of
// them is a 64-bit integer, the same in any order.
//
// A row is cut into slices, one workgroup each:
//   1. sample_max_kernel     each slice's first token of the order, and (with rules)
//                            the largest logit of every group of 32 tokens
//   2. sample_bins_kernel    each slice's weights, summed and counted in bins of an
//                            eighth of an octave of w, down to 2^-46 where it rounds
//                            to 0; without rules one sum
//   3. sample_finish_kernel  one workgroup a row: the bins say where the rules cut; the
//                            tokens of the bins that they cut through are listed, from
//                            the groups that reach them, and sorted, and give the
//                            cuts; bins and list each slice's sum of kept weights, u
//                            the slice, the slice read again the token
// A row whose top_k is small (few_kept) has no bins: the k-th largest of its groups'
// largest logits is a logit that k tokens reach, so what it keeps is among the
// tokens that reach it, and those are in the groups that do; k of them, but for
// ties.  They are listed, and that is all that is read again of the row.
// What it takes: 160 rows of 131077 fp32 logits with every rule and top_k of 1 to 1024
// 46 us, 84 MB.  1 reads them at 3.6 TB/s in 23.5; 2 finds nothing to do in 4.6; 3 is
// one memory round trip after the other (rules, groups, tokens, 2 us each) and some
// twenty waits of a workgroup between, 21.  With top_p or min_p alone 89 to 93 us (logits
// of deviation 4, T = 0.8): 2 takes 44, an exp in 64 bits and an atomic in LDS for every
// token.  With a temperature alone 69 (21, 34 and 12).  One row of 50257 with top_p 25 to
// 36 us by how many tokens are listed (4, 6, and 11 to 20), with a temperature alone 16.
// Other ways measured: cuts and list as launches of their own, a slice each, 34 and
// 59 us where one took 29 and 48 (48 rows of 50257, 160 of 131077); a list that scans the
// slice again instead of its groups 21 us at 160 rows, now 2 to 5; 1000 tokens sorted by
// merging 40 us, through buckets 2.
// A row with over kMostListed tokens in the bins that the rules cut through is worked out
// by its workgroup alone: radix selection, some ten passes over the row.  Equal logits are
// such rows (48 of 50257 with top_p 245 us, with top_k of 1000 194), and logits next to
// each other where a cut falls: an eighth of an octave holds over 4096 of 131077 whose
// deviation over T is about 1 (160 rows with top_p of 0.9 514 us, one 325), and of 262144
// at 4/3 (48 rows 833 us, one 571).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "nb_device.h"
#include "nb_internal.h"

namespace nb {
namespace {

typedef __attribute__((ext_vector_type(4), aligned(4))) float f4_any;
typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t u2_any;

constexpr int kBins = 368;          // of an eighth of an octave: 46 octaves; one more below
constexpr int kMostListed = 4096;   // listed tokens of a row
constexpr int kSliceThreads = 512;
constexpr int kMostSlices = 128;
constexpr int kFewKept = 2048;
constexpr int kGroup = 32;          // 128 bytes of fp32 logits

struct SampleArgs {
    const void* logits;
    int64_t ld;
    int V, shift;          // shift: S
    int slices, length;    // of a row; tokens of a slice
    const float *u, *temperature;
    const int32_t* top_k;
    const float *top_p, *min_p;
    int32_t* tokens;
    float* logprobs;
    // workspace, for each row and slice
    uint64_t* first;       // the slice's first token of the order (place_of)
    uint32_t* groups;      // of a row, with rules: the largest key of every kGroup tokens
    uint64_t* sums;        // [kBins + 1] with rules, else one
    uint32_t* counts;      // [kBins + 1]
    __host__ __device__ __forceinline__ bool rules() const { return top_k || top_p || min_p; }
    __host__ __device__ __forceinline__ int groups_of_row() const { return (V + kGroup - 1) / kGroup; }
    // A row whose kept tokens are in few groups: its bins are not needed.  48 rows of
    // 50257 (1571 groups) with k = 50, 500, 1024, 1300 and 1500 and the other rules: 20, 26,
    // 30, 36 and 43 us so, 38, 46, 49, 48 and 48 us by bins; 300 of 10007 (313 groups) 21 and
    // 26 (without the other rules 26 and 24); 160 rows of 131077 with 2048: 57 and 111.
    __device__ __forceinline__ bool few_kept(int64_t b) const {
        const int64_t k = top_k ? as_constant(top_k)[b] : 0;
        return k > 0 && k < V && k <= kFewKept && k <= groups_of_row();
    }
};

// Larger for larger logits; 0 for -inf and NaN.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.f);   // (-0 as 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A token's place in the order (larger: earlier); 0 for -inf and NaN.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int v) {
    return key ? (uint64_t)key << 32 | (0xffffffffu - (uint32_t)v) : 0;
}
__device__ __forceinline__ uint32_t key_of_place(uint64_t place) { return (uint32_t)(place >> 32); }
__device__ __forceinline__ int token_of_place(uint64_t place) {
    return (int)(0xffffffffu - (uint32_t)place);
}

template <int kDtype>
__device__ __forceinline__ uint32_t key_at(const SampleArgs& a, int64_t b, int v) {
    const int64_t at = b * a.ld + v;
    return key_of(kDtype == NB_F32 ? static_cast<const float*>(a.logits)[at]
                                   : bf16_to_f32(static_cast<const bf16_bits*>(a.logits)[at]));
}

// The tokens lo .. hi - 1 of a row by the kThreads threads of a workgroup, groups of
// four, kBatch groups of a thread at once and as many asked for ahead of them.
template <int kDtype, int kThreads>
struct Tokens {
    static constexpr int kBatch = 4, kStep = 4 * kThreads * kBatch;
    using Four = std::conditional_t<kDtype == NB_F32, f4_any, u2_any>;
    const char* row;
    int v0, hi;
    Four x[kBatch];

    __device__ __forceinline__ Tokens(const SampleArgs& a, int64_t b, int lo, int hi_)
        : row(static_cast<const char*>(a.logits) + b * a.ld * (kDtype == NB_F32 ? 4 : 2)),
          v0(lo + 4 * (int)threadIdx.x), hi(hi_) {
        load(v0);
    }
    __device__ __forceinline__ void load(int first) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int v = first + j * 4 * kThreads;
            if (v + 3 < hi) {
                x[j] = *reinterpret_cast<const Four*>(row + (int64_t)v * (kDtype == NB_F32 ? 4 : 2));
            } else {
                float e4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    e4[e] = -INFINITY;
                    if (v + e < hi) {
                        e4[e] = kDtype == NB_F32 ? reinterpret_cast<const float*>(row)[v + e]
                                                 : bf16_to_f32(reinterpret_cast<const bf16_bits*>(row)[v + e]);
                    }
                }
                if constexpr (kDtype == NB_F32) {
                    x[j] = Four{e4[0], e4[1], e4[2], e4[3]};
                } else {
                    x[j] = Four{__float_as_uint(e4[0]) >> 16 | __float_as_uint(e4[1]),
                                __float_as_uint(e4[2]) >> 16 | __float_as_uint(e4[3])};
                }
            }
        }
    }
    // f(token, keys of four from it on), once; lanes of a wave stay together
    template <typename F>
    __device__ __forceinline__ void each_four(F f) {
        for (; (v0 & ~255) < hi; v0 += kStep) {
            Four now[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) now[j] = x[j];
            if (((v0 + kStep) & ~255) < hi) load(v0 + kStep);
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                uint32_t keys[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y;
                    if constexpr (kDtype == NB_F32) y = now[j][e];
                    else y = __uint_as_float(e & 1 ? now[j][e / 2] & 0xffff0000u : now[j][e / 2] << 16);
                    keys[e] = key_of(y);
                }
                f(v0 + j * 4 * kThreads, keys);
            }
        }
    }
    // f(token, key), once (0 past the last)
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        each_four([&](int v, const uint32_t* keys) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f(v + e, keys[e]);
        });
    }
};

// The bin of a weight by its log2.
__device__ __forceinline__ int bin_of(double z) { return z > -kBins / 8 ? (int)(z * -8.0) : kBins; }

constexpr int kFractions = 128;   // entries of 2^(i / 128)

struct Weights {
    double most, turn;   // the row's maximum, log2(e) / T
    const double* table;
    int shift;
    // log2 of a key's weight
    __device__ __forceinline__ double log2_of(uint32_t key) const {
        const double x = logit_of(key);
        return x == most ? 0.0 : fmax((x - most) * turn, -4000.0);   // (of infinities: 0 or less)
    }
    // 2^(n + f): the table's entry by f's upper bits, a polynomial of the rest
    // (|r| <= 1/256: its next term is 2e-12)
    __device__ __forceinline__ uint64_t of(uint32_t key) const {
        return key ? of_log2(log2_of(key)) : 0;
    }
    __device__ __forceinline__ uint64_t of_log2(double z) const {
        constexpr double kMagic = 6755399441055744.0;   // 1.5 * 2^52: rounds to a whole number
        const double y = z * kFractions + kMagic;
        const int n = __double2loint(y);
        const double r = z - (y - kMagic) * (1.0 / kFractions);
        double p = 0.05550410866482158;
        p = fma(p, r, 0.2402265069591007);
        p = fma(p, r, 0.6931471805599453);
        p = fma(p, r, 1.0);
        p = ldexp(p * table[n & (kFractions - 1)], (n >> 7) + shift);
        return (uint64_t)__double_as_longlong(p + 4503599627370496.0) - 0x4330000000000000ull;
    }
};

// Over the lanes of a wave by DPP moves (a 64-bit shuffle is two LDS round trips): rows
// of 16 lanes by shifts, then a row's last lane to the next, and the second's to the
// other half.  All lanes must be active.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {   // 0 where no lane is read
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, kRows, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), kCtrl, kRows, 0xf, true);
    return (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
}
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ uint32_t dpp32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, true);
}
__device__ __forceinline__ uint32_t wave_scan32(uint32_t v) {
    v += dpp32<0x111>(v);
    v += dpp32<0x112>(v);
    v += dpp32<0x114>(v);
    v += dpp32<0x118>(v);
    v += dpp32<0x142, 0xa>(v);
    return v + dpp32<0x143, 0xc>(v);
}
template <typename Join>
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, Join join) {   // of lanes 0 .. this one
    v = join(v, dpp64<0x111, 0xf>(v));   // row_shr 1, 2, 4, 8
    v = join(v, dpp64<0x112, 0xf>(v));
    v = join(v, dpp64<0x114, 0xf>(v));
    v = join(v, dpp64<0x118, 0xf>(v));
    v = join(v, dpp64<0x142, 0xa>(v));   // row_bcast 15 into rows 1 and 3
    return join(v, dpp64<0x143, 0xc>(v));   // row_bcast 31 into rows 2 and 3
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
    return wave_scan(v, [](uint64_t x, uint64_t y) { return x + y; });
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return lane_of(wave_scan(v), 63); }
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    return lane_of(wave_scan(v, [](uint64_t x, uint64_t y) { return x > y ? x : y; }), 63);
}
__device__ __forceinline__ uint64_t lesser(uint64_t x, uint64_t y) { return x < y ? x : y; }

// A row's rules.  (Weights of a greedy row are those of T = 1: nothing uses them.)
struct Rules {
    bool greedy;       // the first of the order: T is not over 0, or one token is kept
    int64_t k;         // 0: all
    float p;           // 1: all
    uint64_t least;    // of a kept weight
    double least_high, least_low;   // log2s around it
    uint64_t first;    // of the row's order; 0: nothing is left
    Weights w;
    __device__ __forceinline__ Rules(const SampleArgs& a, int64_t b, const double* table) {
        const float t = a.temperature ? as_constant(a.temperature)[b] : 1.f;
        k = a.top_k ? as_constant(a.top_k)[b] : 0;
        if (k <= 0 || k >= a.V) k = 0;
        greedy = !(t > 0.f) || k == 1;
        p = a.top_p ? as_constant(a.top_p)[b] : 1.f;
        if (!(p < 1.f)) p = 1.f;
        const float mp = a.min_p ? as_constant(a.min_p)[b] : 0.f;
        const double m = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        least = (uint64_t)ceil(m * (double)(1ull << a.shift));
        if (least <= 1) least = 0;   // (weights of 0 are never drawn)
        if (least) {
            // around it: a unit of the weights' rounding, and of the logarithms'
            const double unit = 1e-9 + 2.0 / (double)least, z = log2(m);
            least_high = fmin(z + unit, 0.0), least_low = z - unit;
        }
        const int lane = threadIdx.x & 63;
        static_assert(kMostSlices <= 128, "two slices a lane");
        const uint64_t o0 = lane < a.slices ? a.first[b * a.slices + lane] : 0;
        const uint64_t o1 = lane + 64 < a.slices ? a.first[b * a.slices + lane + 64] : 0;
        first = wave_max(o0 > o1 ? o0 : o1);
        w.most = (double)logit_of(key_of_place(first));
        w.turn = 1.4426950408889634 / (t > 0.f ? (double)t : 1.0);
        w.table = table;
        w.shift = a.shift;
    }
};
__device__ __forceinline__ void make_table(double* table) {
    if (threadIdx.x < kFractions) table[threadIdx.x] = exp2((double)threadIdx.x / kFractions);
}

// ---------------------------------------------------------------------------
// slices
// ---------------------------------------------------------------------------
template <int kDtype, bool kRules>
__global__ __launch_bounds__(kSliceThreads) void sample_max_kernel(SampleArgs a) {
    __shared__ uint64_t part[kSliceThreads / 64];
    const int64_t b = blockIdx.y;
    const int lo = blockIdx.x * a.length, hi = min(lo + a.length, a.V), tid = threadIdx.x;
    uint64_t first = 0;
    Tokens<kDtype, kSliceThreads>(a, b, lo, hi).each_four([&](int v, const uint32_t* keys) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t place = place_of(keys[e], v + e);
            first = place > first ? place : first;
        }
        if constexpr (kRules) {   // (8 lanes have a group, half a DPP row)
            static_assert(kGroup == 32, "lanes of a group");
            uint32_t most = max(max(keys[0], keys[1]), max(keys[2], keys[3]));
            most = max(most, dpp32<0x111>(most));
            most = max(most, dpp32<0x112>(most));
            most = max(most, dpp32<0x114>(most));
            if ((tid & 7) == 7 && v / kGroup * kGroup < hi) a.groups[b * a.groups_of_row() + v / kGroup] = most;
        }
    });
    first = wave_max(first);
    if ((tid & 63) == 0) part[tid >> 6] = first;
    __syncthreads();
    if (tid) return;
    for (int i = 1; i < kSliceThreads / 64; ++i) first = part[i] > first ? part[i] : first;
    a.first[b * a.slices + blockIdx.x] = first;
}

// Weights up to 2^-11 are most of a row's: in bins of a slice of up to 2^14 tokens
// their sum is at most 2^48, and the count lies above it in the same word (one
// atomic for both).  Four copies of the bins, a lane's by its number: lanes of a wave
// hit the same word less often.
constexpr int kPackedFrom = 88, kCountAt = 49, kCopies = 4;

template <int kDtype, bool kRules>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ double table[kFractions];
    __shared__ unsigned long long sums[(kBins + 1) * kCopies];
    __shared__ uint32_t counts[kBins + 1];
    const int64_t b = blockIdx.y, slice = b * a.slices + blockIdx.x;
    const int lo = blockIdx.x * a.length, hi = min(lo + a.length, a.V), tid = threadIdx.x;
    if (kRules && a.few_kept(b)) return;
    Tokens<kDtype, kSliceThreads> tokens(a, b, lo, hi);   // (its first loads are under way meanwhile)
    make_table(table);
    const Rules r(a, b, table);
    if (r.greedy || r.first == 0) return;   // (nothing reads the row's bins)
    if (kRules) {
        for (int i = tid; i < (kBins + 1) * kCopies; i += kSliceThreads) sums[i] = 0;
        for (int i = tid; i <= kBins; i += kSliceThreads) counts[i] = 0;
    }
    __syncthreads();
    const int packed_from = a.length <= 1 << 14 ? kPackedFrom : kBins;
    uint64_t sum = 0;       // without bins of all, else of the last bin
    uint32_t count = 0;
    tokens.each([&](int, uint32_t key) {
        if (!key) return;
        const double z = r.w.log2_of(key);
        uint64_t w = r.w.of_log2(z);
        const int bin = kRules ? bin_of(z) : kBins;
        if (bin < kBins) {
            if (bin >= packed_from) w += 1ull << kCountAt;
            else atomicAdd(&counts[bin], 1u);
            atomicAdd(&sums[bin * kCopies + (tid & (kCopies - 1))], (unsigned long long)w);
        } else {
            sum += w, ++count;
        }
    });
    if (kRules) {
        sum = wave_sum(sum), count = (uint32_t)wave_sum(count);
        if ((tid & 63) == 0) {
            atomicAdd(&sums[kBins * kCopies], (unsigned long long)sum);
            atomicAdd(&counts[kBins], count);
        }
        __syncthreads();
        for (int i = tid; i <= kBins; i += kSliceThreads) {
            uint64_t all = 0;
            for (int c = 0; c < kCopies; ++c) all += sums[i * kCopies + c];
            const bool packed = i >= packed_from && i < kBins;
            a.sums[slice * (kBins + 1) + i] = packed ? all & ((1ull << kCountAt) - 1) : all;
            a.counts[slice * (kBins + 1) + i] = packed ? (uint32_t)(all >> kCountAt) : counts[i];
        }
    } else {
        sum = wave_sum(sum);
        if ((tid & 63) == 0) sums[tid >> 6] = sum;
        __syncthreads();
        if (tid) return;
        for (int i = 1; i < kSliceThreads / 64; ++i) sum += sums[i];
        a.sums[slice] = sum;
    }
}

// Where the rules cut a row, from its bins.
struct Cuts {
    int k;               // the bin that top_k ends in; past the last: none
    int p_low, p_high;   // those that top_p may end in (what top_k keeps of its bin
                         // is not known yet)
    int m_low, m_high;   // those around min_p
    uint64_t above_k, sum_k, above_p;   // tokens and weights over bin k, weights over p_low
    float low, high;     // the logits of all listed tokens lie between
    // The bin of a listed token by its log2; where all of a row's first tokens are listed
    // (few_kept) they are one bin.
    bool one;
    __device__ __forceinline__ int bin(double z) const { return one ? 0 : bin_of(z); }
    __device__ __forceinline__ bool listed(int bin) const {
        return bin == k || (bin >= p_low && bin <= p_high) || (bin >= m_low && bin <= m_high);
    }
    // all tokens of the bins before it are kept, of those after it only listed ones
    __host__ __device__ __forceinline__ int sure() const { return std::min(k, std::min(p_low, m_low)); }
};
// The least sum of a beginning that makes up p of `total`: at least one unit.
__device__ __forceinline__ uint64_t share_of(float p, uint64_t total) {
    if (!(p > 0.f)) return 1;
    const double s = fmax(ceil((double)p * (double)total), 1.0);
    return s < (double)total ? (uint64_t)s : total;
}
struct CutShared {
    uint64_t sum[kBins + 2], above[kBins + 2];   // of a bin; of those before it
    uint32_t count[kBins + 2], before[kBins + 2];
    uint64_t part[(kBins + 64) / 64];
    uint32_t count_part[(kBins + 64) / 64];
    int found[3];
};
// By all threads of a workgroup of over kBins + 1, each with its bin of the row.
__device__ Cuts find_cuts(const Rules& r, uint64_t sum, uint32_t count, CutShared& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int kAll = kBins + 1, kNone = kBins + 1, kParts = (kAll + 63) / 64;
    uint64_t above = 0;
    uint32_t before = 0;
    if (tid < kParts * 64) {
        above = wave_scan(sum), before = (uint32_t)wave_scan((uint64_t)count);
        if (lane == 63) s.part[wave] = above, s.count_part[wave] = before;
        above -= sum, before -= count;
    }
    if (tid < 3) s.found[tid] = kNone;
    __syncthreads();
    static_assert(kAll < kParts * 64, "one past the last");
    if (tid <= kAll) {   // (and one past the last: all of them)
        for (int i = 0; i < wave; ++i) above += s.part[i], before += s.count_part[i];
        s.sum[tid] = sum, s.above[tid] = above, s.count[tid] = count, s.before[tid] = before;
    }
    __syncthreads();
    if (r.k && tid < kAll && s.before[tid] < r.k && s.before[tid] + (uint64_t)s.count[tid] >= (uint64_t)r.k) {
        s.found[0] = tid;
    }
    __syncthreads();
    Cuts c;
    // (what all threads have alike is kept once for a wave)
    c.k = __builtin_amdgcn_readfirstlane(s.found[0]);
    if (c.k == kBins) c.k = kNone;   // (a cut among weights of 0 changes nothing)
    c.above_k = lane_of(s.before[c.k], 0), c.sum_k = lane_of(s.above[c.k], 0);
    if (r.p < 1.f && tid < kAll) {
        const uint64_t low = share_of(r.p, max(s.above[c.k], (uint64_t)1));
        const uint64_t high = share_of(r.p, s.above[c.k] + s.sum[c.k]);
        if (s.above[tid] < low && s.above[tid] + s.sum[tid] >= low) s.found[1] = tid;
        if (s.above[tid] < high && s.above[tid] + s.sum[tid] >= high) s.found[2] = tid;
    }
    __syncthreads();
    c.p_low = __builtin_amdgcn_readfirstlane(s.found[1]), c.p_high = __builtin_amdgcn_readfirstlane(s.found[2]);
    c.above_p = lane_of(s.above[c.p_low], 0);
    c.m_low = c.m_high = kNone;
    if (r.least) {
        c.m_low = bin_of(r.least_high);
        c.m_high = bin_of(r.least_low);
    }
    // an eighth of an octave and the roundings to either side of the first and the
    // last listed bin (none: no logit is infinite both ways)
    int to = -1;
    if (c.k <= kBins) to = c.k;
    if (c.p_low <= kBins) to = max(to, c.p_high);
    if (c.m_low <= kBins) to = max(to, c.m_high);
    const double octave = 1.0 / r.w.turn, slack = 1e-6 * fabs(r.w.most);
    c.high = to < 0 ? -INFINITY : (float)(r.w.most - (c.sure() - 1) * 0.125 * octave + slack);
    c.low = to < 0 ? INFINITY : to == kBins ? -INFINITY : (float)(r.w.most - (to + 2) * 0.125 * octave - slack);
    c.one = false;
    return c;
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
constexpr int kThreads = 1024, kWaves = kThreads / 64, kDigits = 2048;
constexpr int kHeld = 4, kMostGroups = kHeld * kThreads;   // groups of a row at once, kHeld a thread

struct Shared {
    double table[kFractions];
    uint64_t list[kMostListed];              // the listed tokens
    union {
        struct {
            union {
                uint64_t digits[kDigits];    // radix selection
                CutShared cuts;
            };
            uint32_t groups[kMostGroups];    // those that are looked into
        };
        struct {
            uint64_t sorted[kMostListed];    // sort_list's
        };
    };
    uint32_t bucket[kDigits];
    uint64_t part[kWaves], ties[kWaves];
    uint64_t found[2];
    uint32_t some_groups, some, key_low, key_high;
};

// What is kept: tokens up to `last` in the order, of weights of `least` or more.
// (0: all of the order.)
struct Kept {
    uint64_t last, least;
    __device__ __forceinline__ uint64_t weight(const Weights& w, uint32_t key, int v) const {
        if (!key || place_of(key, v) < last) return 0;
        const uint64_t n = w.of(key);
        return n >= least ? n : 0;
    }
};

__device__ uint64_t block_sum(Shared& s, uint64_t v) {   // in all threads
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) v += s.part[i];
    return v;
}

// From the largest bin down: the one in which their sum reaches `bound` (> 0, at
// most the sum of all), and the sum of the bins above it.
struct Crossing {
    int bin;
    uint64_t above;
};
__device__ Crossing cross(Shared& s, uint64_t bound) {
    constexpr int kEach = kDigits / kThreads;
    const int tid = threadIdx.x, lane = tid & 63;
    // thread t takes the bins from the t-th largest pair on
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine += s.digits[kDigits - 1 - (tid * kEach + i)];
    const uint64_t upto = wave_scan(mine);
    __syncthreads();
    if (lane == 63) s.part[tid >> 6] = upto;
    if (tid == 0) s.found[0] = 0, s.found[1] = 0;
    __syncthreads();
    uint64_t above = upto - mine;
    for (int i = 0; i < (tid >> 6); ++i) above += s.part[i];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int bin = kDigits - 1 - (tid * kEach + i);
        const uint64_t n = s.digits[bin];
        if (above < bound && above + n >= bound) {
            s.found[0] = (uint64_t)bin, s.found[1] = above;
        }
        above += n;
    }
    __syncthreads();
    return Crossing{(int)s.found[0], s.found[1]};
}

// f(key) for a row's tokens.
template <int kDtype, typename F>
__device__ __forceinline__ void for_row(const SampleArgs& a, int64_t b, F f) {
#pragma unroll 4
    for (int v = threadIdx.x; v < a.V; v += kThreads) f(key_at<kDtype>(a, b, v));
}

// The key at which the order's sum of `value(key)` over keys >= least first
// reaches `bound` (> 0, at most the sum of all), and the sum above that key.
template <int kDtype, typename Value>
__device__ uint64_t select(const SampleArgs& a, int64_t b, Shared& s, uint32_t least, uint64_t bound,
                           Value value, uint32_t& at) {
    uint64_t above = 0;
    uint32_t prefix = 0, mask = 0;
    for (int shift = 21; shift >= -1; shift -= 11) {   // 11, 11 and 10 bits
        const int low = max(shift, 0), bits = shift < 0 ? 10 : 11;
        __syncthreads();
        for (int i = threadIdx.x; i < kDigits; i += kThreads) s.digits[i] = 0;
        __syncthreads();
        for_row<kDtype>(a, b, [&](uint32_t key) {
            if (key && key >= least && (key & mask) == prefix) {
                atomicAdd((unsigned long long*)&s.digits[key >> low & ((1u << bits) - 1)],
                          (unsigned long long)value(key));
            }
        });
        __syncthreads();
        const Crossing c = cross(s, bound - above);
        above += c.above;
        prefix |= (uint32_t)c.bin << low;
        mask |= ((1u << bits) - 1) << low;
    }
    at = prefix;
    return above;
}

// A key that k or more of those that each(f) gives reach, and few more than k do (but for
// equal ones); 1 where they are fewer.  `high`: none is larger.  Counted in buckets of
// neighbouring keys between the least and it (by the keys' upper bits 64 lanes would
// meet in a handful of words: 5 us of a row), once, or again in the bucket of the k-th
// where outliers leave many in it.
template <typename Each>
__device__ __forceinline__ uint32_t edge_of(Shared& s, uint32_t k, uint32_t high, Each each) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t least = ~0u;
    each([&](uint32_t key) { least = min(least, key ? key : ~0u); });
    least = ~(uint32_t)wave_max(~least);
    __syncthreads();
    if (tid == 0) s.key_low = ~0u;
    __syncthreads();
    if (lane == 0) atomicMin(&s.key_low, least);
    __syncthreads();
    uint32_t low = s.key_low;
    if (low > high) return 1;   // (there are none)
    for (;;) {
        const int shift = max(32 - __clz((int)(high - low)) - 11, 0);
        s.bucket[2 * tid] = s.bucket[2 * tid + 1] = 0;
        if (tid == 0) s.found[1] = kDigits;
        __syncthreads();
        each([&](uint32_t key) {
            if (key >= low && key <= high) atomicAdd(&s.bucket[(high - key) >> shift], 1u);
        });
        __syncthreads();
        const uint32_t first = s.bucket[2 * tid], both = first + s.bucket[2 * tid + 1];
        uint32_t before = wave_scan32(both);
        if (lane == 63) s.part[wave] = before;
        __syncthreads();
        for (int i = 0; i < wave; ++i) before += (uint32_t)s.part[i];
        before -= both;
        if (before < k && before + both >= k) {   // one thread
            const bool second = before + first < k;
            s.found[1] = 2 * tid + second;
            s.found[0] = before + (second ? first : 0);
        }
        __syncthreads();
        const uint32_t bucket = (uint32_t)s.found[1], above = (uint32_t)s.found[0];
        if (bucket == kDigits) return 1;
        const uint32_t count = s.bucket[bucket];
        high -= bucket << shift;
        low = max(low, high - min(high, (1u << shift) - 1));
        if (shift == 0 || above + count <= k + k / 8 + 32) return max(low, 1u);
        k -= above;
        __syncthreads();
    }
}

// A row's largest keys of groups, the first kMostGroups in registers.
struct Groups {
    const uint32_t* most;
    int count;
    uint32_t held[kHeld];
    __device__ __forceinline__ Groups(const SampleArgs& a, int64_t b)
        : most(a.groups + b * a.groups_of_row()), count(a.rules() ? a.groups_of_row() : 0) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = at(i * kThreads + threadIdx.x);
    }
    __device__ __forceinline__ uint32_t at(int g) const { return g < count ? most[g] : 0; }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) f(held[i]);
        for (int g = kMostGroups + threadIdx.x; g < count; g += kThreads) f(most[g]);
    }
};

// Where a lane's n entries go in an array that all waves fill: `filled` counts them.
__device__ __forceinline__ uint32_t append(uint32_t* filled, uint32_t n) {
    const uint32_t upto = wave_scan32(n), all = __builtin_amdgcn_readlane((int)upto, 63);
    uint32_t at = 0;
    if ((threadIdx.x & 63) == 63 && all) at = atomicAdd(filled, all);
    return (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + upto - n;
}

// f(tokens, keys of four from each on) for the tokens of the groups whose largest key is
// `least` (not 0) or more, by all threads, lanes of a wave together; waits before it and
// after.
constexpr int kAtOnce = 4;   // groups of a lane
template <int kDtype, typename F>
__device__ __forceinline__ void for_groups(const SampleArgs& a, int64_t b, const Groups& groups, uint32_t least,
                                           Shared& s, F f) {
    const int tid = threadIdx.x;
    constexpr int kLanes = kGroup / 4, kStep = kThreads / kLanes;   // four tokens a lane
    const int64_t size = kDtype == NB_F32 ? 4 : 2;
    const char* row = static_cast<const char*>(a.logits) + b * a.ld * size;
    for (int g0 = 0; g0 < groups.count; g0 += kMostGroups) {
        __syncthreads();
        if (tid == 0) s.some_groups = 0;
        __syncthreads();
        bool reach[kHeld];
        uint32_t count = 0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            reach[i] = (g0 ? groups.at(g0 + i * kThreads + tid) : groups.held[i]) >= least;
            count += reach[i];
        }
        uint32_t at = append(&s.some_groups, count);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (reach[i]) s.groups[at++] = (uint32_t)(g0 + i * kThreads + tid);
        }
        __syncthreads();
        const int some = (int)s.some_groups;
        for (int i0 = tid / kLanes; i0 - i0 % (64 / kLanes) < some; i0 += kStep * kAtOnce) {
            int v[kAtOnce];
            uint32_t keys[kAtOnce][4], x[kAtOnce][kDtype == NB_F32 ? 4 : 2];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const int at = i0 + i * kStep;
                v[i] = at < some ? (int)s.groups[at] * kGroup + tid % kLanes * 4 : a.V;
                if (v[i] + 3 < a.V) {
                    if constexpr (kDtype == NB_F32) {
                        const f4_any four = *reinterpret_cast<const f4_any*>(row + v[i] * size);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[i][e] = __float_as_uint(four[e]);
                    } else {
                        const u2_any four = *reinterpret_cast<const u2_any*>(row + v[i] * size);
                        x[i][0] = four[0], x[i][1] = four[1];
                    }
                } else {   // the row's end
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool there = v[i] + e < a.V;
                        if constexpr (kDtype == NB_F32) {
                            x[i][e] = there ? reinterpret_cast<const uint32_t*>(row)[v[i] + e] : 0xff800000u;
                        } else {
                            const uint32_t y = there ? reinterpret_cast<const bf16_bits*>(row)[v[i] + e] : 0xff80u;
                            x[i][e / 2] = e & 1 ? x[i][e / 2] | y << 16 : y;
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t y;
                    if constexpr (kDtype == NB_F32) y = x[i][e];
                    else y = e & 1 ? x[i][e / 2] & 0xffff0000u : x[i][e / 2] << 16;
                    keys[i][e] = key_of(__uint_as_float(y));
                }
            }
            f(v, keys);
        }
    }
    __syncthreads();
}

// Lists the tokens of groups from `least` on that take(key) names; how many they are,
// more than kMostListed: not all are listed.  kDense: many are, so a wave finds its room
// at once; else each token by itself (a row cut by top_p takes 1 us less of 29 so, rows
// cut by top_k 1.5 to 2 more, of 28 and 47).
template <int kDtype, bool kDense, typename Take>
__device__ __forceinline__ int list_tokens(const SampleArgs& a, int64_t b, const Groups& groups, uint32_t least,
                                           Shared& s, Take take) {
    if (threadIdx.x == 0) s.some = 0;
    for_groups<kDtype>(a, b, groups, least, s, [&](const int (&v)[kAtOnce], const uint32_t (&keys)[kAtOnce][4]) {
        uint32_t taken = 0, at = 0;
        if (kDense) {
#pragma unroll
            for (int i = 0; i < kAtOnce * 4; ++i) {
                if (take(keys[i / 4][i % 4])) taken |= 1u << i;
            }
            if (!__ballot(taken)) return;
            at = append(&s.some, __popc(taken));
        }
#pragma unroll
        for (int i = 0; i < kAtOnce * 4; ++i) {
            const uint32_t key = keys[i / 4][i % 4];
            if (kDense ? !(taken >> i & 1) : !key || !take(key)) continue;
            if (!kDense) at = atomicAdd(&s.some, 1u);
            if (at < kMostListed) s.list[at] = place_of(key, v[i / 4] + i % 4);
            ++at;
        }
    });
    return (int)s.some;
}

// Lists a row's first tokens, k or more of them (all, if they are fewer): a key that the
// largest of k groups reach is one that k tokens do, and all that reach it are in
// those groups.  Returns how many they are, over kMostListed: not all are listed.
template <int kDtype>
__device__ __forceinline__ int list_first(const SampleArgs& a, int64_t b, const Rules& r, const Groups& groups, Shared& s) {
    const uint32_t k = (uint32_t)r.k, high = key_of_place(r.first);
    uint32_t edge = edge_of(s, k, high, [&](auto f) { groups.each(f); });
    for (;;) {
        const int n = list_tokens<kDtype, true>(a, b, groups, edge, s, [&](uint32_t key) { return key >= edge; });
        if (n <= kMostListed) return n;
        // groups with many such tokens (neighbours that are alike): a key that k of those
        // that found room reach
        const uint32_t higher = edge_of(s, k, high, [&](auto f) {
            for (int i = threadIdx.x; i < kMostListed; i += kThreads) f(key_of_place(s.list[i]));
        });
        if (higher <= edge) return n;
        edge = higher;
    }
}

// A row's cuts from its bins, the sums of those that are kept whole into slice_sums.
__device__ __forceinline__ Cuts cuts_of_row(const SampleArgs& a, int64_t b, const Rules& r, Shared& s,
                            unsigned long long* slice_sums) {
    constexpr int kAll = kBins + 1;
    const int tid = threadIdx.x, lane = tid & 63;
    const uint64_t* sums = a.sums + b * a.slices * kAll;
    const uint32_t* counts = a.counts + b * a.slices * kAll;
    uint64_t sum = 0;
    uint32_t count = 0;
    if (tid < kAll) {
#pragma unroll 16
        for (int i = 0; i < a.slices; ++i) sum += sums[i * kAll + tid], count += counts[i * kAll + tid];
    }
    const Cuts c = find_cuts(r, sum, count, s.cuts);
    for (int i = tid >> 6; i < a.slices; i += kWaves) {   // a wave a slice
        uint64_t whole = 0;
#pragma unroll
        for (int bin = 0; bin < kAll; bin += 64) {
            if (bin + lane < min(c.sure(), kAll)) whole += sums[i * kAll + bin + lane];
        }
        whole = wave_sum(whole);
        if (lane == 0) slice_sums[i] = whole;
    }
    return c;
}

// The last kept token of the row (its place), of what top_k and top_p keep, by
// selection over the whole row: any number of tokens in a bin.
template <int kDtype>
__device__ uint64_t last_of_row(const SampleArgs& a, int64_t b, const Rules& r, Shared& s) {
    // kept: keys over `edge`, and the first `edge_ties` of those that equal it
    uint32_t edge = 1;
    uint64_t edge_ties = ~0ull;
    if (r.k) {
        uint64_t some = 0;
        for_row<kDtype>(a, b, [&](uint32_t key) { some += key != 0; });
        if ((uint64_t)r.k < block_sum(s, some)) {
            edge_ties = (uint64_t)r.k -
                        select<kDtype>(a, b, s, 1, (uint64_t)r.k, [](uint32_t) { return 1ull; }, edge);
        }
    }
    uint64_t ties = 0;
    if (r.p < 1.f) {
        uint64_t total = 0;
        for_row<kDtype>(a, b, [&](uint32_t key) {
            if (key > edge) total += r.w.of(key);
            ties += key == edge;
        });
        total = block_sum(s, total);
        ties = block_sum(s, ties);
        total += lesser(ties, edge_ties) * r.w.of(edge);
        const uint64_t bound = share_of(r.p, total);
        uint32_t at = 0;
        const uint64_t above = select<kDtype>(a, b, s, edge, bound, [&](uint32_t key) { return r.w.of(key); }, at);
        const uint64_t each = r.w.of(at);   // (not 0: the sum reached the bound with it)
        const uint64_t need = (bound - above + each - 1) / each;
        edge_ties = at == edge ? lesser(edge_ties, need) : need;
        edge = at;
    }
    if (edge == 1) return 0;
    // the token of the last tie: waves count those of their part of the row
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = ((a.V + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int begin = min(wave * each, a.V), end = min(begin + each, a.V);
    ties = 0;
    for (int v = begin + lane; v < end; v += 64) ties += key_at<kDtype>(a, b, v) == edge;
    ties = wave_sum(ties);
    __syncthreads();
    if (lane == 0) s.ties[wave] = ties;
    if (tid == 0) s.found[0] = 0xffffffffu;   // (all ties are kept)
    __syncthreads();
    uint64_t before = 0;
    for (int i = 0; i < wave; ++i) before += s.ties[i];
    if (before < edge_ties && before + ties >= edge_ties) {   // one wave
        for (int v0 = begin; v0 < end; v0 += 64) {
            const int v = v0 + lane;
            const uint64_t tied = __ballot(v < end && key_at<kDtype>(a, b, min(v, end - 1)) == edge);
            const uint64_t rank = before + __popcll(tied & ((1ull << lane) - 1));
            if ((tied >> lane & 1) && rank + 1 == edge_ties) s.found[0] = (uint64_t)v;
            before += __popcll(tied);
            if (before >= edge_ties) break;
        }
    }
    __syncthreads();
    const uint64_t v = s.found[0];
    return v == 0xffffffffu ? (uint64_t)edge << 32 : place_of(edge, (int)v);
}

// Sorts n listed tokens into the order: into buckets of neighbouring keys, and by
// counting in a bucket.
__device__ void sort_list(Shared& s, int n) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    static_assert(kDigits == 2 * kThreads, "two buckets a thread");
    s.bucket[2 * tid] = s.bucket[2 * tid + 1] = 0;
    if (tid == 0) s.key_low = ~0u, s.key_high = 0;
    __syncthreads();
    uint32_t low = ~0u, high = 0;
    for (int i = tid; i < n; i += kThreads) {
        const uint32_t key = key_of_place(s.list[i]);
        low = min(low, key), high = max(high, key);
    }
    low = ~(uint32_t)wave_max(~low), high = (uint32_t)wave_max(high);
    if (lane == 0) atomicMin(&s.key_low, low), atomicMax(&s.key_high, high);
    __syncthreads();
    high = s.key_high;
    const int shift = max(32 - __clz((int)(high - s.key_low)) - 11, 0);
    auto bucket_of = [&](uint64_t place) { return (high - key_of_place(place)) >> shift; };
    for (int i = tid; i < n; i += kThreads) atomicAdd(&s.bucket[bucket_of(s.list[i])], 1u);
    __syncthreads();
    const uint32_t first = s.bucket[2 * tid], both = first + s.bucket[2 * tid + 1];
    uint32_t upto = wave_scan32(both);
    if (lane == 63) s.part[wave] = upto;
    __syncthreads();
    for (int i = 0; i < wave; ++i) upto += (uint32_t)s.part[i];
    s.bucket[2 * tid] = upto - both, s.bucket[2 * tid + 1] = upto - both + first;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t place = s.list[i];
        s.sorted[atomicAdd(&s.bucket[bucket_of(place)], 1u)] = place;   // (in the end a bucket's end)
    }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t place = s.sorted[i];
        const int bucket = (int)bucket_of(place), end = (int)s.bucket[bucket];
        const int begin = bucket ? (int)s.bucket[bucket - 1] : 0;
        int rank = begin;
        for (int j = begin; j < end; ++j) rank += s.sorted[j] > place;
        s.list[rank] = place;
    }
    __syncthreads();
}

// Listed tokens of a thread, and their weights: 0 if they are not kept.
constexpr int kEach = kMostListed / kThreads;
struct Own {
    uint64_t place[kEach], weight[kEach];
};

// The same by up to 64 listed tokens, by one wave; their kept weights are added to their
// slices' sums.
__device__ uint64_t last_of_few(const SampleArgs& a, const Rules& r, const Cuts& c, uint64_t* list, int n,
                                unsigned long long* slice_sums, Own& own) {
    const int lane = threadIdx.x & 63;
    uint64_t place = lane < n ? list[lane] : 0;
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += list[j] > place;
    // into the order
    wave_lds_order();
    if (lane < n) list[rank] = place;
    wave_lds_order();
    place = lane < n ? list[lane] : 0;
    const uint32_t key = key_of_place(place);
    const double z = key ? r.w.log2_of(key) : 0.0;
    const uint64_t weight = key ? r.w.of_log2(z) : 0;
    const int bin = key ? c.bin(z) : kBins + 2;
    const uint64_t number = c.above_k + lane - __popcll(__ballot(bin < c.k));   // (of bin k's)
    const bool in_k = bin < c.k || (bin == c.k && number < (uint64_t)r.k);
    bool kept = place && in_k;
    if (r.p < 1.f) {
        const uint64_t bound = share_of(r.p, c.sum_k + wave_sum(bin == c.k && in_k ? weight : 0));
        const bool inside = bin >= c.p_low && bin <= c.p_high;
        const uint64_t upto = wave_scan(inside ? weight : 0);
        kept = kept && (bin < c.p_low || (inside && c.above_p + upto - weight < bound));
    }
    if (kept && weight >= r.least) {
        atomicAdd(&slice_sums[token_of_place(place) / a.length], (unsigned long long)weight);
        own.place[0] = place, own.weight[0] = weight;
    }
    if (c.k > kBins && !(r.p < 1.f)) return 0;   // (min_p alone)
    const uint64_t all = __ballot(kept);
    return all ? lane_of(place, 63 - __clzll((long long)all)) : 0;
}

// The same by the listed tokens of a workgroup, kMine a thread.
template <int kMine>
__device__ uint64_t last_of_list(const SampleArgs& a, const Rules& r, const Cuts& c, Shared& s, int n,
                                 unsigned long long* slice_sums) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    sort_list(s, n);
    uint64_t place[kMine], weight[kMine];
    int bin[kMine];
    uint64_t first_k = 0, in_p = 0;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const int i = tid * kMine + e;
        place[e] = i < n ? s.list[i] : 0;
        const uint32_t key = key_of_place(place[e]);
        const double z = key ? r.w.log2_of(key) : 0.0;
        weight[e] = key ? r.w.of_log2(z) : 0;
        bin[e] = key ? bin_of(z) : kBins + 2;
        first_k += bin[e] < c.k;   // listed tokens before bin k
        if (bin[e] >= c.p_low && bin[e] <= c.p_high) in_p += weight[e];
    }
    uint64_t kept_k = 0;
    if (c.k <= kBins) {
        first_k = block_sum(s, first_k);
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            const uint64_t rank = c.above_k + (uint64_t)(tid * kMine + e) - first_k;
            if (bin[e] == c.k && rank < (uint64_t)r.k) kept_k += weight[e];
        }
    }
    kept_k = block_sum(s, kept_k);
    const uint64_t bound = r.p < 1.f ? share_of(r.p, c.sum_k + kept_k) : 0;
    // weights of the order before a token, over p_low's bin
    uint64_t upto = wave_scan(in_p);
    __syncthreads();
    if (lane == 63) s.part[wave] = upto;
    __syncthreads();
    uint64_t before = c.above_p + upto - in_p;
    for (int i = 0; i < wave; ++i) before += s.part[i];
    uint64_t last = 0;    // the largest number of a token that top_k and top_p keep
    bool kept[kMine];
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const uint64_t i = (uint64_t)(tid * kMine + e), rank = c.above_k + i - first_k;
        kept[e] = place[e] && (bin[e] < c.k || (bin[e] == c.k && rank < (uint64_t)r.k));
        if (r.p < 1.f) {
            const bool inside = bin[e] >= c.p_low && bin[e] <= c.p_high;
            kept[e] = kept[e] && (bin[e] < c.p_low || (inside && before < bound));
            if (inside) before += weight[e];
        }
        if (kept[e]) last = i + 1;
        if (kept[e] && weight[e] >= r.least && bin[e] >= c.sure()) {
            atomicAdd(&slice_sums[token_of_place(place[e]) / a.length], (unsigned long long)weight[e]);
        }
    }
    if (c.k > kBins && !(r.p < 1.f)) return 0;   // (min_p alone)
    last = wave_max(last);
    __syncthreads();
    if (lane == 0) s.part[wave] = last;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) last = s.part[i] > last ? s.part[i] : last;
    return s.list[last - 1];
}

__device__ __forceinline__ float logprob_of(const Rules& r, uint32_t key, uint64_t total) {
    return (float)(r.w.log2_of(key) * 0.6931471805599453 - log((double)total / (double)(1ull << r.w.shift)));
}

// The kept ones of the n first tokens of a row (few_kept), of a thread kMine; their weights
// are added to their slices' sums.
template <int kMine>
__device__ void keep_first(const SampleArgs& a, const Rules& r, Shared& s, int n, unsigned long long* slice_sums,
                           Own& own) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t weight[kMine], sum = 0;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        const int i = tid * kMine + e;
        own.place[e] = i < n && i < r.k ? s.list[i] : 0;
        weight[e] = own.place[e] ? r.w.of(key_of_place(own.place[e])) : 0;
        sum += weight[e];
    }
    uint64_t upto = wave_scan(sum), total = 0;
    if (lane == 63) s.part[wave] = upto;
    __syncthreads();
    uint64_t before = upto - sum;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const uint64_t part = s.part[i];
        total += part;
        if (i < wave) before += part;
    }
    const uint64_t bound = r.p < 1.f ? share_of(r.p, total) : ~0ull;
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        own.weight[e] = before < bound && weight[e] >= r.least ? weight[e] : 0;
        before += weight[e];
        if (own.weight[e]) {
            atomicAdd(&slice_sums[token_of_place(own.place[e]) / a.length], (unsigned long long)own.weight[e]);
        }
    }
}

template <int kDtype>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a) {
    __shared__ Shared s;
    __shared__ unsigned long long slice_sums[kMostSlices];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t b = blockIdx.x, slice0 = b * a.slices;
    const float u = as_constant(a.u)[b];
    const bool rules = a.rules(), few = a.few_kept(b);
    const Groups most(a, b);   // (asked for ahead of the rules)
    if (tid < kMostSlices) slice_sums[tid] = !rules && tid < a.slices ? a.sums[slice0 + tid] : 0;
    make_table(s.table);
    const Rules r(a, b, s.table);
    if (r.first == 0 || r.greedy) {
        if (tid == 0) {
            a.tokens[b] = r.first ? token_of_place(r.first) : -1;
            if (a.logprobs) a.logprobs[b] = r.first ? 0.f : -INFINITY;
        }
        return;
    }
    Kept kept{0, r.least};
    bool known = true;   // slice_sums are those of kept weights
    Cuts c{};
    Own own{};
    if (rules) {
        __syncthreads();
        int listed = 0;
        if (few) {
            listed = list_first<kDtype>(a, b, r, most, s);
            c.one = true;
        } else {
            c = cuts_of_row(a, b, r, s, slice_sums);
            if (!(c.low > c.high)) {
                listed = list_tokens<kDtype, false>(a, b, most, max(key_of(c.low), 1u), s, [&](uint32_t key) {
                    const float x = logit_of(key);
                    return !(x < c.low || x > c.high) && c.listed(bin_of(r.w.log2_of(key)));   // (T = inf: no high)
                });
            } else {
                __syncthreads();
            }
        }
        known = listed <= kMostListed;
        if (!known) {
            kept.last = last_of_row<kDtype>(a, b, r, s);
        } else if (listed <= 64) {
            if (wave == 0) {
                const uint64_t last = last_of_few(a, r, c, s.list, listed, slice_sums, own);
                if (lane == 0) s.found[0] = last;
            }
            __syncthreads();
            kept.last = s.found[0];
        } else if (few) {
            sort_list(s, listed);
            if (r.k <= kThreads) keep_first<1>(a, r, s, listed, slice_sums, own);
            else keep_first<kFewKept / kThreads>(a, r, s, listed, slice_sums, own);
        } else {
            kept.last = listed <= kThreads ? last_of_list<1>(a, r, c, s, listed, slice_sums)
                                           : last_of_list<kEach>(a, r, c, s, listed, slice_sums);
        }
    }
    __syncthreads();
    if (!known) {   // the slices' sums, a wave a slice
        for (int i = wave; i < a.slices; i += kWaves) {
            const int lo = i * a.length, hi = min(lo + a.length, a.V);
            uint64_t sum = 0;
            for (int v = lo + lane; v < hi; v += 64) sum += kept.weight(r.w, key_at<kDtype>(a, b, v), v);
            sum = wave_sum(sum);
            if (lane == 0) slice_sums[i] = sum;
        }
        __syncthreads();
    }
    // the slice that u falls in: two slices a lane, every wave by itself
    const uint64_t s0 = slice_sums[2 * lane], s1 = slice_sums[2 * lane + 1];
    const uint64_t sums = wave_scan(s0 + s1), total = lane_of(sums, 63);
    // u of it, rounded down: u in 64 bits of fraction, exact
    const uint64_t fraction = u >= 1.f ? ~0ull : u > 0.f ? (uint64_t)((double)u * 18446744073709551616.0) : 0;
    uint64_t rest = __umul64hi(fraction, total);
    const int pair = __popcll(__ballot(sums <= rest));   // (under 64: rest is under the total)
    const uint64_t before = lane_of(sums - s0 - s1, pair), first = lane_of(s0, pair);
    rest -= before;
    int part = 2 * pair;
    if (rest >= first) rest -= first, ++part;
    if (c.one && known) {
        // all kept tokens are at hand: those of the slice, with the weights before them
        if (tid == 0) s.some = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (!own.weight[e] || token_of_place(own.place[e]) / a.length != part) continue;
            const uint32_t at = atomicAdd(&s.some, 1u);
            s.list[2 * at] = ~own.place[e] & 0xffffffffu, s.list[2 * at + 1] = own.weight[e];
        }
        __syncthreads();
        const int n = (int)s.some;
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t v = s.list[2 * i], weight = s.list[2 * i + 1];
            uint64_t upto = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) upto += s.list[2 * j] < v ? s.list[2 * j + 1] : 0;
            if (upto <= rest && rest - upto < weight) {   // one token
                a.tokens[b] = (int)v;
                if (a.logprobs) a.logprobs[b] = logprob_of(r, key_at<kDtype>(a, b, (int)v), total);
            }
        }
        return;
    }
    // the slice is split over the waves, a large one's part with the token again
    int lo = part * a.length, hi = min(lo + a.length, a.V);
    constexpr int kInHand = 16;   // groups of 64 tokens of a wave
    while (hi - lo > kThreads * kInHand) {
        const int each = ((hi - lo + kWaves - 1) / kWaves + 63) / 64 * 64;
        const int begin = min(lo + wave * each, hi), end = min(begin + each, hi);
        uint64_t sum = 0;
#pragma unroll 4
        for (int v = begin + lane; v < end; v += 64) sum += kept.weight(r.w, key_at<kDtype>(a, b, v), v);
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) s.part[wave] = sum;
        __syncthreads();
        for (part = 0; part < kWaves - 1 && rest >= s.part[part]; ++part) rest -= s.part[part];
        lo = min(lo + part * each, hi);
        hi = min(lo + each, hi);
    }
    // then its weights are in registers, 64 neighbours in those of a number
    const int groups = (hi - lo + kThreads - 1) / kThreads;   // of a wave
    const int begin = lo + wave * groups * 64;
    uint64_t weights[kInHand], sum = 0;
    {
        uint32_t keys[kInHand];
#pragma unroll
        for (int g = 0; g < kInHand; ++g) {
            const int v = begin + g * 64 + lane;
            keys[g] = g < groups && v < hi ? key_at<kDtype>(a, b, v) : 0;
        }
#pragma unroll
        for (int g = 0; g < kInHand; ++g) {
            weights[g] = g < groups ? kept.weight(r.w, keys[g], begin + g * 64 + lane) : 0;
            sum += weights[g];
        }
    }
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) s.part[wave] = sum;
    __syncthreads();
    for (part = 0; part < kWaves - 1 && rest >= s.part[part]; ++part) rest -= s.part[part];
    if (wave != part) return;
#pragma unroll
    for (int g = 0; g < kInHand; ++g) {
        const uint64_t upto = wave_scan(weights[g]), all = lane_of(upto, 63);
        if (rest < all) {
            if (upto > rest && upto - weights[g] <= rest) {   // one lane
                const int v = begin + g * 64 + lane;
                a.tokens[b] = v;
                if (a.logprobs) a.logprobs[b] = logprob_of(r, key_at<kDtype>(a, b, v), total);
            }
            return;
        }
        rest -= all;
    }
}

// Slices of a row: up to 16 of at least 4096 tokens (a batch of loads is 8192, and a
// thread of the cuts reads a bin of 16 slices at once), of at most 16384 while that
// makes no more than kMostSlices.
struct Slices {
    int count, length;
};
Slices slices_of(int V) {
    int64_t length = std::min<int64_t>(std::max<int64_t>(((V + 15) / 16 + 2047) / 2048 * 2048, 4096), 1 << 14);
    while (((int64_t)V + length - 1) / length > kMostSlices) length *= 2;
    return {(int)(((int64_t)V + length - 1) / length), (int)length};
}

int shift_of(int V) {   // a row's sum stays under 2^63
    int bits = 0;
    while ((int64_t)1 << bits < V) ++bits;
    return std::min(45, 62 - bits);
}

}  // namespace

int64_t sample_bytes(int rows, int V) {
    const int64_t slices = (int64_t)rows * slices_of(V).count;
    return rows * (((int64_t)V + kGroup - 1) / kGroup) * 4 + slices * (8 + (kBins + 1) * (8 + 4));
}

int launch_sample(const void* logits, int dtype, int64_t ld, int rows, int V, const float* u,
                  const float* temperature, const int32_t* top_k, const float* top_p,
                  const float* min_p, int32_t* tokens, float* logprobs, void* workspace,
                  hipStream_t stream) {
    const Slices cut = slices_of(V);
    const int64_t slices = (int64_t)rows * cut.count;
    SampleArgs a{logits, ld, V, shift_of(V), cut.count, cut.length, u, temperature, top_k, top_p, min_p,
                 tokens, logprobs};
    a.first = static_cast<uint64_t*>(workspace);
    a.sums = a.first + slices;
    a.counts = reinterpret_cast<uint32_t*>(a.sums + slices * (kBins + 1));
    a.groups = a.counts + slices * (kBins + 1);
    const dim3 grid(cut.count, rows);
    auto run = [&](auto type) {
        constexpr int kDtype = decltype(type)::value;
        auto* most = a.rules() ? sample_max_kernel<kDtype, true> : sample_max_kernel<kDtype, false>;
        hipLaunchKernelGGL(most, grid, dim3(kSliceThreads), 0, stream, a);
        auto* bins = a.rules() ? sample_bins_kernel<kDtype, true> : sample_bins_kernel<kDtype, false>;
        hipLaunchKernelGGL(bins, grid, dim3(kSliceThreads), 0, stream, a);
        hipLaunchKernelGGL(sample_finish_kernel<kDtype>, dim3(rows), dim3(kThreads), 0, stream, a);
    };
    if (dtype == NB_F32) run(std::integral_constant<int, NB_F32>{});
    else run(std::integral_constant<int, NB_BF16>{});
    return check_launch("nb_sample");
}

}  // namespace nb
