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
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "nb_device.h"
#include "nb_internal.h"

namespace nb {
namespace {

struct SampleArgs {
    const void* logits;
    int64_t ld;
    int dtype, V, shift;   // shift: S
    const float *u, *temperature;
    const int32_t* top_k;
    const float *top_p, *min_p;
    int32_t* tokens;
    float* logprobs;
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

__device__ __forceinline__ uint32_t key_at(const SampleArgs& a, int64_t b, int v) {
    const int64_t at = b * a.ld + v;
    return key_of(a.dtype == NB_F32 ? static_cast<const float*>(a.logits)[at]
                                    : bf16_to_f32(static_cast<const bf16_bits*>(a.logits)[at]));
}

constexpr int kFractions = 32;   // entries of 2^(i / 32)

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
    // (|r| <= 1/64: its next term is 2e-15)
    __device__ __forceinline__ uint64_t of(uint32_t key) const {
        if (key == 0) return 0;
        const double z = log2_of(key);
        constexpr double kMagic = 6755399441055744.0;   // 1.5 * 2^52: rounds to a whole number
        const double y = z * kFractions + kMagic;
        const int n = __double2loint(y);
        const double r = z - (y - kMagic) * (1.0 / kFractions);
        double p = 0.0013333558146428443;
        p = fma(p, r, 0.009618129107628477);
        p = fma(p, r, 0.05550410866482158);
        p = fma(p, r, 0.2402265069591007);
        p = fma(p, r, 0.6931471805599453);
        p = fma(p, r, 1.0);
        p = ldexp(p * table[n & (kFractions - 1)], (n >> 5) + shift);
        return (uint64_t)__double_as_longlong(p + 4503599627370496.0) - 0x4330000000000000ull;
    }
};

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

struct Shared {
    double table[kFractions];
    uint64_t bins[kBins];
    uint64_t part[kWaves], ties[kWaves];
    uint64_t found[3];
};

__device__ __forceinline__ uint64_t lesser(uint64_t x, uint64_t y) { return x < y ? x : y; }
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor((unsigned long long)v, d);
    return v;
}
// The sum over the workgroup, in all threads.
__device__ uint64_t block_sum(Shared& s, uint64_t v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
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
    constexpr int kEach = kBins / kThreads;
    const int tid = threadIdx.x, lane = tid & 63;
    // thread t takes the bins from the t-th largest pair on
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine += s.bins[kBins - 1 - (tid * kEach + i)];
    uint64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)upto, d);
        if (lane >= d) upto += o;
    }
    __syncthreads();
    if (lane == 63) s.part[tid >> 6] = upto;
    if (tid == 0) s.found[0] = 0, s.found[1] = 0;
    __syncthreads();
    uint64_t above = upto - mine;
    for (int i = 0; i < (tid >> 6); ++i) above += s.part[i];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int bin = kBins - 1 - (tid * kEach + i);
        const uint64_t n = s.bins[bin];
        if (above < bound && above + n >= bound) {
            s.found[0] = (uint64_t)bin, s.found[1] = above;
        }
        above += n;
    }
    __syncthreads();
    return Crossing{(int)s.found[0], s.found[1]};
}

// The key at which the order's sum of `value(key)` over keys >= least first
// reaches `bound` (> 0, at most the sum of all), and the sum above that key.
template <typename Value>
__device__ uint64_t select(const SampleArgs& a, int64_t b, Shared& s, uint32_t least, uint64_t bound,
                           Value value, uint32_t& at) {
    uint64_t above = 0;
    uint32_t prefix = 0, mask = 0;
    for (int shift = 21; shift >= -1; shift -= 11) {   // 11, 11 and 10 bits
        const int low = max(shift, 0), bits = shift < 0 ? 10 : 11;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins[i] = 0;
        __syncthreads();
        for (int v = threadIdx.x; v < a.V; v += kThreads) {
            const uint32_t key = key_at(a, b, v);
            if (key && key >= least && (key & mask) == prefix) {
                atomicAdd((unsigned long long*)&s.bins[key >> low & ((1u << bits) - 1)],
                          (unsigned long long)value(key));
            }
        }
        __syncthreads();
        const Crossing c = cross(s, bound - above);
        above += c.above;
        prefix |= (uint32_t)c.bin << low;
        mask |= ((1u << bits) - 1) << low;
    }
    at = prefix;
    return above;
}

// One row.
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t b = blockIdx.x;
    const float t = a.temperature ? a.temperature[b] : 1.f;
    const bool greedy = !(t > 0.f);
    if (tid < kFractions) s.table[tid] = exp2((double)tid / kFractions);
    // the maximum
    uint32_t top = 0;
    for (int v = tid; v < a.V; v += kThreads) top = max(top, key_at(a, b, v));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if (lane == 0) s.part[wave] = top;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) top = max(top, (uint32_t)s.part[i]);
    if (top == 0) {   // nothing is left
        if (tid == 0) {
            a.tokens[b] = -1;
            if (a.logprobs) a.logprobs[b] = -INFINITY;
        }
        return;
    }
    Weights w;
    w.most = (double)logit_of(top);
    w.turn = 1.4426950408889634 / (greedy ? 1.0 : (double)t);
    w.table = s.table;
    w.shift = a.shift;
    // kept: keys over `edge`, and the first `edge_ties` of those that equal it
    uint32_t edge = 1;
    uint64_t edge_ties = ~0ull;
    const int64_t k = greedy ? 1 : a.top_k ? a.top_k[b] : 0;
    if (k > 0 && k < a.V) {
        uint64_t some = 0;
        for (int v = tid; v < a.V; v += kThreads) some += key_at(a, b, v) != 0;
        some = block_sum(s, some);
        if ((uint64_t)k < some) {
            const uint64_t above = select(a, b, s, 1, (uint64_t)k, [](uint32_t) { return 1ull; }, edge);
            edge_ties = (uint64_t)k - above;
        }
    }
    const float p = a.top_p ? a.top_p[b] : 1.f;
    if (p < 1.f) {
        uint64_t total = 0, ties = 0;
        for (int v = tid; v < a.V; v += kThreads) {
            const uint32_t key = key_at(a, b, v);
            if (key > edge) total += w.of(key);
            ties += key == edge;
        }
        total = block_sum(s, total);
        ties = block_sum(s, ties);
        total += lesser(ties, edge_ties) * w.of(edge);
        // (at least the first of the order)
        const uint64_t bound = p > 0.f ? lesser((uint64_t)fmax(ceil((double)p * (double)total), 1.0), total) : 1;
        uint32_t at = 0;
        const uint64_t above = select(a, b, s, edge, bound, [&](uint32_t key) { return w.of(key); }, at);
        const uint64_t each = w.of(at);   // (not 0: the sum reached the bound with it)
        const uint64_t need = (bound - above + each - 1) / each;
        edge_ties = at == edge ? lesser(edge_ties, need) : need;
        edge = at;
    }
    const float mp = a.min_p ? a.min_p[b] : 0.f;
    const uint64_t one = 1ull << a.shift;
    const uint64_t least = mp > 0.f ? (uint64_t)ceil(fmin((double)mp, 1.0) * (double)one) : 0;
    const uint64_t edge_weight = w.of(edge);
    // the sum of kept weights by index: a range is split over the waves, the part
    // with the token split again
    int lo = 0, hi = a.V;
    uint64_t ties_before = 0, rest = 0, total = 0;
    bool first = true;
    while (hi - lo > 64 || first) {
        const int each = max(((hi - lo + kWaves - 1) / kWaves + 63) / 64 * 64, 64);
        const int begin = min(lo + wave * each, hi), end = min(begin + each, hi);
        uint64_t sum = 0, ties = 0;
        for (int v = begin + lane; v < end; v += 64) {
            const uint32_t key = key_at(a, b, v);
            if (key > edge) {
                const uint64_t n = w.of(key);
                sum += n >= least ? n : 0;
            }
            ties += key == edge;
        }
        sum = wave_sum(sum);
        ties = wave_sum(ties);
        __syncthreads();
        if (lane == 0) s.part[wave] = sum, s.ties[wave] = ties;
        __syncthreads();
        auto kept_ties = [&](uint64_t before, uint64_t n) {   // of n after `before`
            return edge_weight < least || before >= edge_ties ? 0 : lesser(n, edge_ties - before);
        };
        if (first) {
            uint64_t before = 0;
            for (int i = 0; i < kWaves; ++i) {
                total += s.part[i] + kept_ties(before, s.ties[i]) * edge_weight;
                before += s.ties[i];
            }
            // u of it, rounded down: u in 64 bits of fraction, exact
            const float u = a.u[b];
            const uint64_t fraction = u >= 1.f ? ~0ull : u > 0.f ? (uint64_t)((double)u * 18446744073709551616.0) : 0;
            rest = __umul64hi(fraction, total);
            first = false;
        }
        int part = 0;
        for (;; ++part) {
            const uint64_t n = s.part[part] + kept_ties(ties_before, s.ties[part]) * edge_weight;
            if (rest < n || part == kWaves - 1) break;
            rest -= n;
            ties_before += s.ties[part];
        }
        lo = min(lo + part * each, hi);
        hi = min(lo + each, hi);
    }
    if (wave) return;
    const int v = lo + lane;
    const uint32_t key = v < hi ? key_at(a, b, v) : 0;
    const uint64_t tied = __ballot(key == edge);
    const uint64_t rank = ties_before + __popcll(tied & ((1ull << lane) - 1));
    uint64_t mine = key > edge || (key == edge && rank < edge_ties) ? w.of(key) : 0;
    if (mine < least) mine = 0;
    uint64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)upto, d);
        if (lane >= d) upto += o;
    }
    if (upto > rest && upto - mine <= rest) {   // one lane
        a.tokens[b] = v;
        if (a.logprobs) {
            a.logprobs[b] = (float)(w.log2_of(key) * 0.6931471805599453 -
                                    log((double)total / (double)one));
        }
    }
}

}  // namespace

int sample_shift(int V) {   // a row's sum stays under 2^63
    int bits = 0;
    while ((int64_t)1 << bits < V) ++bits;
    return std::min(45, 62 - bits);
}

int64_t sample_bytes(int, int) { return 0; }

int launch_sample(const void* logits, int dtype, int64_t ld, int rows, int V, const float* u,
                  const float* temperature, const int32_t* top_k, const float* top_p,
                  const float* min_p, int32_t* tokens, float* logprobs, void*, hipStream_t stream) {
    const SampleArgs a{logits, ld, dtype, V, sample_shift(V), u, temperature, top_k, top_p, min_p,
                       tokens, logprobs};
    hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(kThreads), 0, stream, a);
    return check_launch("nb_sample");
}

}  // namespace nb
