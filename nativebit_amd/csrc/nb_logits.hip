// Rules on a batch of logits and the greedy choice (gfx950): nb_logits_rules.
//
// For row b and token v, with seen(v): v is in history[b][0 .. len), and n(v)
// its occurrences in history[b][prompt .. len):
//     x = logits[b][v]
//     x = x > 0 ? x / repetition[b] : x * repetition[b]     where seen(v)
//     x = (x - frequency[b] * n(v)) - presence[b] (n(v) > 0)
//     x = x + bias[b][i], i the last with bias_ids[b][i] = v
//     x = -inf                                where bit v of mask[b] is 0
// each operation rounded by itself in fp32, and tokens[b] the lowest v with
// the largest x (-1 where no x is over -inf; a NaN is never chosen).
//
// Bound by memory: one pass over the logits.  A workgroup takes 1024 or 2048
// tokens of a row; it issues the loads of their logits, counts the row's history
// in an LDS word per token and notes the biases beside it while they are under
// way, so that neither counts nor dense biases exist in memory.  Every workgroup
// of a row walks its whole history, from the L2: against 16 KB of logits read
// and written, a history of 1000 is 4 KB.  LDS atomics are on whole numbers
// (sums, or, maximum): no result depends on their order.  160 fp32 rows of
// 131077, three inputs in turn, both launches: 42 us with histories of 1000 (4.1
// TB/s), 49 with 4000; on one input, part of it in the last level cache, 37 and 42
// (40 and 44 with the masks' bits made beside their loads, which waited for
// each); one row of 50257 6.2.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "nb_device.h"
#include "nb_internal.h"

// Products and sums round one by one (no fused multiply-add, which the
// compiler makes of __fmul_rn and __fadd_rn too).
#pragma clang fp contract(off)

namespace nb {
namespace {

typedef __attribute__((ext_vector_type(4))) float f4;
// (logits at any of their elements' places: one access all the same)
typedef __attribute__((ext_vector_type(4), aligned(4))) float f4_any;
typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t u2_any;

constexpr int kThreads = 256;
// Tokens of a workgroup: one group of four for each thread up to 2^20 logits
// (more workgroups, each sooner done), two above (half as many that walk a
// history).  With histories of 700 to 1000, both launches, in us: 1 row of 50257
// 5.7 (two 6.8), 8 rows 6.5 (7.5); 16 rows of 131077 9.9 (one 10.8), 160 rows 40
// (48), with histories of 4000 44 (57; four groups, with 32 KB of LDS, 52).  512
// threads with two groups: 42 for those, but 10.3 for the 16 rows.  (Both sides
// of an earlier step, 3 to 7 % slower than now.)
constexpr int tokens_of(int loads) { return 4 * kThreads * loads; }
int loads_of(int rows, int V) { return (int64_t)rows * V <= 1 << 20 ? 1 : 2; }
// An LDS word per token: seen in the history, has a bias, times in the answer.
constexpr uint32_t kSeen = 0x80000000u, kBias = 0x40000000u, kTimes = 0x3fffffffu;

struct LogitsArgs {
    const void* logits;
    int64_t ld, ld_out, ld_history, ld_bias, ld_mask;
    const int32_t *history, *lens, *prompt_lens;
    const float *repetition, *frequency, *presence;
    const int32_t* bias_ids;
    const float* bias;
    const int32_t* mask;
    float* out;
    uint64_t* keys;
    int32_t* tokens;
    int V, max_history, n_bias;
};

// Larger for larger values, and for the lower of equal tokens; 0 for -inf and NaN.
__device__ __forceinline__ uint64_t key_of(float x, int v) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.f);   // (-0 as 0)
    const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)order << 32 | (0xffffffffu - (uint32_t)v);
}
__device__ __forceinline__ int token_of(uint64_t key) {
    return key ? (int)(0xffffffffu - (uint32_t)key) : -1;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t key) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)key, d);
        key = o > key ? o : key;
    }
    return key;
}

// kDtype: the logits' type.  Groups of four begin at 16-byte places of the
// output's row: all but its first and last move as vectors.
template <int kDtype, int kLoads>
__global__ __launch_bounds__(kThreads) void logits_rules_kernel(LogitsArgs a) {
    constexpr int kTokens = tokens_of(kLoads);
    __shared__ __align__(16) uint32_t count[kTokens];
    __shared__ int32_t bias_at[kTokens];   // the place of the token's bias, where it has one
    __shared__ uint64_t wave_keys[kThreads / 64];
    const int b = blockIdx.y, tid = threadIdx.x;
    using In = std::conditional_t<kDtype == NB_F32, float, bf16_bits>;
    const In* in = static_cast<const In*>(a.logits) + b * a.ld;
    float* out = a.out + b * a.ld_out;
    // group q of four elements holds tokens 4 q - shift ..
    const int shift = (int)(reinterpret_cast<uintptr_t>(out) / 4 & 3);
    const int v0 = (int)blockIdx.x * kTokens - shift;   // (V <= 2^30)
    // everything that the row's rules read is asked for before it is used: the
    // lengths, the first history entries and biases, the logits, the masks
    const int32_t* hist = a.history ? a.history + b * a.ld_history : nullptr;
    const int len = hist ? min(max(as_constant(a.lens)[b], 0), a.max_history) : 0;
    const int prompt = hist && a.prompt_lens ? as_constant(a.prompt_lens)[b] : 0;
    const float rep = a.repetition ? as_constant(a.repetition)[b] : 1.f;
    const float freq = a.frequency ? as_constant(a.frequency)[b] : 0.f;
    const float pres = a.presence ? as_constant(a.presence)[b] : 0.f;
    constexpr int kBatch = 8;   // history entries of a thread under way at once
    int ids[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
        ids[j] = a.max_history > 0 && hist ? hist[min(tid + j * kThreads, a.max_history - 1)] : -1;
    }
    const int bias_id = tid < a.n_bias ? a.bias_ids[b * a.ld_bias + tid] : -1;
    f4 x[kLoads];
    uint32_t m0[kLoads], m1[kLoads];   // the mask's words from the group's first token on
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int v = v0 + 4 * (tid + j * kThreads);
        // (bf16 stay pairs until they are needed, so that no load is waited for here)
        if (v >= 0 && v + 3 < a.V) {
            if constexpr (kDtype == NB_F32) {
                x[j] = *reinterpret_cast<const f4_any*>(in + v);
            } else {
                const u2_any w = *reinterpret_cast<const u2_any*>(in + v);
                x[j] = f4{__uint_as_float(w[0]), __uint_as_float(w[1]), 0.f, 0.f};
            }
        } else {
            In e4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) e4[e] = v + e >= 0 && v + e < a.V ? in[v + e] : In{};
            if constexpr (kDtype == NB_F32) {
                x[j] = f4{e4[0], e4[1], e4[2], e4[3]};
            } else {
                x[j] = f4{__uint_as_float(e4[0] | (uint32_t)e4[1] << 16),
                          __uint_as_float(e4[2] | (uint32_t)e4[3] << 16), 0.f, 0.f};
            }
        }
        m0[j] = m1[j] = 0xffffffffu;
        if (a.mask) {   // (a group that is not aligned may reach into the next word)
            const int32_t* mask = a.mask + b * a.ld_mask;
            const int last = (a.V - 1) >> 5, w = max(v, 0) >> 5;
            m0[j] = mask[min(w, last)];
            m1[j] = mask[min(w + 1, last)];
        }
    }
    const bool marked = hist || a.n_bias;   // whether there are words to look at
    const uint4 none = make_uint4(0, 0, 0, 0);
    if (marked) {
        for (int i = tid; i < kTokens / 4; i += kThreads) reinterpret_cast<uint4*>(count)[i] = none;
    }
    __syncthreads();
    // place of a token in this workgroup's, where it is under `span`
    const int low = max(v0, 0);
    const uint32_t span = (uint32_t)max(min(a.V, v0 + kTokens) - low, 0);
    auto is_here = [&](int id) { return (uint32_t)(id - low) < span; };   // (id >= 0: low is)
    for (int i0 = tid; i0 < len; i0 += kBatch * kThreads) {
        int next[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {   // (past the end: the last again, unused)
            next[j] = hist[min(i0 + (kBatch + j) * kThreads, len - 1)];
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = i0 + j * kThreads;
            if (is_here(ids[j]) && i < len) {
                if (i >= prompt) atomicAdd(&count[ids[j] - v0], 1u);
                else atomicOr(&count[ids[j] - v0], kSeen);
            }
            ids[j] = next[j];
        }
    }
    auto id_of = [&](int i) { return i == tid ? bias_id : a.bias_ids[b * a.ld_bias + i]; };
    for (int i = tid; i < a.n_bias; i += kThreads) {
        const int id = id_of(i);
        if (is_here(id)) atomicOr(&count[id - v0], kBias), bias_at[id - v0] = 0;
    }
    __syncthreads();
    if (a.n_bias) {   // the last of a token's places
        for (int i = tid; i < a.n_bias; i += kThreads) {
            const int id = id_of(i);
            if (is_here(id)) atomicMax(&bias_at[id - v0], i);
        }
        __syncthreads();
    }
    float best = -INFINITY;
    int best_v = -1;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int at = 4 * (tid + j * kThreads);
        const int v = v0 + at;
        if constexpr (kDtype == NB_BF16) {
            const uint32_t w0 = __float_as_uint(x[j][0]), w1 = __float_as_uint(x[j][1]);
            x[j] = f4{__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u),
                      __uint_as_float(w1 << 16), __uint_as_float(w1 & 0xffff0000u)};
        }
        // bits of the group's four tokens (a row's first may begin before token 0)
        const uint64_t m = (uint64_t)m1[j] << 32 | m0[j];
        const uint32_t allowed = v >= 0 ? (uint32_t)(m >> (v & 31)) : m0[j] << -v;
        uint4 c4 = none;
        if (marked) c4 = *reinterpret_cast<const uint4*>(&count[at]);
        // the marked tokens of the group, one a turn: few lanes have any, hardly
        // one has two
        uint32_t left = (c4.x ? 1 : 0) | (c4.y ? 2 : 0) | (c4.z ? 4 : 0) | (c4.w ? 8 : 0);
        while (left) {
            const int e = __ffs((int)left) - 1;
            left &= left - 1;
            const uint32_t c = e < 2 ? (e ? c4.y : c4.x) : (e == 2 ? c4.z : c4.w);
            float y = e < 2 ? (e ? x[j][1] : x[j][0]) : (e == 2 ? x[j][2] : x[j][3]);
            const uint32_t n = c & kTimes;
            if (n || c & kSeen) y = y > 0.f ? y / rep : y * rep;
            if (n) y = (y - freq * (float)n) - pres;
            if (c & kBias) y = y + a.bias[b * a.ld_bias + bias_at[at + e]];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = e == i ? y : x[j][i];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = allowed >> e & 1 ? x[j][e] : -INFINITY;
            x[j][e] = y;
            const bool in_row = v + e >= 0 && v + e < a.V;
            if (y > best && in_row) best = y, best_v = v + e;   // (a NaN is not over it)
        }
        if (v >= 0 && v + 3 < a.V) {
            *reinterpret_cast<f4*>(out + v) = x[j];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v + e >= 0 && v + e < a.V) out[v + e] = x[j][e];
            }
        }
    }
    if (!a.tokens) return;
    uint64_t key = wave_max(key_of(best, best_v));
    if ((tid & 63) == 0) wave_keys[tid >> 6] = key;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) key = wave_keys[w] > key ? wave_keys[w] : key;
        if (gridDim.x == 1) a.tokens[b] = token_of(key);
        else a.keys[(int64_t)b * gridDim.x + blockIdx.x] = key;
    }
}

// The choice over a row's workgroups, one wave a row.
__global__ __launch_bounds__(64) void logits_choose_kernel(const uint64_t* keys, int parts,
                                                           int32_t* tokens) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < parts; i += 64) {
        const uint64_t key = keys[(int64_t)blockIdx.x * parts + i];
        best = key > best ? key : best;
    }
    best = wave_max(best);
    if (threadIdx.x == 0) tokens[blockIdx.x] = token_of(best);
}

// One workgroup more where a row's first group is not whole.
int parts_of(int rows, int V) {
    const int tokens = tokens_of(loads_of(rows, V));
    return (int)(((int64_t)V + 3 + tokens - 1) / tokens);
}

}  // namespace

int64_t logits_rules_bytes(int rows, int V) {
    const int parts = parts_of(rows, V);
    return parts == 1 ? 0 : (int64_t)rows * parts * 8;
}

int launch_logits_rules(const void* logits, int dtype, int64_t ld, int rows, int V,
                        const int32_t* history, int64_t ld_history, int max_history,
                        const int32_t* lens, const int32_t* prompt_lens, const float* repetition,
                        const float* frequency, const float* presence, const int32_t* bias_ids,
                        const float* bias, int64_t ld_bias, int n_bias, const int32_t* mask,
                        int64_t ld_mask, float* out, int64_t ld_out, int32_t* tokens,
                        void* workspace, hipStream_t stream) {
    const LogitsArgs a{logits, ld, ld_out, ld_history, ld_bias, ld_mask, history, lens,
                       prompt_lens, repetition, frequency, presence, bias_ids, bias, mask, out,
                       static_cast<uint64_t*>(workspace), tokens, V, max_history, n_bias};
    const int parts = parts_of(rows, V);
    const bool one = loads_of(rows, V) == 1;
    auto* kernel = dtype == NB_F32
                       ? (one ? logits_rules_kernel<NB_F32, 1> : logits_rules_kernel<NB_F32, 2>)
                       : (one ? logits_rules_kernel<NB_BF16, 1> : logits_rules_kernel<NB_BF16, 2>);
    hipLaunchKernelGGL(kernel, dim3(parts, rows), dim3(kThreads), 0, stream, a);
    if (tokens && parts > 1) {
        hipLaunchKernelGGL(logits_choose_kernel, dim3(rows), dim3(64), 0, stream,
                           a.keys, parts, tokens);
    }
    return check_launch("nb_logits_rules");
}

}  // namespace nb
