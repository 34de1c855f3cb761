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
// Bound by memory: one pass over the logits.  A workgroup takes 4096 tokens of
// a row; it issues the loads of their logits, counts the row's history in an
// LDS word per token (bit 31: seen, the rest: n) and notes the biases there
// while they are under way, so that neither counts nor dense biases exist in
// memory.  Every workgroup of a row walks its whole history, from the L2:
// against 32 KB of logits read and written, a history of 1000 is 4 KB.  LDS
// atomics are on whole numbers (sums, or, maximum): no result depends on their
// order.
#include <math.h>

#include <algorithm>

#include "nb_device.h"
#include "nb_internal.h"

// Products and sums round one by one (no fused multiply-add, which the
// compiler makes of __fmul_rn and __fadd_rn too).
#pragma clang fp contract(off)

namespace nb {
namespace {

typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(4))) uint16_t h4;

constexpr int kThreads = 256;
constexpr int kLoads = 4;                          // groups of four tokens a thread
constexpr int kTokens = 4 * kThreads * kLoads;     // of a workgroup
constexpr uint32_t kSeen = 0x80000000u;

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
    int dtype, V, max_history, n_bias;
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

// kVec: input and output rows begin at the same place of a group of four
// elements, so that all groups but a row's first and last move as vectors.
template <bool kVec>
__global__ __launch_bounds__(kThreads) void logits_rules_kernel(LogitsArgs a) {
    __shared__ uint32_t count[kTokens];
    __shared__ int32_t bias_at[kTokens];   // 1 + the place of the token's bias
    __shared__ uint64_t wave_keys[kThreads / 64];
    const int b = blockIdx.y, tid = threadIdx.x;
    const int esize = a.dtype == NB_F32 ? 4 : 2;
    const char* in = static_cast<const char*>(a.logits) + b * a.ld * esize;
    float* out = a.out + b * a.ld_out;
    // group q of four elements holds tokens 4 q - shift ..
    const int shift = kVec ? (int)(reinterpret_cast<uintptr_t>(in) / esize & 3) : 0;
    const int64_t v0 = (int64_t)blockIdx.x * kTokens - shift;
    f4 x[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int64_t v = v0 + 4 * (tid + j * kThreads);
        if (kVec && v >= 0 && v + 3 < a.V) {
            if (a.dtype == NB_F32) {
                x[j] = *reinterpret_cast<const f4*>(in + 4 * v);
            } else {
                const h4 w = *reinterpret_cast<const h4*>(in + 2 * v);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = bf16_to_f32(w[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool ok = v + e >= 0 && v + e < a.V;
                x[j][e] = !ok ? 0.f
                          : a.dtype == NB_F32 ? reinterpret_cast<const float*>(in)[v + e]
                                              : bf16_to_f32(reinterpret_cast<const bf16_bits*>(in)[v + e]);
            }
        }
    }
    if (a.history) {
        for (int i = tid; i < kTokens; i += kThreads) count[i] = 0;
    }
    if (a.n_bias) {
        for (int i = tid; i < kTokens; i += kThreads) bias_at[i] = 0;
    }
    __syncthreads();
    if (a.history) {
        const int32_t* hist = a.history + b * a.ld_history;
        const int len = min(max(a.lens[b], 0), a.max_history);
        const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
        for (int i = tid; i < len; i += kThreads) {
            const int id = hist[i];
            const int64_t at = id - v0;
            if (id >= 0 && id < a.V && at >= 0 && at < kTokens) {
                if (i >= prompt) atomicAdd(&count[at], 1u);
                else atomicOr(&count[at], kSeen);
            }
        }
    }
    for (int i = tid; i < a.n_bias; i += kThreads) {
        const int id = a.bias_ids[b * a.ld_bias + i];
        const int64_t at = id - v0;
        if (id >= 0 && id < a.V && at >= 0 && at < kTokens) atomicMax(&bias_at[at], i + 1);
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[b] : 1.f;
    const float freq = a.frequency ? a.frequency[b] : 0.f;
    const float pres = a.presence ? a.presence[b] : 0.f;
    const int32_t* mask = a.mask ? a.mask + b * a.ld_mask : nullptr;
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int at = 4 * (tid + j * kThreads);
        const int64_t v = v0 + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (v + e < 0 || v + e >= a.V) continue;
            float y = x[j][e];
            const uint32_t c = a.history ? count[at + e] : 0;
            if (c) {
                y = y > 0.f ? y / rep : y * rep;
                const uint32_t n = c & ~kSeen;
                if (n) y = (y - freq * (float)n) - pres;
            }
            const int i = a.n_bias ? bias_at[at + e] : 0;
            if (i) y = y + a.bias[b * a.ld_bias + i - 1];
            if (mask && !((uint32_t)mask[(v + e) >> 5] >> ((v + e) & 31) & 1)) y = -INFINITY;
            x[j][e] = y;
            const uint64_t key = key_of(y, (int)(v + e));
            best = key > best ? key : best;
        }
        if (kVec && v >= 0 && v + 3 < a.V) {
            *reinterpret_cast<f4*>(out + v) = x[j];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v + e >= 0 && v + e < a.V) out[v + e] = x[j][e];
            }
        }
    }
    if (!a.tokens) return;
    best = wave_max(best);
    if ((tid & 63) == 0) wave_keys[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) best = wave_keys[w] > best ? wave_keys[w] : best;
        if (gridDim.x == 1) a.tokens[b] = token_of(best);
        else a.keys[(int64_t)b * gridDim.x + blockIdx.x] = best;
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
int parts_of(int V) { return (int)(((int64_t)V + 3 + kTokens - 1) / kTokens); }

}  // namespace

int64_t logits_rules_bytes(int rows, int V) {
    const int parts = parts_of(V);
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
                       static_cast<uint64_t*>(workspace), tokens, dtype, V, max_history, n_bias};
    const int esize = dtype == NB_F32 ? 4 : 2;
    const int parts = parts_of(V);
    const bool vec = ((reinterpret_cast<uintptr_t>(logits) / esize) & 3) ==
                         ((reinterpret_cast<uintptr_t>(out) / 4) & 3) && (ld - ld_out) % 4 == 0;
    hipLaunchKernelGGL(vec ? logits_rules_kernel<true> : logits_rules_kernel<false>,
                       dim3(parts, rows), dim3(kThreads), 0, stream, a);
    if (tokens && parts > 1) {
        hipLaunchKernelGGL(logits_choose_kernel, dim3(rows), dim3(64), 0, stream,
                           a.keys, parts, tokens);
    }
    return check_launch("nb_logits_rules");
}

}  // namespace nb
