// What the kernels of nb_linear8 share: the tiles of a layer, the weights of a
// unit, and the epilogue.
//
//     y[m][n] = f(x_scale[m] * scale[n] * sum_k x[m][k] * c[n][k] + bias[n]) + residual[m][n]
//
// x and c int8: c[n][k] is the entry that weight k's 3-bit index picks of its
// block's eight codes.  The sums are whole numbers below 2^31 (K <= 2^17), the
// same in any order; the rest is fp32, rounded to y's type once.
//
// Layer in tiles of 16 outputs x 128 inputs (nb_linear8_layout), a row of tiles
// one after the other.  A tile is 64 units of 12 bytes, unit 16 g + r holding the
// 32 indices of output r's inputs 32 g .. 32 g + 31 (selector-ordered,
// nb_stream_common.h; selector s has indices 4 s .. 4 s + 3), and then the 16
// outputs' 8 codes: 0.4375 bytes a weight against 0.625 with fp32 codebooks.
// Lane 16 g + r of a wave takes unit 16 g + r and output r's codes, as 12 and 8
// bytes, all lanes' side by side.  Eight codes are one v_perm_b32's table: a
// selector becomes four weights in one instruction, 25 for the 32 of a unit.
// These are the lane's operands of two v_mfma_i32_16x16x64_i8, whose other
// operand is 16 rows' codes at inputs 32 g + 16 h .. + 15: 16 bytes of x as it is.
#pragma once

#include <math.h>

#include <type_traits>

#include "nb_device.h"
#include "nb_internal.h"
#include "nb_stream_common.h"

namespace nb {
namespace linear8 {

typedef __attribute__((ext_vector_type(4))) int32_t i4;
typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(4))) uint32_t u4;
typedef __attribute__((ext_vector_type(3), aligned(4))) uint32_t u3;   // (one access of 12 bytes)
typedef __attribute__((ext_vector_type(2))) uint32_t u2;

constexpr int kTileBytes = 896, kTileCodes = 768;

struct Args {
    const int8_t* x;
    int64_t ld_x;
    const float* x_scale;
    const uint8_t* tiles;
    const float *scale, *bias;
    const void* residual;   // of y's type
    int64_t ld_residual;
    void* y;
    int64_t ld_y;
    int M, N, K;
    int activation;   // nb_activation
};

// A lane's unit of a tile and the codes of its output.
struct Unit {
    uint32_t d0, d1, d2, c0, c1;
};
__device__ __forceinline__ Unit load_unit(const uint8_t* tile, int lane) {
    const u3 d = *reinterpret_cast<const __attribute__((address_space(1))) u3*>(
        as_global(tile) + lane * 12);
    const u2 c = *reinterpret_cast<const __attribute__((address_space(1))) u2*>(
        as_global(tile) + kTileCodes + (lane & 15) * 8);
    return Unit{d[0], d[1], d[2], c[0], c[1]};
}

// Its 32 weights: inputs 0 .. 15 of the unit, then 16 .. 31.
__device__ __forceinline__ void unit_weights(const Unit& u, i4 (&w)[2]) {
    uint32_t sel[8];
    stream::unit_selectors_sel(u.d0, u.d1, u.d2, sel);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        w[s >> 2][s & 3] = (int32_t)__builtin_amdgcn_perm(u.c1, u.c0, sel[s]);
    }
}

__device__ __forceinline__ i4 mfma(i4 w, i4 x, i4 sum) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, sum, 0, 0, 0);
}

// (the reciprocal within a step: an IEEE quotient takes a dozen instructions, in
// an epilogue whose instructions are a third of a prompt's time)
__device__ __forceinline__ float silu(float v) {
    return v * __builtin_amdgcn_rcpf(1.f + __expf(-v));
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    typedef __attribute__((ext_vector_type(2))) __bf16 pair;
    return __builtin_bit_cast(uint32_t, pair{(__bf16)lo, (__bf16)hi});
}

// f(the activation as a constant): its code has no branches inside loops.
template <typename F>
__device__ __forceinline__ void by_activation(int activation, F f) {
    if (activation == NB_ACT_NONE) f(std::integral_constant<int, NB_ACT_NONE>{});
    else if (activation == NB_ACT_SWIGLU) f(std::integral_constant<int, NB_ACT_SWIGLU>{});
    else if (activation == NB_ACT_SILU) f(std::integral_constant<int, NB_ACT_SILU>{});
    else f(std::integral_constant<int, NB_ACT_GELU>{});
}

// kCount (4 or 2) neighbouring values of a row, `left` of them in the row.
template <int kCount, bool kBf16>
__device__ __forceinline__ void load_some(const void* row, int64_t at, int left, float (&v)[kCount]) {
    if constexpr (kBf16) {
        const bf16_bits* p = static_cast<const bf16_bits*>(row) + at;
        typedef __attribute__((ext_vector_type(kCount / 2), aligned(2))) uint32_t any;
        if (left >= kCount) {
            const any w = *reinterpret_cast<const any*>(p);
#pragma unroll
            for (int e = 0; e < kCount; e += 2) {
                const uint32_t u = reinterpret_cast<const uint32_t*>(&w)[e / 2];
                v[e] = __uint_as_float(u << 16);
                v[e + 1] = __uint_as_float(u & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) v[e] = e < left ? bf16_to_f32(p[e]) : 0.f;
        }
    } else {
        const float* p = static_cast<const float*>(row) + at;
        typedef __attribute__((ext_vector_type(kCount), aligned(4))) float any;
        if (left >= kCount) {
            const any w = *reinterpret_cast<const any*>(p);
#pragma unroll
            for (int e = 0; e < kCount; ++e) v[e] = w[e];
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) v[e] = e < left ? p[e] : 0.f;
        }
    }
}

template <int kCount, bool kBf16>
__device__ __forceinline__ void store_some(void* row, int64_t at, int left, const float (&v)[kCount]) {
    if constexpr (kBf16) {
        bf16_bits* p = static_cast<bf16_bits*>(row) + at;
        typedef __attribute__((ext_vector_type(kCount / 2), aligned(2))) uint32_t any;
        if (left >= kCount) {
            uint32_t w[kCount / 2];
#pragma unroll
            for (int e = 0; e < kCount; e += 2) {
                w[e / 2] = bf16_pair(v[e], v[e + 1]);
            }
            *reinterpret_cast<any*>(p) = *reinterpret_cast<const any*>(w);
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) {
                if (e < left) p[e] = f32_to_bf16_rne(v[e]);
            }
        }
    } else {
        float* p = static_cast<float*>(row) + at;
        typedef __attribute__((ext_vector_type(kCount), aligned(4))) float any;
        if (left >= kCount) {
            *reinterpret_cast<any*>(p) = *reinterpret_cast<const any*>(v);
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) {
                if (e < left) p[e] = v[e];
            }
        }
    }
}

// Scales and biases of layer outputs n .. n + 3 (n a multiple of 4), the last
// output's past the layer.
struct Column {
    float scale[4], bias[4];
};
__device__ __forceinline__ Column column(const Args& a, int n) {
    Column c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int at = min(n + e, a.N - 1);
        c.scale[e] = a.scale[at];
        c.bias[e] = a.bias ? a.bias[at] : 0.f;
    }
    return c;
}

// v Phi(v).  Phi(-a) = exp(-a^2 / 2) P(u) for a >= 0 with u = 0.21 a / (1 + 0.21 a), the
// form of Abramowitz and Stegun 7.1.26 in 1 - t: what is left beside the exponential is
// smooth in u from 1/2 at 0 to its end, and a polynomial of degree 9 (least largest
// relative error, fitted in 64 bits for a up to 15, where the exponential is below fp32)
// is within 1.4e-8 of it.  (In t = 1 / (1 + 0.21 a) the polynomial is as short, but its
// value near 0 moves four times as far as t does.)
// Nothing cancels: a product on the left, at most half of v taken off on the right
// (by a finite factor: of an infinity nothing is, where v tail would be inf * 0).
// Errors of 2^20 outputs in fp32 against 64 bits, of v of deviation 0.1, 0.3, 1 and 3:
// 4.0e-8, 3.8e-8, 2.9e-8 and 2.2e-8; v (1 + erf) / 2 in fp32 3.8e-8, 4.1e-8, 3.9e-8 and 3.0e-8.
// No branch: 500 rows of 5003 x 1280 in bf16 12.6 us, without an activation 11.0, with
// erfcf 3 more (launches of a graph).
__device__ __forceinline__ float gelu(float v) {
    const float a = __builtin_fminf(__builtin_fabsf(v), 3.4e38f);
    const float u = 0.21f * a * __builtin_amdgcn_rcpf(__builtin_fmaf(0.21f, a, 1.f));
    float p = 0.07293546944856644f;
    p = __builtin_fmaf(p, u, -0.3659140467643738f);
    p = __builtin_fmaf(p, u, 0.6481500864028931f);
    p = __builtin_fmaf(p, u, -0.04684164747595787f);
    p = __builtin_fmaf(p, u, -1.916527509689331f);
    p = __builtin_fmaf(p, u, 4.159022331237793f);
    p = __builtin_fmaf(p, u, -4.920256614685059f);
    p = __builtin_fmaf(p, u, 3.7691614627838135f);
    p = __builtin_fmaf(p, u, -1.8997241258621216f);
    p = __builtin_fmaf(p, u, 0.5f);
    const float tail = __builtin_amdgcn_exp2f(a * a * -0.72134752f) * p;
    return v < 0.f ? v * tail : __builtin_fmaf(-a, tail, v);
}

// The outputs of four sums: row m, layer outputs n .. n + 3.  Loads, arithmetic and
// stores are apart, so that a loop can put several in flight (stores count among
// the loads that a wait is for).
template <int kAct>
struct Finished {
    static constexpr int kCount = kAct == NB_ACT_SWIGLU ? 2 : 4;   // (swiglu: N is even)
    float v[kCount];

    template <bool kBf16>
    __device__ __forceinline__ void load_residual(const Args& a, int m, int n) {
        if (m < a.M && n < a.N) {
            load_some<kCount, kBf16>(a.residual, m * a.ld_residual + n * kCount / 4,
                                     (a.N - n) * kCount / 4, v);
        }
    }
    // xs: the row's scale; kResidual: v holds the residual.  Which products and sums
    // are one step is written out: a row's outputs are the same in every form.
    template <bool kResidual>
    __device__ __forceinline__ void finish(const Column& c, float xs, i4 sum) {
#pragma clang fp contract(off)
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf((float)sum[e], xs * c.scale[e], c.bias[e]);
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            float out = y[e];
            if constexpr (kAct == NB_ACT_SWIGLU) out = silu(y[2 * e]) * y[2 * e + 1];
            else if constexpr (kAct == NB_ACT_SILU) out = silu(y[e]);
            else if constexpr (kAct == NB_ACT_GELU) out = gelu(y[e]);
            v[e] = kResidual ? out + v[e] : out;
        }
    }
    template <bool kBf16>
    __device__ __forceinline__ void store(const Args& a, int m, int n) const {
        if (m < a.M && n < a.N) {
            store_some<kCount, kBf16>(a.y, m * a.ld_y + n * kCount / 4, (a.N - n) * kCount / 4, v);
        }
    }
};

}  // namespace linear8
}  // namespace nb
