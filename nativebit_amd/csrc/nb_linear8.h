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
    int y_dtype;
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

__device__ __forceinline__ float silu(float v) { return v / (1.f + __expf(-v)); }

__device__ __forceinline__ float read_as(const void* p, int dtype, int64_t i) {
    return dtype == NB_BF16 ? bf16_to_f32(static_cast<const bf16_bits*>(p)[i])
                            : static_cast<const float*>(p)[i];
}

// `count` (4 or 2) neighbouring values of a row from element `at` on, `left` of
// them in the row.
template <int kCount>
__device__ __forceinline__ void finish_row(const Args& a, int m, int n, int left, float (&v)[kCount]) {
    if (a.residual) {
        const int64_t at = m * a.ld_residual + n;
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            if (e < left) v[e] += read_as(a.residual, a.y_dtype, at + e);
        }
    }
    const int64_t at = m * a.ld_y + n;
    if (a.y_dtype == NB_BF16) {
        bf16_bits* y = static_cast<bf16_bits*>(a.y) + at;
        typedef __attribute__((ext_vector_type(kCount / 2), aligned(2))) uint32_t any;
        if (left >= kCount) {
            any p;
#pragma unroll
            for (int e = 0; e < kCount; e += 2) {
                p[e / 2] = f32_to_bf16_rne(v[e]) | (uint32_t)f32_to_bf16_rne(v[e + 1]) << 16;
            }
            *reinterpret_cast<any*>(y) = p;
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) {
                if (e < left) y[e] = f32_to_bf16_rne(v[e]);
            }
        }
    } else {
        float* y = static_cast<float*>(a.y) + at;
        typedef __attribute__((ext_vector_type(kCount), aligned(4))) float any;
        if (left >= kCount) {
            any p;
#pragma unroll
            for (int e = 0; e < kCount; ++e) p[e] = v[e];
            *reinterpret_cast<any*>(y) = p;
        } else {
#pragma unroll
            for (int e = 0; e < kCount; ++e) {
                if (e < left) y[e] = v[e];
            }
        }
    }
}

// The outputs of four sums: of row m, layer outputs n .. n + 3 (n a multiple of 4).
__device__ __forceinline__ void finish(const Args& a, int m, int n, i4 sum) {
    if (m >= a.M || n >= a.N) return;
    const float xs = a.x_scale[m];
    const int left = a.N - n;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int at = n + min(e, left - 1);
        v[e] = (float)sum[e] * (xs * a.scale[at]);
        if (a.bias) v[e] += a.bias[at];
    }
    if (a.activation == NB_ACT_SWIGLU) {   // (N is even)
        float g[2] = {silu(v[0]) * v[1], silu(v[2]) * v[3]};
        return finish_row<2>(a, m, n / 2, left / 2, g);
    }
    if (a.activation == NB_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = silu(v[e]);
    } else if (a.activation == NB_ACT_GELU) {
        // v Phi(v) by erfc: no cancellation for negative v
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = 0.5f * v[e] * erfcf(-0.70710678f * v[e]);
    }
    finish_row<4>(a, m, n, left, v);
}

}  // namespace linear8
}  // namespace nb
