// Rows in 8 bits times packed 3-bit weights with 8-bit codebooks (gfx950):
// nb_linear8_layout, and nb_linear8 for few rows.  Formulas and layout:
// nb_linear8.h.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "nb_linear8.h"

namespace nb {
namespace {

using namespace linear8;

// ---------------------------------------------------------------------------
// layout, once a layer
// ---------------------------------------------------------------------------
// scale[n] = max |entry of output n| / 127, one wave an output.
__global__ __launch_bounds__(64) void linear8_scale_kernel(const float* codebook, int entries,
                                                           float* scale) {
    const float* row = codebook + (int64_t)blockIdx.x * entries;
    uint32_t most = 0;   // (of the values' bits: a NaN is over infinity)
    for (int i = threadIdx.x; i < entries; i += 64) {
        most = max(most, __float_as_uint(row[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
    if (threadIdx.x == 0) {
        scale[blockIdx.x] = most < 0x7f800000u ? (float)((double)__uint_as_float(most) / 127.0)
                                               : __builtin_nanf("");
    }
}

// Index i of a unit's 96 bits.
__device__ __forceinline__ uint32_t unit_index(const uint32_t (&d)[3], int i) {
    const int bit = 3 * i, w = bit >> 5, off = bit & 31;
    const uint64_t v = (uint64_t)(w < 2 ? d[w + 1] : 0) << 32 | d[w];
    return (uint32_t)(v >> off) & 7u;
}

// A wave a tile, a lane a unit; the first 16 lanes an output's codes too: the
// entries times 127 / max |entry|, rounded, in 64 bits.  Outputs past the layer
// are zeros.
__global__ __launch_bounds__(64) void linear8_layout_kernel(const uint8_t* packed,
                                                            const float* codebook, int N, int bpr,
                                                            uint8_t* tiles) {
    const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
    const int64_t tile = blockIdx.x;
    const int n = (int)(tile / bpr) * 16 + r, kb = (int)(tile % bpr);
    const int64_t block = (int64_t)n * bpr + kb;
    uint32_t o[3] = {0, 0, 0}, c[2] = {0, 0};
    if (n < N) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(packed + block * 48 + g * 12);
        const uint32_t d[3] = {src[0], src[1], src[2]};
        uint32_t sel[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            sel[s] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) sel[s] |= unit_index(d, 4 * s + e) << (8 * e);
        }
        stream::sel_unit_pack(sel, o[0], o[1], o[2]);
    }
    uint8_t* to = tiles + tile * kTileBytes;
    uint32_t* units = reinterpret_cast<uint32_t*>(to + lane * 12);
    units[0] = o[0], units[1] = o[1], units[2] = o[2];
    // the output's largest entry, by four lanes of it
    uint32_t most = 0;
    if (n < N) {
        const float* row = codebook + (int64_t)n * bpr * 8;
        for (int i = g; i < bpr * 8; i += 4) most = max(most, __float_as_uint(row[i]) & 0x7fffffffu);
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    if (g == 0) {
        if (n < N && most > 0 && most < 0x7f800000u) {
            const double turn = 127.0 / (double)__uint_as_float(most);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int q = (int)rint((double)codebook[block * 8 + e] * turn);
                c[e >> 2] |= ((uint32_t)q & 255u) << (8 * (e & 3));
            }
        }
        uint32_t* codes = reinterpret_cast<uint32_t*>(to + kTileCodes + r * 8);
        codes[0] = c[0], codes[1] = c[1];
    }
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
// A workgroup takes 16 outputs and 16 kT rows; its waves take the blocks of K in
// turn and add their sums through LDS.
template <int kWaves, int kT>
__global__ __launch_bounds__(64 * kWaves) void linear8_rows_kernel(Args a) {
    __shared__ i4 part[kWaves][kT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * kT;
    const int bpr = a.K / 128;
    const uint8_t* tiles = a.tiles + (int64_t)blockIdx.x * bpr * kTileBytes;
    const int8_t* x[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) {
        const int m = min(m0 + 16 * t + (lane & 15), a.M - 1);
        x[t] = a.x + m * a.ld_x + (lane >> 4) * 32;
    }
    i4 sum[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) sum[t] = i4{0, 0, 0, 0};
    for (int kb = wave; kb < bpr; kb += kWaves) {
        const Unit u = load_unit(tiles + (int64_t)kb * kTileBytes, lane);
        i4 w[2];
        unit_weights(u, w);
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const i4* p = reinterpret_cast<const i4*>(x[t] + kb * 128);
            sum[t] = mfma(w[0], p[0], sum[t]);
            sum[t] = mfma(w[1], p[1], sum[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < kT; ++t) part[wave][t][lane] = sum[t];
    __syncthreads();
    for (int i = tid; i < kT * 64; i += 64 * kWaves) {
        const int t = i >> 6, l = i & 63;
        i4 s = part[0][t][l];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += part[w][t][l];
        finish(a, m0 + 16 * t + (l & 15), n0 + (l >> 4) * 4, s);
    }
}

}  // namespace

int64_t linear8_tiles_bytes(int N, int K) {
    return ((int64_t)N + 15) / 16 * (K / 128) * kTileBytes;
}

int launch_linear8_layout(const uint8_t* packed, const float* codebook, int N, int K,
                          uint8_t* tiles, float* scale, hipStream_t stream) {
    const int bpr = K / 128;
    hipLaunchKernelGGL(linear8_scale_kernel, dim3(N), dim3(64), 0, stream, codebook, bpr * 8, scale);
    hipLaunchKernelGGL(linear8_layout_kernel, dim3((unsigned)(((int64_t)N + 15) / 16 * bpr)), dim3(64),
                       0, stream, packed, codebook, N, bpr, tiles);
    return check_launch("nb_linear8_layout");
}

int64_t linear8_bytes(int, int, int) { return 0; }

int launch_linear8(const int8_t* x, int64_t ld_x, const float* x_scale, const uint8_t* tiles,
                   const float* scale, const float* bias, int activation, const void* residual,
                   int64_t ld_residual, void* y, int y_dtype, int64_t ld_y, int M, int N, int K,
                   void*, hipStream_t stream) {
    const Args a{x, ld_x, x_scale, tiles, scale, bias, residual, ld_residual, y, ld_y, M, N, K,
                 activation, y_dtype};
    const unsigned columns = ((unsigned)N + 15) / 16;
    if (M <= 16) {
        hipLaunchKernelGGL((linear8_rows_kernel<8, 1>), dim3(columns, 1), dim3(512), 0, stream, a);
    } else {
        hipLaunchKernelGGL((linear8_rows_kernel<8, 4>), dim3(columns, ((unsigned)M + 63) / 64),
                           dim3(512), 0, stream, a);
    }
    return check_launch("nb_linear8");
}

}  // namespace nb
