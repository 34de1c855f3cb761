// Rows in 8 bits with one scale each (gfx950): nb_quantize8, nb_rmsnorm8, and the
// values they stand for: nb_rows8_values.
//
// For a row v of `width` values, a = max |v|:
//     code  = rint(v * (127 / a)),  scale = a / 127            (0 where a = 0)
// nb_rmsnorm8: v = h * w / rms, h = x (+ residual), rms = sqrt(mean h^2 + eps).
// rms is a factor of the whole row: it cancels in the codes, which follow from
// t = h * w alone, and is divided out of the scale.  t, a, sums and quotients are
// in 64 bits: t is exact, and no code falls on the other side of a border because
// of a rounding before it (in fp32 a dozen of 14 million do).  A row with a NaN or
// an infinity has scale NaN and codes 0.
//
// Bound by memory: each value is read once, held in registers (as it was stored)
// over the row's one reduction, and its code written.  2048 rows of 6912 fp32 values
// 14.9 us (71 MB, 4.8 TB/s) and back 12.9 (5.5 TB/s); the norm of 2048 rows of 2560 with
// its residual and the sum written 15.9 (68 MB, 4.3 TB/s), without them 11.2 (9.3 again and
// again on one input), where the 64-bit products and quotients are half of it; one row
// 2 to 4 us, a launch and the reduction's waits.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "nb_device.h"
#include "nb_internal.h"

// Products and sums round one by one (the product with 127 / a before its
// rounding to a whole number, too).
#pragma clang fp contract(off)

namespace nb {
namespace {

typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(4), aligned(4))) float f4_any;
typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t u2_any;
typedef __attribute__((aligned(1))) uint32_t u1_any;

struct RowsArgs {
    const void *x, *residual;   // of one type
    int64_t ld_x, ld_residual, ld_sum;
    void* sum;
    const float* weight;
    int8_t* codes;
    float* scale;
    int width;
    float eps;
};

// Four values from element i of a row on, zeros past its end.
template <int kDtype>
__device__ __forceinline__ f4 load4(const void* row, int i, int width) {
    if constexpr (kDtype == NB_F32) {
        const float* p = static_cast<const float*>(row) + i;
        if (i + 3 < width) return *reinterpret_cast<const f4_any*>(p);
        f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e < width) v[e] = p[e];
        }
        return v;
    } else {
        const bf16_bits* p = static_cast<const bf16_bits*>(row) + i;
        if (i + 3 < width) {
            const u2_any w = *reinterpret_cast<const u2_any*>(p);
            return f4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u),
                      __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
        }
        f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e < width) v[e] = bf16_to_f32(p[e]);
        }
        return v;
    }
}

template <int kDtype>
__device__ __forceinline__ void store4(void* row, int i, int width, f4 v) {
    if constexpr (kDtype == NB_F32) {
        float* p = static_cast<float*>(row) + i;
        if (i + 3 < width) {
            *reinterpret_cast<f4_any*>(p) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e < width) p[e] = v[e];
            }
        }
    } else {   // (values that are bf16 already)
        bf16_bits* p = static_cast<bf16_bits*>(row) + i;
        if (i + 3 < width) {
            const uint32_t u0 = __float_as_uint(v[0]) >> 16 | (__float_as_uint(v[1]) & 0xffff0000u);
            const uint32_t u1 = __float_as_uint(v[2]) >> 16 | (__float_as_uint(v[3]) & 0xffff0000u);
            *reinterpret_cast<u2_any*>(p) = u2_any{u0, u1};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e < width) p[e] = (bf16_bits)(__float_as_uint(v[e]) >> 16);
            }
        }
    }
}

__device__ __forceinline__ double shuffle_xor(double v, int d) { return __shfl_xor(v, d); }

// kNorm: nb_rmsnorm8, else nb_quantize8.  kGroups groups of four values a thread
// at once; rows of over kThreads * 4 * kGroups values are read a second time for
// their codes.
template <int kDtype, bool kNorm, int kThreads, int kGroups>
__global__ __launch_bounds__(kThreads) void rows8_kernel(RowsArgs a) {
    constexpr int kWaves = kThreads / 64, kSpan = kThreads * 4 * kGroups;
    constexpr int kSize = kDtype == NB_F32 ? 4 : 2;
    __shared__ double part[2][kWaves];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x;
    const char* x = static_cast<const char*>(a.x) + b * a.ld_x * kSize;
    const char* residual =
        kNorm && a.residual ? static_cast<const char*>(a.residual) + b * a.ld_residual * kSize : nullptr;
    char* sum = kNorm && a.sum ? static_cast<char*>(a.sum) + b * a.ld_sum * kSize : nullptr;
    f4 h[kGroups], w[kGroups];
    auto load = [&](int first) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int i = first + 4 * (tid + g * kThreads);
            h[g] = i < a.width ? load4<kDtype>(x, i, a.width) : f4{0.f, 0.f, 0.f, 0.f};
            if constexpr (kNorm) {
                w[g] = i < a.width ? load4<NB_F32>(a.weight, i, a.width) : f4{0.f, 0.f, 0.f, 0.f};
            }
        }
        if (!kNorm || !residual) return;
        f4 r[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int i = first + 4 * (tid + g * kThreads);
            r[g] = i < a.width ? load4<kDtype>(residual, i, a.width) : f4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            h[g] = h[g] + r[g];
            if constexpr (kDtype == NB_BF16) {   // (the norm is that of the sum as it is kept)
#pragma unroll
                for (int e = 0; e < 4; ++e) h[g][e] = round_bf16(h[g][e]);
            }
        }
    };
    auto value = [&](int g, int e) {
        return kNorm ? (double)h[g][e] * (double)w[g][e] : (double)h[g][e];
    };
    const bool once = a.width <= kSpan;
    double most = 0.0, squares = 0.0;
    for (int first = 0; first < a.width; first += kSpan) {
        load(first);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double t = fabs(value(g, e));
                most = fmax(most, t < INFINITY ? t : (double)INFINITY);   // (a NaN as infinity)
                if constexpr (kNorm) {
                    const double v = h[g][e];
                    squares = fma(v, v, squares);
                }
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        most = fmax(most, shuffle_xor(most, d));
        if constexpr (kNorm) squares += shuffle_xor(squares, d);
    }
    if constexpr (kWaves > 1) {
        if ((tid & 63) == 0) part[0][tid >> 6] = most, part[1][tid >> 6] = squares;
        __syncthreads();
        most = part[0][0], squares = part[1][0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) most = fmax(most, part[0][i]), squares += part[1][i];
    }
    const bool fine = most < INFINITY && (!kNorm || squares < INFINITY);
    const double turn = most > 0.0 && fine ? 127.0 / most : 0.0;
    if (tid == 0) {
        double s = most / 127.0;
        if constexpr (kNorm) s = most / (127.0 * sqrt(squares / a.width + (double)a.eps));
        a.scale[b] = !fine ? __builtin_nanf("") : most > 0.0 ? (float)s : 0.f;
    }
    int8_t* codes = a.codes + b * a.width;
    for (int first = 0; first < a.width; first += kSpan) {
        if (!once) load(first);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int i = first + 4 * (tid + g * kThreads);
            if (i >= a.width) continue;
            if (sum) store4<kDtype>(sum, i, a.width, h[g]);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (the sum's low word holds the rounded product; rows that are not
                // fine may hold NaNs)
                const double q = fine ? value(g, e) * turn : 0.0;
                c |= ((uint32_t)__double2loint(q + 6755399441055744.0) & 255u) << (8 * e);
            }
            if (i + 3 < a.width) {
                *reinterpret_cast<u1_any*>(codes + i) = c;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i + e < a.width) codes[i + e] = (int8_t)(c >> (8 * e));
                }
            }
        }
    }
}

template <int kDtype, bool kNorm>
void launch(const RowsArgs& a, int rows, hipStream_t stream) {
    auto run = [&](auto threads, auto groups) {
        constexpr int t = decltype(threads)::value, g = decltype(groups)::value;
        hipLaunchKernelGGL((rows8_kernel<kDtype, kNorm, t, g>), dim3(rows), dim3(t), 0, stream, a);
    };
    using std::integral_constant;
    // Threads a row, us for 2048 rows in fp32 (quantize / norm): of 1000 values with 64, 256
    // and 512 threads 4.3, 5.3, 7.4 / 5.2, 7.5, 12.0; of 2560 8.4, 6.3, 8.3 / 10.6, 9.3, 13.4;
    // of 6912 23.8, 19.8, 14.9 / 27.5, 20.6, 20.2.
    if (a.width <= 1024) return run(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    if (a.width <= 4096) return run(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    return run(integral_constant<int, 512>{}, integral_constant<int, 4>{});
}

// The values of a row's codes, four a thread at once.
template <int kDtype, int kThreads>
__global__ __launch_bounds__(kThreads) void rows8_values_kernel(const int8_t* codes, const float* scale,
                                                                int width, void* out, int64_t ld) {
    constexpr int kGroups = 4;
    const int64_t b = blockIdx.y;
    const int first = blockIdx.x * kThreads * 4 * kGroups + 4 * (int)threadIdx.x;
    const int8_t* row = codes + b * width;
    char* to = static_cast<char*>(out) + b * ld * (kDtype == NB_F32 ? 4 : 2);
    const float s = as_constant(scale)[b];
    uint32_t c[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int i = first + g * 4 * kThreads;
        c[g] = 0;
        if (i + 3 < width) {
            c[g] = *reinterpret_cast<const u1_any*>(row + i);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e < width) c[g] |= (uint32_t)(uint8_t)row[i + e] << (8 * e);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int i = first + g * 4 * kThreads;
        if (i >= width) break;
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = (float)(int8_t)(c[g] >> (8 * e)) * s;
            if constexpr (kDtype == NB_BF16) v[e] = round_bf16(v[e]);
        }
        store4<kDtype>(to, i, width, v);
    }
}

}  // namespace

int launch_rows8_values(const int8_t* codes, const float* scale, int rows, int width, void* out,
                        int dtype, int64_t ld, hipStream_t stream) {
    constexpr int threads = 256;
    const int columns = (width + threads * 16 - 1) / (threads * 16);
    auto* kernel = dtype == NB_F32 ? rows8_values_kernel<NB_F32, threads> : rows8_values_kernel<NB_BF16, threads>;
    for (int row = 0; row < rows; row += 65535) {   // (a grid's second dimension)
        const int n = std::min(rows - row, 65535);
        hipLaunchKernelGGL(kernel, dim3(columns, n), dim3(threads), 0, stream, codes + (int64_t)row * width,
                           scale + row, width, static_cast<char*>(out) + row * ld * (dtype == NB_F32 ? 4 : 2), ld);
    }
    return check_launch("nb_rows8_values");
}

int launch_quantize8(const void* x, int dtype, int64_t ld_x, int rows, int width, int8_t* codes,
                     float* scale, hipStream_t stream) {
    const RowsArgs a{x, nullptr, ld_x, 0, 0, nullptr, nullptr, codes, scale, width, 0.f};
    if (dtype == NB_F32) launch<NB_F32, false>(a, rows, stream);
    else launch<NB_BF16, false>(a, rows, stream);
    return check_launch("nb_quantize8");
}

int launch_rmsnorm8(const void* x, int dtype, int64_t ld_x, const void* residual,
                    int64_t ld_residual, void* sum, int64_t ld_sum, const float* weight, float eps,
                    int rows, int width, int8_t* codes, float* scale, hipStream_t stream) {
    const RowsArgs a{x, residual, ld_x, ld_residual, ld_sum, sum, weight, codes, scale, width, eps};
    if (dtype == NB_F32) launch<NB_F32, true>(a, rows, stream);
    else launch<NB_BF16, true>(a, rows, stream);
    return check_launch("nb_rmsnorm8");
}

}  // namespace nb
