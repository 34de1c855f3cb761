// The 8-bit block cache (gfx950): nb_kv8_append and nb_kv8_read.
//
// A block holds 64 consecutive tokens of one request; for each key / value
// head h it has
//     k  [64][D]  int8, a token's codes together        K = k * k_scale
//     v  [D][64]  int8, a dim's codes together          V = v * v_scale
// with one fp32 scale each.  With x the new rows of a chunk (the rows of one
// request inside one block), `before` the tokens that the block already
// holds and s its scale (0 where it holds none)
//     s'   = max(s, max |x| * (1 / 127))
//     code = clamp(rint(x / s'), -127, 127)             of the new rows
//     code = clamp(rint((code * s) / s'), -127, 127)    of the earlier ones
// each operation rounded to nearest in fp32, so that the codes follow from
// the inputs bit for bit; s' = 0 gives codes 0.  A NaN or infinity among the
// new rows makes s' +inf and the block's codes 0: the block then reads as NaN.
//
// What bounds them: memory.  One token writes D bytes of codes a head, and
// reads the earlier codes of its block only when the scale grows.
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

// Four consecutive values from p + i in fp32 (vec: 4-value aligned).
__device__ __forceinline__ f4 load4(const void* p, int dtype, int64_t i, bool vec) {
    f4 r;
    if (dtype == NB_F32) {
        const float* s = static_cast<const float*>(p) + i;
        if (vec) return *reinterpret_cast<const f4*>(s);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = s[e];
        return r;
    }
    const bf16_bits* s = static_cast<const bf16_bits*>(p) + i;
    if (vec) {
        const h4 v = *reinterpret_cast<const h4*>(s);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = bf16_to_f32(v[e]);
        return r;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = bf16_to_f32(s[e]);
    return r;
}

__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, f4 v, bool vec) {
    if (dtype == NB_F32) {
        float* d = static_cast<float*>(p) + i;
        if (vec) {
            *reinterpret_cast<f4*>(d) = v;
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = v[e];
        return;
    }
    bf16_bits* d = static_cast<bf16_bits*>(p) + i;
    h4 b;
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = f32_to_bf16_rne(v[e]);
    if (vec) {
        *reinterpret_cast<h4*>(d) = b;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = b[e];
}

// code of x at scale s (> 0, or 0 / +inf: code 0)
__device__ __forceinline__ int code_of(float x, float s) {
    if (!(s > 0.f && s < INFINITY)) return 0;
    return (int)fminf(fmaxf(rintf(x / s), -127.f), 127.f);
}

__device__ __forceinline__ uint32_t pack_codes(const int* c) {
    return (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 |
           (uint32_t)(c[3] & 255) << 24;
}

// four codes at scale s again at scale s2
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float s, float s2) {
    int c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = code_of((float)(int8_t)(w >> (8 * e)) * s, s2);
    return pack_codes(c);
}

// ---------------------------------------------------------------------------
// append: a workgroup takes one chunk and, of one key / value head, its keys,
// its values or the queries that share it.  A thread holds four consecutive
// dims of every (256 / (D / 4))-th row of the chunk in registers between the
// maximum and the codes.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kMaxD = 256;
constexpr int kMaxPass = kKvBlock * kMaxD / 4 / kThreads;

struct AppendArgs {
    const void* qkv;
    int64_t ld_qkv;
    const int32_t *slots, *positions, *chunks;
    const float *cos_t, *sin_t;
    int8_t *k, *v;
    float *k_scale, *v_scale;
    void* q_out;
    int64_t ld_q;
    int qkv_dtype, q_dtype, vec_in, vec_q;
    int n_pos, n_blocks, n_tokens, n_head, n_kv, D;
    float q_scale;
};

// Pairs (x0, x1), (x2, x3) turned by the angles of dims d, d + 2 at position
// pos: each product and sum rounded by itself, as nb_rope_kv_rows rounds them.
// A position outside the tables has no angle: NaN.
__device__ __forceinline__ f4 turn4(f4 x, const AppendArgs& a, int pos, int d) {
    float c[2], s[2];
    if (pos >= 0 && pos < a.n_pos) {
        const int64_t o = (int64_t)pos * (a.D / 2) + d / 2;
        c[0] = a.cos_t[o], c[1] = a.cos_t[o + 1];
        s[0] = a.sin_t[o], s[1] = a.sin_t[o + 1];
    } else {
        c[0] = c[1] = s[0] = s[1] = __builtin_nanf("");
    }
    f4 r;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float x0 = x[2 * e], x1 = x[2 * e + 1];
        r[2 * e] = x0 * c[e] - x1 * s[e];
        r[2 * e + 1] = x1 * c[e] + x0 * s[e];
    }
    return r;
}

__global__ __launch_bounds__(kThreads) void kv8_append_kernel(AppendArgs a) {
    __shared__ float wave_max[kThreads / 64];
    __shared__ __align__(16) uint8_t vt[kMaxD * kKvBlock];   // new value codes, as a block holds them
    const int32_t* ch = a.chunks + 4 * (int64_t)blockIdx.x;
    const int row0 = ch[0], n = ch[1];
    const int h = blockIdx.y / 3, part = blockIdx.y % 3;   // 0 keys, 1 values, 2 queries
    if (n <= 0 || row0 < 0 || row0 > a.n_tokens - n) return;
    const int D = a.D, per = D / 4, rows = kThreads / per;
    const int tr = threadIdx.x / per, d = 4 * (threadIdx.x - tr * per);
    const bool on = tr < rows;
    if (part == 2) {
        const int G = a.n_head / a.n_kv;
        if (!on) return;
        for (int e = tr; e < n * G; e += rows) {
            const int t = row0 + e / G, head = h * G + e % G;
            if (a.slots[t] < 0) continue;
            const f4 x = load4(a.qkv, a.qkv_dtype, t * a.ld_qkv + head * D + d, a.vec_in);
            const f4 r = turn4(x, a, a.positions[t], d);
            f4 q;
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = r[i] * a.q_scale;
            store4(a.q_out, a.q_dtype, t * a.ld_q + head * D + d, q, a.vec_q);
        }
        return;
    }
    const int slot = a.slots[row0];
    const int block = slot / kKvBlock, before = slot % kKvBlock;
    if (slot < 0 || block >= a.n_blocks || before + n > kKvBlock) return;
    const int64_t bh = (int64_t)block * a.n_kv + h;
    const int64_t col = (int64_t)(a.n_head + part * a.n_kv + h) * D + d;
    f4 x[kMaxPass];
    float most = 0.f;
#pragma unroll
    for (int p = 0; p < kMaxPass; ++p) {
        if (p * rows >= n) break;
        const int i = p * rows + tr;
        if (on && i < n) {
            const int64_t t = row0 + i;
            x[p] = load4(a.qkv, a.qkv_dtype, t * a.ld_qkv + col, a.vec_in);
            if (part == 0) x[p] = turn4(x[p], a, a.positions[t], d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float m = fabsf(x[p][e]);
                most = fmaxf(most, m < INFINITY ? m : INFINITY);   // (NaN counts as infinity)
            }
        }
    }
    most = wave64_max(most);
    if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
    float* scale = (part == 0 ? a.k_scale : a.v_scale) + bh;
    const float s = before > 0 ? *scale : 0.f;
    const float s2 = fmaxf(s, most * (1.f / 127.f));
    const bool again = before > 0 && s2 > s;   // the earlier codes change
    __syncthreads();   // every thread has the old scale
    if (threadIdx.x == 0 && (again || before == 0)) *scale = s2;
    int8_t* codes = (part == 0 ? a.k : a.v) + bh * kKvBlock * D;
    if (part == 0 && again) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes);
        for (int i = threadIdx.x; i < before * per; i += kThreads) w[i] = rescale4(w[i], s, s2);
    }
#pragma unroll
    for (int p = 0; p < kMaxPass; ++p) {
        if (p * rows >= n) break;
        const int i = p * rows + tr;
        if (on && i < n) {
            int c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = code_of(x[p][e], s2);
            if (part == 0) {
                *reinterpret_cast<uint32_t*>(codes + (before + i) * D + d) = pack_codes(c);
            } else if (n == 1 && !again) {
#pragma unroll
                for (int e = 0; e < 4; ++e) codes[(d + e) * kKvBlock + before] = (int8_t)c[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) vt[(d + e) * kKvBlock + before + i] = (uint8_t)c[e];
            }
        }
    }
    if (part == 0 || (n == 1 && !again)) return;
    // Values: 16 tokens of a dim at a time.  The block is this workgroup's
    // alone, so a piece that is new in part is read, completed and written.
    __syncthreads();
    const int end = before + n;
    const int first = again ? 0 : before / 16, last = (end + 15) / 16;   // pieces of a dim
    for (int i = threadIdx.x; i < D * (last - first); i += kThreads) {
        const int dim = i / (last - first), j = 16 * (first + i - dim * (last - first));
        uint4* g = reinterpret_cast<uint4*>(codes + dim * kKvBlock + j);
        const uint4 fresh = *reinterpret_cast<const uint4*>(&vt[dim * kKvBlock + j]);
        uint32_t w[4] = {fresh.x, fresh.y, fresh.z, fresh.w};
        if (j < before || j + 16 > end) {
            const uint4 held = *g;
            const uint32_t o[4] = {held.x, held.y, held.z, held.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t fresh_bytes = 0, held_bytes = 0;   // of the new and of the earlier tokens
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int at = j + 4 * e + b;
                    fresh_bytes |= at >= before && at < end ? 255u << (8 * b) : 0u;
                    held_bytes |= at < before ? 255u << (8 * b) : 0u;
                }
                const uint32_t old = again && held_bytes ? rescale4(o[e], s, s2) : o[e];
                w[e] = (w[e] & fresh_bytes) | (old & held_bytes) | (o[e] & ~(fresh_bytes | held_bytes));
            }
        }
        *g = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---------------------------------------------------------------------------
// read: a workgroup takes 64 slots of one head.  Values pass through LDS: a
// lane reads one slot's byte of a dim (slots of one block lie side by side),
// and the rows are written whole.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(
    const int32_t* slots, int64_t n, const int8_t* k, const int8_t* v, const float* k_scale,
    const float* v_scale, int n_blocks, int n_kv, int D, void* keys, void* values, int dtype,
    int vec) {
    __shared__ int8_t vt[64][kMaxD + 4];   // (rows 65 dwords apart: a row a bank)
    const int64_t i0 = blockIdx.x * 64LL;
    const int h = blockIdx.y;
    const int count = (int)min((int64_t)64, n - i0);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mine = lane < count ? slots[i0 + lane] : -1;
    if (mine >= 0 && mine / kKvBlock < n_blocks) {
        const int8_t* g = v + ((int64_t)(mine / kKvBlock) * n_kv + h) * kKvBlock * D + mine % kKvBlock;
        for (int d = wave; d < D; d += kThreads / 64) vt[lane][d] = g[d * kKvBlock];
    }
    __syncthreads();
    const int per = D / 4;
    for (int i = threadIdx.x; i < count * per; i += kThreads) {
        const int t = i / per, d = 4 * (i - t * per);
        const int slot = slots[i0 + t];
        f4 kr = {0.f, 0.f, 0.f, 0.f}, vr = kr;
        if (slot >= 0 && slot / kKvBlock < n_blocks) {
            const int64_t bh = (int64_t)(slot / kKvBlock) * n_kv + h;
            const uint32_t kw = *reinterpret_cast<const uint32_t*>(
                k + (bh * kKvBlock + slot % kKvBlock) * D + d);
            const uint32_t vw = *reinterpret_cast<const uint32_t*>(&vt[t][d]);
            const float ks = k_scale[bh], vs = v_scale[bh];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kr[e] = (float)(int8_t)(kw >> (8 * e)) * ks;
                vr[e] = (float)(int8_t)(vw >> (8 * e)) * vs;
            }
        }
        const int64_t o = ((i0 + t) * n_kv + h) * D + d;
        store4(keys, dtype, o, kr, vec);
        store4(values, dtype, o, vr, vec);
    }
}

bool four_aligned(const void* p, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % (dtype == NB_F32 ? 16 : 8) == 0;
}

}  // namespace

int kv8_max_head_dim() { return kMaxD; }

int launch_kv8_append(const void* qkv, int qkv_dtype, int64_t ld_qkv, const int32_t* slots,
                      const int32_t* positions, const int32_t* chunks, int n_chunks,
                      const float* cos_t, const float* sin_t, int n_pos, int8_t* k, int8_t* v,
                      float* k_scale, float* v_scale, int n_blocks, void* q_out, int q_dtype,
                      int64_t ld_q, int n_tokens, int n_head, int n_kv, int D,
                      hipStream_t stream) {
    AppendArgs a{qkv, ld_qkv, slots, positions, chunks, cos_t, sin_t, k, v, k_scale, v_scale,
                 q_out, ld_q, qkv_dtype, q_dtype,
                 four_aligned(qkv, qkv_dtype) && ld_qkv % 4 == 0,
                 four_aligned(q_out, q_dtype) && ld_q % 4 == 0,
                 n_pos, n_blocks, n_tokens, n_head, n_kv, D, (float)(1.0 / sqrt((double)D))};
    hipLaunchKernelGGL(kv8_append_kernel, dim3(n_chunks, 3 * n_kv), dim3(kThreads), 0, stream, a);
    return check_launch("nb_kv8_append");
}

int launch_kv8_read(const int32_t* slots, int64_t n, const int8_t* k, const int8_t* v,
                    const float* k_scale, const float* v_scale, int n_blocks, int n_kv, int D,
                    void* keys, void* values, int dtype, hipStream_t stream) {
    const int vec = four_aligned(keys, dtype) && four_aligned(values, dtype);
    hipLaunchKernelGGL(kv8_read_kernel, dim3((unsigned)((n + 63) / 64), n_kv), dim3(kThreads), 0,
                       stream, slots, n, k, v, k_scale, v_scale, n_blocks, n_kv, D, keys, values,
                       dtype, vec);
    return check_launch("nb_kv8_read");
}

}  // namespace nb
