// Attention of a step's queries over the 8-bit block cache on int8 MFMAs
// (gfx950): the kernel of nb_kv8_attention.  nb_kv8_attention_2.hip and _3.hip
// build it for two and three digits, nb_kv8_attention.hip launches it.
//
// Mathematics.  The cache's codes are int8, and a scale belongs to a block of
// 64 tokens and head, so that both products are int8 ones if the other factor
// is cut into signed base-256 digits: a row of q is written as
//     q[d] = inv (a[d] 2^16 + b[d] 2^8 + c[d]),   inv = max |q| / (127 * 2^16)
// (rounded to nearest; digits -128 .. 127) and q . k = inv * k_scale * (A 2^16
// + B 2^8 + C) with A, B, C exact 32-bit sums of int8 products: 24 bits of q
// relative to its row's largest value, what fp32 has of that value.  Likewise the softmax
// weights of a block of 64 tokens, w = exp(s - m) in [0, 1] with m the block's
// largest score of the row, are three digits, and V's dims get
//     O = O exp(M - M') + (A 2^16 + B 2^8 + C) / (127 * 2^16) v_scale exp(m - M')
// with M, M' the running maximum before and after.  Scores, statistics and O
// are fp32.  Two digits (16 bits of q and of w, each relative to the largest of its row)
// serve bf16 outputs, whose own rounding is 2^-9: 2^-17 is lost of q and w.
// The codes go from memory into the MFMAs as they are.
//
// Layout.  Everything is transposed, so that a lane keeps one row from the
// scores to the output and nothing passes through LDS.  Lane (c, g) = (lane %
// 16, lane / 16) holds row c of a tile of 16 rows (a row is a query token and
// a head of those that share the keys).
//   S^T = K Q^T: MFMA mt takes the 16 tokens 16 (i / 4) + 4 mt + i % 4, so that
//     the lane ends with the scores of tokens 16 g + 4 mt + r, the 16
//     consecutive ones whose weights, packed to bytes, are its B operand of
//   O^T = V^T P^T: A = 16 dims x 64 tokens of V's [D][64]; the lane ends with
//     dims 16 dt + 4 g + r of its row.
// A wave walks whole blocks; the next block's keys are loaded while the
// softmax and the second product run, its values during the first.
//
// Split.  A workgroup takes one chunk and key / value head.  Up to 16 rows
// (single tokens) all its waves take the blocks in turn and are joined through
// LDS at the end; more rows go to the waves 16 each, which then walk the same
// blocks (one trip through the L1 for all).  Few chunks over long caches are
// split over workgroups too (gridDim.z), with partial results in a workspace
// that a second launch joins.
#pragma once

#include <math.h>

#include "nb_device.h"
#include "nb_internal.h"

namespace nb {

struct Kv8AttentionArgs {
    const void* q;
    int64_t ld_q;
    const int32_t *chunks, *lens, *table;
    int64_t table_stride;
    const int8_t *k, *v;
    const float *k_scale, *v_scale;
    void* out;
    int64_t ld_out;
    const float* slopes;
    const int32_t* prefix;
    float* part;        // split results: [rows][heads][splits][D], then (m, l) pairs
    int q_dtype, out_dtype, vec_q, vec_out;
    int n_chunks, n_tokens, R, max_blocks, n_blocks, n_head, n_kv, D, window;
    float softcap;
};

// A chunk that holds rows of the call (else n = 0).
struct Kv8Chunk { int row0, n, request, pos0; };
__device__ __forceinline__ Kv8Chunk kv8_chunk(const Kv8AttentionArgs& a, int i) {
    const int32_t* c = a.chunks + 4 * (int64_t)i;
    Kv8Chunk h{c[0], c[1], c[2], c[3]};
    if (h.n < 0 || h.n > kKvBlock || h.row0 < 0 || h.row0 > a.n_tokens - h.n || h.request < 0 ||
        h.request >= a.R || h.pos0 < 0 || h.pos0 > a.max_blocks * kKvBlock - h.n) {
        h.n = 0;
    }
    return h;
}

namespace {

typedef __attribute__((ext_vector_type(4))) int i4;
typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(4))) uint16_t h4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.0e38f;   // stands for a maximum of -inf in differences

// The maximum / sum over the four lanes (c, 0 .. 3) of a row.
__device__ __forceinline__ float rows_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Four numbers I + 0x8080 (three digits) or I + 0x80 (two), the digits' bytes
// gathered by digit: d[0] the lowest.
template <int ND>
__device__ __forceinline__ void digits4(const uint32_t* w, uint32_t* d) {
    const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x05010400);   // w0.0 w1.0 w0.1 w1.1
    const uint32_t hi = __builtin_amdgcn_perm(w[3], w[2], 0x05010400);
    d[0] = __builtin_amdgcn_perm(hi, lo, 0x05040100) ^ 0x80808080u;
    d[1] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
    if constexpr (ND == 3) {
        d[1] ^= 0x80808080u;
        d[2] = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0602) |
               __builtin_amdgcn_perm(w[3], w[2], 0x06020c0c);
    }
}

template <int ND>
struct Digits {
    static constexpr float kTop = ND == 3 ? 127.f * 65536.f : 127.f * 256.f;   // of |value| = 1
    static constexpr int kBias = ND == 3 ? 0x8080 : 0x80;
};

// tanh to 3e-7 of its value: the odd series up to 0.3 (next term 1.3e-10 of
// it), above it 1 - 2 / (e^2t + 1), whose 6e-8 are 2e-7 of 0.29.  For bf16
// outputs the latter alone: 6e-8 of the cap in the exponent.
template <int ND>
__device__ __forceinline__ float tanh_of(float t) {
    const float e = __builtin_amdgcn_exp2f(t * (2.f * kLog2e));
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
    if constexpr (ND == 2) return far;
    const float z = t * t;
    float p = 0.0035921280f;
    p = fmaf(p, z, -0.0088632356f);
    p = fmaf(p, z, 0.0218694885f);
    p = fmaf(p, z, -0.0539682540f);
    p = fmaf(p, z, 0.1333333333f);
    p = fmaf(p, z, -0.3333333333f);
    const float near = fmaf(t * z, p, t);
    return z < 0.09f ? near : far;
}

template <int DT, int ND, bool kRules, int NW>
__global__ __launch_bounds__(NW * 64, (DT <= 8 ? 2 : 1)) void kv8_attention_kernel(
    Kv8AttentionArgs a) {
    constexpr int DS = (DT + 3) / 4;   // steps of 64 dims of the first product
    constexpr float kTop = Digits<ND>::kTop;
    constexpr int kSlot = (DT * 4 + 2) * 64;   // floats of a wave's result
    __shared__ float joined[NW / 2 * kSlot];
    // Heads vary fastest (neighbouring workgroups, dealt to the XCDs in turn,
    // then share no keys, and with heads a multiple of 8 an XCD's L2 holds its
    // own heads only); the last chunks, which see the longest caches, go first.
    const int h = blockIdx.x % a.n_kv;
    const Kv8Chunk ch = kv8_chunk(a, a.n_chunks - 1 - blockIdx.x / a.n_kv);
    if (ch.n == 0) return;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.n_head / a.n_kv, D = a.D;
    const int rows = ch.n * G, tiles = (rows + 15) / 16;
    // waves of a row group (rw) and of a row's blocks (kw)
    int rw = 1;
    while (rw < NW && rw < tiles) rw *= 2;
    const int kw = NW / rw, wr = wave & (rw - 1), wk = wave / rw;
    const int split = blockIdx.z, splits = gridDim.z;
    const int32_t* blocks = a.table + ch.request * a.table_stride;
    const int cached = min(max(a.lens[ch.request], 0), a.max_blocks * kKvBlock);

    for (int group = blockIdx.y; group * rw < tiles; group += gridDim.y) {
        const int tile = group * rw + wr;
        const bool idle = tile >= tiles;
        const int row = min(tile * 16 + c, rows - 1);   // (rows past the last repeat it)
        const int tok = row / G, head = h * G + row - tok * G;
        const int pos = ch.pos0 + tok;
        const int64_t q_row = ch.row0 + tok;

        // ---- the row's digits -------------------------------------------------
        i4 qd[ND][DS];
        float inv;
        {
            float x[DS][16];
            float most = 0.f, odd = 0.f;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const int d0 = 64 * s + 16 * g;
                const int64_t at = q_row * a.ld_q + head * D + d0;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[s][e] = 0.f;
                if (d0 < D) {   // (D is a multiple of 16)
                    if (a.q_dtype == NB_F32) {
                        const float* p = static_cast<const float*>(a.q) + at;
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            if (a.vec_q) {
                                const f4 v = *reinterpret_cast<const f4*>(p + e);
                                x[s][e] = v[0], x[s][e + 1] = v[1], x[s][e + 2] = v[2], x[s][e + 3] = v[3];
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[s][e + i] = p[e + i];
                            }
                        }
                    } else {
                        const bf16_bits* p = static_cast<const bf16_bits*>(a.q) + at;
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            if (a.vec_q) {
                                const h4 v = *reinterpret_cast<const h4*>(p + e);
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[s][e + i] = bf16_to_f32(v[i]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[s][e + i] = bf16_to_f32(p[e + i]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    most = fmaxf(most, fabsf(x[s][e]));
                    odd += x[s][e] * 0.f;   // NaN if any is NaN or infinite
                }
            }
            // (rows below 2^-100 keep their size: 127 * 2^16 / most stays finite)
            most = fmaxf(rows_max(most), 0x1p-100f);
            odd = rows_sum(odd);
            const float f = kTop / most;
            inv = most / kTop + odd;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    uint32_t w[4], d[3];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y = fminf(fmaxf(rintf(x[s][e + i] * f), -kTop), kTop);
                        w[i] = (uint32_t)((int)y + Digits<ND>::kBias);
                    }
                    digits4<ND>(w, d);
#pragma unroll
                    for (int n = 0; n < ND; ++n) qd[n][s][e / 4] = (int)d[n];
                }
            }
        }
        const float to_log2 = inv * kLog2e;
        const float slope = kRules && a.slopes ? a.slopes[head] : 0.f;

        // ---- what the tile's rows see -----------------------------------------
        // row: positions [lo, hi) and [0, pre); the tile: blocks [0, pt) and
        // [wt, t_end)
        const int tok_lo = min(tile * 16, rows - 1) / G, tok_hi = min(tile * 16 + 15, rows - 1) / G;
        const int pos_lo = ch.pos0 + tok_lo, pos_hi = ch.pos0 + tok_hi;
        const int pre = kRules && a.prefix ? min(max(a.prefix[ch.request], 0), cached) : 0;
        const bool windowed = kRules && a.window > 0;
        const int hi = pos + 1, lo = windowed ? max(0, hi - a.window) : 0;
        const int lo_max = windowed ? max(0, pos_hi + 1 - a.window) : 0;
        const int t_end = (max(pos_hi + 1, pre) + kKvBlock - 1) / kKvBlock;
        int wt = windowed ? max(0, pos_lo + 1 - a.window) / kKvBlock : 0;
        int pt = (pre + kKvBlock - 1) / kKvBlock;
        if (wt <= pt) wt = pt = 0;
        const int count = idle ? 0 : pt + t_end - wt;
        const int i_end = (int)((int64_t)count * (split + 1) / splits);
        int i = (int)((int64_t)count * split / splits) + wk;

        f4 o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = f4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;   // l: of the lane's own tokens

        i4 kf[4][DS], vf[DT];
        // lane's places in a block: dims past D are read at the row's start
        // (their digits of q are zero), value dims past D at the last one (not
        // stored)
        int k_at[DS];
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            const int d0 = 64 * s + 16 * g;
            k_at[s] = (16 * (c >> 2) + (c & 3)) * D + (d0 < D ? d0 : 0);
        }
        auto place = [&](int n) { return n < pt ? n : n - pt + wt; };
        auto block_at = [&](int n) {
            return __builtin_amdgcn_readfirstlane(blocks[place(min(n, i_end - 1))]);
        };
        auto valid = [&](int b) { return b >= 0 && b < a.n_blocks; };
        auto load_keys = [&](int b) {
            const auto* p = as_global(a.k + ((int64_t)(valid(b) ? b : 0) * a.n_kv + h) * kKvBlock * D);
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
                for (int s = 0; s < DS; ++s) {
                    kf[mt][s] = *reinterpret_cast<const __attribute__((address_space(1))) i4*>(
                        p + k_at[s] + 4 * mt * D);
                }
            }
        };
        auto load_values = [&](int b) {
            const auto* p = as_global(a.v + ((int64_t)(valid(b) ? b : 0) * a.n_kv + h) * kKvBlock * D);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                vf[dt] = *reinterpret_cast<const __attribute__((address_space(1))) i4*>(
                    p + min(16 * dt + c, D - 1) * kKvBlock + 16 * g);
            }
        };
        int b = 0, b_next = 0;
        if (i < i_end) {
            b = block_at(i);
            b_next = block_at(i + kw);
            load_keys(b);
            load_values(b);
        }
        for (; i < i_end; i += kw) {
            const int64_t bh = (int64_t)(valid(b) ? b : 0) * a.n_kv + h;
            const float ks = a.k_scale[bh], vs = a.v_scale[bh];
            const int j0 = place(i) * kKvBlock;
            const bool more = i + kw < i_end;
            // ---- scores -------------------------------------------------------
            float x[16];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                i4 acc = {0, 0, 0, 0}, low = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < DS; ++s)
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[mt][s], qd[ND - 1][s], acc, 0, 0, 0);
                acc <<= 8;
#pragma unroll
                for (int s = 0; s < DS; ++s)
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[mt][s], qd[ND - 2][s], acc, 0, 0, 0);
                if constexpr (ND == 3) {
#pragma unroll
                    for (int s = 0; s < DS; ++s)
                        low = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[mt][s], qd[0][s], low, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[4 * mt + r] = ND == 3 ? fmaf((float)acc[r], 256.f, (float)low[r]) : (float)acc[r];
                }
            }
            const int b_now = b;
            b = b_next;
            if (more) {
                load_keys(b);
                b_next = block_at(i + 2 * kw);
            }
            if constexpr (kRules) {
                const float f = inv * ks;
                const float per_cap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;
                const float from = (float)(j0 + 16 * g - pos);   // distance of the lane's first token
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float s = x[e] * f;
                    if (a.softcap > 0.f) s = a.softcap * tanh_of<ND>(s * per_cap);
                    x[e] = fmaf(slope, from + (float)e, s) * kLog2e;
                }
            } else {
                const float f = to_log2 * ks;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] *= f;
            }
            // some row of the tile does not see the whole block
            if (!valid(b_now) ||
                !((j0 + kKvBlock <= pos_lo + 1 && j0 >= lo_max) || j0 + kKvBlock <= pre)) {
                const int jl = j0 + 16 * g;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = jl + e;
                    const bool seen = valid(b_now) && ((j < hi && j >= lo) || j < pre);
                    x[e] = seen ? x[e] : -INFINITY;
                }
            }
            // ---- weights ------------------------------------------------------
            float top = x[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
            top = rows_max(top);
            const float base = fmaxf(top, kLowest);
            float sum = 0.f;
            i4 pd[ND];
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                uint32_t w[4], d[3];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(x[e + r] - base);
                    sum += p;
                    // 2^23 + bias + rint(p kTop): the low mantissa bits
                    w[r] = __float_as_uint(fmaf(p, kTop, 8388608.f + (float)Digits<ND>::kBias));
                }
                digits4<ND>(w, d);
#pragma unroll
                for (int n = 0; n < ND; ++n) pd[n][e / 4] = (int)d[n];
            }
            const float m_new = fmaxf(m, top), safe = fmaxf(m_new, kLowest);
            const float beta = __builtin_amdgcn_exp2f(m - safe);
            const float share = __builtin_amdgcn_exp2f(top - safe);
            l = fmaf(l, beta, sum * share);
            m = m_new;
            // (a row that sees nothing of the block takes nothing of its scale)
            const float gamma = top == -INFINITY ? 0.f : share * vs * (1.f / kTop);
            // ---- O ------------------------------------------------------------
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                i4 acc = {0, 0, 0, 0}, low = {0, 0, 0, 0};
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[dt], pd[ND - 1], acc, 0, 0, 0);
                acc <<= 8;
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[dt], pd[ND - 2], acc, 0, 0, 0);
                if constexpr (ND == 3)
                    low = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[dt], pd[0], low, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float t =
                        ND == 3 ? fmaf((float)acc[r], 256.f, (float)low[r]) : (float)acc[r];
                    o[dt][r] = fmaf(gamma, t, o[dt][r] * beta);
                }
            }
            if (more) load_values(b);
        }
        l = rows_sum(l);

        // ---- the waves of a row joined, halves to halves ----------------------
        for (int half = kw / 2; half > 0; half /= 2) {
            float* slot = joined + ((wk >= half ? wk - half : wk) * rw + wr) * kSlot + lane;
            if (wk >= half && wk < 2 * half) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) slot[(4 * dt + r) * 64] = o[dt][r];
                }
                slot[4 * DT * 64] = m;
                slot[(4 * DT + 1) * 64] = l;
            }
            __syncthreads();
            if (wk < half) {
                const float m2 = slot[4 * DT * 64], l2 = slot[(4 * DT + 1) * 64];
                const float m_new = fmaxf(m, m2), safe = fmaxf(m_new, kLowest);
                const float w1 = __builtin_amdgcn_exp2f(m - safe), w2 = __builtin_amdgcn_exp2f(m2 - safe);
                l = l * w1 + l2 * w2;
                m = m_new;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[dt][r] = o[dt][r] * w1 + slot[(4 * dt + r) * 64] * w2;
                }
            }
            __syncthreads();
        }
        if (wk > 0 || tile * 16 + c >= rows) continue;   // (no barrier below)
        if (splits > 1) {
            const int64_t at = (q_row * a.n_head + head) * splits + split;
            float* ml = a.part + (int64_t)a.n_tokens * a.n_head * splits * D + 2 * at;
            if (g == 0) ml[0] = m, ml[1] = l;
            if (l == 0.f) continue;   // nothing seen: the join does not read its dims
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const int d = 16 * dt + 4 * g;
                if (d < D) *reinterpret_cast<f4*>(a.part + at * D + d) = o[dt];
            }
            continue;
        }
        const float norm = l == 0.f ? 0.f : 1.f / l;   // (a row that sees nothing is 0)
        const int64_t to = q_row * a.ld_out + head * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = 16 * dt + 4 * g;
            if (d >= D) continue;
            const f4 v = o[dt] * norm;
            if (a.out_dtype == NB_F32) {
                float* p = static_cast<float*>(a.out) + to + d;
                if (a.vec_out) {
                    *reinterpret_cast<f4*>(p) = v;
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[r] = v[r];
                }
            } else {
                bf16_bits* p = static_cast<bf16_bits*>(a.out) + to + d;
                h4 w;
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = f32_to_bf16_rne(v[r]);
                if (a.vec_out) {
                    *reinterpret_cast<h4*>(p) = w;
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[r] = w[r];
                }
            }
        }
    }
}

template <int DT, int ND, int NW>
void launch_kv8_form(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    if (rules) {
        hipLaunchKernelGGL((kv8_attention_kernel<DT, ND, true, NW>), grid, dim3(NW * 64), 0, stream, a);
    } else {
        hipLaunchKernelGGL((kv8_attention_kernel<DT, ND, false, NW>), grid, dim3(NW * 64), 0, stream, a);
    }
}

template <int ND>
void launch_kv8_digits(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    if (a.D <= 64) {
        launch_kv8_form<4, ND, 4>(a, grid, rules, stream);
    } else if (a.D <= 96) {
        launch_kv8_form<6, ND, 4>(a, grid, rules, stream);
    } else if (a.D <= 128) {
        launch_kv8_form<8, ND, 4>(a, grid, rules, stream);
    } else {
        launch_kv8_form<16, ND, 4>(a, grid, rules, stream);
    }
}

}  // namespace

void launch_kv8_attention_2(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream);
void launch_kv8_attention_3(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream);

}  // namespace nb
