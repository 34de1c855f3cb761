// Attention of a step's queries over the 8-bit block cache on int8 MFMAs
// (gfx950): the kernel of nb_kv8_attention.  nb_kv8_attention_tokens_2.hip,
// _tokens_3.hip, _prompts_2.hip and _prompts_3.hip build it, nb_kv8_attention.hip
// launches it.
//
// Mathematics.  The cache's codes are int8, and a scale belongs to a block of
// 64 tokens and head, so that both products are int8 ones if the other factor
// is cut into signed base-256 digits: a row of q is written as
//     q[d] = inv (a[d] 2^16 + b[d] 2^8 + c[d]),   inv = max |q| / (127 * 2^16)
// (rounded to nearest; digits -128 .. 127) and q . k = inv * k_scale * 2^8 (A 2^8
// + B + C / 2^8) with A, B, C exact 32-bit sums of int8 products, C / 2^8 rounded
// to a whole number: 24 bits of q relative to its row's largest value, what fp32
// has of that value, and half a unit of 2^-15 of it in the sum.  Likewise the softmax
// weights of a block of 64 tokens, w = exp(s - m) in [0, 1] with m the block's
// largest score of the row, are three digits, and V's dims get
//     O = O + (A 2^8 + B + C / 2^8) / (127 * 2^8) v_scale exp(m - M)
// with M the row's running reference, its largest score or up to 16 binary
// orders less (O is scaled when it moves).  Scores, statistics and O are fp32.
// Two digits (16 bits of q and of w, each relative to the largest of its row)
// serve bf16 outputs, whose own rounding is 2^-9: 2^-17 is lost of q and w.
// Rows of q with a few large dims need more: where the largest value is over
// kEven times the mean one, q has a digit more (32 bits, bf16 outputs 24), and
// with 32 the sum's halves A 2^8 + B and C 2^8 + E are added in fp32.  One dim 3000
// times the others, keys small there, 512 tokens: errors of 1.9e-5 without it and
// 1.1e-7 with (products in fp32 2.6e-7), with bf16 outputs 4.1e-3 and 4.8e-4 (their
// rounding).  The rule is a row's own and so is its result; a tile without such
// rows skips the digit.  8003 prompt tokens, 20 heads of 128: 365 us, 409 with the
// digit in all rows.  The codes go into the MFMAs as they are.
//
// Layout.  Everything is transposed, so that a lane keeps one row from the
// scores to the output and no row's numbers pass through LDS.  Lane (c, g) =
// (lane % 16, lane / 16) holds row c of a tile of 16 rows (a row is a query
// token and a head of those that share the keys).
//   S^T = K Q^T: MFMA mt takes the 16 tokens 16 (i / 4) + 4 mt + i % 4, so that
//     the lane ends with the scores of tokens 16 g + 4 mt + r, the 16
//     consecutive ones whose weights, packed to bytes, are its B operand of
//   O^T = V^T P^T: A = 16 dims x 64 tokens of V's [D][64]; the lane ends with
//     dims 16 dt + 4 g + r of its row.
//
// Chunks of up to 32 rows (single tokens): a wave takes whole blocks of one or
// two tiles of rows, codes straight to registers, a block's values on their way
// during the softmax and the next one's keys during the second product; the
// waves of a tile take the blocks in turn and are joined through LDS at the end.
// More rows: the four waves take 16 each and walk the blocks together, two at a
// time, whose codes each wave brings a quarter of to LDS (directly, with no
// register between) while the product before runs.  Without LDS every wave
// fetches all codes through the L1: 8003 prompt tokens of two requests, 20
// heads of 128, 505 us then; 375 with LDS, scalar loads of tables and scales
// and the reference that moves seldom; two blocks a turn (one maximum, one step
// of O) instead of one: 384 to 371 in turn on one card.  Now 337 to 389 by the drawn
// lengths.
//
// Split.  A workgroup takes one chunk and key / value head (and 64 rows of it, 32
// of single tokens).  Few of them over long caches are split over workgroups too
// (gridDim.y), with partial results in a workspace that a second launch joins.
//
// What bounds it.  Single tokens: the codes, 2 D bytes a cached token and head.
// 64 requests of 960 positions at most, 20 heads of 128: 51 us, 4.8 TB/s from
// memory (44 where they come from the last level cache); 128 of 2000, 8 heads:
// 77 us, 5.1 TB/s; six of 40000, 8 heads: 74 us with the join, 5.0 TB/s.
// Prompts: the issue of vector instructions and MFMAs, which overlap only in
// part.  16384 tokens, 16 heads on 2: 546 TFLOP/s (of 4 D a score; each takes
// three int8 MFMA products in fp32, two for bf16 outputs: 729).  Of 360 us for
// 8003 tokens 125 go with the second product, 85 with the first, 10 with the
// exponentials.
#pragma once

#include <math.h>

#include <type_traits>

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
    int q_dtype, out_dtype;
    int n_chunks, n_tokens, R, max_blocks, n_blocks, n_head, n_kv, D, window;
    float softcap;
};

// A chunk that holds rows of the call (else n = 0).
struct Kv8Chunk { int row0, n, request, pos0; };
__device__ __forceinline__ Kv8Chunk kv8_chunk(const Kv8AttentionArgs& a, int i) {
    const auto* c = as_constant(a.chunks) + 4 * (int64_t)i;
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
// (rows of q and out at any of their elements' places: one access all the same)
typedef __attribute__((ext_vector_type(4), aligned(4))) float f4_any;
typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t u2_any;
typedef __attribute__((ext_vector_type(4), aligned(2))) uint16_t h4_any;

constexpr float kLog2e = 1.44269504088896340736f;
// Rows of q whose largest value is over this many times their mean one have a
// digit more (of 128 normal ones it is 3.5 times).
constexpr float kEven = 8.f;
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

// Four numbers I + 0x808080 (four digits), I + 0x8080 (three) or I + 0x80 (two),
// the digits' bytes gathered by digit: d[0] the lowest.
template <int ND>
__device__ __forceinline__ void digits4(const uint32_t* w, uint32_t* d) {
    const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x05010400);   // w0.0 w1.0 w0.1 w1.1
    const uint32_t hi = __builtin_amdgcn_perm(w[3], w[2], 0x05010400);
    d[0] = __builtin_amdgcn_perm(hi, lo, 0x05040100) ^ 0x80808080u;
    d[1] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
    if constexpr (ND >= 3) d[1] ^= 0x80808080u;
    if constexpr (ND == 3) {
        d[2] = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0602) |
               __builtin_amdgcn_perm(w[3], w[2], 0x06020c0c);
    }
    if constexpr (ND == 4) {
        const uint32_t lo2 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);   // w0.2 w1.2 w0.3 w1.3
        const uint32_t hi2 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
        d[2] = __builtin_amdgcn_perm(hi2, lo2, 0x05040100) ^ 0x80808080u;
        d[3] = __builtin_amdgcn_perm(hi2, lo2, 0x07060302);
    }
}

// The largest of three; as one instruction (fmaxf of a number that came by
// several ways quiets it first, with an instruction more for each).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <int ND>
struct Digits {
    // (of |value| = 1)
    static constexpr float kTop = ND == 4 ? 127.f * 16777216.f : ND == 3 ? 127.f * 65536.f : 127.f * 256.f;
    static constexpr int kBias = ND == 4 ? 0x808080 : ND == 3 ? 0x8080 : 0x80;
};

// o *= beta where flag (the same in all lanes) is not 0.  One instruction to
// the compiler: a branch in the program makes it keep O twice, with a copy of
// all of it on the way round.
__device__ __forceinline__ void scale_if(int flag, float beta, float (&o)[4]) {
    asm("s_cmp_eq_u32 %5, 0\n\t"
        "s_cbranch_scc1 .Lkv8_kept_%=\n\t"
        "v_mul_f32 %0, %0, %4\n\t"
        "v_mul_f32 %1, %1, %4\n\t"
        "v_mul_f32 %2, %2, %4\n\t"
        "v_mul_f32 %3, %3, %4\n"
        ".Lkv8_kept_%=:"
        : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3])
        : "v"(beta), "s"(flag)
        : "scc");
}

// cap * tanh(x f) + add, to_cap = add + cap.  The tanh to 3e-7 of its value: the
// odd series up to 0.3 (next term 1.3e-10 of it), above it 1 - 2 / (e^2t + 1),
// whose 6e-8 are 2e-7 of 0.29.  For bf16 outputs and caps up to kNearCap the
// latter alone: 2^-22 of the cap in the exponent, 2^-14 at most.
constexpr float kNearCap = 256.f;
template <int ND>
__device__ __forceinline__ float capped(float x, float f, float cap, float add, float to_cap) {
    const float e = __builtin_amdgcn_exp2f(x * (f * (2.f * kLog2e)));
    const float far = fmaf(__builtin_amdgcn_rcpf(e + 1.f), -2.f * cap, to_cap);
    if constexpr (ND == 2) return far;
    const float t = x * f;
    const float z = t * t;
    float p = 0.0035921280f;
    p = fmaf(p, z, -0.0088632356f);
    p = fmaf(p, z, 0.0218694885f);
    p = fmaf(p, z, -0.0539682540f);
    p = fmaf(p, z, 0.1333333333f);
    p = fmaf(p, z, -0.3333333333f);
    return z < 0.09f ? fmaf(fmaf(t * z, p, t), cap, add) : far;
}

// The same for bf16 outputs and larger caps, to 2^-16 of its value: t - t^3 / 3 up
// to 2^-6.
__device__ __forceinline__ float capped_wide(float x, float f, float cap) {
    const float t = x * f, z = t * t;
    const float e = __builtin_amdgcn_exp2f(t * (2.f * kLog2e));
    const float far = fmaf(__builtin_amdgcn_rcpf(e + 1.f), -2.f * cap, cap);
    return z < 0x1p-12f ? t * cap * fmaf(z, -0.33333333f, 1.f) : far;
}

// 16 bytes a lane from `src` to LDS at m0 + 16 * lane, m0 = `lds`; counted by
// vmcnt, unseen by the compiler.  (s_nop: the wait state between a scalar write
// of m0 and a load to LDS.)
__device__ __forceinline__ void to_lds16(uint32_t lds, const void* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds), "v"(src)
                 : "memory", "m0");
}

// Waves of a workgroup: four where chunks share codes, else two.  Four for single
// tokens cost their start and end: one of 200 requests of 300 positions, 20
// heads of 128, 69 us against 57; of 128 of 2000, 8 heads 86 and 80, of 64 of 960,
// 20 heads 55 and 53 (one wave: 56, 82, 52, but 51 against 39 for 40 of 1000, 8
// heads of 256).
constexpr int kv8_waves(bool prompts) { return prompts ? 4 : 2; }

// LDS of a workgroup: the waves' results to join, or two blocks' codes.
template <int DT, bool kShared>
constexpr int kv8_lds_bytes() {
    const int join = kv8_waves(kShared) / 2 * (DT * 4 + 2) * 64 * 4, codes = 4 * 64 * 16 * DT;
    return kShared && codes > join ? codes : join;
}

// Behind it the waves' lowest digits of q, each lane its own, read back by the
// first products that need them.  In registers (4 for 64 dims) they cost the
// others: 4096 prompt tokens, 16 heads of 256 on 4, 218 us so and 235; 1500 with
// every rule, 20 heads of 128, 162 and 176.
template <int DT, bool kShared>
constexpr int kv8_low_bytes() {
    return kv8_waves(kShared) * ((DT + 3) / 4) * 64 * 16;
}

// ND: digits of the weights and of most rows of q, NQ of the others.
template <int DT, int ND, bool kRules, bool kWhole, int NW, bool kShared>
__device__ __forceinline__ void kv8_rows(const Kv8AttentionArgs& a, const Kv8Chunk& ch, int h, char* lds,
                                         char* low_lds) {
    constexpr int DS = (DT + 3) / 4;   // steps of 64 dims of the first product
    constexpr int NQ = ND + 1;
    constexpr float kTop = Digits<ND>::kTop, kTopQ = Digits<NQ>::kTop;
    constexpr int kSlot = (DT * 4 + 2) * 64;      // floats of a wave's result
    constexpr int kCodes = 64 * 16 * DT;          // bytes of a block's keys or values
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int D = kWhole ? 16 * DT : a.D;
    const int per = kWhole ? DT : D / 16;   // 16-byte pieces of a key
    const int G = a.n_head / a.n_kv;
    const int rows = ch.n * G, tiles = (rows + 15) / 16;
    // waves of a row group (rw) and of a row's blocks (kw)
    const int rw = kShared || tiles > 2 ? NW : tiles, kw = NW / rw;
    const int wr = wave & (rw - 1), wk = wave / rw;
    const int split = blockIdx.y, splits = gridDim.y;
    const auto* blocks = as_constant(a.table) + ch.request * a.table_stride;
    const int cached = min(max(as_constant(a.lens)[ch.request], 0), a.max_blocks * kKvBlock);
    const int pre = kRules && a.prefix ? min(max(as_constant(a.prefix)[ch.request], 0), cached) : 0;
    const bool windowed = kRules && a.window > 0;

    for (int group = blockIdx.z; group * rw < tiles; group += gridDim.z) {
        const int tile = group * rw + wr;
        const int row = min(tile * 16 + c, rows - 1);   // (rows past the last repeat it)
        const int tok = row / G, head = h * G + row - tok * G;
        const int pos = ch.pos0 + tok;
        const int q_row = ch.row0 + tok;

        // ---- what the rows see --------------------------------------------------
        // a row: positions [lo, hi) and [0, pre); the tile's rows pos_lo .. pos_hi;
        // the waves that walk together: blocks [0, pt) and [wt, t_end)
        auto position = [&](int r) { return ch.pos0 + min(r, rows - 1) / G; };
        const int pos_lo = position(tile * 16), pos_hi = position(tile * 16 + 15);
        const int hi = pos + 1, lo = windowed ? max(0, hi - a.window) : 0;
        const int lo_max = windowed ? max(0, pos_hi + 1 - a.window) : 0;
        const int first = kShared ? position(group * NW * 16) : pos_lo;
        const int last = kShared ? position(group * NW * 16 + NW * 16 - 1) : pos_hi;
        const int t_end = (max(last + 1, pre) + kKvBlock - 1) / kKvBlock;
        int wt = windowed ? max(0, first + 1 - a.window) / kKvBlock : 0;
        int pt = (pre + kKvBlock - 1) / kKvBlock;
        if (wt <= pt) wt = pt = 0;
        const int count = !kShared && tile >= tiles ? 0 : pt + t_end - wt;
        const int i_end = (int)((int64_t)count * (split + 1) / splits);
        int i = (int)((int64_t)count * split / splits) + wk;

        // ---- the row of q, and the first block on its way -----------------------
        // (its bits: pairs of bf16 stay as they are until the block's loads are
        // out, and dims past D are read at the head's start)
        float x[DS][16];
        if (a.q_dtype == NB_F32) {
            const float* p = static_cast<const float*>(a.q) + q_row * a.ld_q + head * D;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const int d0 = 64 * s + 16 * g, at = d0 < D ? d0 : 0;   // (D is a multiple of 16)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f4 v = *reinterpret_cast<const f4_any*>(p + at + e);
                    x[s][e] = v[0], x[s][e + 1] = v[1], x[s][e + 2] = v[2], x[s][e + 3] = v[3];
                }
            }
        } else {
            const bf16_bits* p = static_cast<const bf16_bits*>(a.q) + q_row * a.ld_q + head * D;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const int d0 = 64 * s + 16 * g, at = d0 < D ? d0 : 0;
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const u2_any v = *reinterpret_cast<const u2_any*>(p + at + e);
                    x[s][e] = __uint_as_float(v[0]), x[s][e + 2] = __uint_as_float(v[1]);
                    x[s][e + 1] = x[s][e + 3] = 0.f;
                }
            }
        }
        // Lane's places in a block, in memory: dims past D are read at the row's
        // start (their digits of q are zero), value dims past D at the last one
        // (not stored).
        const int key_row = 16 * (c >> 2) + (c & 3);   // (+ 4 mt)
        auto place = [&](int n) { return n < pt ? n : n - pt + wt; };
        auto block_at = [&](int n) { return blocks[place(min(n, i_end - 1))]; };
        auto valid = [&](int b) { return b >= 0 && b < a.n_blocks; };
        auto codes_at = [&](const int8_t* p, int b) {
            return p + ((int64_t)(valid(b) ? b : 0) * a.n_kv + h) * kKvBlock * D;
        };
        i4 kf[4][DS], vf[DT];
        auto load_keys = [&](int b) {
            const auto* p = as_global(codes_at(a.k, b));
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
                for (int s = 0; s < DS; ++s) {
                    const int d0 = 64 * s + 16 * g;
                    kf[mt][s] = *reinterpret_cast<const __attribute__((address_space(1))) i4*>(
                        p + key_row * D + (d0 < D ? d0 : 0) + 4 * mt * D);
                }
            }
        };
        auto load_values = [&](int b) {
            const auto* p = as_global(codes_at(a.v, b));
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                vf[dt] = *reinterpret_cast<const __attribute__((address_space(1))) i4*>(
                    p + (kWhole ? 16 * dt + c : min(16 * dt + c, D - 1)) * kKvBlock + 16 * g);
            }
        };
        // In LDS the 16-byte pieces of a key (and of a dim's values) are exchanged
        // by its row, so that the 8 lanes that are served together (rows c ..
        // c + 7, one piece) reach all 32 banks: keys of 8 or 16 pieces by c & 7
        // (token bits 0, 1, 4), of 4 by token bits 1, 4; values by dim bits 1, 2.
        // (No conflicts counted at 128 dims.  Other sizes stay in order.)
        auto key_swap = [&](int token) {
            return per % 8 == 0 ? (token & 3) | (token >> 4 & 1) << 2
                   : per == 4   ? (token >> 1 & 1) | (token >> 4 & 1) << 1
                                : 0;
        };
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        constexpr int kIns = (DT + NW - 1) / NW;   // loads of a wave for a block's keys
        // (keys of two blocks, then the values of two)
        auto stage_keys = [&](int b, int slot) {
            const int8_t* p = codes_at(a.k, b);
#pragma unroll
            for (int n = 0; n < kIns; ++n) {
                const int ins = wave + NW * n;   // 64 pieces each
                if (DT % NW != 0 || !kWhole) {
                    if (ins >= per) break;
                }
                const int l = 64 * ins + lane;
                const int token = l / per, piece = l - token * per;
                to_lds16(lds0 + slot * kCodes + 1024 * ins, p + token * D + 16 * (piece ^ key_swap(token)));
            }
        };
        auto stage_values = [&](int b, int slot) {
            const int8_t* p = codes_at(a.v, b);
#pragma unroll
            for (int n = 0; n < kIns; ++n) {
                const int ins = wave + NW * n;
                if (DT % NW != 0 || !kWhole) {
                    if (ins >= per) break;
                }
                const int l = 64 * ins + lane, dim = l >> 2;
                to_lds16(lds0 + (2 + slot) * kCodes + 1024 * ins,
                         p + dim * kKvBlock + 16 * ((l & 3) ^ (dim >> 1 & 3)));
            }
        };
        // the block, or two, under way and the next
        constexpr int kAtOnce = kShared ? 2 : 1;
        int now[kAtOnce], next[kAtOnce];
        if (i < i_end) {
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) now[e] = block_at(i + e), next[e] = block_at(i + kAtOnce * kw + e);
            if constexpr (kShared) {
                stage_keys(now[0], 0);
                if (i + 1 < i_end) stage_keys(now[1], 1);
            } else {
                load_keys(now[0]);
            }
        }

        // ---- the row's digits -------------------------------------------------
        i4 qd[ND][DS];   // but the lowest digit
        volatile i4* low_q = reinterpret_cast<volatile i4*>(low_lds) + wave * DS * 64 + lane;
        float inv;
        bool fine;   // the row has a lowest digit
        {
            if (a.q_dtype != NB_F32) {
#pragma unroll
                for (int s = 0; s < DS; ++s) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const uint32_t w = __float_as_uint(x[s][e]);
                        x[s][e] = __uint_as_float(w << 16);
                        x[s][e + 1] = __uint_as_float(w & 0xffff0000u);
                    }
                }
            }
            float most = 0.f, odd = 0.f, size = 0.f;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                if (64 * s + 16 * g >= D) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[s][e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    most = fmaxf(most, fabsf(x[s][e]));
                    size += fabsf(x[s][e]);
                    odd += x[s][e] * 0.f;   // NaN if any is NaN or infinite
                }
            }
            most = rows_max(most);
            fine = most * (float)D > kEven * rows_sum(size);
            // (rows below 2^-90 keep their size: 127 * 2^24 / most stays finite)
            most = fmaxf(most, 0x1p-90f);
            odd = rows_sum(odd);
            const float top = fine ? kTopQ : kTopQ / 256.f;
            const int shift = fine ? 0 : 8;
            const float f = top / most;
            inv = most / kTopQ + odd;
            inv *= NQ == 4 ? 65536.f : 256.f;   // (the first product's units)
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                i4 low;
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    uint32_t w[4], d[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float y = fminf(fmaxf(rintf(x[s][e + r] * f), -top), top);
                        w[r] = ((uint32_t)(int)y << shift) + (uint32_t)Digits<NQ>::kBias;
                    }
                    digits4<NQ>(w, d);
                    low[e / 4] = (int)d[0];
#pragma unroll
                    for (int n = 0; n < ND; ++n) qd[n][s][e / 4] = (int)d[n + 1];
                }
                low_q[64 * s] = low;
            }
        }
        const int any_fine = __builtin_amdgcn_readfirstlane(__any(fine));
        const float to_log2 = inv * kLog2e;
        // (for exponents of 2)
        const float slope = kRules && a.slopes ? a.slopes[head] * kLog2e : 0.f;
        const float cap = a.softcap * kLog2e, per_cap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;

        float o[DT][4];   // (no vectors: their elements would move in and out of them)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][0] = o[dt][1] = o[dt][2] = o[dt][3] = 0.f;
        float m = -INFINITY, l = 0.f;   // l: of the lane's own tokens

        // Waves at their weights go before those at a product, whose MFMAs run on
        // meanwhile: four prompts of 500 tokens, 24 heads of 64 on 8: 37.8 to 36.2
        // us (bf16 outputs 31.5 to 30.1), 4096 tokens, 16 heads of 256 on 4: 326 to
        // 308.  Not with two digits for longer heads: 233 to 245 there.
        constexpr bool kAhead = kShared && (DT <= 4 || ND == 3);
        // Blocks n .. n + NB - 1 of the walk, one or two, at once: key(e, mt, s) and
        // value(e, dt) give the codes of the e-th, between() runs after the first
        // product.  Two share their weights' largest score and one step of O; their
        // value scales are factors of the weights' digits.
        auto walk = [&](auto nb, int n, auto&& key, auto&& between, auto&& value)
                        __attribute__((always_inline)) {
            constexpr int NB = decltype(nb)::value;
            // ---- scores -------------------------------------------------------
            float x[NB][16], unit[NB], vs[NB], top[NB];
            bool there[NB];
#pragma unroll
            for (int e = 0; e < NB; ++e) {
                there[e] = valid(now[e]);
                const int64_t bh = (int64_t)(there[e] ? now[e] : 0) * a.n_kv + h;
                // scores in units of 1 / unit: x * unit is the exponent of 2
                unit[e] = as_constant(a.k_scale)[bh];
                vs[e] = as_constant(a.v_scale)[bh];
            }
            auto product = [&](auto lowest) __attribute__((always_inline)) {
                i4 q0[DS];
                if constexpr (lowest.value) {
#pragma unroll
                    for (int s = 0; s < DS; ++s) q0[s] = low_q[64 * s];
                }
#pragma unroll
                for (int e = 0; e < NB; ++e) {
#pragma unroll
                    for (int mt = 0; mt < 4; ++mt) {
                        i4 acc = {0, 0, 0, 0}, low = {0, 0, 0, 0}, f[DS];
                        auto sum = [&](i4 to, const i4* q) {
#pragma unroll
                            for (int s = 0; s < DS; ++s)
                                to = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[s], q[s], to, 0, 0, 0);
                            return to;
                        };
#pragma unroll
                        for (int s = 0; s < DS; ++s) f[s] = key(e, mt, s);
                        float* y = &x[e][4 * mt];
                        acc = sum(acc, qd[ND - 1]) << 8;
                        if constexpr (ND == 3) low = sum(low, qd[0]);
                        if constexpr (!lowest.value) {
                            if constexpr (ND == 3) acc += (low + 128) >> 8;
                            acc = sum(acc, qd[ND - 2]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) y[r] = (float)acc[r];
                        } else {
                            low = sum(low << 8, q0);
                            if constexpr (ND == 2) acc += (low + 128) >> 8;
                            acc = sum(acc, qd[ND - 2]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                y[r] = (float)acc[r];
                                if constexpr (ND == 3)   // (the others as without)
                                    y[r] = fine ? fmaf((float)low[r], 0x1p-16f, y[r])
                                                : (float)(acc[r] + ((low[r] + 32768) >> 16));
                            }
                        }
                    }
                }
            };
            if (any_fine) product(std::true_type{});
            else product(std::false_type{});
            between();
#pragma unroll
            for (int e = 0; e < NB; ++e) {
                const int j0 = place(n + e) * kKvBlock, j_lane = j0 + 16 * g;
                if constexpr (kRules) {
                    // slope * distance, from the lane's first token on
                    const float at = slope * (float)(j_lane - pos);
                    if (a.softcap > 0.f) {
                        const float f = inv * unit[e] * per_cap;
                        if (ND == 2 && a.softcap > kNearCap) {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                x[e][i] = fmaf(slope, (float)i, capped_wide(x[e][i], f, cap) + at);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                x[e][i] = capped<ND>(x[e][i], f, cap, fmaf(slope, (float)i, at),
                                                     fmaf(slope, (float)i, at + cap));
                        }
                    } else {
                        const float f = to_log2 * unit[e];
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[e][i] = fmaf(x[e][i], f, fmaf(slope, (float)i, at));
                    }
                    unit[e] = 1.f;
                } else {
                    unit[e] *= to_log2;
                }
                // some row of the tile does not see the whole block
                if (!there[e] ||
                    !((j0 + kKvBlock <= pos_lo + 1 && j0 >= lo_max) || j0 + kKvBlock <= pre)) {
                    const int end = there[e] ? hi : 0, pre_end = there[e] ? pre : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = j_lane + i;
                        const bool seen = ((j < end) & (j >= lo)) | (j < pre_end);
                        x[e][i] = seen ? x[e][i] * unit[e] : -INFINITY;
                    }
                    unit[e] = 1.f;   // (a unit of 0 or infinity times -inf is NaN)
                }
                float most = x[e][0];
#pragma unroll
                for (int i = 1; i < 15; i += 2) most = max3(most, x[e][i], x[e][i + 1]);
                most = max3(most, x[e][15], x[e][15]);
                top[e] = rows_max(most) * unit[e];
            }
            if constexpr (kAhead) __builtin_amdgcn_s_setprio(1);
            // ---- weights ------------------------------------------------------
            float all = top[0];
            if constexpr (NB == 2) all = fmaxf(all, top[1]);
            const float base = fmaxf(all, kLowest);
            // p is at most 1 + 2^-24 |base|, which its digits hold up to 2^12
            const bool far = fabsf(base) > 4096.f;
            if (__any(far)) {
#pragma unroll
                for (int e = 0; e < NB; ++e) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[e][i] *= far ? unit[e] : 1.f;
                    unit[e] = far ? 1.f : unit[e];
                }
            }
            // (a row that sees nothing of a block takes nothing of its scale)
            float v_scale = top[0] == -INFINITY ? 0.f : vs[0];
            float digits_of_1[NB] = {kTop};
            if constexpr (NB == 2) {
                // v_scale: what the largest weights of a block bring at most, of
                // the block that brings more, so that p * digits_of_1 is up to
                // kTop (the larger scale alone would cost the other block's weights
                // the scales' ratio where the row hardly weighs its block).  A
                // scale that is NaN or infinite makes it NaN.
                const float v0 = v_scale, v1 = top[1] == -INFINITY ? 0.f : vs[1];
                const float c0 = v0 * __builtin_amdgcn_exp2f(top[0] - base);
                const float c1 = v1 * __builtin_amdgcn_exp2f(top[1] - base);
                v_scale = fmaxf(c0, c1) + (c0 + c1) * 0.f;
                // (a ratio over 2^100 has weights under 2^-100)
                digits_of_1[0] = kTop * fminf(v0 / v_scale, 0x1p100f);
                digits_of_1[1] = kTop * fminf(v1 / v_scale, 0x1p100f);
            }
            float sum = 0.f;
            i4 pd[NB][ND];
#pragma unroll
            for (int e = 0; e < NB; ++e) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    uint32_t w[4], d[3];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(x[e][i + r], unit[e], -base));
                        sum += p;
                        // 2^23 + bias + rint(p kTop): the low mantissa bits
                        w[r] = __float_as_uint(
                            fmaf(p, digits_of_1[e], 8388608.f + (float)Digits<ND>::kBias));
                    }
                    digits4<ND>(w, d);
#pragma unroll
                    for (int j = 0; j < ND; ++j) pd[e][j][i / 4] = (int)d[j];
                }
            }
            // m follows a row's largest score only when that is 2^16 ahead:
            // shares up to 2^16 cost fp32 sums nothing, scaling O does (by 1 in
            // the rows that stay: a row's result is its own)
            const bool ahead = all > m + 16.f;
            const float m_new = ahead ? all : m;
            const float beta = ahead ? __builtin_amdgcn_exp2f(m - fmaxf(m_new, kLowest)) : 1.f;
            const int any_ahead = __builtin_amdgcn_readfirstlane(__any(ahead));
            l *= beta;
            m = m_new;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) scale_if(any_ahead, beta, o[dt]);
            const float share = __builtin_amdgcn_exp2f(all - fmaxf(m, kLowest));
            l = fmaf(sum, share, l);
            const float gamma = v_scale == 0.f ? 0.f : share * v_scale * (ND == 3 ? 256.f / kTop : 1.f / kTop);
            if constexpr (kAhead) __builtin_amdgcn_s_setprio(0);
            // ---- O ------------------------------------------------------------
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                i4 acc = {0, 0, 0, 0}, low = {128, 128, 128, 128}, f[NB];
#pragma unroll
                for (int e = 0; e < NB; ++e) f[e] = value(e, dt);
#pragma unroll
                for (int e = 0; e < NB; ++e)
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[e], pd[e][ND - 1], acc, 0, 0, 0);
                if constexpr (ND == 3) {
#pragma unroll
                    for (int e = 0; e < NB; ++e)
                        low = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[e], pd[e][0], low, 0, 0, 0);
                    acc = (acc << 8) + (low >> 8);
                } else {
                    acc <<= 8;
                }
#pragma unroll
                for (int e = 0; e < NB; ++e)
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[e], pd[e][ND - 2], acc, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[dt][r] = fmaf(gamma, (float)acc[r], o[dt][r]);
            }
        };
        if constexpr (kShared) {
            // Two blocks a turn: their values load during the first product, the
            // next two's keys during the rest.
            const i4* mine = reinterpret_cast<const i4*>(lds);
            const int swap = key_swap(key_row);   // (the same for all mt)
            auto key = [&](int e, int mt, int s) {
                const int piece = 4 * s + g < per ? 4 * s + g : 0;
                return mine[e * (kCodes / 16) + (key_row + 4 * mt) * per + (piece ^ swap)];
            };
            auto value = [&](int e, int dt) {
                return mine[(2 + e) * (kCodes / 16) + (16 * dt + c) * 4 + (g ^ (c >> 1 & 3))];
            };
            // this wave's loads are there, then everybody's, and what was read
            // before is free
            auto arrive = [] {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            };
            for (; i < i_end; i += 2) {
                const bool two = i + 1 < i_end;
                arrive();
                stage_values(now[0], 0);
                if (two) stage_values(now[1], 1);
                auto between = [&] {
                    arrive();
                    if (i + 2 < i_end) stage_keys(next[0], 0);
                    if (i + 3 < i_end) stage_keys(next[1], 1);
                };
                if (two) walk(std::integral_constant<int, 2>{}, i, key, between, value);
                else walk(std::integral_constant<int, 1>{}, i, key, between, value);
                now[0] = next[0], now[1] = next[1];
                next[0] = block_at(i + 4), next[1] = block_at(i + 5);
            }
            __syncthreads();   // the last values are read
        } else {
            // `more`: the next block's loads are issued (a constant, so that every
            // path to the next block has them in flight and waits for no more)
            auto direct = [&](auto more) __attribute__((always_inline)) {
                walk(
                    std::integral_constant<int, 1>{}, i, [&](int, int mt, int s) { return kf[mt][s]; },
                    [&] { load_values(now[0]); }, [&](int, int dt) { return vf[dt]; });
                if constexpr (decltype(more)::value) {
                    now[0] = next[0];
                    next[0] = block_at(i + 2 * kw);
                    load_keys(now[0]);
                }
            };
            for (; i + kw < i_end; i += kw) direct(std::true_type{});
            if (i < i_end) direct(std::false_type{});
        }
        l = rows_sum(l);

        // ---- the waves of a row joined, halves to halves ----------------------
        for (int half = kw / 2; half > 0; half /= 2) {
            float* slot = reinterpret_cast<float*>(lds) + ((wk >= half ? wk - half : wk) * rw + wr) * kSlot + lane;
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
            const int64_t at = ((int64_t)q_row * a.n_head + head) * splits + split;
            float* ml = a.part + (int64_t)a.n_tokens * a.n_head * splits * D + 2 * at;
            if (g == 0) ml[0] = m, ml[1] = l;
            if (l == 0.f) continue;   // nothing seen: the join does not read its dims
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const int d = 16 * dt + 4 * g;
                if (d < D) *reinterpret_cast<f4*>(a.part + at * D + d) = f4{o[dt][0], o[dt][1], o[dt][2], o[dt][3]};
            }
            continue;
        }
        const float norm = l == 0.f ? 0.f : 1.f / l;   // (a row that sees nothing is 0)
        const int64_t to = q_row * a.ld_out + head * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = 16 * dt + 4 * g;
            if (d >= D) continue;
            const f4 v = f4{o[dt][0], o[dt][1], o[dt][2], o[dt][3]} * norm;
            if (a.out_dtype == NB_F32) {
                *reinterpret_cast<f4_any*>(static_cast<float*>(a.out) + to + d) = v;
            } else {
                h4_any w;
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = f32_to_bf16_rne(v[r]);
                *reinterpret_cast<h4_any*>(static_cast<bf16_bits*>(a.out) + to + d) = w;
            }
        }
    }
}

// kPrompts: chunks of over two tiles of 16 rows share their blocks' codes
// through LDS, the others of the launch go as without.
// Registers: those of three waves a SIMD, for heads of over 128 dims (O alone is
// 64 of them) of two.  4096 prompt tokens, 16 heads of 256 on 4: 327 us, 230
// for bf16 outputs; with all registers, one a SIMD, 374 and 310.
template <int DT, int ND, bool kRules, bool kWhole, bool kPrompts>
__global__ __launch_bounds__(kv8_waves(kPrompts) * 64, (DT <= 8 ? 3 : 2)) void kv8_attention_kernel(
    Kv8AttentionArgs a) {
    constexpr int kWaves = kv8_waves(kPrompts);
    // (the codes first: loads to LDS take addresses of 16 bits)
    constexpr int kBytes = kv8_lds_bytes<DT, kPrompts>();
    __shared__ __align__(16) char lds[kBytes + kv8_low_bytes<DT, kPrompts>()];
    // Heads vary fastest (neighbouring workgroups, dealt to the XCDs in turn,
    // then share no keys, and with heads a multiple of 8 an XCD's L2 holds its
    // own heads only); the last chunks, which see the longest caches, go first.
    const int h = blockIdx.x % a.n_kv;
    const Kv8Chunk ch = kv8_chunk(a, a.n_chunks - 1 - blockIdx.x / a.n_kv);
    if (ch.n == 0) return;
    if constexpr (kPrompts) {
        if (ch.n * (a.n_head / a.n_kv) > 32) {
            kv8_rows<DT, ND, kRules, kWhole, kWaves, true>(a, ch, h, lds, lds + kBytes);
            return;
        }
    }
    kv8_rows<DT, ND, kRules, kWhole, kWaves, false>(a, ch, h, lds, lds + kBytes);
}

template <int DT, int ND, bool kWhole, bool kPrompts>
void launch_kv8_form(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    if (rules) {
        hipLaunchKernelGGL((kv8_attention_kernel<DT, ND, true, kWhole, kPrompts>), grid,
                           dim3(kv8_waves(kPrompts) * 64), 0, stream, a);
    } else {
        hipLaunchKernelGGL((kv8_attention_kernel<DT, ND, false, kWhole, kPrompts>), grid,
                           dim3(kv8_waves(kPrompts) * 64), 0, stream, a);
    }
}

// The head dim as a constant where it fills the tiles, else the next tiles' form.
template <int ND, bool kPrompts>
void launch_kv8_digits(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    if (a.D == 64) launch_kv8_form<4, ND, true, kPrompts>(a, grid, rules, stream);
    else if (a.D < 64) launch_kv8_form<4, ND, false, kPrompts>(a, grid, rules, stream);
    else if (a.D == 96) launch_kv8_form<6, ND, true, kPrompts>(a, grid, rules, stream);
    else if (a.D == 128) launch_kv8_form<8, ND, true, kPrompts>(a, grid, rules, stream);
    else if (a.D < 128) launch_kv8_form<8, ND, false, kPrompts>(a, grid, rules, stream);
    else if (a.D == 256) launch_kv8_form<16, ND, true, kPrompts>(a, grid, rules, stream);
    else launch_kv8_form<16, ND, false, kPrompts>(a, grid, rules, stream);
}

}  // namespace

// Two or three digits; with or without chunks that share codes through LDS.
using Kv8AttentionLaunch = void(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream);
Kv8AttentionLaunch launch_kv8_tokens_2, launch_kv8_tokens_3, launch_kv8_prompts_2, launch_kv8_prompts_3;

}  // namespace nb
