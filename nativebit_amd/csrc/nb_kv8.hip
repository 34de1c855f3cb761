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
// reads the earlier codes of its block only when the scale grows.  Over three
// inputs in turn: append of 96 tokens of 96 requests, 32 query and 8 key / value
// heads of 128 in bf16: 6.5 us; of 8000 prompt tokens of those heads 71 us in fp32
// for 344 MB in and out (4.9 TB/s), 48 in bf16; of 6001 of 20 heads 69 in fp32 for
// 276 MB (4.0), 47 in bf16.  The latter on one input, part of it in the last level
// cache: 58 and 44 (one form for both types: 62 and 64, with each bf16 load waited
// for by its conversion).  Read, fp32 out: 6240 slots of 8 heads 15 us, 6577 of 20
// heads 33.
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
// (rows at any of their elements' places: one access all the same)
typedef __attribute__((ext_vector_type(4), aligned(4))) float f4_any;
typedef __attribute__((ext_vector_type(2), aligned(4))) float f2_any;
typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t u2_any;
typedef __attribute__((ext_vector_type(4), aligned(2))) uint16_t h4_any;

// The bits of four consecutive values from p + i: fp32, or two pairs of bf16 in
// the first two.  values4 makes fp32 of them, when all loads are out (a
// conversion beside its load would wait for each).
__device__ __forceinline__ f4 load4(const void* p, int dtype, int64_t i) {
    if (dtype == NB_F32) return *reinterpret_cast<const f4_any*>(static_cast<const float*>(p) + i);
    const u2_any w = *reinterpret_cast<const u2_any*>(static_cast<const bf16_bits*>(p) + i);
    return f4{__uint_as_float(w[0]), __uint_as_float(w[1]), 0.f, 0.f};
}
__device__ __forceinline__ f4 values4(f4 r, int dtype) {
    if (dtype == NB_F32) return r;
    const uint32_t a = __float_as_uint(r[0]), b = __float_as_uint(r[1]);
    return f4{__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16),
              __uint_as_float(b & 0xffff0000u)};
}

__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, f4 v) {
    if (dtype == NB_F32) {
        *reinterpret_cast<f4_any*>(static_cast<float*>(p) + i) = v;
        return;
    }
    h4_any b;
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = f32_to_bf16_rne(v[e]);
    *reinterpret_cast<h4_any*>(static_cast<bf16_bits*>(p) + i) = b;
}

// A block's scale as the codes need it.
struct Scale {
    float s, inv;
    bool usable;   // else (0 or +inf) codes are 0
};
__device__ __forceinline__ Scale scale_of(float s) {
    // (with an infinite reciprocal all quotients divide: where 1 / s or s is no
    // normal number)
    const bool usable = s > 0.f && s < INFINITY;
    return {s, s > 0x1p-120f && s < 0x1p120f ? __builtin_amdgcn_rcpf(s) : INFINITY, usable};
}

// clamp(rint(x / s), -127, 127).  x times the reciprocal is the quotient to
// 2^-21 of it, under 2^-13 where it counts, so a product that is further than
// that from the middle between two whole numbers rounds as the quotient does;
// the others divide (about one in 10^4).
__device__ __forceinline__ int code_of(float x, const Scale& s) {
    if (!s.usable) return 0;
    float q = x * s.inv;
    float r = rintf(q);
    if (!(fabsf(q - r) < 0.4995f)) r = rintf(x / s.s);
    return (int)fminf(fmaxf(r, -127.f), 127.f);
}

__device__ __forceinline__ uint32_t pack_codes(const int* c) {
    return (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 |
           (uint32_t)(c[3] & 255) << 24;
}

// four codes at scale s again at scale s2
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float s, const Scale& s2) {
    int c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = code_of((float)(int8_t)(w >> (8 * e)) * s, s2);
    return pack_codes(c);
}

// ---------------------------------------------------------------------------
// append: a workgroup takes one chunk and, of one key / value head, its keys,
// its values or the queries that share it.  A thread takes four consecutive
// dims of every (256 / (D / 4))-th row, all of whose loads are issued before
// the first is used, and holds them in registers between the maximum and the
// codes.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kMaxD = 256;
// LDS row of a dim's new value codes: 17 dwords, so that the 16 dims that a
// half row of lanes writes (4 apart) lie in 16 banks.
constexpr int kVtPitch = kKvBlock + 4;

struct AppendArgs {
    const void* qkv;
    int64_t ld_qkv;
    const int32_t *slots, *positions, *chunks;
    const float *cos_t, *sin_t;
    int8_t *k, *v;
    float *k_scale, *v_scale;
    void* q_out;
    int64_t ld_q;
    int q_dtype;
    int n_pos, n_blocks, n_tokens, n_head, n_kv, D;
    int shares;   // workgroups of a chunk's and head's queries
    float q_scale;
};

// Angles of dims d, d + 2 at a position; one outside the tables has none: NaN.
struct Angles { float c[2], s[2]; };
__device__ __forceinline__ Angles angles_at(const AppendArgs& a, int pos, int d) {
    Angles r;
    const bool in = pos >= 0 && pos < a.n_pos;
    const int64_t o = (int64_t)(in ? pos : 0) * (a.D / 2) + d / 2;
    if (!in) {
        r.c[0] = r.c[1] = r.s[0] = r.s[1] = __builtin_nanf("");
    } else {
        const f2_any c = *reinterpret_cast<const f2_any*>(a.cos_t + o);
        const f2_any s = *reinterpret_cast<const f2_any*>(a.sin_t + o);
        r.c[0] = c[0], r.c[1] = c[1], r.s[0] = s[0], r.s[1] = s[1];
    }
    return r;
}

// Pairs (x0, x1), (x2, x3) turned: each product and sum rounded by itself, as
// nb_rope_kv_rows rounds them.
__device__ __forceinline__ f4 turn4(f4 x, const Angles& w) {
    f4 r;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float x0 = x[2 * e], x1 = x[2 * e + 1];
        r[2 * e] = x0 * w.c[e] - x1 * w.s[e];
        r[2 * e + 1] = x1 * w.c[e] + x0 * w.s[e];
    }
    return r;
}

// The slot is looked at only when the first rows are on their way.
struct AppendChunk {
    int row0, n, slot;
    __device__ __forceinline__ int block() const { return slot / kKvBlock; }
    __device__ __forceinline__ int before() const { return slot % kKvBlock; }
    __device__ __forceinline__ bool stored(int n_blocks) const {
        return slot >= 0 && block() < n_blocks && before() + n <= kKvBlock;
    }
};

// The queries of a chunk's rows that share key / value head h, kRows of a
// thread at once; every shares-th batch from the share-th on.
template <int kDtype, int kRows>
__device__ __forceinline__ void append_queries(const AppendArgs& a, const AppendChunk& ch, int h,
                                               int share, int tr, int d, int rows) {
    // row e of the n G: token e / G, head e % G of theirs; e goes on by `rows`
    const int G = a.n_head / a.n_kv, total = ch.n * G;
    const int by_t = rows / G, by_g = rows - by_t * G;
    for (int e0 = kRows * rows * share + tr; e0 < total; e0 += kRows * rows * a.shares) {
        f4 x[kRows];
        int t[kRows], g[kRows], pos[kRows];
        Angles w[kRows];
        t[0] = e0 / G, g[0] = e0 - t[0] * G;
#pragma unroll
        for (int i = 1; i < kRows; ++i) {
            const bool wraps = g[i - 1] + by_g >= G;
            t[i] = t[i - 1] + by_t + (wraps ? 1 : 0);
            g[i] = g[i - 1] + by_g - (wraps ? G : 0);
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int64_t row = ch.row0 + min(t[i], ch.n - 1);   // (past the last: unused)
            pos[i] = a.positions[row];
            x[i] = load4(a.qkv, kDtype, row * a.ld_qkv + (h * G + g[i]) * a.D + d);
        }
        if (!ch.stored(a.n_blocks)) return;
#pragma unroll
        for (int i = 0; i < kRows; ++i) w[i] = angles_at(a, pos[i], d);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (t[i] >= ch.n) break;
            const f4 r = turn4(values4(x[i], kDtype), w[i]);
            f4 q;
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = r[j] * a.q_scale;
            store4(a.q_out, a.q_dtype, (ch.row0 + (int64_t)t[i]) * a.ld_q + (h * G + g[i]) * a.D + d, q);
        }
    }
}

// The keys (kKeys) or values of a chunk, kRows rows a thread.
template <int kDtype, int kRows, bool kKeys>
__device__ __forceinline__ void append_codes(const AppendArgs& a, const AppendChunk& ch, int h,
                                             int tr, int d, int rows, float* wave_max, uint8_t* vt) {
    const int D = a.D, n = ch.n;
    const bool on = tr < rows;
    const int64_t col = (int64_t)(a.n_head + (kKeys ? 0 : a.n_kv) + h) * D + d;
    // keys: rows tr, tr + rows, ..; values: kRows consecutive ones, whose codes
    // go to the transposed block by the dword
    auto row_of = [&](int p) { return kKeys ? p * rows + tr : tr * kRows + p; };
    f4 x[kRows];
    int pos[kRows];
#pragma unroll
    for (int p = 0; p < kRows; ++p) {
        const int64_t t = ch.row0 + min(row_of(p), n - 1);   // (past the last: the last again)
        if (kKeys) pos[p] = a.positions[t];
        x[p] = load4(a.qkv, kDtype, t * a.ld_qkv + col);
    }
    if (!ch.stored(a.n_blocks)) return;
    const int before = ch.before();
    const int64_t bh = (int64_t)ch.block() * a.n_kv + h;
    float* scale = (kKeys ? a.k_scale : a.v_scale) + bh;
    const float s = before > 0 ? *scale : 0.f;
#pragma unroll
    for (int p = 0; p < kRows; ++p) x[p] = values4(x[p], kDtype);
    if (kKeys) {
        constexpr int kBatch = kRows < 4 ? kRows : 4;
#pragma unroll
        for (int p0 = 0; p0 < kRows; p0 += kBatch) {
            Angles w[kBatch];
#pragma unroll
            for (int p = 0; p < kBatch; ++p) w[p] = angles_at(a, pos[p0 + p], d);
#pragma unroll
            for (int p = 0; p < kBatch; ++p) x[p0 + p] = turn4(x[p0 + p], w[p]);
        }
    }
    float most = 0.f;
#pragma unroll
    for (int p = 0; p < kRows; ++p) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float m = fabsf(x[p][e]);
            most = fmaxf(most, m < INFINITY ? m : INFINITY);   // (NaN counts as infinity)
        }
    }
    most = wave64_max(most);
    if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = most;
    __syncthreads();   // (and every thread has the old scale)
    most = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
    const float grown = fmaxf(s, most * (1.f / 127.f));
    const bool again = before > 0 && grown > s;   // the earlier codes change
    const Scale s2 = scale_of(grown);
    if (threadIdx.x == 0 && (again || before == 0)) *scale = grown;
    int8_t* codes = (kKeys ? a.k : a.v) + bh * kKvBlock * D;
    if (kKeys && again) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes);
        for (int i = threadIdx.x; i < before * (D / 4); i += kThreads) w[i] = rescale4(w[i], s, s2);
    }
    if constexpr (kKeys) {
#pragma unroll
        for (int p = 0; p < kRows; ++p) {
            const int i = row_of(p);
            if (!on || i >= n) continue;
            int c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = code_of(x[p][e], s2);
            *reinterpret_cast<uint32_t*>(codes + (before + i) * D + d) = pack_codes(c);
        }
        return;
    }
    if (n == 1 && !again) {   // a column of bytes
        if (tr == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) codes[(d + e) * kKvBlock + before] = (int8_t)code_of(x[0][e], s2);
        }
        return;
    }
    // vt[dim][i]: the code of new row i
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (!on || row_of(0) >= n) break;
        if constexpr (kRows % 4 == 0) {
#pragma unroll
            for (int p = 0; p < kRows; p += 4) {
                int c[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) c[r] = code_of(x[p + r][e], s2);
                *reinterpret_cast<uint32_t*>(&vt[(d + e) * kVtPitch + row_of(p)]) = pack_codes(c);
            }
        } else {
#pragma unroll
            for (int p = 0; p < kRows; ++p) vt[(d + e) * kVtPitch + row_of(p)] = (uint8_t)code_of(x[p][e], s2);
        }
    }
    // 16 tokens of a dim at a time.  The block is this workgroup's alone, so a
    // piece that is new in part is read, completed and written.
    __syncthreads();
    const int end = before + n;
    const int first = again ? 0 : before / 16, last = (end + 15) / 16;   // pieces of a dim
    for (int i = threadIdx.x; i < D * (last - first); i += kThreads) {
        const int dim = i / (last - first), j = 16 * (first + i - dim * (last - first));
        uint4* g = reinterpret_cast<uint4*>(codes + dim * kKvBlock + j);
        const uint8_t* row = &vt[dim * kVtPitch];
        uint32_t w[4];
        if (before % 4 == 0 && j >= before && j + 16 <= end) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(row + j - before + 4 * e);
        } else {
            const uint4 held = *g;
            const uint32_t o[4] = {held.x, held.y, held.z, held.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = j + 4 * e;
                const uint32_t old = again && at < before ? rescale4(o[e], s, s2) : o[e];
                w[e] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const uint32_t byte = at + b >= end      ? o[e] >> (8 * b)
                                          : at + b >= before ? row[at + b - before]
                                                             : old >> (8 * b);
                    w[e] |= (byte & 255) << (8 * b);
                }
            }
        }
        *g = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int kDtype, int kRows>
__device__ __forceinline__ void append_part(const AppendArgs& a, const AppendChunk& ch, int h,
                                            int part, int tr, int d, int rows, float* wave_max,
                                            uint8_t* vt) {
    if (part == 0) append_codes<kDtype, kRows, true>(a, ch, h, tr, d, rows, wave_max, vt);
    else append_codes<kDtype, kRows, false>(a, ch, h, tr, d, rows, wave_max, vt);
}

// kDtype: qkv's type.  kMost: head dims up to it (the most rows of a thread go by
// them).
template <int kDtype, int kMost>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(AppendArgs a) {
    __shared__ float wave_max[kThreads / 64];
    __shared__ __align__(16) uint8_t vt[kMost * kVtPitch];
    // the parts and heads of a chunk vary fastest: together they read its rows whole
    const int parts = (2 + a.shares) * a.n_kv;
    const int chunk = blockIdx.x / parts, which = blockIdx.x - chunk * parts;
    const int part = which / a.n_kv, h = which - part * a.n_kv;   // 0 keys, 1 values, 2 .. queries
    const auto* c = as_constant(a.chunks) + 4 * (int64_t)chunk;
    const int row0 = c[0], n = c[1];
    if (n <= 0 || row0 < 0 || n > kKvBlock || row0 > a.n_tokens - n) return;
    const AppendChunk ch{row0, n, as_constant(a.slots)[row0]};
    const int per = a.D / 4, rows = kThreads / per;
    const int tr = threadIdx.x / per, d = 4 * (threadIdx.x - tr * per);
    if (part >= 2) {
        if (tr >= rows) return;
        if (n * (a.n_head / a.n_kv) <= rows) append_queries<kDtype, 1>(a, ch, h, part - 2, tr, d, rows);
        else append_queries<kDtype, 4>(a, ch, h, part - 2, tr, d, rows);
        return;
    }
    // rows of a thread: a single token's, or up to 64 / rows (rows >= 8 up to 128
    // dims, >= 4 up to 256)
    if (n <= rows) append_part<kDtype, 1>(a, ch, h, part, tr, d, rows, wave_max, vt);
    else if (n <= 4 * rows) append_part<kDtype, 4>(a, ch, h, part, tr, d, rows, wave_max, vt);
    else if (n <= 8 * rows) append_part<kDtype, 8>(a, ch, h, part, tr, d, rows, wave_max, vt);
    else if constexpr (kMost > 128) append_part<kDtype, 16>(a, ch, h, part, tr, d, rows, wave_max, vt);
}

// ---------------------------------------------------------------------------
// read: a workgroup takes 32 slots of one head.  Values pass through LDS: half
// a wave's lanes read the slots' bytes of a dim (slots of one block lie side by
// side), and the rows are written whole.
// ---------------------------------------------------------------------------
constexpr int kReadSlots = 32;

__global__ __launch_bounds__(kThreads) void kv8_read_kernel(
    const int32_t* slots, int64_t n, const int8_t* k, const int8_t* v, const float* k_scale,
    const float* v_scale, int n_blocks, int n_kv, int D, void* keys, void* values, int dtype) {
    // (rows 65 dwords apart: a row a bank; read by the dword)
    __shared__ __align__(4) int8_t vt[kReadSlots][kMaxD + 4];
    const int64_t i0 = (int64_t)blockIdx.x * kReadSlots;
    const int h = blockIdx.y;
    const int count = (int)min((int64_t)kReadSlots, n - i0);
    const int lane = threadIdx.x % kReadSlots, half = threadIdx.x / kReadSlots;
    constexpr int kHalves = kThreads / kReadSlots;
    const int mine = lane < count ? slots[i0 + lane] : -1;
    const bool held = mine >= 0 && mine / kKvBlock < n_blocks;
    const int8_t* g = v + ((int64_t)(held ? mine / kKvBlock : 0) * n_kv + h) * kKvBlock * D +
                      (held ? mine % kKvBlock : 0);
    // a thread's first rows of keys and scales, under way with the values
    const int per = D / 4, rows = kThreads / per;
    const int tr = threadIdx.x / per, d = 4 * (threadIdx.x - tr * per);
    constexpr int kRows = 4;
    uint32_t kw[kRows];
    float ks[kRows], vs[kRows];
    bool ok[kRows];
    auto ask = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int slot = slots[i0 + min(t0 + i * rows, count - 1)];
            ok[i] = slot >= 0 && slot / kKvBlock < n_blocks;
            const int64_t bh = (int64_t)(ok[i] ? slot / kKvBlock : 0) * n_kv + h;
            kw[i] = *reinterpret_cast<const uint32_t*>(
                k + (bh * kKvBlock + (ok[i] ? slot % kKvBlock : 0)) * D + min(d, D - 4));
            ks[i] = k_scale[bh], vs[i] = v_scale[bh];
        }
    };
    ask(tr);
    for (int d0 = half; d0 < D; d0 += 16 * kHalves) {   // 16 dims of a lane's slot at once
        int8_t c[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) c[e] = g[min(d0 + kHalves * e, D - 1) * kKvBlock];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if (d0 + kHalves * e < D) vt[lane][d0 + kHalves * e] = c[e];
        }
    }
    __syncthreads();
    if (tr >= rows) return;
    for (int t0 = tr; t0 < count; t0 += kRows * rows) {
        if (t0 != tr) ask(t0);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int t = t0 + i * rows;
            if (t >= count) break;
            const uint32_t vw = *reinterpret_cast<const uint32_t*>(&vt[t][d]);
            f4 kr, vr;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kr[e] = ok[i] ? (float)(int8_t)(kw[i] >> (8 * e)) * ks[i] : 0.f;
                vr[e] = ok[i] ? (float)(int8_t)(vw >> (8 * e)) * vs[i] : 0.f;
            }
            const int64_t o = ((i0 + t) * n_kv + h) * D + d;
            store4(keys, dtype, o, kr);
            store4(values, dtype, o, vr);
        }
    }
}

}  // namespace

int kv8_max_head_dim() { return kMaxD; }

// Workgroups of a chunk's queries that share a head's keys: two batches of four
// rows a thread each, for the most rows that a chunk may have where some must have
// more than a token (but no more of all than a grid holds).  The list's length is a
// plan's bound, so that is not seen of a prompt of up to about twice as many tokens
// as there are requests: one workgroup takes its chunks' queries.  8000 bf16 tokens,
// 32 heads on 8 of 128: 84 us with one for all, 68 so; 6001 fp32, 16 on 4 of
// 256: 80 and 60 (one batch each 64).  64 single tokens and a prompt of 1000, 32
// heads on 8: 15.7 us, for the mean rows 22.1; the 64 alone 5.4, for the most
// rows 6.8.
static int query_shares(int n_chunks, int n_tokens, int n_head, int n_kv, int D) {
    const int64_t rows =
        (int64_t)(n_tokens > n_chunks ? std::min(n_tokens, kKvBlock) : 1) * (n_head / n_kv);
    const int batch = 8 * (kThreads / (D / 4));
    const int64_t most = ((1LL << 24) - 1) / ((int64_t)n_chunks * n_kv) - 2;
    return (int)std::max<int64_t>(1, std::min((rows + batch - 1) / batch, most));
}

int launch_kv8_append(const void* qkv, int qkv_dtype, int64_t ld_qkv, const int32_t* slots,
                      const int32_t* positions, const int32_t* chunks, int n_chunks,
                      const float* cos_t, const float* sin_t, int n_pos, int8_t* k, int8_t* v,
                      float* k_scale, float* v_scale, int n_blocks, void* q_out, int q_dtype,
                      int64_t ld_q, int n_tokens, int n_head, int n_kv, int D,
                      hipStream_t stream) {
    AppendArgs a{qkv, ld_qkv, slots, positions, chunks, cos_t, sin_t, k, v, k_scale, v_scale,
                 q_out, ld_q, q_dtype,
                 n_pos, n_blocks, n_tokens, n_head, n_kv, D,
                 query_shares(n_chunks, n_tokens, n_head, n_kv, D), (float)(1.0 / sqrt((double)D))};
    auto* kernel = qkv_dtype == NB_F32
                       ? (D <= 128 ? kv8_append_kernel<NB_F32, 128> : kv8_append_kernel<NB_F32, kMaxD>)
                       : (D <= 128 ? kv8_append_kernel<NB_BF16, 128> : kv8_append_kernel<NB_BF16, kMaxD>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_chunks * (2 + a.shares) * n_kv), dim3(kThreads), 0,
                       stream, a);
    return check_launch("nb_kv8_append");
}

int launch_kv8_read(const int32_t* slots, int64_t n, const int8_t* k, const int8_t* v,
                    const float* k_scale, const float* v_scale, int n_blocks, int n_kv, int D,
                    void* keys, void* values, int dtype, hipStream_t stream) {
    hipLaunchKernelGGL(kv8_read_kernel, dim3((unsigned)((n + kReadSlots - 1) / kReadSlots), n_kv), dim3(kThreads), 0,
                       stream, slots, n, k, v, k_scale, v_scale, n_blocks, n_kv, D, keys, values,
                       dtype);
    return check_launch("nb_kv8_read");
}

}  // namespace nb
