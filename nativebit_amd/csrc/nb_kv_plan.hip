// The plan of a serving step over a block cache, from the requests' lengths
// (gfx950): nb_kv_plan and nb_kv_release.
//
//   nb_kv_plan      request r has lens[r] tokens cached and brings new[r].  The
//                   rows of the step are the requests' new tokens in order;
//                   with L = lens, N = new (clipped to the rows that exist), E =
//                   L + N (clipped to the table and the longest request)
//                     first[r] = sum N[< r]             row of its first token
//                     need[r]  = ceil(E / 64) - ceil(L / 64)
//                     base[r]  = sum need[< r]
//                   and new block number k of the step (k < free count) is the
//                   free list's entry free count - 1 - k.  Row first[r] + i
//                   lies at position L + i, slot 64 * block + position % 64.
//                   A chunk is a run of rows of one request inside one block.
//   nb_kv_release   blocks of finished requests back on the free list.
//
// Bound by latency: a step of 8 requests moves 400 bytes, one of 700 requests
// and 30000 rows 290 KB.  So one launch, without a pass over the requests in
// front of it: every workgroup forms the three sums over all requests itself
// (4096 at most, 4 KB of lengths from the L2 and three scans) and then writes
// its share of the rows, chunks and table entries, each found by a binary
// search in the sums, which stay in LDS.  Inputs and outputs are different
// memory (of the table only entries past a request's cached blocks are
// written, which no workgroup reads), so the workgroups need no order.
// 3.6 us for 8 requests, 5.8 for 700 (24 with the sums by 64-bit LDS
// atomics, which go one at a time).
#include <algorithm>

#include "nb_device.h"
#include "nb_internal.h"

namespace nb {
namespace {

constexpr int kMaxRequests = 4096;
constexpr int kPlanThreads = 256;

// Inclusive sum over a wave's lanes, by row shifts and row broadcasts.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast 31 into rows 2, 3
    return v;
}

// Exclusive sum over the workgroup's threads; `total` that of all.
template <int kWaves>
__device__ __forceinline__ int block_scan(int v, int* wave_sums, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = wave_scan(v);
    __syncthreads();   // the sums of an earlier call are read
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const int s = wave_sums[w];
        before += w < wave ? s : 0;
        all += s;
    }
    total = all;
    return before + sum - v;
}

// The first of n ascending inclusive sums that is over i (n if none is).
__device__ __forceinline__ int find(const int* upto, int n, int i) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

struct PlanArgs {
    int32_t* table;
    int64_t table_stride;
    const int32_t *lens, *asked, *free_blocks, *state;
    int R, max_blocks, n_blocks, n_tokens, n_chunks, max_len;
    int32_t *slots, *positions, *chunks, *lens_out, *state_out;
};

__device__ __forceinline__ int blocks_of(int tokens) {
    return (int)(((int64_t)tokens + kKvBlock - 1) / kKvBlock);
}

// kItems consecutive requests a thread.
template <int kItems>
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a) {
    constexpr int kMost = kItems * kPlanThreads, kWaves = kPlanThreads / 64;
    __shared__ int rows_upto[kMost];     // inclusive sums over the requests: rows,
    __shared__ int need_upto[kMost];     // blocks they need,
    __shared__ int chunks_upto[kMost];   // chunks
    __shared__ int wave_sums[kWaves];
    __shared__ long long wave_dropped[kWaves];
    const int tid = threadIdx.x, nt = kPlanThreads;
    const int cap = a.max_blocks * kKvBlock;
    // where a request of len tokens and n new ones ends, blocks allowing (one that
    // is longer than it may be stays as it is)
    auto end_of = [&](int len, int n) {
        return max(len, (int)min((int64_t)len + n, (int64_t)min(cap, a.max_len)));
    };
    const int left = min(max(a.state[0], 0), a.n_blocks);
    const int r0 = tid * kItems;
    int len[kItems], asked[kItems], n[kItems], want[kItems], count[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const bool in = r0 + i < a.R;
        len[i] = in ? min(max(a.lens[r0 + i], 0), cap) : 0;
        asked[i] = in ? max(a.asked[r0 + i], 0) : 0;
    }
    // rows: what is asked, up to the rows that exist (clipped to n_tokens each,
    // which changes no result and keeps the sums in 31 bits)
    int sum = 0, total;
#pragma unroll
    for (int i = 0; i < kItems; ++i) sum += min(asked[i], a.n_tokens);
    int upto = block_scan<kWaves>(sum, wave_sums, total);
    sum = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int first = min(upto, a.n_tokens);
        upto += min(asked[i], a.n_tokens);
        n[i] = min(upto, a.n_tokens) - first;
        rows_upto[r0 + i] = first + n[i];
        want[i] = blocks_of(end_of(len[i], n[i])) - blocks_of(len[i]);
        sum += want[i];
    }
    long long dropped = 0;   // tokens asked for and not stored
    int need;   // blocks of the step
    upto = block_scan<kWaves>(sum, wave_sums, need);
    sum = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int have = blocks_of(len[i]), got = min(want[i], max(left - upto, 0));
        upto += want[i];
        need_upto[r0 + i] = upto;
        const int end = max(len[i], min(end_of(len[i], n[i]), (have + got) * kKvBlock));
        count[i] = end > len[i] ? (end - 1) / kKvBlock - len[i] / kKvBlock + 1 : 0;
        sum += count[i];
        dropped += (long long)asked[i] - (end - len[i]);
        if (blockIdx.x == 0 && r0 + i < a.R) a.lens_out[r0 + i] = end;
    }
    if (blockIdx.x == 0) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) dropped += __shfl_xor(dropped, d);
        if ((tid & 63) == 0) wave_dropped[tid >> 6] = dropped;
    }
    int chunks;   // of the step
    upto = block_scan<kWaves>(sum, wave_sums, chunks);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        upto += count[i];
        chunks_upto[r0 + i] = upto;
    }
    __syncthreads();
    // what request r has stored after the step: its end, its blocks before it
    // and the rank of its first new block
    struct Request { int len, first, end, have, base; };
    auto request = [&](int r) {
        Request q;
        q.len = min(max(a.lens[r], 0), cap);
        q.first = r ? rows_upto[r - 1] : 0;
        q.base = r ? need_upto[r - 1] : 0;
        q.have = blocks_of(q.len);
        const int want = need_upto[r] - q.base;
        const int got = min(want, max(left - q.base, 0));
        q.end = max(q.len, min(end_of(q.len, rows_upto[r] - q.first), (q.have + got) * kKvBlock));
        return q;
    };
    auto new_block = [&](int rank) { return a.free_blocks[left - 1 - rank]; };   // rank < left
    const int stride = gridDim.x * nt, id = blockIdx.x * nt + tid;
    const int given = min(need, left);
    for (int e = id; e < given; e += stride) {
        const int r = find(need_upto, a.R, e);
        const Request q = request(r);
        a.table[r * a.table_stride + q.have + e - q.base] = new_block(e);
    }
    for (int i = id; i < a.n_chunks; i += stride) {
        int4 c = make_int4(0, 0, 0, 0);
        if (i < chunks) {
            const int r = find(chunks_upto, a.R, i);
            const Request q = request(r);
            const int b = q.len / kKvBlock + i - (r ? chunks_upto[r - 1] : 0);
            const int begin = max(q.len, b * kKvBlock);
            const int end = (int)min((int64_t)q.end, ((int64_t)b + 1) * kKvBlock);
            c = make_int4(q.first + begin - q.len, end - begin, r, begin);
        }
        int32_t* o = a.chunks + 4 * (int64_t)i;
        o[0] = c.x, o[1] = c.y, o[2] = c.z, o[3] = c.w;
    }
    for (int t = id; t < a.n_tokens; t += stride) {
        int slot = -1, pos = 0;
        const int r = find(rows_upto, a.R, t);
        if (r < a.R) {
            const Request q = request(r);
            const int p = (int)min((int64_t)q.len + t - q.first, (int64_t)cap);
            if (p < q.end) {
                pos = p;
                const int j = p / kKvBlock;
                const int b = j < q.have ? a.table[r * a.table_stride + j]
                                         : new_block(q.base + j - q.have);
                if (b >= 0 && b < a.n_blocks) slot = b * kKvBlock + p % kKvBlock;
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    if (id == 0) {
        a.state_out[0] = left - given;
        dropped = 0;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 64; ++w) dropped += wave_dropped[w];
        a.state_out[1] = (int)min(dropped, 0x7fffffffLL);
    }
}

constexpr int kReleaseWaves = 16;

// One workgroup: a wave counts the blocks of a finished request, their sum
// over the requests says where each one's go, a wave copies them.  64 requests of
// 16 blocks 2.5 us, 256 of 626 103 (its chains of loads, 64 entries a turn).
__global__ __launch_bounds__(kReleaseWaves * 64) void kv_release_kernel(
    int32_t* table, int64_t table_stride, int32_t* lens, const int32_t* finished,
    int32_t* free_blocks, int32_t* state, int R, int max_blocks, int n_blocks) {
    __shared__ int upto[kMaxRequests];
    __shared__ int wave_sums[kReleaseWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = kReleaseWaves;
    const int left = min(max(state[0], 0), n_blocks);
    // the valid entries of a row, 64 at a time: f(bit set of valid lanes, entry)
    auto row = [&](int r, auto&& f) {
        for (int j0 = 0; j0 < max_blocks; j0 += 64) {
            const int j = j0 + lane;
            const int b = j < max_blocks ? table[r * table_stride + j] : -1;
            f(__ballot(b >= 0 && b < n_blocks), j, b);
        }
    };
    for (int r = wave; r < R; r += waves) {
        int n = 0;
        if (finished[r]) row(r, [&](uint64_t valid, int, int) { n += __popcll(valid); });
        if (lane == 0) upto[r] = n;
    }
    __syncthreads();
    int before = 0;
    for (int r0 = 0; r0 < R; r0 += kReleaseWaves * 64) {
        const int r = r0 + tid;
        const int mine = r < R ? upto[r] : 0;
        int total;
        const int sum = before + mine + block_scan<kReleaseWaves>(mine, wave_sums, total);
        if (r < R) upto[r] = sum;
        before += total;
    }
    __syncthreads();
    for (int r = wave; r < R; r += waves) {
        if (!finished[r]) continue;
        int at = left + (r ? upto[r - 1] : 0);
        row(r, [&](uint64_t valid, int j, int b) {
            const int o = at + __popcll(valid & ((1ULL << lane) - 1));
            if ((valid >> lane & 1) && o < n_blocks) free_blocks[o] = b;
            if (j < max_blocks) table[r * table_stride + j] = -1;
            at += __popcll(valid);
        });
        if (lane == 0) lens[r] = 0;
    }
    if (tid == 0) state[0] = min(left + before, n_blocks);
}

}  // namespace

int kv_plan_max_requests() { return kMaxRequests; }

int launch_kv_plan(int32_t* table, int64_t table_stride, const int32_t* lens,
                   const int32_t* new_tokens, const int32_t* free_blocks, const int32_t* state,
                   int R, int max_blocks, int n_blocks, int n_tokens, int n_chunks, int max_len,
                   int32_t* slots, int32_t* positions, int32_t* chunks, int32_t* lens_out,
                   int32_t* state_out, hipStream_t stream) {
    const PlanArgs a{table, table_stride, lens, new_tokens, free_blocks, state, R, max_blocks,
                     n_blocks, n_tokens, n_chunks, max_len, slots, positions, chunks, lens_out, state_out};
    const int groups = std::min(256, std::max(1, (n_tokens + kPlanThreads - 1) / kPlanThreads));
    auto* kernel = R <= kPlanThreads ? kv_plan_kernel<1>
                   : R <= 4 * kPlanThreads ? kv_plan_kernel<4>
                                           : kv_plan_kernel<kMaxRequests / kPlanThreads>;
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(kPlanThreads), 0, stream, a);
    return check_launch("nb_kv_plan");
}

int launch_kv_release(int32_t* table, int64_t table_stride, int32_t* lens, const int32_t* finished,
                      int32_t* free_blocks, int32_t* state, int R, int max_blocks, int n_blocks,
                      hipStream_t stream) {
    hipLaunchKernelGGL(kv_release_kernel, dim3(1), dim3(kReleaseWaves * 64), 0, stream, table,
                       table_stride, lens, finished, free_blocks, state, R, max_blocks, n_blocks);
    return check_launch("nb_kv_release");
}

}  // namespace nb
