// The plan of a serving step over a block cache, from the requests' lengths
// (gfx950): nb_kv_plan and nb_kv_release.
//
//   nb_kv_plan      request r has lens[r] tokens cached and brings new[r].  The
//                   rows of the step are the requests' new tokens in order;
//                   with L = lens, N = new (clipped to the rows that exist)
//                     first[r] = sum N[< r]             row of its first token
//                     need[r]  = ceil((L + N) / 64) - ceil(L / 64)
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
#include <algorithm>

#include "nb_device.h"
#include "nb_internal.h"

namespace nb {
namespace {

constexpr int kMaxRequests = 4096;
constexpr int kWaves = 16;   // of the largest workgroup

// Inclusive sum over the workgroup's threads; `total` its last value.
__device__ __forceinline__ int block_scan(int v, int* wave_sums, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();   // the sums of an earlier call are read
    if (lane == 63) wave_sums[wave] = v;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < waves; ++w) {
        const int s = wave_sums[w];
        before += w < wave ? s : 0;
        all += s;
    }
    total = all;
    return v + before;
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
    int R, max_blocks, n_blocks, n_tokens, n_chunks;
    int32_t *slots, *positions, *chunks, *lens_out, *state_out;
};

__device__ __forceinline__ int blocks_of(int tokens) {
    return (int)(((int64_t)tokens + kKvBlock - 1) / kKvBlock);
}

__global__ __launch_bounds__(kWaves * 64) void kv_plan_kernel(PlanArgs a) {
    __shared__ int rows_upto[kMaxRequests];     // inclusive sums over the requests: rows,
    __shared__ int need_upto[kMaxRequests];     // blocks they need,
    __shared__ int chunks_upto[kMaxRequests];   // chunks
    __shared__ int wave_sums[kWaves];
    __shared__ unsigned long long asked_sum, stored_sum;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int cap = a.max_blocks * kKvBlock;
    const int left = min(max(a.state[0], 0), a.n_blocks);
    if (tid == 0) asked_sum = stored_sum = 0;
    __syncthreads();
    int rows = 0, need = 0, chunks = 0;   // of the requests before this strip
    for (int r0 = 0; r0 < a.R; r0 += nt) {
        const int r = r0 + tid;
        const bool in = r < a.R;
        const int len = in ? min(max(a.lens[r], 0), cap) : 0;
        const int asked = in ? max(a.asked[r], 0) : 0;
        int total;
        // rows: what is asked, up to the rows that exist (clipped to n_tokens
        // each, which changes no result and keeps the sums in 31 bits)
        const int clipped = min(asked, a.n_tokens);
        const int upto = rows + block_scan(clipped, wave_sums, total);
        const int first = min(upto - clipped, a.n_tokens);
        const int n = min(clipped, a.n_tokens - first);
        rows += total;
        const int have = blocks_of(len);
        int end = (int)min((int64_t)len + n, (int64_t)cap);
        const int want = blocks_of(end) - have;
        const int base = need + block_scan(want, wave_sums, total) - want;
        need += total;
        const int got = min(want, max(left - base, 0));
        end = max(len, min(end, (have + got) * kKvBlock));
        const int c = end > len ? (end - 1) / kKvBlock - len / kKvBlock + 1 : 0;
        const int cu = chunks + block_scan(c, wave_sums, total);
        chunks += total;
        if (in) {
            rows_upto[r] = first + n;
            need_upto[r] = base + want;
            chunks_upto[r] = cu;
            if (blockIdx.x == 0) {
                a.lens_out[r] = end;
                if (asked) atomicAdd(&asked_sum, (unsigned long long)asked);
                if (end > len) atomicAdd(&stored_sum, (unsigned long long)(end - len));
            }
        }
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
        const int end = (int)min((int64_t)q.len + rows_upto[r] - q.first, (int64_t)cap);
        q.end = max(q.len, min(end, (q.have + got) * kKvBlock));
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
        a.state_out[1] = (int)min(asked_sum - stored_sum, 0x7fffffffULL);
    }
}

// One workgroup: a wave counts the blocks of a finished request, their sum
// over the requests says where each one's go, a wave copies them.
__global__ __launch_bounds__(kWaves * 64) void kv_release_kernel(
    int32_t* table, int64_t table_stride, int32_t* lens, const int32_t* finished,
    int32_t* free_blocks, int32_t* state, int R, int max_blocks, int n_blocks) {
    __shared__ int upto[kMaxRequests];
    __shared__ int wave_sums[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
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
    for (int r0 = 0; r0 < R; r0 += blockDim.x) {
        const int r = r0 + tid;
        int total;
        const int sum = before + block_scan(r < R ? upto[r] : 0, wave_sums, total);
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
                   int R, int max_blocks, int n_blocks, int n_tokens, int n_chunks, int32_t* slots,
                   int32_t* positions, int32_t* chunks, int32_t* lens_out, int32_t* state_out,
                   hipStream_t stream) {
    const PlanArgs a{table, table_stride, lens, new_tokens, free_blocks, state, R, max_blocks,
                     n_blocks, n_tokens, n_chunks, slots, positions, chunks, lens_out, state_out};
    const int threads = R <= 256 ? 256 : 1024;
    const int groups = std::min(64, std::max(1, (n_tokens + 2 * threads - 1) / (2 * threads)));
    hipLaunchKernelGGL(kv_plan_kernel, dim3(groups), dim3(threads), 0, stream, a);
    return check_launch("nb_kv_plan");
}

int launch_kv_release(int32_t* table, int64_t table_stride, int32_t* lens, const int32_t* finished,
                      int32_t* free_blocks, int32_t* state, int R, int max_blocks, int n_blocks,
                      hipStream_t stream) {
    hipLaunchKernelGGL(kv_release_kernel, dim3(1), dim3(R <= 16 ? 256 : 1024), 0, stream, table,
                       table_stride, lens, finished, free_blocks, state, R, max_blocks, n_blocks);
    return check_launch("nb_kv_release");
}

}  // namespace nb
