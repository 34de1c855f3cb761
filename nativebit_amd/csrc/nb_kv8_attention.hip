// nb_kv8_attention: the launch (its shape and split) and the join of split
// results.  The kernel and its mathematics: nb_kv8_attention.h.
#include <algorithm>

#include "nb_kv8_attention.h"

namespace nb {
namespace {

// (Waves of a workgroup and rows of a chunk by the list's length, a plan's bound:
// with up to about twice as many tokens as requests the launch below may start
// prompts' workgroups of twice the waves, with half the blocks for each.)
// Workgroups over a row's blocks: three a CU (heads of over 128 dims two), over
// tables of 32 blocks or more, two blocks a wave at least.  One token of six
// requests of 40000 positions, 8 heads of 128 (48 workgroups unsplit): 16 splits
// 78 us, 10 (two a CU) 85, 21 (four) 80, 32 (six) 81; of 32 of 4000 50, 52, 49,
// 51; of one of 8000 16.8 against 18 with four blocks a wave.  512 prompt tokens
// after 8000 (180 workgroups): 4 splits 114 us, one 229; 300 of two requests
// after 3000, 2 heads of 256: two blocks a wave 45 us, four 63, one split 129.
// More than fill the CUs cost their partial results: 2048 prompt tokens 60 us,
// in two splits 95.
int splits_of(int n_chunks, int n_tokens, int max_blocks, int n_head, int n_kv, int D) {
    const int waves = kv8_waves(n_tokens > n_chunks);
    const int64_t rows = ((int64_t)n_tokens + n_chunks - 1) / n_chunks * (n_head / n_kv);
    const int64_t groups = (int64_t)n_chunks * n_kv * ((rows + 16 * waves - 1) / (16 * waves));
    const int64_t want = (D <= 128 ? 3 : 2) * device_cu_count();
    if (groups >= want || max_blocks < 32) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want / groups, max_blocks / (2 * waves), 64}));
}

constexpr int kJoinWaves = 4;

// A wave takes a row and head at a time: the splits' maxima and sums in its
// lanes, then the dims.  A chunk's tokens go to the waves of gridDim.z workgroups.
__global__ __launch_bounds__(kJoinWaves * 64) void kv8_join_kernel(Kv8AttentionArgs a, int splits) {
    const Kv8Chunk ch = kv8_chunk(a, blockIdx.x);
    const int head = blockIdx.y, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int t = blockIdx.z * kJoinWaves + wave; t < ch.n; t += gridDim.z * kJoinWaves) {
        const int64_t row = ch.row0 + t, at = (row * a.n_head + head) * splits;
        const float* ml = a.part + (int64_t)a.n_tokens * a.n_head * splits * a.D + 2 * at;
        const float m = lane < splits ? ml[2 * lane] : -INFINITY;
        const float l = lane < splits ? ml[2 * lane + 1] : 0.f;
        const float top = fmaxf(wave64_max(m), kLowest);
        const float w = __builtin_amdgcn_exp2f(m - top);
        const float sum = wave64_sum(l * w);
        const float scaled = l == 0.f ? 0.f : w * (sum == 0.f ? 0.f : 1.f / sum);
        const uint64_t used = __ballot(lane < splits && l != 0.f);
        for (int d = lane; d < a.D; d += 64) {
            float v = 0.f;
            for (int s0 = 0; s0 < splits; s0 += 16) {
                float p[16];   // (16 loads at once; splits that saw nothing were not written)
#pragma unroll
                for (int s = 0; s < 16; ++s) p[s] = a.part[(at + min(s0 + s, splits - 1)) * a.D + d];
#pragma unroll
                for (int s = 0; s < 16; ++s) {
                    if (used >> (s0 + s) & 1) v = fmaf(p[s], lane_value(scaled, s0 + s), v);
                }
            }
            const int64_t to = row * a.ld_out + head * a.D + d;
            if (a.out_dtype == NB_F32) static_cast<float*>(a.out)[to] = v;
            else static_cast<bf16_bits*>(a.out)[to] = f32_to_bf16_rne(v);
        }
    }
}

}  // namespace

int64_t kv8_attention_bytes(int n_chunks, int n_tokens, int max_blocks, int n_head, int n_kv, int D) {
    const int splits = splits_of(n_chunks, n_tokens, max_blocks, n_head, n_kv, D);
    return splits == 1 ? 0 : (int64_t)n_tokens * n_head * splits * (D + 2) * 4;
}

int launch_kv8_attention(const void* q, int q_dtype, int64_t ld_q, const int32_t* chunks,
                         int n_chunks, const int32_t* lens, const int32_t* table,
                         int64_t table_stride, int R, int max_blocks, const int8_t* k,
                         const int8_t* v, const float* k_scale, const float* v_scale, int n_blocks,
                         void* out, int out_dtype, int64_t ld_out, int n_tokens, int n_head,
                         int n_kv, int D, float softcap, int window, const float* slopes,
                         const int32_t* prefix, void* workspace, hipStream_t stream) {
    const int splits = splits_of(n_chunks, n_tokens, max_blocks, n_head, n_kv, D);
    Kv8AttentionArgs a{q, ld_q, chunks, lens, table, table_stride, k, v, k_scale, v_scale, out,
                       ld_out, slopes, prefix, static_cast<float*>(workspace), q_dtype, out_dtype,
                       n_chunks, n_tokens, R, max_blocks, n_blocks, n_head, n_kv, D, window, softcap};
    // whether there may be chunks of over 32 rows, by what the host knows
    const bool prompts = n_tokens > R && (int64_t)std::min(n_tokens, kKvBlock) * (n_head / n_kv) > 32;
    // groups of rows of a chunk: the most that one may have (a prompt's beside
    // single tokens would else go one after the other; those that a chunk does not
    // have end at once, and come last in the grid: 32 tokens of 4000 positions 49
    // us with them, 54 between the splits)
    const int64_t rows = (int64_t)std::min(n_tokens, kKvBlock) * (n_head / n_kv);
    const int of = 16 * kv8_waves(prompts);
    const int groups = (int)std::min<int64_t>((rows + of - 1) / of, 64);
    const dim3 grid((unsigned)(n_chunks * n_kv), splits, groups);
    const bool rules = softcap > 0.f || window > 0 || slopes || prefix;
    Kv8AttentionLaunch* launch =
        out_dtype == NB_BF16 ? (prompts ? launch_kv8_prompts_2 : launch_kv8_tokens_2)
                             : (prompts ? launch_kv8_prompts_3 : launch_kv8_tokens_3);
    launch(a, grid, rules, stream);
    if (splits > 1) {
        const int mean = std::min(kKvBlock, (n_tokens + n_chunks - 1) / n_chunks);
        hipLaunchKernelGGL(kv8_join_kernel,
                           dim3(n_chunks, n_head, (mean + kJoinWaves - 1) / kJoinWaves),
                           dim3(kJoinWaves * 64), 0, stream, a, splits);
    }
    return check_launch("nb_kv8_attention");
}

}  // namespace nb
