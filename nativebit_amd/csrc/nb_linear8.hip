// Rows in 8 bits times packed 3-bit weights with 8-bit codebooks (gfx950):
// nb_linear8_layout and nb_linear8.  Formulas and layout: nb_linear8.h.
//
// Few rows: bound by latency (a launch, one trip to the weights, the sum over the
// waves; 2560 x 2560 at one row 3.6 us, 13824 x 2560 5.1 for 15.5 MB).  Many rows: bound
// by the LDS reads of rows and units beside the products (about 1700 of the 2048
// cycles that a 256 x 256 x 128 step's products take, in a step of 3000; without
// barriers 2600, without operands made 2400, loads alone 100), and at the ends by
// whole rounds of tiles and the epilogue: 13824 x 2560 at 2048 rows 78 to 81 us in
// launches of a graph (1790 to 1860 TOP/s), 82 under the profiler.  Measured and not faster there: units straight to registers (88 us against
// 82 with 128 x 128 tiles: 12 and 8 bytes a lane are many small requests), waits a block
// later, tiles of an XCD in the other order.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "nb_linear8.h"
#include "nb_linear8_forms.h"

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
// A workgroup takes 16 kI outputs and 16 kJ rows; its waves take the blocks of K
// in turn, each all outputs and rows, and add their sums through LDS.  Units and
// rows come straight from memory, the next block's ahead of this one's products.
template <int kWaves, int kI, int kJ, bool kBf16>
__global__ __launch_bounds__(64 * kWaves, 2) void linear8_rows_kernel(Args a) {
    extern __shared__ __align__(16) i4 part[];   // [kWaves][kI][kJ][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bpr = a.K / 128, last = (a.N + 15) / 16 - 1;
    const int n0 = blockIdx.x * 16 * kI, m0 = blockIdx.y * 16 * kJ;
    const uint8_t* tiles[kI];
#pragma unroll
    for (int i = 0; i < kI; ++i) {
        tiles[i] = a.tiles + (int64_t)min((int)blockIdx.x * kI + i, last) * bpr * kTileBytes;
    }
    const int8_t* x[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
        x[j] = a.x + min(m0 + 16 * j + (lane & 15), a.M - 1) * a.ld_x + (lane >> 4) * 32;
    }
    struct Block {
        Unit u[kI];
        i4 x[kJ][2];
    };
    auto load = [&](int kb, Block& b) {
#pragma unroll
        for (int i = 0; i < kI; ++i) b.u[i] = load_unit(tiles[i] + (int64_t)kb * kTileBytes, lane);
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
            const i4* p = reinterpret_cast<const i4*>(x[j] + kb * 128);
            b.x[j][0] = p[0], b.x[j][1] = p[1];
        }
    };
    i4 sum[kI][kJ];
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) sum[i][j] = i4{0, 0, 0, 0};
    auto multiply = [&](const Block& b) {
#pragma unroll
        for (int i = 0; i < kI; ++i) {
            i4 w[2];
            unit_weights(b.u[i], w);
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                sum[i][j] = mfma(w[0], b.x[j][0], sum[i][j]);
                sum[i][j] = mfma(w[1], b.x[j][1], sum[i][j]);
            }
        }
    };
    Block b0, b1;
    if (wave < bpr) load(wave, b0);
    for (int kb = wave; kb < bpr; kb += 2 * kWaves) {
        if (kb + kWaves < bpr) load(kb + kWaves, b1);
        multiply(b0);
        if (kb + kWaves >= bpr) break;
        if (kb + 2 * kWaves < bpr) load(kb + 2 * kWaves, b0);
        multiply(b1);
    }
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) part[((wave * kI + i) * kJ + j) * 64 + lane] = sum[i][j];
    __syncthreads();
    for (int at = tid; at < kI * kJ * 64; at += 64 * kWaves) {
        const int i = at / (kJ * 64), j = at / 64 % kJ, l = at & 63;
        const int m = m0 + 16 * j + (l & 15), n = n0 + 16 * i + (l >> 4) * 4;
        const Column c = column(a, n);
        const float xs = a.x_scale[min(m, a.M - 1)];
        i4 s = part[at];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += part[w * kI * kJ * 64 + at];
        by_activation(a.activation, [&](auto act) {
            Finished<decltype(act)::value> f;
            if (a.residual) {
                f.template load_residual<kBf16>(a, m, n);
                f.template finish<true>(c, xs, s);
            } else {
                f.template finish<false>(c, xs, s);
            }
            f.template store<kBf16>(a, m, n);
        });
    }
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
// (s_nop: the wait state between a scalar write of m0 and a load to LDS)
__device__ __forceinline__ void load_to_lds(uint32_t lds, const void* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(offset), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)p;
}

// A lane's unit of a tile in LDS.
__device__ __forceinline__ Unit read_unit(const unsigned char* tile, int lane) {
    const uint32_t* d = reinterpret_cast<const uint32_t*>(tile + lane * 12);
    const u2 c = *reinterpret_cast<const u2*>(tile + kTileCodes + (lane & 15) * 8);
    return Unit{d[0], d[1], d[2], c[0], c[1]};
}
// Half h of its weights (10 and 15 instructions).
template <int kHalf>
__device__ __forceinline__ i4 half_weights(const Unit& u) {
    i4 w[2];
    unit_weights(u, w);
    return w[kHalf];
}

constexpr int kAhead = 2;   // reads of rows under way in front of the products

// Sizes of a workgroup of kN x kM waves with kI x kJ products of 16 x 16 each and
// kStages blocks in LDS, kSplit times.
template <int kI, int kJ, int kN, int kM, int kStages, int kSplit>
struct Tile {
    static constexpr int kWaves = kN * kM, kOutputs = 16 * kI * kN, kRows = 16 * kJ * kM;
    static constexpr int kRowLoads = kRows / (8 * kWaves);   // of a wave, 1 KB each: eight rows
    static constexpr int kTileLoads = (kI * kN * kTileBytes + 1024 * kWaves - 1) / (1024 * kWaves);
    static constexpr int kStage = kRows * 128 + kTileLoads * kWaves * 1024;
    static constexpr int kHalf = kJ < 4 ? kJ : 4;            // groups of 16 rows that leave at once
    static constexpr int kPitch = 16 * kI + 4;
    static constexpr int kSums = kWaves * 16 * kHalf * kPitch * 4;
    static constexpr int kLds = kSplit * (kStages * kStage > kSums ? kStages * kStage : kSums);
    static constexpr int kThreads = 64 * kWaves * kSplit;
    static constexpr int kLoads = kRowLoads + kTileLoads;    // of a wave and block
    static_assert(kRows % (8 * kWaves) == 0, "rows of a wave's loads");
    static_assert(kStages >= 3 && (kStages - 2) * kLoads < 64, "loads under way");
};

// All but the last kLoads loads of the wave are there.  (The compiler does not track
// those to LDS.)
template <int kLoads>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLoads) : "memory");
}

// A workgroup of kN x kM waves takes 16 kI kN outputs and 16 kJ kM rows and walks K
// a block at a time, wave (n, m) with kI x kJ products of 16 x 16.  Rows and tiles
// are loaded straight to LDS, kStages blocks of them, 16-byte chunk c of row r in place
// c ^ (r & 7), so that eight rows' reads of a chunk hit eight groups of banks.
// In the middle of a block the next one is waited for, and one is asked for into the
// place of the last one, which the barrier there says all waves have left: kStages
// - 1 blocks ahead, past the end the last block again (every wave has the same
// number of loads under way at every wait).  While a half block's products run, the
// next half's operands are made.
// kSplit > 1: so many groups of waves take the blocks of K in turn, each with LDS of
// its own; their sums are added as they leave.
template <int kI, int kJ, int kN, int kM, int kStages, int kSplit, bool kBf16>
__global__ __launch_bounds__(64 * kN * kM * kSplit, 2) void linear8_tiles_kernel(Args a) {
    using T = Tile<kI, kJ, kN, kM, kStages, kSplit>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, all = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = all % T::kWaves, group = all / T::kWaves;
    const int fr = lane & 15, fq = lane >> 4;
    const int bpr = a.K / 128, last = (a.N + 15) / 16 - 1;
    // workgroups are dealt to the 8 XCDs in turn; an XCD takes a contiguous run of
    // tiles, so that its L2 holds the rows of one or two of them
    const int columns = (a.N + T::kOutputs - 1) / T::kOutputs;
    const int total = gridDim.x, g = blockIdx.x, xcd = g % 8;
    const int tile = xcd * (total / 8) + min(xcd, total % 8) + g / 8;
    const int n0 = tile % columns * T::kOutputs, m0 = tile / columns * T::kRows;
    const int wn = wave % kN, wm = wave / kN;

    // what the wave loads of a block, as offsets that every block shares (under
    // 2^31: ld_x is at most 2^22); rows and tiles past the last one are that again
    const int8_t* rows = a.x + m0 * a.ld_x;
    const uint8_t* tiles = a.tiles + (int64_t)(n0 / 16) * bpr * kTileBytes;
    uint32_t row_at[T::kRowLoads], tile_at[T::kTileLoads];
#pragma unroll
    for (int i = 0; i < T::kRowLoads; ++i) {
        const int r = (wave * T::kRowLoads + i) * 8 + (lane >> 3);
        row_at[i] = (uint32_t)(min(r, a.M - 1 - m0) * (int)a.ld_x) + (((lane & 7) ^ (r & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < T::kTileLoads; ++i) {
        const int at = (wave * T::kTileLoads + i) * 1024 + lane * 16;
        tile_at[i] = (uint32_t)(min(at / kTileBytes, last - n0 / 16) * bpr * kTileBytes + at % kTileBytes);
    }
    unsigned char* lds = smem + group * kStages * T::kStage;
    const uint32_t lds_rows = lds_address(lds) + wave * T::kRowLoads * 1024;
    const uint32_t lds_tiles = lds_address(lds) + T::kRows * 128 + wave * T::kTileLoads * 1024;
    auto load = [&](int turn, int stage) {
        const int kb = min(turn * kSplit + group, bpr - 1);
#pragma unroll
        for (int i = 0; i < T::kRowLoads; ++i) {
            load_to_lds(__builtin_amdgcn_readfirstlane(lds_rows + stage * T::kStage + i * 1024),
                        rows + kb * 128, row_at[i]);
        }
#pragma unroll
        for (int i = 0; i < T::kTileLoads; ++i) {
            load_to_lds(__builtin_amdgcn_readfirstlane(lds_tiles + stage * T::kStage + i * 1024),
                        tiles + kb * kTileBytes, tile_at[i]);
        }
    };
    i4 sum[kI][kJ];
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) sum[i][j] = i4{0, 0, 0, 0};
    const unsigned char* own_rows = lds + (wm * 16 * kJ + fr) * 128;
    const unsigned char* own_tiles = lds + T::kRows * 128 + wn * kI * kTileBytes;
    // The products of half h of the block in `stage`.  The next half's operands are
    // made meanwhile: after half 0 those of half 1, of the units in registers; after
    // half 1 those of half 0 of the block in `after`, whose units are read first.
    // (Left alone, the compiler puts all operands in front of the products that use
    // them, and reads next to their use.)
    Unit u[kI];
    auto half = [&](auto h_, int stage, int after, const i4 (&w)[kI], i4 (&next)[kI]) {
        constexpr int h = decltype(h_)::value;
        const unsigned char* s = own_rows + stage * T::kStage + (((2 * fq + h) ^ (fr & 7)) << 4);
        const unsigned char* t = own_tiles + after * T::kStage;
        i4 x[kJ];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) x[j] = *reinterpret_cast<const i4*>(s + j * 2048);
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
            if (j + kAhead < kJ) x[j + kAhead] = *reinterpret_cast<const i4*>(s + (j + kAhead) * 2048);
#pragma unroll
            for (int i = 0; i < kI; ++i) {
                if (h == 1 && i * kJ / kI == j) u[i] = read_unit(t + i * kTileBytes, lane);
            }
#pragma unroll
            for (int i = 0; i < kI; ++i) sum[i][j] = mfma(w[i], x[j], sum[i][j]);
#pragma unroll
            for (int i = 0; i < kI; ++i) {
                if ((i + 1) * kJ / kI - 1 == j) next[i] = half_weights<1 - h>(u[i]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < kI; ++i) asm volatile("" : "+v"(next[i]));   // (made here, not later)
    };
    using zero = std::integral_constant<int, 0>;
    using one = std::integral_constant<int, 1>;
    i4 w0[kI], w1[kI];
#pragma unroll
    for (int turn = 0; turn < kStages - 1; ++turn) load(turn, turn);
    wait_loads<(kStages - 2) * T::kLoads>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kI; ++i) {
        u[i] = read_unit(own_tiles + i * kTileBytes, lane);
        w0[i] = half_weights<0>(u[i]);
    }
    int stage = 0;
    for (int turn = 0; turn * kSplit < bpr; ++turn) {
        const int after = stage == kStages - 1 ? 0 : stage + 1;
        const bool mine = kSplit == 1 || turn * kSplit + group < bpr;
        if (mine) half(zero{}, stage, after, w0, w1);
        wait_loads<(kStages - 3) * T::kLoads>();
        __syncthreads();
        load(turn + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
        // (past the last block: operands that nothing uses)
        if (mine) half(one{}, stage, after, w1, w0);
        stage = after;
    }
    wait_loads<0>();
    __syncthreads();
    // The sums go through LDS, kHalf of the wave's 16-row groups at a time, so that a
    // row's outputs leave side by side, in a loop that is not unrolled over them
    // (sums in registers have no index).
    constexpr int kLanes = 4 * kI, kRegion = 16 * T::kHalf * T::kPitch;
    int* sums = reinterpret_cast<int*>(smem);
    const int n = n0 + wn * 16 * kI + lane % kLanes * 4;
    const Column c = column(a, n);
#pragma unroll
    for (int j0 = 0; j0 < kJ; j0 += T::kHalf) {
        const int first = m0 + (wm * kJ + j0) * 16;
        const float xs = a.x_scale[min(first + lane, a.M - 1)];   // of 16 kHalf <= 64 rows
        // (of one group: written and read by the wave itself)
        if (j0) {
            if (kSplit > 1) __syncthreads();
            else wave_lds_order();
        }
#pragma unroll
        for (int i = 0; i < kI; ++i)
#pragma unroll
            for (int j = 0; j < T::kHalf; ++j) {
                *reinterpret_cast<i4*>(sums + all * kRegion + (j * 16 + fr) * T::kPitch + i * 16 +
                                       fq * 4) = sum[i][j0 + j];
            }
        if (kSplit > 1) __syncthreads();
        else wave_lds_order();
        by_activation(a.activation, [&](auto act) {
            constexpr int kAct = decltype(act)::value;
            auto leave = [&](auto residual) {
                constexpr int kStep = 64 / kLanes, kTurns = T::kHalf * 16 / kStep / kSplit;
                constexpr int kAtOnce = kTurns < 4 ? kTurns : 4;
                static_assert(kTurns > 0 && kTurns % kAtOnce == 0, "turns of the epilogue");
                const int r0 = group * kTurns * kStep + lane / kLanes;
#pragma unroll 1
                for (int turn = 0; turn < kTurns; turn += kAtOnce) {
                    Finished<kAct> f[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        if constexpr (decltype(residual)::value) {
                            f[i].template load_residual<kBf16>(a, first + r0 + (turn + i) * kStep, n);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int r = r0 + (turn + i) * kStep;
                        const int* at = sums + wave * kRegion + r * T::kPitch + lane % kLanes * 4;
                        i4 v = *reinterpret_cast<const i4*>(at);
#pragma unroll
                        for (int k = 1; k < kSplit; ++k) {
                            v += *reinterpret_cast<const i4*>(at + k * T::kWaves * kRegion);
                        }
                        f[i].template finish<decltype(residual)::value>(c, __shfl(xs, r), v);
                    }
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        f[i].template store<kBf16>(a, first + r0 + (turn + i) * kStep, n);
                    }
                }
            };
            if (a.residual) leave(std::true_type{});
            else leave(std::false_type{});
        });
    }
}

template <int kForm, int kWaves, int kI, int kJ>
void launch_rows(const Args& a, bool bf16, hipStream_t stream) {
    constexpr Form f = kForms[kForm];
    static_assert(!f.tiles && f.outputs == 16 * kI && f.rows == 16 * kJ && f.split == kWaves, "the form");
    const dim3 grid((unsigned)output_groups(f, a.N), (unsigned)row_groups(f, a.M));
    constexpr size_t lds = (size_t)kWaves * kI * kJ * 64 * 16;
    auto* kernel = bf16 ? linear8_rows_kernel<kWaves, kI, kJ, true> : linear8_rows_kernel<kWaves, kI, kJ, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), lds, stream, a);
}

template <int kForm, int kI, int kJ, int kN, int kM, int kStages, int kSplit>
void launch_tiles(const Args& a, bool bf16, hipStream_t stream) {
    using T = Tile<kI, kJ, kN, kM, kStages, kSplit>;
    constexpr Form f = kForms[kForm];
    static_assert(f.tiles && f.outputs == T::kOutputs && f.rows == T::kRows && f.split == kSplit, "the form");
    const dim3 grid((unsigned)(output_groups(f, a.N) * row_groups(f, a.M)));
    auto* kernel = bf16 ? linear8_tiles_kernel<kI, kJ, kN, kM, kStages, kSplit, true>
                        : linear8_tiles_kernel<kI, kJ, kN, kM, kStages, kSplit, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(T::kThreads), T::kLds, stream, a);
}

void (*const kRun[kFormCount])(const Args&, bool, hipStream_t) = {
    launch_rows<0, 8, 1, 1>,           launch_rows<1, 8, 2, 2>,           launch_tiles<2, 1, 2, 4, 1, 4, 2>,
    launch_tiles<3, 1, 4, 4, 1, 4, 2>, launch_tiles<4, 2, 4, 4, 1, 3, 2>, launch_tiles<5, 2, 4, 4, 1, 3, 1>,
    launch_tiles<6, 2, 8, 4, 1, 3, 2>, launch_tiles<7, 2, 8, 4, 1, 3, 1>, launch_tiles<8, 4, 8, 4, 2, 3, 1>,
};

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

int launch_linear8(const int8_t* x, int64_t ld_x, const float* x_scale, const uint8_t* tiles,
                   const float* scale, const float* bias, int activation, const void* residual,
                   int64_t ld_residual, void* y, int y_dtype, int64_t ld_y, int M, int N, int K,
                   hipStream_t stream) {
    const Args a{x, ld_x, x_scale, tiles, scale, bias, residual, ld_residual, y, ld_y, M, N, K,
                 activation};
    kRun[form_of(M, N, K, device_cu_count())](a, y_dtype == NB_BF16, stream);
    return check_launch("nb_linear8");
}

}  // namespace nb
