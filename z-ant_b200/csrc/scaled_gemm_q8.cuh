// Products of int8 operands with a scale for each token and each output channel, dense or grouped by expert:
//   y[m, n] = float(sum over k of a[m, k] w[n, k]) * a_scale[m] * w_scale[n] + bias[n]
// The sums are exact (int32), so neither their order nor a split of k changes a result.
//
// Chosen by the tokens of a group, the tiles that there are, and the operands' addresses:
//
//   scaled_few_kernel    few tokens: warp-level MMAs on operands straight from global memory
//   scaled_gemm_kernel   tcgen05, 128 channels x 64, 128 or 256 tokens, operands by TMA
//   scaled_pair_kernel   tcgen05 on pairs of CTAs, 256 channels x 256 tokens
//   scaled_any_kernel    tcgen05, 128 x 128, rows that the TMA cannot read: calls that may not use the arena
//   scaled_align_kernel  lays such rows out in the arena for the kernels above
//
// On tcgen05 (kind::i8) the weights are the MMA's A operand: 128 output channels on the lanes of an accumulator, NT tokens in its
// columns.  A warp that reads one column then holds 32 neighbouring channels of one token and stores them as one line, w_scale and bias
// belong to the lane, and a last tile of few tokens costs few MMA clocks.  A stage is 128 bytes of k: 128 rows of weights and NT of tokens,
// K-major operands in the 128-byte swizzle.
//
// The kernels start while the one before them still writes their tokens (ptx::grid_wait), so that operands are read by plain loads: the
// non-coherent ones (__ldg) are for what nobody writes while the kernel runs, and may be moved in front of the wait.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "context.cuh"
#include "fused_cnn.cuh"
#include "irb_band.cuh"
#include "ptx_sm100.cuh"
#include "quantize_rows.cuh"
#include "tc_conv_nhwc.cuh"

namespace zb {

constexpr int kScaledMaxGroups = 1024;
constexpr int kScaledMaxK = 131071;      // 2^17 products of -128 and -128 would leave int32

struct ScaledGemmArgs {
    const int8_t* a; const float* a_scale; long long a_stride;
    const int8_t* w; const float* w_scale; long long w_stride;
    const float* bias;
    void* y; long long y_stride;
    const int32_t* offsets;              // [groups + 1], or nullptr: one group of all rows
    int rows, n, k, groups;
    int y_dtype;
    // how it is run
    int n_tiles, k_blocks, stages;
    int a_tma, w_tma;
    int off_scales, off_groups, off_bar;        // shared memory
    int* status;
    long long wait_budget;               // clocks after which a wait gives up
    int give_up;                         // self test: a CTA whose first wait counts as run out (-1: none)
};

__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Groups of rows as the kernel takes them: row[g] = the largest of offsets[0 .. g], clamped to the rows there are; group g is the rows
// row[g] .. row[g + 1] - 1, and its tiles are first[g] .. first[g + 1] - 1.  Both hold groups + 1 entries.  The tiles are at most
// rows / tile_rows + groups, whatever the offsets hold.  Called by the whole CTA.
__device__ __forceinline__ void group_tiles(const int32_t* offsets, int groups, int rows, int tile_rows, int* row, int* first) {
    for (int g = threadIdx.x; g <= groups; g += blockDim.x) row[g] = min(max(offsets[g], 0), rows);
    __syncthreads();
    if (threadIdx.x < 32) {                              // a lane takes `per` neighbouring entries
        const int lane = threadIdx.x, per = (groups + 32) / 32, g0 = min(lane * per, groups + 1), g1 = min(g0 + per, groups + 1);
        int top = 0;
        for (int g = g0; g < g1; ++g) top = max(top, row[g]);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, top, d); if (lane >= d) top = max(top, o); }
        int run = __shfl_up_sync(0xffffffffu, top, 1);
        if (lane == 0) run = 0;
        int tiles = 0, before = run;                      // `before`: the running maximum in front of the lane's entries
        for (int g = g0; g < g1; ++g) {
            run = max(run, row[g]);
            row[g] = run;
            if (g > 0) tiles += (run - before + tile_rows - 1) / tile_rows;      // of group g - 1
            before = run;
        }
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, sum, d); if (lane >= d) sum += o; }
        sum -= tiles;
        __syncwarp();
        for (int g = g0; g < g1; ++g) {
            if (g > 0) sum += (row[g] - row[g - 1] + tile_rows - 1) / tile_rows;
            first[g] = sum;
        }
    }
    __syncthreads();
}

struct RowTile { int group, row, rows; };      // rows: how many of the tile's rows there are

__device__ __forceinline__ RowTile row_tile_of(const ScaledGemmArgs& a, const int* row, const int* first, int tile, int tile_rows) {
    if (!a.offsets) return RowTile{0, tile * tile_rows, min(tile_rows, a.rows - tile * tile_rows)};
    int lo = 0, hi = a.groups - 1;                    // the last group that starts at or before the tile
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= tile) lo = mid; else hi = mid - 1;
    }
    const int r = row[lo] + (tile - first[lo]) * tile_rows;
    return RowTile{lo, r, min(tile_rows, row[lo + 1] - r)};
}

// Order of the tiles: bands of 8 row tiles, in a band channels outside and rows inside, so that CTAs that run at the same time share weights
// and a band's tokens stay in L2 while all weights pass.
struct TileAt { int m, n; };
__device__ __forceinline__ TileAt tile_at(int t, int row_tiles, int n_tiles) {
    const int band = t / (8 * n_tiles), in = t - band * 8 * n_tiles, wide = min(8, row_tiles - band * 8), n = in / wide;
    return TileAt{band * 8 + in - n * wide, n};
}

template <int NT>
struct ScaledCfg {
    static constexpr int STAGE_W = 128 * 128, STAGE = STAGE_W + NT * 128;
    static constexpr int TMEM_COLS = 2 * NT;
    static constexpr int PARTS = 2, EPI = 4 * PARTS;                // warps that share a lane quarter's columns
    static constexpr int COLS = NT / PARTS;
    static constexpr int THREADS = 64 + 32 * EPI;
    static_assert(NT % 64 == 0 && NT <= 256, "tile width");
};

// 32 neighbouring tokens (`cols` of them exist) for the lane's channel n: float(sum) * a_scale * w_scale + bias, one rounding to Y.  `scales`: the
// tokens' a_scale, in shared memory, read four at a time.  (Every shuffle, shared-memory access and store takes a clock of the pipe
// that feeds the tensor core: with a shuffle for each column 2048 x 2048 x 8192 took 32.1 us, with words of two channels, exchanged
// by shuffles, as long.)
template <typename Y>
__device__ __forceinline__ void store_columns(const ScaledGemmArgs& a, const uint32_t* v, long long row, int n, int cols, const float* scales, float ws, float bias, bool has_bias) {
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride + n;
    if (n >= a.n) cols = 0;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 as = *reinterpret_cast<const float4*>(scales + j);
        const float f[4] = {as.x, as.y, as.z, as.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float r = __int2float_rn((int)v[j + i]) * f[i] * ws;
            if (has_bias) r += bias;
            if (j + i < cols) store_as(y, r);
            y += a.y_stride;
        }
    }
}
__device__ __forceinline__ void store_columns_any(const ScaledGemmArgs& a, const uint32_t* v, long long row, int n, int cols, const float* scales, float ws, float bias) {
    const bool has_bias = a.bias != nullptr;
    if (a.y_dtype == ZANT_F32) store_columns<float>(a, v, row, n, cols, scales, ws, bias, has_bias);
    else if (a.y_dtype == ZANT_F16) store_columns<__half>(a, v, row, n, cols, scales, ws, bias, has_bias);
    else store_columns<__nv_bfloat16>(a, v, row, n, cols, scales, ws, bias, has_bias);
}

// The barriers at the end of the dynamic shared memory, and the roles that both tcgen05 kernels share.
struct ScaledBars {
    uint32_t at;
    __device__ __forceinline__ uint32_t full(int s) const { return at + 8u * (uint32_t)s; }
    __device__ __forceinline__ uint32_t empty(int s) const { return at + 128u + 8u * (uint32_t)s; }
    __device__ __forceinline__ uint32_t tfull(int b) const { return at + 256u + 8u * (uint32_t)b; }
    __device__ __forceinline__ uint32_t tempty(int b) const { return at + 272u + 8u * (uint32_t)b; }
    static constexpr int SLOT = 400, FLAG = 404, BYTES = 512;       // TMEM address, abort flag
};

// A wait of a whole warp.  Its lanes leave it together and with one answer: behind it stand instructions and barriers that want all of them (tcgen05.ld,
// shuffles, the next wait of a ring, in which a lane a phase behind the others would wait for good).
template <bool CLUSTER = false>
__device__ __forceinline__ bool scaled_wait(const ScaledGemmArgs& a, uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, ptx::mbar_wait<CLUSTER>(bar, parity, abort_flag, a.wait_budget)) != 0;
}

// The MMA issuer (a whole warp): NT columns per tile of the walk t0, t0 + step, ..
template <int NT>
__device__ __forceinline__ void scaled_mma_role(const ScaledGemmArgs& a, const ScaledBars& bar, uint32_t s0, uint32_t tmem_base, const int* grow, const int* gfirst,
                                                int row_tiles, int t0, int step, volatile int* abort_flag) {
    using Cfg = ScaledCfg<NT>;
    const int tiles = row_tiles * a.n_tiles;
    const uint32_t leader = ptx::elect_one() ? 1u : 0u;
    const uint32_t hi = (uint32_t)(smem_desc_kmajor_swizzled(0, 128) >> 32), lo = (uint32_t)smem_desc_kmajor_swizzled(0, 128);
    int s = 0, ti = 0;
    uint32_t ph = 0;
    for (int t = t0; t < tiles; t += step, ++ti) {
        const int b = ti & 1;
        if (!scaled_wait(a, bar.tempty(b), ((uint32_t)(ti >> 1) & 1u) ^ 1u, abort_flag)) return;
        ptx::tc_fence_after();
        const RowTile rt = row_tile_of(a, grow, gfirst, tile_at(t, row_tiles, a.n_tiles).m, NT);
        const uint32_t idesc = ptx::idesc_i8(128, (rt.rows + 15) & ~15, true, true), d = tmem_base + (uint32_t)(b * NT);
        for (int kb = 0; kb < a.k_blocks; ++kb) {
            if (!scaled_wait(a, bar.full(s), ph, abort_flag)) return;
            ptx::tc_fence_after();
            const uint32_t wa = lo + ((s0 + (uint32_t)(s * Cfg::STAGE)) >> 4), ta = wa + (Cfg::STAGE_W >> 4);
            const int steps = min(4, (a.k - kb * 128 + 31) >> 5);
            for (int i = 0; i < steps; ++i) ptx::mma_i8_if(leader, d, wa + 2u * i, hi, ta + 2u * i, hi, idesc, (kb | i) ? 1u : 0u);
            ptx::mma_commit_if(leader, bar.empty(s));
            if (++s == a.stages) { s = 0; ph ^= 1u; }
        }
        ptx::mma_commit_if(leader, bar.tfull(b));
    }
}

// The end of a producer's ring: the tensor core has arrived on every stage's barrier.  Nothing else waits for the last round of these arrivals, and
// one of them must not come when the shared memory (in a pair, the other CTA's) is the next kernel's.
__device__ __forceinline__ void scaled_drain(const ScaledGemmArgs& a, const ScaledBars& bar, int s, uint32_t ph, volatile int* abort_flag) {
    for (int i = 0; i < a.stages; ++i) {
        if (!ptx::mbar_wait(bar.empty(s), ph ^ 1u, abort_flag, a.wait_budget)) return;      // (a stage that was never filled is free)
        if (++s == a.stages) { s = 0; ph ^= 1u; }
    }
}

// An epilogue warp: lane quarter `warp & 3`, the `part`-th of the tile's column ranges.  PAIR: the CTA has half `rank` of the tile's 256 channels,
// and rank 0 is told when the accumulators are free.  A warp whose wait has given up still walks its tiles, from part barrier to part barrier: the other
// warps of the part may have had the accumulator, and would stand there.
template <int NT, bool PAIR>
__device__ __forceinline__ void scaled_epilogue_role(const ScaledGemmArgs& a, const ScaledBars& bar, uint32_t tmem_base, const int* grow, const int* gfirst, int row_tiles,
                                                     int t0, int step, int quarter, int part, int rank, float* scale_ring, volatile int* abort_flag) {
    using Cfg = ScaledCfg<NT>;
    const int tiles = row_tiles * a.n_tiles, lane = threadIdx.x & 31;
    int ti = 0;
    bool ok = true;
    for (int t = t0; t < tiles; t += step, ++ti) {
        const TileAt at = tile_at(t, row_tiles, a.n_tiles);
        const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
        const int n = (PAIR ? at.n * 256 + rank * 128 : at.n * 128) + quarter * 32 + lane, b = ti & 1;
        const bool live = n < a.n, all_live = n - lane + 32 <= a.n;
        const long long wat = (long long)rt.group * a.n + n;
        const float ws = live ? a.w_scale[wat] : 0.0f, bias = live && a.bias ? a.bias[wat] : 0.0f;
        const int col0 = part * Cfg::COLS, cols = min(Cfg::COLS, rt.rows - col0), own = quarter * (Cfg::COLS / 4) + lane;
        // the part's a_scale, by its four warps; the other buffer is the next tile's, and none of them writes this one again before all
        // have come to the next tile
        float* scales = scale_ring + b * NT + col0;
        if (lane < Cfg::COLS / 4) scales[own] = own < cols ? a.a_scale[rt.row + col0 + own] : 0.0f;
        ptx::named_barrier_sync(1 + part, 128);
        ok = ok && scaled_wait(a, bar.tfull(b), (uint32_t)(ti >> 1) & 1u, abort_flag);
        if (!ok) continue;
        ptx::tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * NT + col0);
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
            uint32_t v[32];
            ptx::tmem_ld32(taddr + (uint32_t)c, v);
            ptx::tmem_wait_ld32(v);
            store_columns_any(a, v, (long long)rt.row + col0 + c, n, cols - c, scales + c, ws, bias);
            if (!all_live) __syncwarp();              // (lanes without a channel store nothing; the next load wants them all)
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            if (PAIR) ptx::mbar_arrive_cluster(ptx::cluster_addr(bar.tempty(b), 0));
            else ptx::mbar_arrive(bar.tempty(b));
        }
    }
}

// Set-up and end that the tcgen05 kernels share.
template <int COLS, bool PAIR = false>
__device__ __forceinline__ uint32_t scaled_setup(uint8_t* smem, const ScaledGemmArgs& a, const ScaledBars& bar, int full_arrivals, int epilogue_warps) {
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + a.off_bar + ScaledBars::SLOT);
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) { ptx::mbar_init(bar.full(s), (uint32_t)full_arrivals); ptx::mbar_init(bar.empty(s), 1); }
        for (int b = 0; b < 2; ++b) { ptx::mbar_init(bar.tfull(b), 1); ptx::mbar_init(bar.tempty(b), (uint32_t)epilogue_warps); }
        *reinterpret_cast<volatile int*>(smem + a.off_bar + ScaledBars::FLAG) = (int)blockIdx.x == a.give_up ? 1 : 0;
        ptx::mbar_fence_init();
    }
    if (threadIdx.x >> 5 == 1) {
        if (PAIR) ptx::tmem_alloc_pair(ptx::smem_u32(slot), COLS);
        else { ptx::tmem_alloc(ptx::smem_u32(slot), COLS); ptx::tmem_relinquish(); }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (PAIR) { ptx::cluster_arrive(); ptx::cluster_wait(); }         // both CTAs' barriers are there
    ptx::tc_fence_after();
    ptx::grid_trigger();
    ptx::grid_wait();
    return *slot;
}
template <int COLS, bool PAIR = false>
__device__ __forceinline__ void scaled_end(const ScaledGemmArgs& a, uint32_t tmem_base, volatile int* abort_flag) {
    if (*abort_flag) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);      // copies in flight land
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (PAIR) { ptx::cluster_arrive(); ptx::cluster_wait(); }         // nobody leaves while its memory is read or its barriers are arrived on
    if (threadIdx.x >> 5 == 1) {
        if (PAIR) ptx::tmem_dealloc_pair(tmem_base, COLS);
        else ptx::tmem_dealloc(tmem_base, COLS);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, (int)DEV_ERR_WAIT_TIMEOUT);
}

//   warp 0  TMA        warp 1  TMEM owner, MMA issuer        warps 2 .. 9  epilogue
template <int NT>
__global__ void __launch_bounds__(ScaledCfg<NT>::THREADS, 1) scaled_gemm_kernel(const __grid_constant__ ScaledGemmArgs a, const __grid_constant__ CUtensorMap w_map,
                                                                                const __grid_constant__ CUtensorMap a_map) {
    using Cfg = ScaledCfg<NT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t s0 = ptx::smem_u32(smem);
    int* grow = reinterpret_cast<int*>(smem + a.off_groups);
    int* gfirst = grow + kScaledMaxGroups + 1;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + a.off_bar + ScaledBars::FLAG);
    const ScaledBars bar{s0 + (uint32_t)a.off_bar};
    const int warp = threadIdx.x >> 5;
    const uint32_t tmem_base = scaled_setup<Cfg::TMEM_COLS>(smem, a, bar, 1, Cfg::EPI);

    int row_tiles = (a.rows + NT - 1) / NT;
    if (a.offsets) { group_tiles(a.offsets, a.groups, a.rows, NT, grow, gfirst); row_tiles = gfirst[a.groups]; }
    const int step = (int)gridDim.x, t0 = (int)blockIdx.x;

    if (warp == 0) {
        if (ptx::elect_one()) {
            int s = 0; uint32_t ph = 0;
            for (int t = t0; t < row_tiles * a.n_tiles; t += step) {
                const TileAt at = tile_at(t, row_tiles, a.n_tiles);
                const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
                const int wrow = rt.group * a.n + at.n * 128;
                for (int kb = 0; kb < a.k_blocks; ++kb) {
                    if (!ptx::mbar_wait(bar.empty(s), ph ^ 1u, abort_flag, a.wait_budget)) goto producer_done;
                    ptx::mbar_arrive_expect_tx(bar.full(s), Cfg::STAGE);
                    const uint32_t dst = s0 + (uint32_t)(s * Cfg::STAGE);
                    ptx::tma_load_2d(dst, &w_map, kb * 128, wrow, bar.full(s));
                    ptx::tma_load_2d(dst + Cfg::STAGE_W, &a_map, kb * 128, rt.row, bar.full(s));
                    if (++s == a.stages) { s = 0; ph ^= 1u; }
                }
            }
            scaled_drain(a, bar, s, ph, abort_flag);
        producer_done:;
        }
    } else if (warp == 1) {
        scaled_mma_role<NT>(a, bar, s0, tmem_base, grow, gfirst, row_tiles, t0, step, abort_flag);
    } else {
        scaled_epilogue_role<NT, false>(a, bar, tmem_base, grow, gfirst, row_tiles, t0, step, warp & 3, (warp - 2) >> 2, 0, reinterpret_cast<float*>(smem + a.off_scales), abort_flag);
    }
    scaled_end<Cfg::TMEM_COLS>(a, tmem_base, abort_flag);
}

// ------------------------------------------------------------------------------------------------------------------------------
// Rows that start anywhere.  Sixteen warps read the aligned 16-byte blocks that a row's 16-byte chunks begin in (only blocks that hold a byte of the
// row), two or three stages ahead in registers, get the following block from the lane that has it, shift the two and write the chunk where the TMA
// would have.  An operand that the TMA can read comes by TMA all the same.  (257 x 4095 x 5001: 30 us with odd weights, 43 with odd tokens too;
// 30 also with asynchronous copies to a ring of raw rows and other warps that shift from there; the loads bound both.  Calls that may use the
// context's arena lay such rows out first, scaled_align_kernel, and take the TMA's kernels: 20 us.)
//
//   warp 0  TMA        warp 1  TMEM owner, MMA issuer        warps 2 .. 9  epilogue        10 .. 25  loaders
struct ScaledAny {
    static constexpr int NT = 128, LOADERS = 16, THREADS = ScaledCfg<NT>::THREADS + 32 * LOADERS;
};

// A loader warp's rows of an operand's tile: eight lanes a row, R rows for each of them; D stages in registers.
template <int R, int D>
struct AnyRows {
    const uint4* src[R];
    int sh[R], end[R];                                 // end: the row's bytes from the lane's first block on (0 and less: none)
    uint4 b[D][R];                                     // blocks of D stages, in turn (a copy between them would wait for the load)
    __device__ __forceinline__ void begin(const int8_t* all, long long row0, long long stride, int there, int k, int lane) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = i * 4 + (lane >> 3), c = lane & 7;
            const int8_t* p = all + (row0 + r) * stride + c * 16;
            sh[i] = (int)(reinterpret_cast<uintptr_t>(p) & 15);
            src[i] = reinterpret_cast<const uint4*>(p - sh[i]);
            end[i] = r < there ? k - c * 16 + sh[i] : 0;
        }
#pragma unroll
        for (int i = 0; i < D; ++i) fetch(b[i]);
    }
    __device__ __forceinline__ void fetch(uint4 (&to)[R]) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            to[i] = end[i] > 0 ? *src[i] : make_uint4(0, 0, 0, 0);
            src[i] += 8;
            end[i] -= 128;
        }
    }
    // Stage AT of each D, of which `left` bytes are left, to the swizzled rows at `tile`; and the loads for the one D further.
    template <int AT>
    __device__ __forceinline__ void stage(uint8_t* tile, int left, int lane) {
        const int c = lane & 7, from = (lane & 24) | ((c + 1) & 7);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint4 &own = b[AT][i], &then = b[(AT + 1) % D][i], o = c == 0 ? then : own;       // the block behind a row's eighth is the next stage's first
            uint32_t w[8] = {own.x, own.y, own.z, own.w, __shfl_sync(0xffffffffu, o.x, from), __shfl_sync(0xffffffffu, o.y, from), __shfl_sync(0xffffffffu, o.z, from),
                             __shfl_sync(0xffffffffu, o.w, from)};
#pragma unroll
            for (int k = 0; k < 6; ++k) w[k] = (sh[i] & 8) ? w[k + 2] : w[k];
#pragma unroll
            for (int k = 0; k < 5; ++k) w[k] = (sh[i] & 4) ? w[k + 1] : w[k];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], (sh[i] & 3) * 8);
            uint4 v = make_uint4(w[0], w[1], w[2], w[3]);
            if (left < 128) v = first_bytes(v, left - c * 16);      // the last stage: zeros behind the rows
            const int r = i * 4 + (lane >> 3);
            *reinterpret_cast<uint4*>(tile + r * 128 + ((c ^ (r & 7)) << 4)) = v;
        }
        fetch(b[AT]);
    }
};

// BOTH: the loaders bring both operands, 16 rows a warp; else one of them, 8 rows a warp.
template <bool BOTH>
__global__ void __launch_bounds__(ScaledAny::THREADS, 1) scaled_any_kernel(const __grid_constant__ ScaledGemmArgs a, const __grid_constant__ CUtensorMap w_map,
                                                                           const __grid_constant__ CUtensorMap a_map) {
    constexpr int NT = ScaledAny::NT;
    using Cfg = ScaledCfg<NT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t s0 = ptx::smem_u32(smem);
    int* grow = reinterpret_cast<int*>(smem + a.off_groups);
    int* gfirst = grow + kScaledMaxGroups + 1;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + a.off_bar + ScaledBars::FLAG);
    const ScaledBars bar{s0 + (uint32_t)a.off_bar};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t tmem_base = scaled_setup<Cfg::TMEM_COLS>(smem, a, bar, 1 + ScaledAny::LOADERS, Cfg::EPI);

    int row_tiles = (a.rows + NT - 1) / NT;
    if (a.offsets) { group_tiles(a.offsets, a.groups, a.rows, NT, grow, gfirst); row_tiles = gfirst[a.groups]; }
    const int step = (int)gridDim.x, t0 = (int)blockIdx.x;

    if (warp == 0) {
        if (ptx::elect_one()) {
            const uint32_t bytes = (a.w_tma ? Cfg::STAGE_W : 0) + (a.a_tma ? NT * 128 : 0);
            int s = 0; uint32_t ph = 0;
            for (int t = t0; t < row_tiles * a.n_tiles; t += step) {
                const TileAt at = tile_at(t, row_tiles, a.n_tiles);
                const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
                const int wrow = rt.group * a.n + at.n * 128;
                for (int kb = 0; kb < a.k_blocks; ++kb) {
                    if (!ptx::mbar_wait(bar.empty(s), ph ^ 1u, abort_flag, a.wait_budget)) goto producer_done;
                    ptx::mbar_arrive_expect_tx(bar.full(s), bytes);
                    const uint32_t dst = s0 + (uint32_t)(s * Cfg::STAGE);
                    if (a.w_tma) ptx::tma_load_2d(dst, &w_map, kb * 128, wrow, bar.full(s));
                    if (a.a_tma) ptx::tma_load_2d(dst + Cfg::STAGE_W, &a_map, kb * 128, rt.row, bar.full(s));
                    if (++s == a.stages) { s = 0; ph ^= 1u; }
                }
            }
            scaled_drain(a, bar, s, ph, abort_flag);
        producer_done:;
        }
    } else if (warp == 1) {
        scaled_mma_role<NT>(a, bar, s0, tmem_base, grow, gfirst, row_tiles, t0, step, abort_flag);
    } else if (warp < 2 + Cfg::EPI) {
        scaled_epilogue_role<NT, false>(a, bar, tmem_base, grow, gfirst, row_tiles, t0, step, warp & 3, (warp - 2) >> 2, 0, reinterpret_cast<float*>(smem + a.off_scales), abort_flag);
    } else {
        constexpr int R = BOTH ? 4 : 2, D = BOTH ? 2 : 3;
        const int loader = warp - 2 - Cfg::EPI, row0 = (BOTH ? loader & 7 : loader) * R * 4;
        const bool weights = BOTH ? loader < 8 : a.w_tma == 0;
        AnyRows<R, D> rows;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = t0; t < row_tiles * a.n_tiles && ok; t += step) {
            const TileAt at = tile_at(t, row_tiles, a.n_tiles);
            const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
            if (weights) rows.begin(a.w, (long long)rt.group * a.n + at.n * 128 + row0, a.w_stride, a.n - at.n * 128 - row0, a.k, lane);
            else rows.begin(a.a, rt.row + row0, a.a_stride, rt.rows - row0, a.k, lane);
            auto stage = [&](auto at_stage, int kb) {
                if (kb >= a.k_blocks || !ok) return;
                ok = scaled_wait(a, bar.empty(s), ph ^ 1u, abort_flag);
                if (!ok) return;
                rows.template stage<decltype(at_stage)::value>(smem + s * Cfg::STAGE + (weights ? 0 : Cfg::STAGE_W) + row0 * 128, a.k - kb * 128, lane);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(bar.full(s));
                if (++s == a.stages) { s = 0; ph ^= 1u; }
            };
            for (int kb = 0; kb < a.k_blocks; kb += D) {
                stage(std::integral_constant<int, 0>(), kb);
                stage(std::integral_constant<int, 1>(), kb + 1);
                if constexpr (D == 3) stage(std::integral_constant<int, 2>(), kb + 2);
            }
        }
    }
    scaled_end<Cfg::TMEM_COLS>(a, tmem_base, abort_flag);
}

// ------------------------------------------------------------------------------------------------------------------------------
// Pairs of CTAs: tiles of 256 channels x 256 tokens, each CTA loads half of either operand.  What bounds both forms is shared memory, 128 bytes a
// clock: for 512 clocks of MMA a CTA of a pair takes 32 KB in and 32 KB out to the tensor core, one CTA with 128 x 256 takes 48 KB each way
// (8192 x 8192 x 8192: 334 us, 3300 TOPS, against 371; the tensor pipe is active 80 % of a tile's time).
__global__ void __launch_bounds__(ScaledCfg<256>::THREADS, 1) scaled_pair_kernel(const __grid_constant__ ScaledGemmArgs a, const __grid_constant__ CUtensorMap w_map,
                                                                                const __grid_constant__ CUtensorMap a_map) {
    constexpr int NT = 256;
    using Cfg = ScaledCfg<NT>;
    constexpr int STAGE = Cfg::STAGE_W + NT / 2 * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t s0 = ptx::smem_u32(smem);
    int* grow = reinterpret_cast<int*>(smem + a.off_groups);
    int* gfirst = grow + kScaledMaxGroups + 1;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + a.off_bar + ScaledBars::FLAG);
    const ScaledBars bar{s0 + (uint32_t)a.off_bar};
    const int warp = threadIdx.x >> 5, rank = (int)ptx::cluster_rank();
    const uint32_t tmem_base = scaled_setup<Cfg::TMEM_COLS, true>(smem, a, bar, 1, 2 * Cfg::EPI);

    int row_tiles = (a.rows + NT - 1) / NT;
    if (a.offsets) { group_tiles(a.offsets, a.groups, a.rows, NT, grow, gfirst); row_tiles = gfirst[a.groups]; }
    const int step = (int)gridDim.x / 2, t0 = (int)blockIdx.x / 2, tiles = row_tiles * a.n_tiles;
    // columns of a tile: its tokens rounded up to 32; the first half of them are rank 0's rows of the operand, the second rank 1's
    auto half_of = [](int rows) { return ((rows + 31) & ~31) / 2; };

    if (warp == 0) {
        if (ptx::elect_one()) {
            int s = 0; uint32_t ph = 0;
            for (int t = t0; t < tiles; t += step) {
                const TileAt at = tile_at(t, row_tiles, a.n_tiles);
                const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
                const int wrow = rt.group * a.n + at.n * 256 + rank * 128, xrow = rt.row + rank * half_of(rt.rows);
                for (int kb = 0; kb < a.k_blocks; ++kb) {
                    if (!ptx::mbar_wait(bar.empty(s), ph ^ 1u, abort_flag, a.wait_budget)) goto producer_done;
                    if (rank == 0) ptx::mbar_arrive_expect_tx(bar.full(s), 2 * STAGE);
                    const uint32_t dst = s0 + (uint32_t)(s * STAGE), full = ptx::cluster_addr(bar.full(s), 0);
                    ptx::tma_load_2d_pair(dst, &w_map, kb * 128, wrow, full);
                    ptx::tma_load_2d_pair(dst + Cfg::STAGE_W, &a_map, kb * 128, xrow, full);
                    if (++s == a.stages) { s = 0; ph ^= 1u; }
                }
            }
            scaled_drain(a, bar, s, ph, abort_flag);
        producer_done:;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t leader = ptx::elect_one() ? 1u : 0u;
            const uint32_t hi = (uint32_t)(smem_desc_kmajor_swizzled(0, 128) >> 32), lo = (uint32_t)smem_desc_kmajor_swizzled(0, 128);
            int s = 0, ti = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = t0; t < tiles && ok; t += step, ++ti) {
                const int b = ti & 1;
                ok = scaled_wait<true>(a, bar.tempty(b), ((uint32_t)(ti >> 1) & 1u) ^ 1u, abort_flag);       // both CTAs' epilogues have read this accumulator
                if (!ok) break;
                ptx::tc_fence_after();
                const RowTile rt = row_tile_of(a, grow, gfirst, tile_at(t, row_tiles, a.n_tiles).m, NT);
                const uint32_t idesc = ptx::idesc_i8(256, 2 * half_of(rt.rows), true, true), d = tmem_base + (uint32_t)(b * NT);
                for (int kb = 0; kb < a.k_blocks; ++kb) {
                    ok = scaled_wait(a, bar.full(s), ph, abort_flag);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint32_t wa = lo + ((s0 + (uint32_t)(s * STAGE)) >> 4), ta = wa + (Cfg::STAGE_W >> 4);
                    const int steps = min(4, (a.k - kb * 128 + 31) >> 5);
                    for (int i = 0; i < steps; ++i) ptx::mma_i8_pair_if(leader, d, wa + 2u * i, hi, ta + 2u * i, hi, idesc, (kb | i) ? 1u : 0u);
                    ptx::mma_commit_pair_if(leader, bar.empty(s));
                    if (++s == a.stages) { s = 0; ph ^= 1u; }
                }
                if (ok) ptx::mma_commit_pair_if(leader, bar.tfull(b));
            }
        }
    } else {
        scaled_epilogue_role<NT, true>(a, bar, tmem_base, grow, gfirst, row_tiles, t0, step, warp & 3, (warp - 2) >> 2, rank, reinterpret_cast<float*>(smem + a.off_scales), abort_flag);
    }
    scaled_end<Cfg::TMEM_COLS, true>(a, tmem_base, abort_flag);
}

// ------------------------------------------------------------------------------------------------------------------------------
// Up to 32 tokens a tile.  Bound by the weights' bytes, and by latency where they are few: no shared memory in front of the MMAs, no barriers but
// one.  A CTA has 16 MT channels; its 8 warps share k, 128 bytes at a time, and their sums meet in shared memory.  A lane reads 16
// neighbouring bytes of a row; as operands of m16n8k32 these stand for other k than the instruction's order says, but for the same ones in both
// operands, and the order of a sum is free.  One token, 4096 x 4096: 4.9 us, 3.4 TB/s; 8192 x 8192: 14.5 us, 4.6 TB/s.  PER: CTAs an SM.
template <int NTL, int MT>
struct ScaledFew {
    static constexpr int TOK = 8 * NTL, CH = 16 * MT, THREADS = 256;
};

// 16 bytes p[0..15] of which the first `valid` exist, zeros behind them.  Only words that hold an existing byte are read.
__device__ __forceinline__ uint4 load16_any(const int8_t* p, int valid) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const int sh = (int)(at & 3);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(at - sh);
    uint32_t w[5], v[4];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = (valid > 0 && i * 4 < valid + sh) ? q[i] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = __funnelshift_r(w[i], w[i + 1], sh * 8);
        const int left = valid - i * 4;
        if (left < 4) v[i] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <int NTL, int MT, bool ANY, int PER>
__global__ void __launch_bounds__(256, PER) scaled_few_kernel(const __grid_constant__ ScaledGemmArgs a) {
    using F = ScaledFew<NTL, MT>;
    __shared__ int part[8][F::TOK][F::CH];
    __shared__ int grow[kScaledMaxGroups + 1], gfirst[kScaledMaxGroups + 1];
    ptx::grid_start();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    int row_tiles = (a.rows + F::TOK - 1) / F::TOK;
    if (a.offsets) { group_tiles(a.offsets, a.groups, a.rows, F::TOK, grow, gfirst); row_tiles = gfirst[a.groups]; }
    const int tiles = row_tiles * a.n_tiles, whole = a.k >> 7;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
        const TileAt at = tile_at(t, row_tiles, a.n_tiles);
        const RowTile rt = row_tile_of(a, grow, gfirst, at.m, F::TOK);
        const int n0 = at.n * F::CH;
        // rows that do not exist: the last one again, its results are not stored
        const int8_t* w[MT][2];
        const int8_t* x[NTL];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[m][h] = a.w + ((long long)rt.group * a.n + min(n0 + m * 16 + h * 8 + g, a.n - 1)) * a.w_stride + q * 16;
#pragma unroll
        for (int i = 0; i < NTL; ++i) x[i] = a.a + (long long)(rt.row + min(i * 8 + g, rt.rows - 1)) * a.a_stride + q * 16;
        int acc[MT][NTL][4] = {};
        auto step = [&](int c, bool all) {
            uint4 wv[2][MT][2], xv[2][NTL];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = c * 128 + h * 64, valid = all ? 16 : a.k - k - q * 16;
                auto get = [&](const int8_t* p, bool once) {
                    if constexpr (ANY) return load16_any(p + k, min(valid, 16));
                    else return all || valid >= 16 ? (once ? ptx::ld_global_once(reinterpret_cast<const uint4*>(p + k)) : *reinterpret_cast<const uint4*>(p + k)) : load16_any(p + k, valid);
                };
#pragma unroll
                for (int m = 0; m < MT; ++m) { wv[h][m][0] = get(w[m][0], true); wv[h][m][1] = get(w[m][1], true); }
#pragma unroll
                for (int i = 0; i < NTL; ++i) xv[h][i] = get(x[i], false);
            }
            if (ANY || !all) __syncwarp();            // (which words a lane reads is its own; the MMAs want all lanes)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < NTL; ++i) {
                        const uint4 &w0 = wv[h][m][0], &w1 = wv[h][m][1], &b = xv[h][i];
                        mma_m16n8k32_s8(acc[m][i], make_uint4(w0.x, w1.x, w0.y, w1.y), b.x, b.y);
                        mma_m16n8k32_s8(acc[m][i], make_uint4(w0.z, w1.z, w0.w, w1.w), b.z, b.w);
                    }
        };
        int c = warp;
#pragma unroll (ANY ? 2 : 4)
        for (; c < whole; c += 8) step(c, true);
        if (c * 128 < a.k) step(c, false);
        __syncthreads();                              // the sums of the tile before have been read
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < NTL; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[warp][i * 8 + 2 * q + (j & 1)][m * 16 + g + (j >> 1) * 8] = acc[m][i][j];
        __syncthreads();
        for (int o = tid; o < F::TOK * F::CH; o += F::THREADS) {
            const int tok = o / F::CH, ch = o - tok * F::CH, n = n0 + ch;
            if (tok >= rt.rows || n >= a.n) continue;
            int sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += part[i][tok][ch];
            const long long wat = (long long)rt.group * a.n + n, yat = (long long)(rt.row + tok) * a.y_stride + n;
            float r = __int2float_rn(sum) * a.a_scale[rt.row + tok] * a.w_scale[wat];
            if (a.bias) r += a.bias[wat];
            if (a.y_dtype == ZANT_F32) static_cast<float*>(a.y)[yat] = r;
            else if (a.y_dtype == ZANT_F16) store_as(static_cast<__half*>(a.y) + yat, r);
            else store_as(static_cast<__nv_bfloat16*>(a.y) + yat, r);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------- host
// Rows of bytes as boxes of 128 x `box_rows`, 128-byte swizzle, zeros outside.
inline int32_t encode_rows_map(CUtensorMap* map, const void* p, size_t row_bytes, size_t rows, size_t stride, int box_rows) {
    using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<EncodeFn> known{nullptr};
    EncodeFn encode = known.load(std::memory_order_acquire);
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) {
            cudaGetLastError();
            return fail(ZANT_E_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
        }
        encode = reinterpret_cast<EncodeFn>(fn);
        known.store(encode, std::memory_order_release);
    }
    const cuuint64_t dims[2] = {row_bytes, rows}, strides[1] = {rows > 1 ? stride : align_up(row_bytes, 16)};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ZANT_OK : fail(ZANT_E_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
}

// Rows that the TMA can read.
inline bool tma_rows(const void* p, size_t rows, size_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && rows <= 0x7fffffffULL && (rows == 1 || ((stride & 15) == 0 && stride < (1ULL << 39)));
}

// Row tiles of `nt` rows: all of a dense product's, of a grouped one those that there are if the rows are spread evenly (the kernels walk what there is).
inline long long scaled_row_tiles(const ScaledGemmArgs& a, int nt) {
    if (!a.offsets) return ((long long)a.rows + nt - 1) / nt;
    const long long groups = std::min(a.rows, a.groups), per = (a.rows + groups - 1) / groups;
    return groups * ((per + nt - 1) / nt);
}

template <int NTL, int MT>
inline int32_t launch_scaled_few(zant_ctx* ctx, ScaledGemmArgs a) {
    using F = ScaledFew<NTL, MT>;
    a.n_tiles = (a.n + F::CH - 1) / F::CH;
    const long long tiles = scaled_row_tiles(a, F::TOK) * a.n_tiles;
    const unsigned grid = (unsigned)std::min<long long>(tiles, (long long)ctx->sm_count * 16);
    auto go = [&](auto kernel) { launch(ctx, kernel, dim3(grid), F::THREADS, 0, a); };
    // No more tiles than SMs: one CTA an SM with twice the registers, for loads further ahead (40 x 9040 x 1856: 12.8 us, with two 17.8; 16 x 4096 x
    // 2048: 4.0, 5.1; 30 x 4095 x 2001: 12.2, 18.9; but 18 x 3381 x 8256, 258 tiles: 19.3, 15.1).  One token at an odd address needs no more.
    const bool tma = a.a_tma && a.w_tma, one = tiles <= ctx->sm_count;
    if (tma) {
        if constexpr (NTL == 4) go(scaled_few_kernel<NTL, MT, false, 1>);         // (comes here with so few tiles only)
        else one ? go(scaled_few_kernel<NTL, MT, false, 1>) : go(scaled_few_kernel<NTL, MT, false, 2>);
    } else if constexpr (NTL == 1) {
        go(scaled_few_kernel<NTL, MT, true, 2>);
    } else {
        one ? go(scaled_few_kernel<NTL, MT, true, 1>) : go(scaled_few_kernel<NTL, MT, true, 2>);
    }
    return check_launch(ctx, "scaled_few_kernel");
}

// A tcgen05 kernel: shared memory (stages, scales, groups, barriers), tensor maps with boxes of w_box and a_box rows, the
// launch.  (The kernel is a template argument: the attribute of its shared memory is set once for each.)
template <auto KERNEL>
inline int32_t launch_scaled_tc(zant_ctx* ctx, const char* name, ScaledGemmArgs a, int stage, int threads, int tile_rows, int tile_n, int w_box, int a_box, int cluster) {
    constexpr int LIMIT = 232448;
    a.n_tiles = (a.n + tile_n - 1) / tile_n;
    a.k_blocks = (a.k + 127) / 128;
    const int groups = a.offsets ? (kScaledMaxGroups + 1) * 8 : 0, scales = 2 * tile_rows * 4;
    a.stages = std::min(16, (LIMIT - scales - groups - ScaledBars::BYTES - 16) / stage);
    a.off_scales = a.stages * stage;
    a.off_groups = a.off_scales + scales;
    a.off_bar = (int)align_up((size_t)(a.off_groups + groups), 16);
    alignas(64) CUtensorMap w_map{}, a_map{};
    if (a.w_tma) ZB_TRY(encode_rows_map(&w_map, a.w, (size_t)a.k, (size_t)a.groups * a.n, (size_t)a.w_stride, w_box));
    if (a.a_tma) ZB_TRY(encode_rows_map(&a_map, a.a, (size_t)a.k, (size_t)a.rows, (size_t)a.a_stride, a_box));
    ZB_SMEM_ATTR(ctx, KERNEL, LIMIT);
    const long long tiles = std::max<long long>(1, scaled_row_tiles(a, tile_rows)) * a.n_tiles;
    const unsigned grid = (unsigned)std::min<long long>(tiles, ctx->sm_count / cluster) * (unsigned)cluster;
    a.give_up = ctx->give_up_cta < 0 ? -1 : ctx->give_up_cta % (int)grid;
    ctx->give_up_cta = -1;
    a.wait_budget = a.give_up < 0 ? ptx::kWaitBudgetCycles : 4000000;       // self test: 2 ms, which the CTA's pair waits for it
    launch_cluster(ctx, KERNEL, dim3(grid), threads, (size_t)a.off_bar + ScaledBars::BYTES, (unsigned)cluster, a, w_map, a_map);
    return check_launch(ctx, name);
}
template <int NT>
inline int32_t launch_scaled_gemm(zant_ctx* ctx, const ScaledGemmArgs& a) {
    return launch_scaled_tc<scaled_gemm_kernel<NT>>(ctx, NT == 64 ? "scaled_gemm_kernel<64>" : NT == 128 ? "scaled_gemm_kernel<128>" : "scaled_gemm_kernel<256>", a, ScaledCfg<NT>::STAGE, ScaledCfg<NT>::THREADS, NT, 128, 128, NT, 1);
}
inline int32_t launch_scaled_pair(zant_ctx* ctx, const ScaledGemmArgs& a) {
    return launch_scaled_tc<scaled_pair_kernel>(ctx, "scaled_pair_kernel", a, ScaledCfg<256>::STAGE_W + 128 * 128, ScaledCfg<256>::THREADS, 256, 256, 128, 128, 2);
}
template <bool BOTH>
inline int32_t launch_scaled_any(zant_ctx* ctx, const ScaledGemmArgs& a) {
    constexpr int NT = ScaledAny::NT;
    return launch_scaled_tc<scaled_any_kernel<BOTH>>(ctx, "scaled_any_kernel", a, ScaledCfg<NT>::STAGE, ScaledAny::THREADS, NT, 128, 128, NT, 1);
}

// Rows laid out for the TMA: `k` bytes each, at multiples of `to_stride` (16), zeros behind them.  A warp a row.
__global__ void __launch_bounds__(256) scaled_align_kernel(const int8_t* from, long long stride, int k, long long rows, int8_t* to, long long to_stride) {
    ptx::grid_start();
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= rows) return;
    const char* row = reinterpret_cast<const char*>(from + r * stride);
    const int sh = (int)(reinterpret_cast<uintptr_t>(row) & 15), chunks = (int)(to_stride >> 4);
    uint4* out = reinterpret_cast<uint4*>(to + r * to_stride);
    for (int c0 = 0; c0 < chunks; c0 += 128) {
        uint32_t w[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) row_chunk<int8_t, true, int>(row, sh, k, c0 + i * 32 + (int)(threadIdx.x & 31), w[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + i * 32 + (int)(threadIdx.x & 31);
            if (c < chunks) out[c] = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
        }
    }
}
inline int32_t run_scaled_align(zant_ctx* ctx, const int8_t* from, long long stride, int k, long long rows, int8_t* to) {
    const uint64_t launched = ctx->launches;
    launch(ctx, scaled_align_kernel, dim3((unsigned)((rows + 7) / 8)), 256, 0, from, stride, k, rows, to, (long long)align_up((size_t)k, 16));
    ZB_TRY(check_launch(ctx, "scaled_align_kernel"));
    ctx->launches = launched;                         // (not an operator launch)
    return ZANT_OK;
}

// Which kernel: clocks of an SM (or a pair) for 128 bytes of k of a tile, from products of 128 to 8192 rows, times the tiles that one of them gets.  They
// are what shared memory delivers: operands in and out again, 64 tokens 24 KB each way, 128 32 KB, 256 48 KB, in a pair 32 KB.
// Up to 128 tokens a group the few-token kernel wins where there are no more tiles of 32 x 32 than SMs (40 x 9040 x 1856: 12.8 us, as tiles of 128
// channels 20.7; 96 x 4096 x 1024: 6.2, 9.6; 128 x 1024 x 512: 4.0, 4.4; but 113 x 9792 x 1472, 184 tiles: 23, 19.4; 128 x 512 x 512: 3.6, 3.5), at odd
// addresses with any k (37 x 970 x 1065: 5.0 us, 7.9).
struct ScaledChoice { int nt; bool pair, few; };
inline ScaledChoice scaled_choice(const ScaledGemmArgs& a, int sm_count) {
    struct Kind { int nt, wide, clocks; };
    constexpr Kind kinds[4] = {{64, 128, 370}, {128, 128, 450}, {256, 128, 720}, {256, 256, 620}};
    const double groups = std::min(a.rows, a.groups), per = a.rows / groups;
    ScaledChoice best{64, false, false};
    double least = 0;
    for (const Kind& k : kinds) {
        const double row_tiles = a.offsets ? groups * std::max(1.0, per / k.nt + 0.5) : (double)((a.rows + k.nt - 1) / k.nt);      // groups end inside a tile
        const double tiles = row_tiles * ((a.n + k.wide - 1) / k.wide) / (sm_count * 128 / k.wide);
        const double cost = (a.offsets ? std::max(1.0, tiles) : std::ceil(tiles)) * k.clocks;
        if (least == 0 || cost < least) { least = cost; best = ScaledChoice{k.nt, k.wide == 256, false}; }
    }
    const bool tma = tma_rows(a.a, (size_t)a.rows, (size_t)a.a_stride) && tma_rows(a.w, (size_t)a.groups * a.n, (size_t)a.w_stride);
    best.few = per <= 128 && scaled_row_tiles(a, 32) * ((a.n + 31) / 32) <= sm_count && (!tma || a.k > 512);
    return best;
}

// Tokens of a group, at most, that go to scaled_few_kernel when an operand cannot be read by the TMA.
constexpr int kScaledFewAny = 32;
inline long long scaled_rows_per_group(const ScaledGemmArgs& a) {
    const long long groups = std::min(a.rows, a.groups);
    return (a.rows + groups - 1) / groups;
}
// Bytes of the arena that operands want to be laid out in: none where they are read as they are.
inline size_t scaled_align_bytes(const ScaledGemmArgs& a, bool weights, int sm_count) {
    const size_t rows = weights ? (size_t)a.groups * a.n : (size_t)a.rows;
    if (scaled_rows_per_group(a) <= kScaledFewAny || scaled_choice(a, sm_count).few || tma_rows(weights ? a.w : a.a, rows, (size_t)(weights ? a.w_stride : a.a_stride)) || rows > 0x7fffffffULL) return 0;
    return rows * align_up((size_t)a.k, 16);
}

inline int32_t run_scaled_gemm(zant_ctx* ctx, int32_t y_dtype, ScaledGemmArgs a) {
    a.y_dtype = y_dtype;
    a.a_tma = tma_rows(a.a, (size_t)a.rows, (size_t)a.a_stride);
    a.w_tma = tma_rows(a.w, (size_t)a.groups * a.n, (size_t)a.w_stride);
    a.status = ctx->status_word;
    const long long per = scaled_rows_per_group(a);
    // (the narrowest tiles of any kernel; fewer than an int holds unless y is larger than any memory)
    if (((long long)a.rows / 8 + a.groups) * ((a.n + 15LL) / 16) > 0x7fffffffLL) return fail(ZANT_E_TOO_LARGE, "%d rows in %d groups and %d columns", a.rows, a.groups, a.n);
    const bool tma = a.a_tma && a.w_tma;
    const ScaledChoice c = scaled_choice(a, ctx->sm_count);
    // Few tokens, and so few tiles of 128 channels that they leave half of the SMs idle (1 x 4096 x 4096: 4.9 us, as tiles 9.9; 1 x 8192 x 8192: 15,
    // 20; but 16 x 2048 x 12288: 10, 8.2, and 64 experts of one or two rows: 38, 20).  Rows at odd addresses: up to 32 tokens always
    // (1 x 4095 x 4096: 7.5 us, as tiles 16).
    if (c.few || (tma ? per <= 16 && scaled_row_tiles(a, 64) * ((a.n + 127) / 128) <= ctx->sm_count / 2 : per <= kScaledFewAny)) {
        if (per <= 8) return launch_scaled_few<1, 1>(ctx, a);
        if (per <= 16) return launch_scaled_few<2, 1>(ctx, a);
        return launch_scaled_few<4, 2>(ctx, a);
    }
    if (!tma) return a.a_tma || a.w_tma ? launch_scaled_any<false>(ctx, a) : launch_scaled_any<true>(ctx, a);
    if (c.pair) return launch_scaled_pair(ctx, a);
    if (c.nt == 64) return launch_scaled_gemm<64>(ctx, a);
    if (c.nt == 128) return launch_scaled_gemm<128>(ctx, a);
    return launch_scaled_gemm<256>(ctx, a);
}

}  // namespace zb
