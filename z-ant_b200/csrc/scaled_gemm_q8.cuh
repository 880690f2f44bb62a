// Products of int8 operands with a scale for each token and each output channel, dense or grouped by expert:
//   y[m, n] = float(sum over k of a[m, k] w[n, k]) * a_scale[m] * w_scale[n] + bias[n]
// The sums are exact (int32), so neither their order nor a split of k changes a result.
//
// tcgen05 kind::i8.  The weights are the MMA's A operand: 128 output channels on the lanes of an accumulator, NT tokens in its
// columns.  A warp that reads one column then holds 32 neighbouring channels of one token and stores them as one line, w_scale and bias
// belong to the lane, and few tokens (16 columns) cost few MMA clocks, while the weights stream by at their full 128 rows.
//
// Stages of 128 bytes of k: 128 rows of weights and NT rows of tokens, each a K-major operand in the 128-byte swizzle.  Operands whose rows
// start at multiples of 16 bytes come by TMA; others are brought by four loader warps, which shift 16-byte blocks into place and write them
// where the TMA would have.
//
//   warp 0  TMA        warp 1  TMEM owner, MMA issuer        then 4 or 8 epilogue warps, then (ANY) 4 loader warps
//
// Few tiles: a cluster of 2, 4 or 8 CTAs shares a tile, each takes a part of k; the partial sums go to the CTA that owns the columns through
// distributed shared memory.  No workspace, nothing to clear, the same bits.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "context.cuh"
#include "fused_cnn.cuh"
#include "ptx_sm100.cuh"
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
    int n_tiles, k_blocks, splits, stages;
    int a_tma, w_tma;
    int off_red, off_groups, off_bar;    // shared memory
    int* status;
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
    static constexpr int TMEM_COLS = 2 * NT < 32 ? 32 : 2 * NT;
    static constexpr int PARTS = NT >= 64 ? 2 : 1;                  // warps that share a lane quarter's columns
    static constexpr int COLS = NT / PARTS, CHUNK = COLS < 32 ? COLS : 32;
    static constexpr int EPI = 4 * PARTS;
    static constexpr int LOADERS = 4;
    static constexpr int threads(bool any) { return 64 + 32 * EPI + (any ? 32 * LOADERS : 0); }
};

template <int C>
__device__ __forceinline__ void tmem_ld_cols(uint32_t at, uint32_t* v) {
    if constexpr (C == 32) ptx::tmem_ld32(at, v);
    else ptx::tmem_ld16(at, v);
}

// Results of `cols` neighbouring tokens for the lane's channel: float(sum) * a_scale * w_scale + bias, one rounding to Y.
template <typename Y, int C>
__device__ __forceinline__ void store_columns(const ScaledGemmArgs& a, const uint32_t* v, long long row, int n, bool live, int cols, float as, float ws, float bias, bool has_bias) {
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride + n;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        float r = __int2float_rn((int)v[j]) * __shfl_sync(0xffffffffu, as, j) * ws;
        if (has_bias) r += bias;
        if (live && j < cols) store_as(y, r);
        y += a.y_stride;
    }
}
template <int C>
__device__ __forceinline__ void store_columns_any(const ScaledGemmArgs& a, const uint32_t* v, long long row, int n, bool live, int cols, float as, float ws, float bias) {
    const bool has_bias = a.bias != nullptr;
    if (a.y_dtype == ZANT_F32) store_columns<float, C>(a, v, row, n, live, cols, as, ws, bias, has_bias);
    else if (a.y_dtype == ZANT_F16) store_columns<__half, C>(a, v, row, n, live, cols, as, ws, bias, has_bias);
    else store_columns<__nv_bfloat16, C>(a, v, row, n, live, cols, as, ws, bias, has_bias);
}

// A loader thread's share of one operand's stage: `rows` rows of 128 bytes from `src`, of which `live` exist and `left` bytes of k.  Eight
// lanes take a row: each reads the aligned 16-byte block that its 16 bytes begin in (only blocks that hold a byte of the row are read), gets
// the following block from its neighbour, and shifts the two.
__device__ __forceinline__ void load_stage_any(uint8_t* dst, const int8_t* src, long long stride, int rows, int live, int left, int thread, int threads) {
    const int c = thread & 7, lane = threadIdx.x & 31;
    constexpr int B = 4;
    for (int r0 = thread >> 3; r0 < rows; r0 += B * (threads >> 3)) {
        uint4 cur[B], nxt[B];
        int sh[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int r = r0 + i * (threads >> 3);
            const int8_t* p = src + (long long)r * stride + c * 16;
            const uintptr_t at = reinterpret_cast<uintptr_t>(p);
            sh[i] = (int)(at & 15);
            const uint4* q = reinterpret_cast<const uint4*>(at - sh[i]);
            const int ahead = left - c * 16 + sh[i];              // bytes from the block's start to the row's end
            cur[i] = r < live && ahead > 0 ? __ldg(q) : make_uint4(0, 0, 0, 0);
            nxt[i] = make_uint4(0, 0, 0, 0);
            if (c == 7 && r < live && sh[i] && ahead > 16) nxt[i] = __ldg(q + 1);
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int r = r0 + i * (threads >> 3);
            uint32_t w[8] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w, 0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t o = __shfl_sync(0xffffffffu, w[k], (lane + 1) & 31);
                w[4 + k] = c == 7 ? (k == 0 ? nxt[i].x : (k == 1 ? nxt[i].y : (k == 2 ? nxt[i].z : nxt[i].w))) : o;
            }
            if (sh[i] & 8) {
#pragma unroll
                for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
            }
            if (sh[i] & 4) {
#pragma unroll
                for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
            }
            uint4 v;
            uint32_t* o = reinterpret_cast<uint32_t*>(&v);
            const int bits = (sh[i] & 3) * 8, bytes = left - c * 16;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] = __funnelshift_r(w[k], w[k + 1], bits);
                const int b = bytes - 4 * k;
                if (b < 4) o[k] &= b <= 0 ? 0u : (1u << (8 * b)) - 1u;
            }
            if (r < rows) *reinterpret_cast<uint4*>(dst + r * 128 + ((c ^ (r & 7)) << 4)) = v;
        }
    }
}

template <int NT, bool ANY>
__global__ void __launch_bounds__(ScaledCfg<NT>::threads(ANY), 1) scaled_gemm_kernel(const __grid_constant__ ScaledGemmArgs a, const __grid_constant__ CUtensorMap w_map,
                                                                                     const __grid_constant__ CUtensorMap a_map) {
    using Cfg = ScaledCfg<NT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t s0 = ptx::smem_u32(smem);
    int* grow = reinterpret_cast<int*>(smem + a.off_groups);
    int* gfirst = grow + kScaledMaxGroups + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + a.off_bar + 400);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + a.off_bar + 404);
    const uint32_t bar0 = s0 + (uint32_t)a.off_bar;
    auto full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    auto empty = [&](int s) { return bar0 + 128u + 8u * (uint32_t)s; };
    auto tfull = [&](int b) { return bar0 + 256u + 8u * (uint32_t)b; };
    auto tempty = [&](int b) { return bar0 + 272u + 8u * (uint32_t)b; };
    auto parts_in = [&](int b) { return bar0 + 288u + 8u * (uint32_t)b; };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = a.splits, rank = S > 1 ? (int)ptx::cluster_rank() : 0;
    if (tid == 0) {
        for (int s = 0; s < a.stages; ++s) { ptx::mbar_init(full(s), ANY ? 1 + Cfg::LOADERS : 1); ptx::mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; ++b) { ptx::mbar_init(tfull(b), 1); ptx::mbar_init(tempty(b), Cfg::EPI); ptx::mbar_init(parts_in(b), S * Cfg::EPI); }
        *abort_flag = 0;
        ptx::mbar_fence_init();
    }
    if (warp == 1) { ptx::tmem_alloc(ptx::smem_u32(tmem_slot), Cfg::TMEM_COLS); ptx::tmem_relinquish(); }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (S > 1) { ptx::cluster_arrive(); ptx::cluster_wait(); }        // every CTA's barriers are there
    ptx::grid_trigger();
    ptx::grid_wait();

    int row_tiles = (a.rows + NT - 1) / NT;
    if (a.offsets) { group_tiles(a.offsets, a.groups, a.rows, NT, grow, gfirst); row_tiles = gfirst[a.groups]; }
    const int tiles = row_tiles * a.n_tiles, step = (int)gridDim.x / S, t0 = (int)blockIdx.x / S;
    const int kb0 = a.k_blocks * rank / S, kb1 = a.k_blocks * (rank + 1) / S;

    if (warp == 0) {
        if (ptx::elect_one()) {
            const uint32_t bytes = (!ANY || a.w_tma ? Cfg::STAGE_W : 0) + (!ANY || a.a_tma ? NT * 128 : 0);
            int s = 0; uint32_t ph = 0;
            for (int t = t0; t < tiles; t += step) {
                const TileAt at = tile_at(t, row_tiles, a.n_tiles);
                const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
                const int wrow = rt.group * a.n + at.n * 128;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!ptx::mbar_wait(empty(s), ph ^ 1u, abort_flag)) goto producer_done;
                    ptx::mbar_arrive_expect_tx(full(s), bytes);
                    const uint32_t dst = s0 + (uint32_t)(s * Cfg::STAGE);
                    if (!ANY || a.w_tma) ptx::tma_load_2d(dst, &w_map, kb * 128, wrow, full(s));
                    if (!ANY || a.a_tma) ptx::tma_load_2d(dst + Cfg::STAGE_W, &a_map, kb * 128, rt.row, full(s));
                    if (++s == a.stages) { s = 0; ph ^= 1u; }
                }
            }
        producer_done:;
        }
    } else if (warp == 1) {
        const uint32_t leader = ptx::elect_one() ? 1u : 0u;
        const uint32_t hi = (uint32_t)(smem_desc_kmajor_swizzled(0, 128) >> 32), lo = (uint32_t)smem_desc_kmajor_swizzled(0, 128);
        int s = 0, ti = 0; uint32_t ph = 0;
        for (int t = t0; t < tiles; t += step, ++ti) {
            const int b = ti & 1;
            if (!ptx::mbar_wait(tempty(b), ((uint32_t)(ti >> 1) & 1u) ^ 1u, abort_flag)) break;
            ptx::tc_fence_after();
            const RowTile rt = row_tile_of(a, grow, gfirst, tile_at(t, row_tiles, a.n_tiles).m, NT);
            const uint32_t idesc = ptx::idesc_i8(128, (rt.rows + 15) & ~15, true, true), d = tmem_base + (uint32_t)(b * NT);
            bool ok = true;
            for (int kb = kb0; kb < kb1 && ok; ++kb) {
                ok = ptx::mbar_wait(full(s), ph, abort_flag);
                if (!ok) break;
                ptx::tc_fence_after();
                const uint32_t wa = lo + ((s0 + (uint32_t)(s * Cfg::STAGE)) >> 4), ta = wa + (Cfg::STAGE_W >> 4);
                const int steps = min(4, (a.k - kb * 128 + 31) >> 5);
                for (int i = 0; i < steps; ++i) ptx::mma_i8_if(leader, d, wa + 2u * i, hi, ta + 2u * i, hi, idesc, (kb > kb0 || i > 0) ? 1u : 0u);
                ptx::mma_commit_if(leader, empty(s));
                if (++s == a.stages) { s = 0; ph ^= 1u; }
            }
            if (!ok) break;
            ptx::mma_commit_if(leader, tfull(b));
        }
    } else if (warp < 2 + Cfg::EPI) {
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        int ti = 0;
        for (int t = t0; t < tiles; t += step, ++ti) {
            const TileAt at = tile_at(t, row_tiles, a.n_tiles);
            const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
            const int n = at.n * 128 + quarter * 32 + lane, b = ti & 1;
            const bool live = n < a.n;
            const long long wat = (long long)rt.group * a.n + n;
            const float ws = live ? a.w_scale[wat] : 0.0f, bias = live && a.bias ? a.bias[wat] : 0.0f;
            if (!ptx::mbar_wait(tfull(b), (uint32_t)(ti >> 1) & 1u, abort_flag)) break;
            ptx::tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * NT);
            if (S == 1) {
                for (int c = part * Cfg::COLS; c < (part + 1) * Cfg::COLS && c < rt.rows; c += Cfg::CHUNK) {
                    const float as = c + lane < rt.rows ? a.a_scale[rt.row + c + lane] : 0.0f;
                    uint32_t v[Cfg::CHUNK];
                    tmem_ld_cols<Cfg::CHUNK>(taddr + (uint32_t)c, v);
                    ptx::tmem_wait_ld();
                    store_columns_any<Cfg::CHUNK>(a, v, (long long)rt.row + c, n, live, rt.rows - c, as, ws, bias);
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(tempty(b));
            } else {
                // columns own * j .. own * j + own - 1 are finished by CTA j: every CTA sends it its sums of them, [CTA][column][channel]
                const int own = NT / S;
                const uint32_t red = s0 + (uint32_t)a.off_red + (uint32_t)(b * NT * 512);
                const uint32_t mine = red + (uint32_t)(rank * own * 512 + (quarter * 32 + lane) * 4);
                for (int c = part * Cfg::COLS; c < (part + 1) * Cfg::COLS && c < rt.rows; c += Cfg::CHUNK) {
                    uint32_t v[Cfg::CHUNK];
                    tmem_ld_cols<Cfg::CHUNK>(taddr + (uint32_t)c, v);
                    ptx::tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < Cfg::CHUNK; ++j)
                        if (c + j < rt.rows) ptx::st_cluster_u32(ptx::cluster_addr(mine + (uint32_t)(((c + j) % own) * 512), (uint32_t)((c + j) / own)), v[j]);
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(tempty(b));
                    for (int j = 0; j < S; ++j) ptx::mbar_arrive_cluster(ptx::cluster_addr(parts_in(b), (uint32_t)j));
                }
                if (!ptx::mbar_wait(parts_in(b), (uint32_t)(ti >> 1) & 1u, abort_flag)) break;
                ptx::fence_acquire_cluster();
                const int* sums = reinterpret_cast<const int*>(smem + a.off_red + b * NT * 512) + quarter * 32 + lane;
                for (int c = part; c < own; c += Cfg::PARTS) {
                    const int col = rank * own + c;
                    if (col >= rt.rows) break;
                    int sum = 0;
                    for (int j = 0; j < S; ++j) sum += sums[(j * own + c) * 128];
                    const float as = a.a_scale[rt.row + col];
                    float r = __int2float_rn(sum) * as * ws;
                    if (a.bias) r += bias;
                    const long long at_y = (long long)(rt.row + col) * a.y_stride + n;
                    if (live) {
                        if (a.y_dtype == ZANT_F32) static_cast<float*>(a.y)[at_y] = r;
                        else if (a.y_dtype == ZANT_F16) store_as(static_cast<__half*>(a.y) + at_y, r);
                        else store_as(static_cast<__nv_bfloat16*>(a.y) + at_y, r);
                    }
                }
            }
        }
    } else if constexpr (ANY) {
        const int thread = tid - 64 - 32 * Cfg::EPI;
        int s = 0; uint32_t ph = 0;
        bool ok = true;
        for (int t = t0; t < tiles && ok; t += step) {
            const TileAt at = tile_at(t, row_tiles, a.n_tiles);
            const RowTile rt = row_tile_of(a, grow, gfirst, at.m, NT);
            const int8_t* w = a.w + ((long long)rt.group * a.n + at.n * 128) * a.w_stride;
            const int8_t* x = a.a + (long long)rt.row * a.a_stride;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = ptx::mbar_wait(empty(s), ph ^ 1u, abort_flag);
                if (!ok) break;
                uint8_t* dst = smem + s * Cfg::STAGE;
                const int left = min(128, a.k - kb * 128);
                if (!a.w_tma) load_stage_any(dst, w + kb * 128, a.w_stride, 128, a.n - at.n * 128, left, thread, 32 * Cfg::LOADERS);
                if (!a.a_tma) load_stage_any(dst + Cfg::STAGE_W, x + kb * 128, a.a_stride, NT, rt.rows, left, thread, 32 * Cfg::LOADERS);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(full(s));
                if (++s == a.stages) { s = 0; ph ^= 1u; }
            }
        }
    }

    if (*abort_flag) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);      // copies in flight land
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) ptx::tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    if (S > 1) { ptx::cluster_arrive(); ptx::cluster_wait(); }        // nobody leaves while its memory or barriers are written to
    if (tid == 0 && *abort_flag) atomicExch(a.status, (int)DEV_ERR_WAIT_TIMEOUT);
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

template <int NT, bool ANY>
inline int32_t launch_scaled_gemm(zant_ctx* ctx, ScaledGemmArgs a, long long row_tiles) {
    using Cfg = ScaledCfg<NT>;
    constexpr int LIMIT = 232448;
    a.n_tiles = (a.n + 127) / 128;
    a.k_blocks = (a.k + 127) / 128;
    const long long tiles = std::max<long long>(1, row_tiles) * a.n_tiles;
    a.splits = 1;
    if (NT <= 64) while (a.splits < 8 && tiles * a.splits * 2 <= ctx->sm_count && a.splits * 2 <= a.k_blocks) a.splits *= 2;
    const int red = a.splits > 1 ? 2 * NT * 512 : 0, groups = a.offsets ? (kScaledMaxGroups + 1) * 8 : 0;
    a.stages = std::min(16, (LIMIT - red - groups - 528) / Cfg::STAGE);
    a.off_red = a.stages * Cfg::STAGE;
    a.off_groups = a.off_red + red;
    a.off_bar = (int)align_up((size_t)(a.off_groups + groups), 16);
    const size_t smem = (size_t)a.off_bar + 512;
    alignas(64) CUtensorMap w_map{}, a_map{};
    if (a.w_tma) ZB_TRY(encode_rows_map(&w_map, a.w, (size_t)a.k, (size_t)a.groups * a.n, (size_t)a.w_stride, 128));
    if (a.a_tma) ZB_TRY(encode_rows_map(&a_map, a.a, (size_t)a.k, (size_t)a.rows, (size_t)a.a_stride, NT));
    auto kernel = scaled_gemm_kernel<NT, ANY>;
    ZB_SMEM_ATTR(ctx, kernel, LIMIT);
    const long long clusters = std::min<long long>(tiles, ctx->sm_count / a.splits);
    launch_cluster(ctx, kernel, dim3((unsigned)(clusters * a.splits)), Cfg::threads(ANY), smem, (unsigned)a.splits, a, w_map, a_map);
    return check_launch(ctx, "scaled_gemm_kernel");
}

template <bool ANY>
inline int32_t run_scaled_gemm_nt(zant_ctx* ctx, const ScaledGemmArgs& a) {
    const long long per_group = std::max<long long>(1, (a.rows + a.groups - 1) / a.groups), groups = std::min(a.rows, a.groups);
    auto tiles = [&](int nt) { return a.offsets ? std::max<long long>(groups, a.rows / nt) : (a.rows + nt - 1) / nt; };
    if (per_group <= 16) return launch_scaled_gemm<16, ANY>(ctx, a, tiles(16));
    if (per_group <= 32) return launch_scaled_gemm<32, ANY>(ctx, a, tiles(32));
    if (per_group <= 64) return launch_scaled_gemm<64, ANY>(ctx, a, tiles(64));
    if (per_group <= 128) return launch_scaled_gemm<128, ANY>(ctx, a, tiles(128));
    return launch_scaled_gemm<256, ANY>(ctx, a, tiles(256));
}

inline int32_t run_scaled_gemm(zant_ctx* ctx, int32_t y_dtype, ScaledGemmArgs a) {
    a.y_dtype = y_dtype;
    a.a_tma = tma_rows(a.a, (size_t)a.rows, (size_t)a.a_stride);
    a.w_tma = tma_rows(a.w, (size_t)a.groups * a.n, (size_t)a.w_stride);
    a.status = ctx->status_word;
    return a.a_tma && a.w_tma ? run_scaled_gemm_nt<false>(ctx, a) : run_scaled_gemm_nt<true>(ctx, a);
}

}  // namespace zb
