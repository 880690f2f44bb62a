// Products of int8 operands with a scale for each token and each output channel, dense or grouped by expert:
//   y[m, n] = float(sum over k of a[m, k] w[n, k]) * a_scale[m] * w_scale[n] + bias[n]
// The sums are exact, so neither the order nor a split of k changes a result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "context.cuh"
#include "ptx_sm100.cuh"

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
};

__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float scaled_value(int sum, float a_scale, float w_scale) { return __int2float_rn(sum) * a_scale * w_scale; }

// Row tiles of all groups, counted per group: tile t of the launch belongs to the group with first[g] <= t < first[g + 1].
// Called by the whole CTA; `first` holds groups + 1 entries.
template <int THREADS>
__device__ __forceinline__ void group_tiles(const ScaledGemmArgs& a, int tile_rows, int* first) {
    const int tid = threadIdx.x;
    for (int g = tid; g < a.groups; g += THREADS) {
        const int b = min(max(a.offsets[g], 0), a.rows), e = min(max(a.offsets[g + 1], 0), a.rows);
        first[g + 1] = e > b ? (e - b + tile_rows - 1) / tile_rows : 0;
    }
    __syncthreads();
    if (tid < 32) {                                   // running sums, 32 groups at a time
        int sum = 0;
        for (int g0 = 0; g0 < a.groups; g0 += 32) {
            int v = g0 + tid < a.groups ? first[g0 + tid + 1] : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, v, d); if (tid >= d) v += o; }
            if (g0 + tid < a.groups) first[g0 + tid + 1] = sum + v;
            sum += __shfl_sync(0xffffffffu, v, 31);
        }
        if (tid == 0) first[0] = 0;
    }
    __syncthreads();
}

struct RowTile { int group, row, rows; };      // rows: how many of the tile's rows there are

__device__ __forceinline__ RowTile row_tile_of(const ScaledGemmArgs& a, const int* first, int tile, int tile_rows) {
    if (!a.offsets) return RowTile{0, tile * tile_rows, min(tile_rows, a.rows - tile * tile_rows)};
    int lo = 0, hi = a.groups - 1;                    // the last group that starts at or before the tile
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= tile) lo = mid; else hi = mid - 1;
    }
    const int b = min(max(a.offsets[lo], 0), a.rows), e = min(max(a.offsets[lo + 1], 0), a.rows);
    const int row = b + (tile - first[lo]) * tile_rows;
    return RowTile{lo, row, min(tile_rows, e - row)};
}

// ------------------------------------------------------------------------------------------------------------------------------
// Operands at any address: 64 rows x 64 channels a CTA, warp-level MMAs, 64 bytes of k at a time.  Each thread brings 16 bytes of an
// operand row at a time as the aligned words around them, shifted into place.
struct AnyGemm {
    static constexpr int BM = 64, BN = 64, BK = 64, PITCH = 80, THREADS = 128;
};

// 16 bytes p[0..15] of which the first `valid` exist, zeros behind them.  Only words that hold an existing byte are read.
__device__ __forceinline__ uint4 load16_any(const int8_t* p, int valid) {
    uint32_t w[5];
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const int sh = (int)(at & 3);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(at - sh);
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = (valid > 0 && i * 4 < valid + sh) ? q[i] : 0u;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = __funnelshift_r(w[i], w[i + 1], sh * 8);
        const int left = valid - i * 4;
        if (left < 4) v[i] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename Y>
__global__ void __launch_bounds__(AnyGemm::THREADS) scaled_gemm_any_kernel(const ScaledGemmArgs a) {
    using G = AnyGemm;
    __shared__ __align__(16) uint8_t sa[G::BM * G::PITCH], sw[G::BN * G::PITCH];
    __shared__ int first[kScaledMaxGroups + 1];
    ptx::grid_start();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n_tiles = (a.n + G::BN - 1) / G::BN;
    if (a.offsets) group_tiles<G::THREADS>(a, G::BM, first);
    const long long tiles = (long long)(a.offsets ? first[a.groups] : (a.rows + G::BM - 1) / G::BM) * n_tiles;
    for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const RowTile rt = row_tile_of(a, first, (int)(t / n_tiles), G::BM);
        const int n0 = (int)(t % n_tiles) * G::BN;
        const int8_t* ga = a.a + (long long)rt.row * a.a_stride;
        const int8_t* gw = a.w + ((long long)rt.group * a.n + n0) * a.w_stride;
        int acc[8][4] = {};
        for (int k0 = 0; k0 < a.k; k0 += G::BK) {
            __syncthreads();
            for (int i = tid; i < 256; i += G::THREADS) {
                const int r = i >> 2, c = (i & 3) * 16, valid = min(16, a.k - k0 - c);
                *reinterpret_cast<uint4*>(sa + r * G::PITCH + c) = load16_any(ga + (long long)r * a.a_stride + k0 + c, r < rt.rows ? valid : 0);
                *reinterpret_cast<uint4*>(sw + r * G::PITCH + c) = load16_any(gw + (long long)r * a.w_stride + k0 + c, n0 + r < a.n ? valid : 0);
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < G::BK; kk += 32) {
                const uint8_t* pa = sa + (warp * 16 + (lane >> 2)) * G::PITCH + kk + (lane & 3) * 4;
                const uint32_t a0 = *reinterpret_cast<const uint32_t*>(pa), a1 = *reinterpret_cast<const uint32_t*>(pa + 8 * G::PITCH);
                const uint32_t a2 = *reinterpret_cast<const uint32_t*>(pa + 16), a3 = *reinterpret_cast<const uint32_t*>(pa + 8 * G::PITCH + 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint8_t* pw = sw + (j * 8 + (lane >> 2)) * G::PITCH + kk + (lane & 3) * 4;
                    const uint32_t b0 = *reinterpret_cast<const uint32_t*>(pw), b1 = *reinterpret_cast<const uint32_t*>(pw + 16);
                    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                                 : "+r"(acc[j][0]), "+r"(acc[j][1]), "+r"(acc[j][2]), "+r"(acc[j][3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = warp * 16 + (lane >> 2) + 8 * h;
            if (r >= rt.rows) continue;
            const float as = a.a_scale[rt.row + r];
            Y* y = static_cast<Y*>(a.y) + (long long)(rt.row + r) * a.y_stride;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int n = n0 + j * 8 + (lane & 3) * 2 + i;
                    if (n >= a.n) continue;
                    const long long at = (long long)rt.group * a.n + n;
                    float v = scaled_value(acc[j][2 * h + i], as, a.w_scale[at]);
                    if (a.bias) v += a.bias[at];
                    store_as(y + n, v);
                }
        }
    }
}

inline int32_t run_scaled_gemm(zant_ctx* ctx, int32_t y_dtype, const ScaledGemmArgs& a) {
    const dim3 grid((unsigned)ctx->sm_count * 4);
    if (y_dtype == ZANT_F32) launch(ctx, scaled_gemm_any_kernel<float>, grid, AnyGemm::THREADS, 0, a);
    else if (y_dtype == ZANT_F16) launch(ctx, scaled_gemm_any_kernel<__half>, grid, AnyGemm::THREADS, 0, a);
    else launch(ctx, scaled_gemm_any_kernel<__nv_bfloat16>, grid, AnyGemm::THREADS, 0, a);
    return check_launch(ctx, "scaled_gemm_any_kernel");
}

}  // namespace zb
