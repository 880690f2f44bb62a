// Codes and scales of rows of activations: the left operand of the scaled int8 products.
//
//   s[r] = max |x[r, :]| / 127        q[r, c] = nearest integer to x[r, c] / s[r], ties to even
//
// Bound by memory, and instructions close behind: a row is read once and waits in registers, one to eight 16-byte chunks a thread, while its
// threads agree on the maximum.  A warp takes a short row (8 rows a CTA), a CTA of up to 32 warps a longer one; rows beyond 64 KB are read
// twice.  8192 x 8192 bf16: 36 us, 5.6 TB/s; f32 rows 6.1 TB/s; rows that begin at odd addresses about 60 % of that.
//
// Rows may begin at any element: a thread reads the aligned 16-byte block that its chunk begins in, gets the following block from its
// neighbour and shifts the two, so that codes leave in whole words whatever the address of x.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "context.cuh"
#include "ptx_sm100.cuh"
#include "row_codes.cuh"

namespace zb {

struct QuantizeRowsArgs {
    const void* x; long long x_rows, x_stride; int cols;
    const int32_t* index; long long rows;
    int8_t* q; long long q_stride; float* scale;
};

// The first `n` of 16 bytes.  (This and store_some run at the end of a row only, and out of line for the reason that codes_again has.)
__device__ __noinline__ uint4 first_bytes(uint4 v, int n) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = n - 4 * i;
        w[i] &= b <= 0 ? 0u : (b < 4 ? (1u << (8 * b)) - 1u : 0xffffffffu);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __noinline__ void store_some(int8_t* q, uint32_t c0, uint32_t c1, int n) {
    const unsigned long long c = ((unsigned long long)c1 << 32) | c0;
    for (int i = 0; i < n; ++i) q[i] = (int8_t)(c >> (8 * i));
}

// Chunk `at` (its 16 bytes) of a row of `bytes` bytes (none: negative) at `row`, zeros behind its end.  SHIFT: the row does not begin at a
// multiple of 16 bytes but `sh` behind one; called by whole warps, lanes with neighbouring chunks.  Only blocks that hold a byte of the row
// are read.
template <typename T, bool SHIFT, typename I>
__device__ __forceinline__ void row_chunk(const char* row, int sh, I bytes, I at, uint32_t* w) {
    const I left = bytes - at * 16;
    const uint4* p = reinterpret_cast<const uint4*>(row - (SHIFT ? sh : 0)) + at;
    uint4 cur = make_uint4(0, 0, 0, 0);
    if (SHIFT ? left + sh > 0 : left > 0) cur = *p;
    if (SHIFT) {
        uint32_t e[8] = {cur.x, cur.y, cur.z, cur.w, 0, 0, 0, 0};
        const bool last = (threadIdx.x & 31) == 31;
        uint4 nxt = make_uint4(0, 0, 0, 0);
        if (last && left + sh > 16) nxt = p[1];
        const uint32_t* n = reinterpret_cast<const uint32_t*>(&nxt);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const uint32_t o = __shfl_down_sync(0xffffffffu, e[i], 1); e[4 + i] = last ? n[i] : o; }
#pragma unroll
        for (int i = 0; i < 6; ++i) e[i] = (sh & 8) ? e[i + 2] : e[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) e[i] = (sh & 4) ? e[i + 1] : e[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = sizeof(T) < 4 ? __funnelshift_r(e[i], e[i + 1], (sh & 3) * 8) : e[i];
        cur = make_uint4(e[0], e[1], e[2], e[3]);
    }
    if (left < 16 && left + (SHIFT ? sh : 0) > 0) cur = first_bytes(cur, (int)left);
    w[0] = cur.x; w[1] = cur.y; w[2] = cur.z; w[3] = cur.w;
}

template <typename T>
__device__ __forceinline__ void store_codes(int8_t* q, const uint32_t* c, int n, bool whole_words) {
    constexpr int N = RowChunk<T>::N;
    if (n >= N && whole_words) {
        if constexpr (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(c[0], c[1]);
        else *reinterpret_cast<uint32_t*>(q) = c[0];
    } else {
        store_some(q, c[0], N == 8 ? c[N / 4 - 1] : 0u, min(n, N));
    }
}

// `warps` warps a row: 1 (a CTA has 8 rows then) or the whole CTA.  AGAIN: rows longer than the registers of a CTA, read twice.
template <typename T, int CHUNKS, bool AGAIN>
__global__ void __launch_bounds__(CHUNKS == 8 ? 512 : 1024) quantize_rows_kernel(const QuantizeRowsArgs a, int warps) {
    using C = RowChunk<T>;
    using I = std::conditional_t<AGAIN, long long, int>;
    __shared__ uint32_t part[32];
    ptx::grid_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long r = warps == 1 ? (long long)blockIdx.x * 8 + warp : (long long)blockIdx.x;
    if (r >= a.rows) return;                          // (whole warps; a CTA of one row never)
    const int t = warps == 1 ? lane : (int)threadIdx.x, threads = warps * 32;
    const long long from = a.index ? (long long)a.index[r] : r;
    const bool there = from >= 0 && from < a.x_rows;
    const char* row = static_cast<const char*>(a.x) + (there ? from : 0) * a.x_stride * (long long)sizeof(T);
    const int sh = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    const I all = (I)a.cols * (I)sizeof(T), bytes = there ? all : -16, step = threads * CHUNKS;
    const I rounds = AGAIN ? ((all + 15) / 16 + step - 1) / step : 1;
    uint32_t w[CHUNKS][4];
    uint32_t m = 0;
    for (I n = 0; n < rounds; ++n) {
        if (sh == 0) {
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) row_chunk<T, false, I>(row, 0, bytes, n * step + i * threads + t, w[i]);
        } else {                                      // (the same for the whole row)
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) row_chunk<T, true, I>(row, sh, bytes, n * step + i * threads + t, w[i]);
        }
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) m = C::top(m, w[i][j]);
    }
    m = __reduce_max_sync(0xffffffffu, __float_as_uint(C::top_value(m)));
    if (warps > 1) {
        if (lane == 0) part[warp] = m;
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
    }
    const bool finite = m < 0x7f800000u;
    const RowScale k(__uint_as_float(m));
    if (t == 0) a.scale[r] = finite ? k.scale : __uint_as_float(0x7fffffffu);
    const bool none = !finite || k.none();
    const bool exactly = k.tiny || (sizeof(T) == 2 && (__float_as_uint(k.s) & 0xfffu) == 0);
    int8_t* q = a.q + r * a.q_stride;
    const bool whole = (reinterpret_cast<uintptr_t>(q) & (C::N - 1)) == 0;
    for (I n = 0; n < rounds; ++n) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const I at = n * step + i * threads + t;
            if (AGAIN) row_chunk<T, true, I>(row, sh, bytes, at, w[i]);
            const I left = a.cols - at * C::N;
            if (left <= 0) continue;
            uint32_t c[C::N / 4] = {};
            if (!none) {
                codes_of<T>(w[i], k, exactly, c);
            }
            store_codes<T>(q + at * C::N, c, left < C::N ? (int)left : C::N, whole);
        }
    }
}

template <typename T>
inline int32_t launch_quantize_rows(zant_ctx* ctx, const QuantizeRowsArgs& a) {
    const long long chunks = ((long long)a.cols * (long long)sizeof(T) + 15) / 16;
    auto go = [&](auto kernel, int warps) -> int32_t {
        const long long grid = warps == 1 ? (a.rows + 7) / 8 : a.rows;
        launch(ctx, kernel, dim3((unsigned)grid), warps == 1 ? 256 : warps * 32, 0, a, warps);
        return check_launch(ctx, "quantize_rows_kernel");
    };
    auto warps = [&](int per_thread) { return (int)((chunks + 32 * per_thread - 1) / (32 * per_thread)); };
    // Chunks a thread: one for latency while the GPU holds that many threads (8 x 4096 bf16: 1.6, 1.7, 2.1, 2.9 us with 1, 2, 4, 8; 512 x 4096:
    // 3.2, 3.1, 4.5, 5.5), more where there are millions, which saves the instructions that each thread spends on its row (8192 x 4096: 30,
    // 25, 20, 21; 8192 x 8192: 62, 57, 38, 36), and no more than a warp needs for a row (65536 x 1024: 68, 68, 35, 46).
    auto many = [&](int per_thread) { return a.rows * chunks > (long long)ctx->sm_count * (per_thread == 4 ? 40960 : 3000 * per_thread); };
    int per = 1;
    while (per < 8 && (warps(per) > 32 || (warps(per) > 1 && many(per)))) per *= 2;
    if (warps(per) > (per == 8 ? 16 : 32)) return go(quantize_rows_kernel<T, 4, true>, 32);
    if (per == 1) return go(quantize_rows_kernel<T, 1, false>, warps(1));
    if (per == 2) return go(quantize_rows_kernel<T, 2, false>, warps(2));
    if (per == 4) return go(quantize_rows_kernel<T, 4, false>, warps(4));
    return go(quantize_rows_kernel<T, 8, false>, warps(8));
}

inline int32_t run_quantize_rows(zant_ctx* ctx, int32_t dtype, const QuantizeRowsArgs& a) {
    if (dtype == ZANT_F32) return launch_quantize_rows<float>(ctx, a);
    if (dtype == ZANT_F16) return launch_quantize_rows<__half>(ctx, a);
    return launch_quantize_rows<__nv_bfloat16>(ctx, a);
}

}  // namespace zb
