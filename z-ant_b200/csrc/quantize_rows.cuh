// Codes and scales of rows of activations: the left operand of the scaled int8 products.
//
//   s[r] = max |x[r, :]| / 127        q[r, c] = nearest integer to x[r, c] / s[r], ties to even
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "context.cuh"
#include "ptx_sm100.cuh"

namespace zb {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

struct QuantizeRowsArgs {
    const void* x; long long x_rows, x_stride; int cols;
    const int32_t* index; long long rows;
    int8_t* q; long long q_stride; float* scale;
};

// A row's scale, and what turns values into codes.  Rows of tiny values (below 2^-60) are scaled up by 2^80 on the way, which is exact:
// neither the reciprocal nor a remainder leaves the normal numbers then.
struct RowScale {
    float scale, up, s, inv;
    __device__ __forceinline__ explicit RowScale(float amax) {
        scale = amax / 127.0f;
        up = amax < 8.6736174e-19f ? 1.2089258e24f : 1.0f;
        s = scale * up;
        inv = 1.0f / s;
    }
    __device__ __forceinline__ bool none() const { return !(s > 0.0f) || s > 3.4e38f; }
    // The nearest integer to the exact quotient v / s: the product with the reciprocal is off by less than one code, and the remainder
    // of the nearest code, v - t s, is exact in fp32 (a multiple of the last place of s or v, and at most about s), so that comparing it
    // with s / 2 decides.
    __device__ __forceinline__ int code(float v) const {
        v *= up;
        float t = rintf(v * inv);
        const float rem = fmaf(-t, s, v), half = 0.5f * s;
        const bool odd = (static_cast<int>(t) & 1) != 0;
        if (rem > half || (rem == half && odd)) t += 1.0f;
        if (rem < -half || (rem == -half && odd)) t -= 1.0f;
        return static_cast<int>(fminf(fmaxf(t, -127.0f), 127.0f));
    }
};

// One CTA a row, two passes over it.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeRowsArgs a) {
    __shared__ float part[8];
    ptx::grid_start();
    const long long r = blockIdx.x;
    const long long from = a.index ? (long long)a.index[r] : r;
    int8_t* q = a.q + r * a.q_stride;
    if (from < 0 || from >= a.x_rows) {
        for (int c = threadIdx.x; c < a.cols; c += 256) q[c] = 0;
        if (threadIdx.x == 0) a.scale[r] = 0.0f;
        return;
    }
    const T* x = static_cast<const T*>(a.x) + from * a.x_stride;
    uint32_t m = 0;                                  // magnitudes compare as integers, NaN above infinity
    for (int c = threadIdx.x; c < a.cols; c += 256) m = max(m, __float_as_uint(as_float(x[c])) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = __uint_as_float(m);
    __syncthreads();
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(part[i]));
    const bool finite = m < 0x7f800000u;
    const RowScale k(__uint_as_float(m));
    if (threadIdx.x == 0) a.scale[r] = finite ? k.scale : __uint_as_float(0x7fffffffu);
    const bool none = !finite || k.none();
    for (int c = threadIdx.x; c < a.cols; c += 256) q[c] = none ? 0 : (int8_t)k.code(as_float(x[c]));
}

inline int32_t run_quantize_rows(zant_ctx* ctx, int32_t dtype, const QuantizeRowsArgs& a) {
    const dim3 grid((unsigned)a.rows);
    if (dtype == ZANT_F32) launch(ctx, quantize_rows_kernel<float>, grid, 256, 0, a);
    else if (dtype == ZANT_F16) launch(ctx, quantize_rows_kernel<__half>, grid, 256, 0, a);
    else launch(ctx, quantize_rows_kernel<__nv_bfloat16>, grid, 256, 0, a);
    return check_launch(ctx, "quantize_rows_kernel");
}

}  // namespace zb
