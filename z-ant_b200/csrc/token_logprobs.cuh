// What logits say of given tokens: log probability, entropy, the likeliest alternatives.
//   m = max x, S = sum exp(x - m), W = sum (x - m) exp(x - m):   log p(t) = x_t - m - log S,   entropy = log S - W / S
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "context.cuh"
#include "ptx_sm100.cuh"
#include "quantize_rows.cuh"

namespace zb {

constexpr int kTopMax = 32;

struct TokenLogprobsArgs {
    const void* x; long long rows, stride; int vocab;
    const int32_t* tokens; float* logprob; float* entropy;
    int top; int32_t* top_ids; float* top_logprobs;
};

// Order of the alternatives as one integer: the greater the logit (NaN first), then the lower the id, the greater the key.
__device__ __forceinline__ uint32_t order_of(float x) {
    x += 0.0f;                                        // -0 ranks with +0
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float x, int id) { return ((unsigned long long)order_of(x) << 32) | (uint32_t)~id; }

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* part, F f) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < (int)blockDim.x / 32; ++i) v = f(v, part[i]);
    return v;
}

// One CTA a row, a pass for each alternative.
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_kernel(const TokenLogprobsArgs a) {
    __shared__ float fpart[8];
    __shared__ unsigned long long kpart[8];
    ptx::grid_start();
    const long long r = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + r * a.stride;
    float m = -INFINITY;
    for (int v = threadIdx.x; v < a.vocab; v += 256) m = fmaxf(m, as_float(x[v]));
    m = block_reduce(m, fpart, [](float p, float q) { return fmaxf(p, q); });
    if (m == -INFINITY) m = 0.0f;
    float S = 0.0f, W = 0.0f;
    for (int v = threadIdx.x; v < a.vocab; v += 256) {
        const float d = as_float(x[v]) - m, e = expf(d);
        S += e;
        W += e == 0.0f ? 0.0f : e * d;
    }
    S = block_reduce(S, fpart, [](float p, float q) { return p + q; });
    W = block_reduce(W, fpart, [](float p, float q) { return p + q; });
    const float ls = S == 0.0f ? 0.0f : logf(S);
    auto logp = [&](float v) { return S == 0.0f && v == v ? -INFINITY : v - m - ls; };
    if (threadIdx.x == 0) {
        if (a.logprob) {
            const int t = a.tokens[r];
            a.logprob[r] = t < 0 ? 0.0f : (t >= a.vocab ? __uint_as_float(0x7fffffffu) : (S != S ? S : logp(as_float(x[t]))));
        }
        if (a.entropy) a.entropy[r] = S == 0.0f ? 0.0f : ls - W / S;
    }
    unsigned long long last = ~0ull;
    for (int i = 0; i < a.top; ++i) {
        unsigned long long best = 0;
        for (int v = threadIdx.x; v < a.vocab; v += 256) {
            const unsigned long long k = key_of(as_float(x[v]), v);
            if ((i == 0 || k < last) && k > best) best = k;
        }
        best = block_reduce(best, kpart, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        last = best;
        if (threadIdx.x == 0) {
            const int id = (int)~(uint32_t)best;
            a.top_ids[r * a.top + i] = id;
            a.top_logprobs[r * a.top + i] = S != S ? S : logp(as_float(x[id]));
        }
    }
}

inline int32_t run_token_logprobs(zant_ctx* ctx, int32_t dtype, const TokenLogprobsArgs& a) {
    const dim3 grid((unsigned)a.rows);
    if (dtype == ZANT_F32) launch(ctx, token_logprobs_kernel<float>, grid, 256, 0, a);
    else if (dtype == ZANT_F16) launch(ctx, token_logprobs_kernel<__half>, grid, 256, 0, a);
    else launch(ctx, token_logprobs_kernel<__nv_bfloat16>, grid, 256, 0, a);
    return check_launch(ctx, "token_logprobs_kernel");
}

}  // namespace zb
