// What logits say of given tokens: log probability, entropy, the likeliest alternatives.
//   m = max x, S = sum exp(x - m), W = sum (x - m) exp(x - m):   log p(t) = x_t - m - log S,   entropy = log S - W / S
//
// One pass over the logits.  A thread keeps its own maximum, S and W, four 16-byte vectors at a time, and rescales when a batch raises its
// maximum; the parts are joined at the end.  Logits of minus infinity are taken as a lowest value that no other term sees (a product of
// zero and infinity would spoil W); rows for which that is not so (their maximum is about as low), and rows with a NaN or plus
// infinity, go through a plain second form, one pass a result.
//
// The alternatives: tau, the n-th largest of the threads' maxima, is a lower bound of the n-th largest logit, and only threads whose maximum
// reaches it have seen a logit that does.  About n threads do; their vectors (V / 512 logits each) are read again, from L2, what reaches tau
// is collected, and each candidate's rank among them is its place in the result.  Equal logits rank by id; where hundreds of them equal
// tau (a mask that leaves fewer than n tokens), the row is read from its start for the lowest ids.
//
// Few rows: a cluster of 2, 4 or 8 CTAs shares a row; the first joins the sums and the lists, which come by distributed shared memory.
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
    int parts;                                        // CTAs of a row
};

// Order of the alternatives as one integer: the greater the logit (NaN first), then the lower the id, the greater the key.
__device__ __forceinline__ uint32_t order_of(float x) {
    x += 0.0f;                                        // -0 ranks with +0
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float((order & 0x80000000u) ? (order & 0x7fffffffu) : ~order); }
__device__ __forceinline__ unsigned long long key_of(uint32_t order, int id) { return ((unsigned long long)order << 32) | (uint32_t)~id; }

// 16 bytes of logits.  LOW: bits of a float that its values leave 0; FLOOR: what stands for minus infinity; LEAST: a maximum that FLOOR is
// far enough below to add nothing.
template <typename T> struct Logits;
template <> struct Logits<float> {
    static constexpr int N = 4, LOW = 0;
    static constexpr float FLOOR = -1e30f, LEAST = -0.9e30f;
    static constexpr uint32_t NONE = 0xff800000u;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float max1(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ float floored(uint32_t a) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(FLOOR)); return r; }
    static __device__ __forceinline__ void values(const uint4& v, float* f) { f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w); }
};
template <> struct Logits<__nv_bfloat16> {
    static constexpr int N = 8, LOW = 16;
    static constexpr float FLOOR = -1e30f, LEAST = -0.9e30f;
    static constexpr uint32_t NONE = 0xff80ff80u, FLOOR2 = 0xf14af14au;       // -1.0002e30
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ uint32_t floored2(uint32_t a) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(FLOOR2)); return r; }
    static __device__ __forceinline__ float2 pair(uint32_t a) { return make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
    static __device__ __forceinline__ float max1(uint32_t a) { const float2 p = pair(a); return fmaxf(p.x, p.y); }
    static __device__ __forceinline__ void values(const uint4& v, float* f) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 p = pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
    }
};
template <> struct Logits<__half> {
    static constexpr int N = 8, LOW = 13;
    static constexpr float FLOOR = -65504.0f, LEAST = -65304.0f;
    static constexpr uint32_t NONE = 0xfc00fc00u, FLOOR2 = 0xfbfffbffu;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t r; asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ uint32_t floored2(uint32_t a) { uint32_t r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(FLOOR2)); return r; }
    static __device__ __forceinline__ float2 pair(uint32_t a) { return __half22float2(*reinterpret_cast<const __half2*>(&a)); }
    static __device__ __forceinline__ float max1(uint32_t a) { const float2 p = pair(a); return fmaxf(p.x, p.y); }
    static __device__ __forceinline__ void values(const uint4& v, float* f) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 p = pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
    }
};

__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
constexpr float kLog2e = 1.4426950408889634f;

// m, S and W of what a thread has seen.
struct ExpSums {
    float m, S, W;
    // To a greater maximum.
    __device__ __forceinline__ void raise(float to) {
        const float d = m - to, f = ex2(d * kLog2e);
        W = f > 0.0f ? (W + S * d) * f : 0.0f;         // (d may be so great that S d is infinite)
        S *= f;
        m = to;
    }
    __device__ __forceinline__ void join(ExpSums o) {
        const float to = fmaxf(m, o.m);
        raise(to); o.raise(to);
        S += o.S; W += o.W;
    }
};

struct TokenLogprobsShared {
    static constexpr int THREADS = 512, WARPS = THREADS / 32, CAP = 1024;
    ExpSums sums[WARPS];
    float top[WARPS];
    unsigned long long over[CAP], equal[CAP];          // candidates above tau and at it
    unsigned long long lists[8][kTopMax];              // of the CTAs of a row, in the first of them
    ExpSums part_sums[8];
    float part_top[8];
    int part_odd[8];
    short seen_by[THREADS];
    int n_seen, n_over, n_equal, odd;
    unsigned long long key_part[WARPS];
    float part[WARPS];
};

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

// The plain form, one CTA, a pass for the maximum, one for the sums and one for each alternative.
template <typename T>
__device__ __noinline__ void token_logprobs_plain(const TokenLogprobsArgs& a, long long r, TokenLogprobsShared& sh) {
    const T* x = static_cast<const T*>(a.x) + r * a.stride;
    const int step = blockDim.x;
    float m = -INFINITY;
    for (int v = threadIdx.x; v < a.vocab; v += step) m = fmaxf(m, as_float(x[v]));
    m = block_reduce(m, sh.part, [](float p, float q) { return fmaxf(p, q); });
    if (m == -INFINITY) m = 0.0f;
    float S = 0.0f, W = 0.0f;
    for (int v = threadIdx.x; v < a.vocab; v += step) {
        const float d = as_float(x[v]) - m, e = expf(d);
        S += e;
        W += e == 0.0f ? 0.0f : e * d;
    }
    S = block_reduce(S, sh.part, [](float p, float q) { return p + q; });
    W = block_reduce(W, sh.part, [](float p, float q) { return p + q; });
    const float ls = S == 0.0f ? 0.0f : logf(S);
    auto logp = [&](float v) { return S != S ? S : (S == 0.0f ? -INFINITY : v - m - ls); };
    if (threadIdx.x == 0) {
        if (a.logprob) {
            const int t = a.tokens[r];
            a.logprob[r] = t < 0 ? 0.0f : (t >= a.vocab ? __uint_as_float(0x7fffffffu) : logp(as_float(x[t])));
        }
        if (a.entropy) a.entropy[r] = S == 0.0f ? 0.0f : ls - W / S;
    }
    unsigned long long last = ~0ull;
    for (int i = 0; i < a.top; ++i) {
        unsigned long long best = 0;
        for (int v = threadIdx.x; v < a.vocab; v += step) {
            const unsigned long long k = key_of(order_of(as_float(x[v])), v);
            if ((i == 0 || k < last) && k > best) best = k;
        }
        best = block_reduce(best, sh.key_part, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        last = best;
        if (threadIdx.x == 0) {
            const int id = (int)~(uint32_t)best;
            a.top_ids[r * a.top + i] = id;
            a.top_logprobs[r * a.top + i] = logp(as_float(x[id]));
        }
    }
}

// The places of `n` (distinct) keys among themselves; the first `top` go to out[].
__device__ __forceinline__ void rank_keys(const unsigned long long* a, int na, const unsigned long long* b, int nb, int top, unsigned long long* out) {
    for (int i = threadIdx.x; i < na + nb; i += blockDim.x) {
        const unsigned long long k = i < na ? a[i] : b[i - na];
        int rank = 0;
        for (int j = 0; j < na; ++j) rank += a[j] > k;
        for (int j = 0; j < nb; ++j) rank += b[j] > k;
        if (rank < top) out[rank] = k;
    }
}

template <typename T>
__global__ void __launch_bounds__(TokenLogprobsShared::THREADS, 2) token_logprobs_kernel(const TokenLogprobsArgs a) {
    using L = Logits<T>;
    using Sh = TokenLogprobsShared;
    constexpr int THREADS = Sh::THREADS, U = 4, N = L::N;
    __shared__ Sh sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, P = a.parts;
    const int part = P > 1 ? (int)ptx::cluster_rank() : 0;
    const long long r = (long long)blockIdx.x / P;
    if (tid == 0) { sh.n_seen = sh.n_over = sh.n_equal = 0; sh.odd = 0; }
    if (P > 1) ptx::cluster_arrive();                 // its shared memory may be written to
    ptx::grid_start();
    const T* row = static_cast<const T*>(a.x) + r * a.stride;
    // this CTA's part of the row: single logits up to a 16-byte boundary, vectors, single ones behind
    const int begin = (int)((long long)a.vocab * part / P), len = (int)((long long)a.vocab * (part + 1) / P) - begin;
    const T* x = row + begin;
    const int head = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int nv = (len - head) / N, body = head + nv * N, single = len - nv * N;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    auto single_at = [&](int i) { return i < head ? i : body + i - head; };       // id in the part of the i-th single logit
    float given = 0.0f;                               // on its way while the row is read
    int token = -1;
    if (tid == 0 && part == 0 && a.logprob) {
        token = a.tokens[r];
        if (token >= 0 && token < a.vocab) given = as_float(row[token]);
    }

    ExpSums s{L::FLOOR, 0.0f, 0.0f};
    float seen = -INFINITY;                           // the largest of the thread's vectors
    for (int i = tid; i < nv; i += THREADS * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = i + u * THREADS < nv ? __ldg(xv + i + u * THREADS) : make_uint4(L::NONE, L::NONE, L::NONE, L::NONE);
        uint32_t best = L::max2(L::max2(v[0].x, v[0].y), L::max2(v[0].z, v[0].w));
#pragma unroll
        for (int u = 1; u < U; ++u) best = L::max2(best, L::max2(L::max2(v[u].x, v[u].y), L::max2(v[u].z, v[u].w)));
        const float top = L::max1(best);
        seen = fmaxf(seen, top);
        if (top > s.m) s.raise(top);
        const unsigned long long minus_m = ptx::pack2(-s.m, -s.m), log2e = ptx::pack2(kLog2e, kLog2e);
        unsigned long long S2 = 0, W2 = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&v[u]);
#pragma unroll
            for (int k = 0; k < N / 2; ++k) {
                float2 p;
                if constexpr (N == 8) p = L::pair(L::floored2(w[k]));
                else p = make_float2(L::floored(w[2 * k]), L::floored(w[2 * k + 1]));
                const unsigned long long d = ptx::add2(ptx::pack2(p.x, p.y), minus_m);
                const float2 t = ptx::unpack2(ptx::mul2(d, log2e));
                const unsigned long long e = ptx::pack2(ex2(t.x), ex2(t.y));
                S2 = ptx::add2(S2, e);
                W2 = ptx::fma2(e, d, W2);
            }
        }
        const float2 S = ptx::unpack2(S2), W = ptx::unpack2(W2);
        s.S += S.x + S.y;
        s.W += W.x + W.y;
    }
    float highest = seen;
    if (tid < single) {
        float v = as_float(x[single_at(tid)]);
        highest = fmaxf(highest, v);
        if (v != v || v > L::FLOOR) {
            if (v > s.m) s.raise(v);
            const float d = v - s.m, e = ex2(d * kLog2e);
            s.S += e;
            s.W += e * d;
        }
    }

    // one S and W for the CTA
    ExpSums c = s;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, d));
        c.join(ExpSums{__shfl_xor_sync(0xffffffffu, c.m, d), __shfl_xor_sync(0xffffffffu, c.S, d), __shfl_xor_sync(0xffffffffu, c.W, d)});
    }
    if (lane == 0) { sh.sums[warp] = c; sh.top[warp] = highest; }
    __syncthreads();

    if (a.top > 0) {
        // tau: the largest value that `top` threads reach (0: every logit does)
        const uint32_t mine = tid < nv ? order_of(seen) : 0u;
        uint32_t tau = 0;
        for (int bit = 31; bit >= L::LOW; --bit)
            if (__syncthreads_count(mine >= (tau | (1u << bit))) >= a.top) tau |= 1u << bit;
        if (L::LOW && !(tau & 0x80000000u)) tau |= (1u << L::LOW) - 1u;          // of negative numbers these bits are set
        auto offer = [&](float v, int id) {
            const uint32_t o = order_of(v);
            if (o < tau) return;
            const bool above = o > tau;
            const int at = atomicAdd(above ? &sh.n_over : &sh.n_equal, 1);
            if (at < Sh::CAP) (above ? sh.over : sh.equal)[at] = key_of(o, id);
        };
        if (tid < nv && mine >= tau) sh.seen_by[atomicAdd(&sh.n_seen, 1)] = (short)tid;
        if (tid < single) offer(as_float(x[single_at(tid)]), begin + single_at(tid));
        __syncthreads();
        const int n_seen = sh.n_seen;
        for (int c = warp; c < n_seen; c += Sh::WARPS)
            for (int i = sh.seen_by[c] + lane * THREADS; i < nv; i += 32 * THREADS) {
                const uint4 v = __ldg(xv + i);
                float f[N];
                L::values(v, f);
#pragma unroll
                for (int k = 0; k < N; ++k) offer(f[k], begin + head + i * N + k);
            }
        __syncthreads();
        const int n_over = sh.n_over;
        int n_equal = sh.n_equal;
        if (n_over > Sh::CAP) { if (tid == 0) sh.odd = 1; }
        else {
            if (n_over >= a.top) n_equal = 0;
            else if (n_equal > Sh::CAP - THREADS) {    // the lowest ids among them
                __syncthreads();
                if (tid == 0) sh.n_equal = 0;
                __syncthreads();
                for (int i = 0; i < len; i += THREADS) {
                    if (i + tid < len && order_of(as_float(x[i + tid])) == tau) sh.equal[atomicAdd(&sh.n_equal, 1)] = key_of(tau, begin + i + tid);
                    __syncthreads();
                    n_equal = sh.n_equal;
                    __syncthreads();
                    if (n_over + n_equal >= a.top) break;
                }
            }
            rank_keys(sh.over, n_over, sh.equal, n_equal, a.top, sh.lists[part]);
        }
        __syncthreads();
    }

    if (warp == 0) {
        ExpSums t = lane < Sh::WARPS ? sh.sums[lane] : ExpSums{L::FLOOR, 0.0f, 0.0f};
        float h = lane < Sh::WARPS ? sh.top[lane] : -INFINITY;
#pragma unroll
        for (int d = 8; d; d >>= 1) {
            h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, d));
            t.join(ExpSums{__shfl_xor_sync(0xffffffffu, t.m, d), __shfl_xor_sync(0xffffffffu, t.S, d), __shfl_xor_sync(0xffffffffu, t.W, d)});
        }
        if (lane == 0) { sh.part_sums[part] = t; sh.part_top[part] = h; sh.part_odd[part] = sh.odd; }
    }
    if (P > 1) {
        __syncthreads();
        ptx::cluster_wait();                          // the first CTA has started
        auto send = [&](const void* p) { ptx::st_cluster_u32(ptx::cluster_addr(ptx::smem_u32(p), 0), *static_cast<const uint32_t*>(p)); };
        if (part > 0) {
            if (tid < 2 * a.top) send(reinterpret_cast<const uint32_t*>(sh.lists[part]) + tid);
            if (tid >= 64 && tid < 67) send(reinterpret_cast<const uint32_t*>(&sh.part_sums[part]) + tid - 64);
            if (tid == 67) send(&sh.part_top[part]);
            if (tid == 68) send(&sh.part_odd[part]);
        }
        __syncwarp();
        ptx::cluster_arrive();
        ptx::cluster_wait();
        if (part > 0) return;
        for (int i = tid; i < P * a.top; i += THREADS) sh.over[i] = sh.lists[i / a.top][i % a.top];
        __syncthreads();
        rank_keys(sh.over, P * a.top, nullptr, 0, a.top, sh.lists[0]);
    }
    __syncthreads();
    ExpSums t = sh.part_sums[0];
    float h = sh.part_top[0];
    int odd = sh.part_odd[0];
    for (int i = 1; i < P; ++i) { t.join(sh.part_sums[i]); h = fmaxf(h, sh.part_top[i]); odd |= sh.part_odd[i]; }
    const bool plain = odd || !(t.S < INFINITY) || !(h > L::LEAST);
    if (plain) { token_logprobs_plain<T>(a, r, sh); return; }
    const float ls = logf(t.S);
    if (tid == 0) {
        if (a.logprob) a.logprob[r] = token < 0 ? 0.0f : (token >= a.vocab ? __uint_as_float(0x7fffffffu) : given - t.m - ls);
        if (a.entropy) a.entropy[r] = ls - t.W / t.S;
    }
    if (tid < a.top) {
        const unsigned long long k = sh.lists[0][tid];
        a.top_ids[r * a.top + tid] = (int)~(uint32_t)k;
        a.top_logprobs[r * a.top + tid] = value_of((uint32_t)(k >> 32)) - t.m - ls;
    }
}

inline int32_t run_token_logprobs(zant_ctx* ctx, int32_t dtype, TokenLogprobsArgs a) {
    // Two CTAs fit an SM.  A row is shared while that leaves nobody idle and each part has a batch of vectors for every thread.
    const int batch = TokenLogprobsShared::THREADS * (dtype == ZANT_F32 ? 4 : 8);
    a.parts = 1;
    while (a.parts < 8 && a.rows * a.parts * 2 <= 2LL * ctx->sm_count && a.vocab / (a.parts * 2) >= batch) a.parts *= 2;
    const dim3 grid((unsigned)(a.rows * a.parts));
    auto go = [&](auto kernel) {
        launch_cluster(ctx, kernel, grid, TokenLogprobsShared::THREADS, 0, (unsigned)a.parts, a);
        return check_launch(ctx, "token_logprobs_kernel");
    };
    if (dtype == ZANT_F32) return go(token_logprobs_kernel<float>);
    if (dtype == ZANT_F16) return go(token_logprobs_kernel<__half>);
    return go(token_logprobs_kernel<__nv_bfloat16>);
}

}  // namespace zb
