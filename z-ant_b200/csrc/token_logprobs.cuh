// What logits say of given tokens: log probability, entropy, the likeliest alternatives.
//   m = max x, S = sum exp(x - m), W = sum (x - m) exp(x - m):   log p(t) = x_t - m - log S,   entropy = log S - W / S
//
// One pass over the logits.  A thread keeps its own maximum, S and W, four 16-byte vectors at a time, and rescales when a batch raises its
// maximum; the parts are joined at the end.  Everything is in units of log 2: d = x log2(e) - m log2(e) is one fused operation for two
// logits, and the rounding of m log2(e), which all terms of a sum share, cancels in log p and the entropy because the token's own d is
// taken the same way, as long as it is a fraction of 1: from a maximum of 2^22 on it would be more than the differences themselves, and the
// powers overflow or vanish (rows of -1e10 throughout, say, as a mask leaves them).  Logits of minus infinity are taken as a lowest value that no
// other term sees (a product of zero and infinity would spoil W).  Rows whose maximum is beyond 2^22 to either side (in f16, so low that the
// lowest value is seen) have their sums taken again in a plain second form, a pass each; rows with a NaN or plus infinity their alternatives
// too, a pass each.
//
// The alternatives: tau, the n-th largest of the threads' maxima, is a lower bound of the n-th largest logit, and only threads whose maximum
// reaches it have seen a logit that does.  About n threads do; their vectors (V / threads logits each) are read again, from L2, what
// reaches tau is collected, and each candidate's rank among them is its place in the result.  Equal logits rank by id; where hundreds of
// them equal tau (a mask that leaves fewer than n tokens), the row is read from its start for the lowest ids.  That is slow: where a CTA has fewer
// than n threads with an unmasked logit, tau is the mask's value (64 x 128000 bf16, n = 20: 12 us with 99 % masked, 69 with 99.99 %).
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

// 16 bytes of logits.  LOW: bits of a float that its values leave 0; FLOOR: a thread's maximum before it has seen one; what stands for minus
// infinity is FLOOR in f16, below it in the others, where the rounding of FLOOR log2(e) leaves a difference whose power would overflow;
// LEAST, MOST: between them a row's maximum leaves the rounding of m log2(e) a quarter at most, and the first two so far below that they add nothing.
template <typename T> struct Logits;
template <> struct Logits<float> {
    static constexpr int N = 4, LOW = 0;
    static constexpr float FLOOR = -1e30f, LEAST = -4194304.0f, MOST = 4194304.0f;
    static constexpr uint32_t NONE = 0xff800000u;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float max1(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ float floored(uint32_t a) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(2.0f * FLOOR)); return r; }
    static __device__ __forceinline__ void values(const uint4& v, float* f) { f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w); }
};
template <> struct Logits<__nv_bfloat16> {
    static constexpr int N = 8, LOW = 16;
    static constexpr float FLOOR = -1e30f, LEAST = -4194304.0f, MOST = 4194304.0f;
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
    static constexpr float FLOOR = -65504.0f, LEAST = -65304.0f, MOST = INFINITY;
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
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// m log2(e), S and W (in log 2) of what a thread has seen.
struct ExpSums {
    float m, S, W;
    // To a greater maximum.
    __device__ __forceinline__ void raise(float to) {
        const float d = m - to, f = ex2(d);
        W = f > 0.0f ? (W + S * d) * f : 0.0f;         // (d may be so great that S d is infinite)
        S *= f;
        m = to;
    }
    // The sums of a warp's lanes, in every lane.
    __device__ __forceinline__ void join_lanes(int lanes) {
        float top = m;
        for (int d = lanes / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        raise(top);
        for (int d = lanes / 2; d; d >>= 1) { S += __shfl_xor_sync(0xffffffffu, S, d); W += __shfl_xor_sync(0xffffffffu, W, d); }
    }
};

template <int T>
struct TokenLogprobsShared {
    static constexpr int THREADS = T, WARPS = THREADS / 32, CAP = 1024;
    ExpSums sums[WARPS];
    float top[WARPS];
    uint32_t seen[THREADS];                            // the threads' maxima, as orders (0: none)
    unsigned long long over[CAP], equal[CAP];          // candidates above tau and at it
    unsigned long long lists[8][kTopMax];              // of the CTAs of a row, in the first of them
    ExpSums part_sums[8];
    float part_top[8];
    int part_odd[8];
    short seen_by[THREADS];
    uint32_t tau;
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

// The plain form, one CTA, a pass for the maximum, one for the sums and one for each alternative.  LISTED: the alternatives are known, sh.lists[0].
template <typename T, typename Sh>
__device__ __noinline__ void token_logprobs_plain(const TokenLogprobsArgs& a, long long r, bool listed, Sh& sh) {
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
    if (listed) {
        if (threadIdx.x < a.top) {
            const int id = (int)~(uint32_t)sh.lists[0][threadIdx.x];
            a.top_ids[r * a.top + threadIdx.x] = id;
            a.top_logprobs[r * a.top + threadIdx.x] = logp(as_float(x[id]));
        }
        return;
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

// tau of a warp that holds R maxima a lane: the largest value that `top` of all reach, in the bits that values have (0: fewer than `top` threads
// have seen a logit).  Bit by bit below what the largest and the least of them have in common.
template <int R, int LOW>
__device__ __forceinline__ uint32_t nth_largest(const uint32_t (&v)[R], int top) {
    uint32_t hi = v[0], lo = v[0];
#pragma unroll
    for (int i = 1; i < R; ++i) { hi = max(hi, v[i]); lo = min(lo, v[i]); }
    hi = __reduce_max_sync(0xffffffffu, hi); lo = __reduce_min_sync(0xffffffffu, lo);
    if (top == 1) return hi;
    if (hi == lo) return lo;
    const int first = 31 - __clz(hi ^ lo);
    uint32_t tau = first == 31 ? 0u : hi & ~((2u << first) - 1u);
    for (int bit = first; bit >= LOW; --bit) {
        const uint32_t at = tau | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) n += v[i] >= at;
        if ((int)__reduce_add_sync(0xffffffffu, (unsigned)n) >= top) tau = at;
    }
    return tau;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const TokenLogprobsArgs a) {
    using L = Logits<T>;
    using Sh = TokenLogprobsShared<THREADS>;
    constexpr int U = 4, N = L::N;
    __shared__ Sh sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, P = a.parts;
    const int part = P > 1 ? (int)ptx::cluster_rank() : 0;
    const long long r = (long long)blockIdx.x / P;
    if (tid == 0) sh.n_seen = sh.n_over = sh.n_equal = 0;
    __syncwarp();
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

    ExpSums s{L::FLOOR * kLog2e, 0.0f, 0.0f};
    float m = L::FLOOR;
    float seen = -INFINITY;                           // the largest of the thread's vectors
    // (Plain loads, here and below: the kernel before this one may have written the logits while this one started.)  Past L1, unless many alternatives are looked for in what has been read (4096 x 65536: 112 -> 103 us with one, 134 -> 140 with 20).
    const bool once = a.top <= 8;
    for (int i = tid; i < nv; i += THREADS * U) {
        uint4 v[U];
        if (once) {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = i + u * THREADS < nv ? ptx::ld_global_once(xv + i + u * THREADS) : make_uint4(L::NONE, L::NONE, L::NONE, L::NONE);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = i + u * THREADS < nv ? xv[i + u * THREADS] : make_uint4(L::NONE, L::NONE, L::NONE, L::NONE);
        }
        uint32_t best = L::max2(L::max2(v[0].x, v[0].y), L::max2(v[0].z, v[0].w));
#pragma unroll
        for (int u = 1; u < U; ++u) best = L::max2(best, L::max2(L::max2(v[u].x, v[u].y), L::max2(v[u].z, v[u].w)));
        const float top = L::max1(best);
        seen = fmaxf(seen, top);
        if (top > m) { m = top; s.raise(m * kLog2e); }
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
                const unsigned long long d = ptx::fma2(ptx::pack2(p.x, p.y), log2e, minus_m);
                const float2 t = ptx::unpack2(d);
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
            if (v > m) s.raise(v * kLog2e);
            const float d = fmaf(v, kLog2e, -s.m), e = ex2(d);
            s.S += e;
            s.W += e * d;
        }
    }

    // one S and W for the CTA
    ExpSums c = s;
    c.join_lanes(32);
#pragma unroll
    for (int d = 16; d; d >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, d));
    if (lane == 0) { sh.sums[warp] = c; sh.top[warp] = highest; }
    const uint32_t mine = tid < nv ? order_of(seen) : 0u;
    if (a.top > 0) sh.seen[tid] = mine;
    __syncthreads();
    if (warp == 0) {
        const bool in = lane < Sh::WARPS;
        ExpSums t = in ? sh.sums[lane] : ExpSums{L::FLOOR * kLog2e, 0.0f, 0.0f};
        float h = in ? sh.top[lane] : -INFINITY;
        t.join_lanes(Sh::WARPS);
#pragma unroll
        for (int d = Sh::WARPS / 2; d; d >>= 1) h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, d));
        if (lane == 0) { sh.part_sums[part] = t; sh.part_top[part] = h; sh.part_odd[part] = 0; }
        if (a.top > 0) {
            uint32_t v[Sh::WARPS];
#pragma unroll
            for (int i = 0; i < Sh::WARPS; ++i) v[i] = sh.seen[i * 32 + lane];
            uint32_t tau = nth_largest<Sh::WARPS, L::LOW>(v, a.top);
            if (L::LOW && !(tau & 0x80000000u)) tau |= (1u << L::LOW) - 1u;      // of negative numbers these bits are set
            if (lane == 0) sh.tau = tau;
        }
    }
    __syncthreads();

    if (a.top > 0) {
        const uint32_t tau = sh.tau;
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
                const uint4 v = xv[i];
                float f[N];
                L::values(v, f);
#pragma unroll
                for (int k = 0; k < N; ++k) offer(f[k], begin + head + i * N + k);
            }
        __syncthreads();
        const int n_over = sh.n_over;
        int n_equal = sh.n_equal;
        if (n_over > Sh::CAP) { if (tid == 0) sh.part_odd[part] = 1; }
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

    if (P > 1) {
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
    for (int i = 1; i < P; ++i) {
        ExpSums o = sh.part_sums[i];
        const float to = fmaxf(t.m, o.m);
        t.raise(to); o.raise(to);
        t.S += o.S; t.W += o.W;
        h = fmaxf(h, sh.part_top[i]);
        odd |= sh.part_odd[i];
    }
    // (Ranked as floats the alternatives are right whatever the sums are, but for a NaN, which makes S one: a thread's maximum does not see it.)
    if (odd || !(t.S < INFINITY) || !(h > L::LEAST) || !(h < L::MOST)) { token_logprobs_plain<T>(a, r, !odd && t.S == t.S, sh); return; }
    const float ls = log2f(t.S);
    auto logp = [&](float v) {
        const float p = (fmaf(v, kLog2e, -t.m) - ls) * kLn2;
        return p > -INFINITY ? p : v - t.m * kLn2;    // (about the lowest value of the type: its product with log2(e) is infinite)
    };
    if (tid == 0) {
        if (a.logprob) a.logprob[r] = token < 0 ? 0.0f : (token >= a.vocab ? __uint_as_float(0x7fffffffu) : logp(given));
        if (a.entropy) a.entropy[r] = (ls - t.W / t.S) * kLn2;
    }
    if (tid < a.top) {
        const unsigned long long k = sh.lists[0][tid];
        a.top_ids[r * a.top + tid] = (int)~(uint32_t)k;
        a.top_logprobs[r * a.top + tid] = logp(value_of((uint32_t)(k >> 32)));
    }
}

template <int THREADS>
inline int32_t launch_token_logprobs(zant_ctx* ctx, int32_t dtype, TokenLogprobsArgs a, int parts) {
    a.parts = parts;
    auto go = [&](auto kernel) {
        launch_cluster(ctx, kernel, dim3((unsigned)(a.rows * parts)), THREADS, 0, (unsigned)parts, a);
        return check_launch(ctx, "token_logprobs_kernel");
    };
    if (dtype == ZANT_F32) return go(token_logprobs_kernel<float, THREADS>);
    if (dtype == ZANT_F16) return go(token_logprobs_kernel<__half, THREADS>);
    return go(token_logprobs_kernel<__nv_bfloat16, THREADS>);
}

inline int32_t run_token_logprobs(zant_ctx* ctx, int32_t dtype, const TokenLogprobsArgs& a) {
    const int vectors = a.vocab / (dtype == ZANT_F32 ? 4 : 8);
    // Many rows: small CTAs, whose ends (about 3 us after the last logit) overlap with other rows (1000 x 5000 bf16: 8.8, 13.0, 25.5 us with
    // 128, 256, 512 threads), but not so small that tau lets much through (4096 x 65536, 20 alternatives: 158, 134, 160).
    if (a.rows > 2LL * ctx->sm_count) return vectors <= 4096 ? launch_token_logprobs<128>(ctx, dtype, a, 1) : launch_token_logprobs<256>(ctx, dtype, a, 1);
    // Few rows: two large CTAs an SM; a row is shared while that leaves nobody idle and a thread has 7 vectors (64 x 128000 bf16: 17.6, 14.1,
    // 12.6, 25.6 us with 1, 2, 4, 8 CTAs a row; 64 x 32000: 5.3, 5.6, 7.1).
    int parts = 1;
    while (parts < 8 && a.rows * parts * 2 <= 2LL * ctx->sm_count && vectors / (parts * 2) >= 7 * 512) parts *= 2;
    return launch_token_logprobs<512>(ctx, dtype, a, parts);
}

}  // namespace zb
