// Attention of new tokens over the cache of kv_cache.cuh, masks by position: token j is seen from position i where j <= i and, with a window,
// j > i - window or j < sinks.
//
//   x_ij = scale q_i . k_j,   out_i = sum over j of exp(x_ij - m) v_j / sum over j of exp(x_ij - m)
//
// One pass over the codes with a running maximum.  The rows of a tile are (new token, head) pairs that share a key head: 8 NT of them.  Codes become
// f16 on the way (exactly) and both products run on the tensor core with the cache as the A operand, transposed: X^T = K Q^T and O^T = V^T P^T, so that
// 8 rows fill an MMA (16 would be needed the other way round).  How codes lie in a thread is free as long as both operands of a product
// agree: a lane takes 16 bytes of a token as they lie and multiplies them with the same dimensions of q, and V's dimensions are put right when results are stored.  So
// nothing is transposed or moved between lanes but P (movmatrix).
//
// q goes in as f16 times a power of two for each row, so that its largest value lies in [2^14, 2^15): f16 and bf16 values lose nothing down to 2^-28 of that one;
// f32 is the sum of two f16 numbers (SPLIT; 2^-39 of the largest value is lost), and so is P.  P is rounded to f16 (2^-12 relative for results in 16 bits), each weight times
// its page's scale over the largest scale so far, times 2^14, so that what is rounded is at most 2^14 and weights down to 2^-28 keep their 11 bits.  Statistics
// and sums are fp32.
//
// Memory is the bound (a cached token of 128 dimensions is 256 bytes for 4 x 8 x 128 operations of 8 rows).  Each warp takes every so many'th 32 tokens and
// brings them by asynchronous copies of 16 bytes into slots of its own lanes, DEPTH steps ahead: a lane reads what it copied itself, in its own order, so that there is no
// bank conflict and no barrier.  The warps of a CTA, and the CTAs of a cluster that share a tile, join their sums at the end.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "context.cuh"
#include "kv_cache.cuh"
#include "ptx_sm100.cuh"
#include "row_codes.cuh"

namespace zb {

struct KvAttendArgs {
    KvArgs c;
    const void* q; long long q_stride; int heads, group, q_type;       // group: heads that share a key head
    void* out; long long out_stride; float* lse;
    float scale_log2;                                 // scale log2(e)
    int window, sinks;
    bool wide_q;                                      // q in whole 16-byte blocks
    int parts, tiles;                                 // CTAs of a tile; row tiles of the grid
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Codes in bytes 0 and 2 of a word as two f16 numbers: 1024 + 128 + c in the bits, less 1152.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t m = (w & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&m), __floats2half2_rn(1152.0f, 1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float kv_value(const void* p, int type, long long at) {
    if (type == ZANT_F32) return static_cast<const float*>(p)[at];
    if (type == ZANT_F16) return __half2float(static_cast<const __half*>(p)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}
__device__ __forceinline__ void kv_store(void* p, int type, long long at, float v) {
    if (type == ZANT_F32) static_cast<float*>(p)[at] = v;
    else if (type == ZANT_F16) static_cast<__half*>(p)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
}
// 16 values from `at` on.
__device__ __forceinline__ void kv_values16(const void* p, int type, bool wide, long long at, float (&f)[16]) {
    if (wide) {
        if (type == ZANT_F32) {
            const uint4* v = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) { const uint4 b = v[i]; f[4 * i] = __uint_as_float(b.x); f[4 * i + 1] = __uint_as_float(b.y); f[4 * i + 2] = __uint_as_float(b.z); f[4 * i + 3] = __uint_as_float(b.w); }
            return;
        }
        const uint4* v = reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + at);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 b = v[i];
            const uint32_t w[4] = {b.x, b.y, b.z, b.w};
            if (type == ZANT_F16) RowChunk<__half>::values(w, f + 8 * i);
            else RowChunk<__nv_bfloat16>::values(w, f + 8 * i);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = kv_value(p, type, at + i);
}

// The tokens that a tile of rows at positions [low, high] sees, in steps of S tokens: sinks first, then the window (or all).
struct KvSteps {
    int sink, first, total;                           // steps of sinks alone, the first step behind them, all
    __device__ __forceinline__ KvSteps(int low, int high, int window, int sinks, int S) {
        sink = first = 0;
        if (high < 0) { total = 0; return; }
        if (window > 0 && low - window + 1 > 0) {
            first = (low - window + 1) / S;
            sink = min((sinks + S - 1) / S, high / S + 1);
            if (sink >= first) sink = first = 0;
        }
        total = sink + high / S + 1 - first;
    }
    __device__ __forceinline__ int at(int k, int S) const { return (k < sink ? k : k - sink + first) * S; }
};

template <int DP_, int NT_, bool SPLIT_>
struct KvAttendCfg {
    static constexpr int DP = DP_, NT = NT_, ROWS = 8 * NT, WARPS = 4, THREADS = 32 * WARPS, STEP = 32;
    static constexpr bool SPLIT = SPLIT_;
    static constexpr int KS = DP / 16;                // MMA steps of the dimensions
    static constexpr int CH = DP < 128 ? 1 : DP / 128;       // a lane's chunks of a token of V
    static constexpr int VB = DP < 128 ? 8 : 16;      // bytes of each
    static constexpr int MT = DP / 16;                // MMA tiles of the dimensions in O^T
    static constexpr int HALF = STEP * DP, STAGE = 2 * HALF + 32;       // K, V, what the pages say
    static constexpr int DEPTH = DP == 256 ? 3 : (DP == 128 ? 3 : 5);
    static constexpr int QF = KS * NT * (SPLIT ? 2 : 1);     // fragments of q, 8 bytes a lane
    static constexpr bool Q_SHARED = QF > 16;
    static constexpr int PITCH = DP + 4;
    static constexpr int RING = WARPS * DEPTH * STAGE;
    static constexpr int JOIN = WARPS * ROWS * PITCH * 4;
    static constexpr int BIG = RING > JOIN ? RING : JOIN;
    static constexpr int OFF_Q = BIG, OFF_STAT = OFF_Q + (Q_SHARED ? QF * 256 : 0);
    static constexpr int SMEM = OFF_STAT + (WARPS * ROWS * 3 + ROWS * 2) * 4;
};

template <int DP, int NT, bool SPLIT>
__global__ void __launch_bounds__(128) kv_attention_kernel(const __grid_constant__ KvAttendArgs a) {
    using F = KvAttendCfg<DP, NT, SPLIT>;
    constexpr int STEP = F::STEP, D = F::DEPTH, KS = F::KS;
    extern __shared__ __align__(128) uint8_t smem[];
    const KvArgs& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l4 = lane >> 2, c4 = lane & 3, P = a.parts;
    const int rank = P > 1 ? (int)ptx::cluster_rank() : 0;
    ptx::grid_start();
    const int work = (int)(blockIdx.x / (unsigned)P), h = work % c.heads;
    KvSeq q; int unit;
    bool any = kv_locate(c, work / c.heads, a.group, F::ROWS, 1, q, unit);
    const int row0 = unit * F::ROWS, rows = any ? min(F::ROWS, q.n * a.group - row0) : 0;
    if (rows <= 0) return;                            // (all CTAs of a cluster)
    const int low = max(q.first + row0 / a.group, -1), high = max(q.first + (row0 + rows - 1) / a.group, -1);      // (below zero: nothing is seen)
    const KvSteps steps(low, high, a.window, a.sinks, STEP);
    const int stride_k = P * F::WARPS, k0 = rank * F::WARPS + warp;

    const uint32_t ring = ptx::smem_u32(smem) + warp * D * F::STAGE;
    uint8_t* ring_p = smem + warp * D * F::STAGE;
    const int pl = c.page_log2, inpage = c.page - 1;
    // pages of both halves of step k (-1: none)
    auto pages_of = [&](int k, long long (&id)[2]) {
        id[0] = id[1] = -1;
        if (k >= steps.total) return;
        const int t = steps.at(k, STEP);
        id[0] = kv_page(c, q.s, t >> pl);
        id[1] = pl == 4 ? kv_page(c, q.s, (t >> pl) + 1) : id[0];
    };
    auto issue = [&](int k, int stage, const long long (&id)[2]) {
        if (k < steps.total) {
            const int t = steps.at(k, STEP);
            const uint32_t dst = ring + stage * F::STAGE + lane * 16;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const bool ok = id[half] >= 0;
                const long long block = (ok ? id[half] : 0) * c.heads + h, off = (block * c.page + ((t + 16 * half) & inpage)) * c.dim;
                const int8_t* pk = c.k + off;
                const int8_t* pv = c.v + off;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < DP / 64; ++j) {
                        const int d = (c4 + 4 * j) * 16;
                        const bool in = ok && d < c.dim;
                        cp_async16(dst + ((half * 2 + b) * (DP / 64) + j) * 512, pk + (in ? (8 * b + l4) * c.dim + d : 0), in);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < F::CH; ++j) {
                        const int tok = (i & 2) * 4 + 2 * c4 + (i & 1), d = l4 * F::VB + 128 * j;
                        const bool in = ok && d < c.dim;
                        if (F::VB == 16) cp_async16(dst + F::HALF + ((half * 4 + i) * F::CH + j) * 512, pv + (in ? tok * c.dim + d : 0), in);
                        else cp_async8(dst - lane * 8 + F::HALF + (half * 4 + i) * 256, pv + (in ? tok * c.dim + d : 0), in);
                    }
                if (lane == half) {
                    cp_async4(ring + stage * F::STAGE + 2 * F::HALF + 8 * half, c.k_scale + block, ok);
                    cp_async4(ring + stage * F::STAGE + 2 * F::HALF + 8 * half + 4, c.v_scale + block, ok);
                    *reinterpret_cast<int*>(ring_p + stage * F::STAGE + 2 * F::HALF + 16 + 4 * half) = ok;
                }
            }
        }
        cp_async_commit();
    };
    long long id[2];
    for (int s = 0; s < D - 1; ++s) { pages_of(k0 + s * stride_k, id); issue(k0 + s * stride_k, s, id); }
    pages_of(k0 + (D - 1) * stride_k, id);

    // q: lane's columns of B are row l4 of each 8, dimensions as its chunks of K have them; its columns of X^T are rows 2 c4 and 2 c4 + 1
    uint2 qf[F::Q_SHARED ? 1 : F::QF];
    uint2* qs = reinterpret_cast<uint2*>(smem + F::OFF_Q);
    float factor[NT][2];
    int seen_to[NT][2];                               // positions of the lane's two rows
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + 8 * n + l4;
        const bool there = 8 * n + l4 < rows;
        const long long at = (long long)(q.row + (there ? r / a.group : 0)) * a.q_stride + (long long)(h * a.group + (there ? r % a.group : 0)) * c.dim;
        float v[DP / 64][16];
        float top = 0.0f;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            const int d = (c4 + 4 * j) * 16;
            if (there && d < c.dim) kv_values16(a.q, a.q_type, a.wide_q, at + d, v[j]);
            else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[j][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) { top = fmaxf(top, fabsf(v[j][i])); odd |= !(fabsf(v[j][i]) < INFINITY); }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        odd = (__ballot_sync(0xffffffffu, odd) >> (lane & 28)) & 15;
        // 2^-e with top 2^-e in [2^14, 2^15); of numbers below 2^-100 what fits
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -114), 127);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = odd ? __uint_as_float(0x7fffffffu) : __uint_as_float((uint32_t)max(127 + e, 1) << 23);
#pragma unroll
        for (int j = 0; j < DP / 64; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[4], y[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) { x[z] = odd ? 0.0f : v[j][4 * i + z] * down; y[z] = x[z] - __half2float(__float2half_rn(x[z])); }
                const uint2 hi = make_uint2(pack_f16(x[0], x[2]), pack_f16(x[1], x[3])), lo = make_uint2(pack_f16(y[0], y[2]), pack_f16(y[1], y[3]));
                const int f = (j * 4 + i) * NT + n;
                if (F::Q_SHARED) {
                    if (warp == 0) { qs[f * 32 + lane] = hi; if (SPLIT) qs[(KS * NT + f) * 32 + lane] = lo; }
                } else {
                    qf[f] = hi;
                    if (SPLIT) qf[KS * NT + f] = lo;
                }
            }
        const float fac = up * a.scale_log2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            factor[n][i] = __shfl_sync(0xffffffffu, fac, (2 * c4 + i) * 4);
            const int row = row0 + min(8 * n + 2 * c4 + i, rows - 1);
            seen_to[n][i] = max(q.first + row / a.group, -1);
        }
    }
    if (F::Q_SHARED) __syncthreads();
    auto q_at = [&](int f) -> uint2 { return F::Q_SHARED ? qs[f * 32 + lane] : qf[F::Q_SHARED ? 0 : f]; };

    float o[F::MT][NT][4];
    float m[NT][2], l[NT][2], vs = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < F::MT; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
    }

    int stage = 0, ahead = D - 1;
    for (int k = k0; k < steps.total; k += stride_k) {
        __syncwarp();                                 // the warp has read the stage that is filled now
        issue(k + (D - 1) * stride_k, ahead, id);
        pages_of(k + D * stride_k, id);
        cp_async_wait<D - 1>();
        __syncwarp();
        const uint8_t* st = ring_p + stage * F::STAGE;
        const float* scales = reinterpret_cast<const float*>(st + 2 * F::HALF);
        const int* ok = reinterpret_cast<const int*>(st + 2 * F::HALF + 16);
        const int t = steps.at(k, STEP);
        // scores of 32 tokens
        float x[2][NT][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) x[half][n][0] = x[half][n][1] = x[half][n][2] = x[half][n][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) {
                const uint4 lo = *reinterpret_cast<const uint4*>(st + ((half * 2) * (DP / 64) + j) * 512 + lane * 16);
                const uint4 hi = *reinterpret_cast<const uint4*>(st + ((half * 2 + 1) * (DP / 64) + j) * 512 + lane * 16);
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t frag[4] = {codes_f16(wl[i]), codes_f16(wh[i]), codes_f16(wl[i] >> 8), codes_f16(wh[i] >> 8)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint2 b = q_at((j * 4 + i) * NT + n);
                        mma_f16(x[half][n], frag, b.x, b.y);
                        if (SPLIT) { const uint2 d = q_at((KS + j * 4 + i) * NT + n); mma_f16(x[half][n], frag, d.x, d.y); }
                    }
                }
            }
        }
        const float ks[2] = {scales[0], scales[2]}, vsc[2] = {scales[1], scales[3]};
        const bool all = ok[0] && ok[1] && t + STEP - 1 <= low && (a.window == 0 || t > high - a.window || t + STEP <= a.sinks);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[half][n][i] *= factor[n][i & 1] * ks[half];
        if (!all) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = t + half * 16 + (i >> 1) * 8 + l4, p = seen_to[n][i & 1];
                        const bool seen = ok[half] && j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
                        if (!seen) x[half][n][i] = -INFINITY;
                    }
        }
        // the running maximum of each row, and the largest scale of V
        float to[NT][2];
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = fmaxf(fmaxf(x[0][n][i], x[0][n][i + 2]), fmaxf(x[1][n][i], x[1][n][i + 2]));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                to[n][i] = fmaxf(m[n][i], v);
                raise |= to[n][i] > m[n][i];
            }
        const float vs_to = fmaxf(vs, fmaxf(fabsf(vsc[0]), fabsf(vsc[1])));
        if (__any_sync(0xffffffffu, raise || vs_to > vs)) {
            const float fv = vs_to > 0.0f ? vs / vs_to : 1.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = m[n][i] == to[n][i] ? 1.0f : ex2(m[n][i] - to[n][i]);
                    l[n][i] *= f;
                    m[n][i] = to[n][i];
#pragma unroll
                    for (int j = 0; j < F::MT; ++j) { o[j][n][i] *= f * fv; o[j][n][i + 2] *= f * fv; }
                }
            vs = vs_to;
        }
        const float over = vs > 0.0f ? 16384.0f / vs : 0.0f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float vf = vsc[half] * over;
            uint32_t b[NT][2], d[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = ex2(x[half][n][i] - (m[n][i & 1] == -INFINITY ? 0.0f : m[n][i & 1]));
                    l[n][i & 1] += e;
                    p[i] = e == 0.0f ? 0.0f : e * vf;
                }
                b[n][0] = pack_f16(p[0], p[1]);
                b[n][1] = pack_f16(p[2], p[3]);
                if (SPLIT) {
                    float r[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[i] = p[i] - __half2float(__float2half_rn(p[i]));
                    d[n][0] = transpose8x8(pack_f16(r[0], r[1]));
                    d[n][1] = transpose8x8(pack_f16(r[2], r[3]));
                }
                b[n][0] = transpose8x8(b[n][0]);
                b[n][1] = transpose8x8(b[n][1]);
            }
#pragma unroll
            for (int j = 0; j < F::CH; ++j) {
                uint32_t w[4][F::VB / 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (F::VB == 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(st + F::HALF + ((half * 4 + i) * F::CH + j) * 512 + lane * 16);
                        w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(st + F::HALF + (half * 4 + i) * 256 + lane * 8);
                        w[i][0] = v.x; w[i][1] = v.y;
                    }
                }
#pragma unroll
                for (int z = 0; z < F::VB / 2; ++z) {
                    const int word = z >> 1, byte = (z & 1) * 2;
                    // a byte of two tokens' words, in bytes 0 and 2
                    auto two = [&](int i, int at) { return codes_f16(__byte_perm(w[i][word], w[i + 1][word], (uint32_t)(at | ((4 + at) << 8)))); };
                    const uint32_t frag[4] = {two(0, byte), two(0, byte + 1), two(2, byte), two(2, byte + 1)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_f16(o[j * 8 + z][n], frag, b[n][0], b[n][1]);
                        if (SPLIT) mma_f16(o[j * 8 + z][n], frag, d[n][0], d[n][1]);
                    }
                }
            }
        }
        stage = stage + 1 == D ? 0 : stage + 1;
        ahead = ahead + 1 == D ? 0 : ahead + 1;
    }
    cp_async_wait<0>();
    __syncthreads();                                  // the ring becomes the place of the warps' sums

    float* sums = reinterpret_cast<float*>(smem);     // [warp][row][dimension]
    float* stat = reinterpret_cast<float*>(smem + F::OFF_STAT);       // [warp][row]: m, l, scale
    float* joined = stat + 3 * F::WARPS * F::ROWS;    // [row]: m, l of the CTA
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 8 * n + 2 * c4 + i;
            float v = l[n][i];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (l4 == 0) {
                float* s = stat + (warp * F::ROWS + r) * 3;
                s[0] = m[n][i]; s[1] = v; s[2] = vs * (1.0f / 16384.0f);
            }
            float* to = sums + (warp * F::ROWS + r) * F::PITCH;
#pragma unroll
            for (int j = 0; j < F::MT; ++j) {
                const int d = (j / 8) * 128 + l4 * F::VB + 2 * (j % 8);
                to[d] = o[j][n][i];
                to[d + 1] = o[j][n][i + 2];
            }
        }
    __syncthreads();
    for (int r = warp; r < F::ROWS; r += F::WARPS) {
        float top = -INFINITY, total = 0.0f, f[F::WARPS];
#pragma unroll
        for (int w = 0; w < F::WARPS; ++w) top = fmaxf(top, stat[(w * F::ROWS + r) * 3]);
#pragma unroll
        for (int w = 0; w < F::WARPS; ++w) {
            const float* s = stat + (w * F::ROWS + r) * 3;
            const float e = s[0] == -INFINITY ? 0.0f : ex2(s[0] - top);
            total += s[0] == -INFINITY && s[1] == 0.0f ? 0.0f : s[1] * (s[0] == -INFINITY ? 1.0f : e);
            f[w] = e * s[2];
        }
        for (int d = lane; d < DP; d += 32) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < F::WARPS; ++w) {
                const float part = sums[(w * F::ROWS + r) * F::PITCH + d];
                v += part == 0.0f ? 0.0f : part * f[w];
            }
            sums[r * F::PITCH + d] = v;               // (only this warp reads row r of any warp)
        }
        if (lane == 0) { joined[2 * r] = top; joined[2 * r + 1] = total; }
    }
    if (P > 1) {
        __syncwarp();
        ptx::cluster_arrive();
        ptx::cluster_wait();
    } else __syncthreads();
    const uint32_t peer_sums = ptx::smem_u32(sums), peer_joined = ptx::smem_u32(joined);
    auto peer = [&](uint32_t addr, int r) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::cluster_addr(addr, (uint32_t)r)) : "memory");
        return v;
    };
    // each CTA of the cluster finishes every so many'th row
    for (int r = rank + P * warp; r < rows; r += P * F::WARPS) {
        float top = -INFINITY, total = 0.0f, f = 0.0f;
        float mine_m = -INFINITY, mine_l = 0.0f;
        if (P > 1) {
            if (lane < P) { mine_m = peer(peer_joined + 8 * r, lane); mine_l = peer(peer_joined + 8 * r + 4, lane); }
        } else if (lane == 0) { mine_m = joined[2 * r]; mine_l = joined[2 * r + 1]; }
        top = mine_m;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        f = mine_m == -INFINITY ? (mine_l == 0.0f ? 0.0f : 1.0f) : ex2(mine_m - top);
        total = mine_l == 0.0f ? 0.0f : mine_l * f;
#pragma unroll
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int row = row0 + r;
        const long long at = (long long)(q.row + row / a.group) * a.out_stride + (long long)(h * a.group + row % a.group) * c.dim;
        for (int d0 = 0; d0 < c.dim; d0 += 32) {      // (whole warps: the parts' factors come by shuffles)
            const int d = d0 + lane;
            float v = 0.0f;
            for (int p = 0; p < P; ++p) {
                const float fp = __shfl_sync(0xffffffffu, f, p);
                const float part = d < c.dim ? (P > 1 ? peer(peer_sums + 4 * (r * F::PITCH + d), p) : sums[r * F::PITCH + d]) : 0.0f;
                v += part == 0.0f ? 0.0f : part * fp;
            }
            if (total != total) v = total;
            if (d < c.dim) kv_store(a.out, a.q_type, at + d, v * inv);
        }
        if (a.lse && lane == 0) a.lse[(long long)(q.row + row / a.group) * a.heads + h * a.group + row % a.group] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
    }
    if (P > 1) {
        __syncwarp();
        ptx::cluster_arrive();
        ptx::cluster_wait();                          // nobody leaves while its sums are read
    }
}

template <int DP, int NT, bool SPLIT>
inline int32_t launch_kv_attention(zant_ctx* ctx, KvAttendArgs a) {
    using F = KvAttendCfg<DP, NT, SPLIT>;
    const long long tiles = kv_units(a.c, a.group, F::ROWS, 1), items = tiles * a.c.heads;
    if (items > 0x7fffffffLL / 16) return fail(ZANT_E_TOO_LARGE, "%lld tiles of attention", items);
    // CTAs that share a tile: while they find room side by side and each warp has steps left to take
    const long long reach = std::min((long long)a.c.width << a.c.page_log2, a.window > 0 ? (long long)a.window + a.sinks + 2 * F::STEP : 0x7fffffffffLL);
    int parts = 1;
    while (parts < 16 && items * parts * 2 <= 2LL * ctx->sm_count && reach >= (long long)parts * 2 * F::WARPS * F::STEP) parts *= 2;
    a.parts = parts; a.tiles = (int)tiles;
    auto kernel = kv_attention_kernel<DP, NT, SPLIT>;
    ZB_SMEM_ATTR(ctx, kernel, F::SMEM);
    static std::atomic<unsigned long long> wide{0ull};
    const unsigned long long bit = 1ull << (ctx->device & 63);
    if (parts > 8 && !(wide.load(std::memory_order_acquire) & bit)) {
        ZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        wide.fetch_or(bit, std::memory_order_release);
    }
    launch_cluster(ctx, kernel, dim3((unsigned)(items * parts)), F::THREADS, F::SMEM, (unsigned)parts, a);
    return check_launch(ctx, "kv_attention_kernel");
}

template <int DP, bool SPLIT>
inline int32_t choose_kv_attention(zant_ctx* ctx, const KvAttendArgs& a) {
    const long long rows = ((long long)a.c.rows + a.c.seqs - 1) / a.c.seqs * a.group;
    if (rows <= 8) return launch_kv_attention<DP, 1, SPLIT>(ctx, a);
    if constexpr (DP <= 128 && !SPLIT)
        if (rows > 16) return launch_kv_attention<DP, 4, SPLIT>(ctx, a);
    return launch_kv_attention<DP, 2, SPLIT>(ctx, a);
}

inline int32_t run_kv_attention(zant_ctx* ctx, const KvAttendArgs& a) {
    const bool split = a.q_type == ZANT_F32;
    if (a.c.dim <= 64) return split ? choose_kv_attention<64, true>(ctx, a) : choose_kv_attention<64, false>(ctx, a);
    if (a.c.dim <= 128) return split ? choose_kv_attention<128, true>(ctx, a) : choose_kv_attention<128, false>(ctx, a);
    return split ? choose_kv_attention<256, true>(ctx, a) : choose_kv_attention<256, false>(ctx, a);
}

}  // namespace zb
