// Attention of new tokens over the cache of kv_cache.cuh, masks by position: token j is seen from position i where j <= i and, with a window,
// j > i - window or j < sinks.
//
//   x_ij = scale q_i . k_j,   out_i = sum over j of exp(x_ij - m) v_j / sum over j of exp(x_ij - m)
//
// One pass over the codes with a running maximum.  The rows of a tile are (new token, head) pairs that share a key head: 8 NT of them.  Both products run on
// the tensor core with the cache as the A operand, transposed: X^T = K Q^T and O^T = V^T P^T, so that 8 rows fill an MMA (16 would be needed the other way round).  How codes lie in
// a thread is free as long as both operands of a product agree: a lane takes 16 bytes of a token as they lie and multiplies them with the same dimensions of q, and
// V's dimensions are put right when results are stored.  So nothing is transposed or moved between lanes but P (movmatrix).
//
// K stays int8: q goes in as whole numbers whose largest in a row is about 2^20 (of F32 2^27), in 3 (4) digits of 7 bits, whose products are int8 products with exact
// sums; a value of q loses 2^-20 of the largest of its row at most (2^-27).  K in f16 took 96 more ALU instructions of 510 for a step, and ALU is the busiest pipe.
// V becomes f16 on the way (exactly) and P is rounded to f16 (2^-11 relative, for results in 16 bits; of F32 the sum of two f16 numbers): each weight times its page's scale, over the largest such
// product M of its row, times 2^9 to 2^15 (M is raised when it has grown by 2^6), so that 2^-23 of a row's largest keeps its 11 bits whatever the scales of pages are that only other rows see.  Statistics and
// sums are fp32; scales below 2^-104 keep fewer bits.
//
// Memory is the bound (a cached token of 128 dimensions is 256 bytes for 4 x 8 x 128 operations of 8 rows).  Each warp takes every so many'th step of 32 tokens (16 of
// 256 dimensions), which its first lane brings by TMA into a ring of the warp's own, swizzled so that the lanes' 16-byte reads meet no bank twice.  No warp waits for
// another until the end, when the warps of a CTA, and the CTAs of a cluster that share a tile, join their sums.  64 x 1 tokens of 40 over 8 heads of 128, 4096 each: 113 us (4.8 TB/s), 760
// instructions a step of 32 tokens at 2.1 a clock; 5 tokens of 16 over 4 heads of 64 in windows of 1024, 24 sequences: 18.2 us with tiles of 24 rows (20.5 with 32, when the former took 17.6).
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "context.cuh"
#include "kv_cache.cuh"
#include "ptx_sm100.cuh"
#include "row_codes.cuh"
#include "tensor_map.cuh"

namespace zb {

struct KvAttendArgs {
    KvArgs c;
    const void* q; long long q_stride; int heads, group, q_type;       // group: heads that share a key head
    void* out; long long out_stride; float* lse;
    float scale_log2;                                 // scale log2(e)
    int window, sinks;
    bool wide_q, wide_out;                            // q, out in whole 16-byte blocks (out: prompts)
    int more_rows_than, rows_up_to;                   // sequences with more rows of a key head than the first, up to the second, are the kernel's
    int parts, tiles_each;                            // CTAs of a tile; tiles of each sequence (0: by its rows)
    bool by_length;                                   // the longest sequences first (as many as a CTA has threads at most)
    float* work; size_t work_bytes;                   // a workspace, if there is one: a tile's CTAs leave their sums there, and need not be a cluster
    int* status; long long wait_budget; int give_up;  // give_up: self test, a CTA whose first wait counts as run out (-1: none)
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// int8 products, 16 x 8 x 32.
__device__ __forceinline__ void mma_i8_16x8(int (&d)[4], const uint32_t (&a)[4], uint2 b, bool first) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(first ? 0 : d[0]), "r"(first ? 0 : d[1]), "r"(first ? 0 : d[2]), "r"(first ? 0 : d[3]));
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

// A page's scale; one that is no finite number is NaN.
__device__ __forceinline__ float kv_scale(float s) { return fabsf(s) < INFINITY ? s : __uint_as_float(0x7fffffffu); }

// The tokens that a tile of rows at positions [low, high] sees, in steps of S tokens: sinks first, then the window (or all).
struct KvSteps {
    int sink, first, total;                           // steps of sinks alone, the first step behind them, all
    __device__ __forceinline__ KvSteps(int low, int high, int window, int sinks, int S) {
        sink = first = 0;
        if (high < 0) { total = 0; return; }
        if (window > 0 && low - window + 1 > 0) {
            first = (low - window + 1) / S;
            sink = min(sinks / S + (sinks % S != 0), high / S + 1);      // (sinks up to the end of int)
            if (sink >= first) sink = first = 0;
        }
        total = sink + high / S + 1 - first;
    }
    __device__ __forceinline__ int at(int k, int S) const { return (k < sink ? k : k - sink + first) * S; }
};
// The rows of a key head that the kernel has to do with in a sequence of n new tokens: all, or none where they are another kernel's.
__device__ __forceinline__ int kv_rows_of(const KvAttendArgs& a, int n) {
    const int rows = n * a.group;
    return rows > a.more_rows_than && rows <= a.rows_up_to ? rows : 0;
}
// Some row at positions [low, high] sees one of the 16 tokens from t on.  (What the table says of others, and their pages' scales, is nobody's business.)
__device__ __forceinline__ bool kv_seen16(int t, int low, int high, int window, int sinks) { return t <= high && (window == 0 || t + 15 > low - window || t < sinks); }

// The maximum of a row that has seen nothing: a number, so that differences are numbers, and below all scores.
constexpr float kKvNothing = -1e30f;

template <int DP_, int NT_, bool SPLIT_>
struct KvAttendCfg {
    static constexpr int DP = DP_, NT = NT_, ROWS = 8 * NT, STEP = DP == 256 ? 16 : 32, HALVES = STEP / 16;
    static constexpr bool SPLIT = SPLIT_;
    static constexpr int MT = DP / 16, KS = DP / 32;  // MMA tiles of the dimensions in O^T, MMA steps of them in X^T
    static constexpr int DIGITS = SPLIT ? 4 : 3;      // of q
    static constexpr int BOX = DP < 128 ? DP : 128, BOXES = DP / BOX;       // bytes of a token in a box
    static constexpr int VB = DP < 128 ? 8 : 16;      // bytes of V that a lane takes of each
    static constexpr int HALF = STEP * DP, STAGE = 2 * HALF;       // K, V
    static constexpr int DEPTH = DP == 64 ? 4 : 2;
    // Warps of an SM: what the ring leaves and registers allow, as CTAs of 4 or as one.
    static constexpr int MOST_WARPS = NT == 1 && DP < 256 ? 12 : 8;
    static constexpr int QF = KS * NT * DIGITS;       // fragments of q, 8 bytes a lane
    static constexpr bool Q_SHARED = QF > 16;
    static constexpr int PITCH = DP + 4;
    static constexpr int Q_BYTES = QF * 256;
    static __host__ __device__ constexpr int big(int warps) {
        const int ring = warps * DEPTH * STAGE, join = warps * ROWS * PITCH * 4;
        return ring > join ? ring : join;
    }
    // ring or sums, q, statistics of warps and of the CTA, factors of rows, barriers, flag
    static __host__ __device__ constexpr int smem(int warps) { return big(warps) + Q_BYTES + (warps * ROWS * 3 + ROWS * 3) * 4 + warps * DEPTH * 8 + 16; }
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
// A part's sum and the factor that brings it to the common maximum: parts that saw nothing add nothing, NaN stays NaN.
__device__ __forceinline__ float join_factor(float m, float l, float top) { return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2(m - top); }
__device__ __forceinline__ float times(float v, float f) { return v == 0.0f ? 0.0f : v * f; }

template <int DP, int NT, bool SPLIT>
__global__ void __launch_bounds__(32 * KvAttendCfg<DP, NT, SPLIT>::MOST_WARPS, 1)
kv_attention_kernel(const __grid_constant__ KvAttendArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using F = KvAttendCfg<DP, NT, SPLIT>;
    constexpr int STEP = F::STEP, H = F::HALVES, D = F::DEPTH, MT = F::MT, DIG = F::DIGITS;
    extern __shared__ __align__(1024) uint8_t smem[];
    const KvArgs& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l4 = lane >> 2, c4 = lane & 3, P = a.parts, W = blockDim.x >> 5;
    const int rank = a.work ? (int)(blockIdx.x % (unsigned)P) : (P > 1 ? (int)ptx::cluster_rank() : 0);
    uint2* qs = reinterpret_cast<uint2*>(smem + F::big(W));
    float* stat = reinterpret_cast<float*>(smem + F::big(W) + F::Q_BYTES);       // [warp][row]: m, l, scale
    float* joined = stat + 3 * W * F::ROWS;           // [row]: m, l of the CTA
    float* row_factor = joined + 2 * F::ROWS;
    uint8_t* tail = reinterpret_cast<uint8_t*>(row_factor + F::ROWS);
    const uint32_t full = ptx::smem_u32(tail) + warp * D * 8;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + W * D * 8);
    if (lane == 0) {
        for (int i = 0; i < D; ++i) ptx::mbar_init(full + 8 * i, 1);
        ptx::mbar_fence_init();
    }
    if (threadIdx.x == 0) *abort_flag = (int)blockIdx.x == a.give_up ? 1 : 0;       // (told at the end, also by a CTA without a step to wait for)
    __syncthreads();
    ptx::grid_start();
    const int work = (int)(blockIdx.x / (unsigned)P), h = work % c.heads;
    KvSeq q; int unit;
    bool any;
    if (a.tiles_each > 0) {
        unit = work / c.heads % a.tiles_each;
        q = kv_seq(c, min(work / c.heads / a.tiles_each, c.seqs - 1));
        any = q.n > 0;
    } else if (a.by_length) {
        // the sequence whose length has the wanted place among all.  (They lie where q's digits come later: the ring is written by TMA alone until its copies have landed, plain stores there would
        // need a fence of proxies in front of the first copy.)
        static_assert(F::Q_BYTES >= (32 * 4 + 1) * 4, "lengths of 128 sequences and a place");
        int* lengths = reinterpret_cast<int*>(qs);
        const int tid = threadIdx.x, each = (int)(((long long)c.per * a.group + F::ROWS - 1) / F::ROWS), want = work / c.heads / each;
        const int mine = tid < c.seqs ? c.lengths[tid] : 0;
        if (tid < c.seqs) lengths[tid] = mine;
        __syncthreads();
        int place = 0;
        for (int i = 0; i < c.seqs; ++i) place += lengths[i] > mine || (lengths[i] == mine && i < tid);
        if (tid < c.seqs && place == want) lengths[128] = tid;
        __syncthreads();
        const int s = lengths[128];
        __syncthreads();                              // (q's digits are written from here on)
        unit = work / c.heads % each;
        q = kv_seq(c, s);
        any = true;
    } else any = kv_locate(c, work / c.heads, a.group, F::ROWS, 1, q, unit);
    const int row0 = unit * F::ROWS, rows = any ? min(F::ROWS, kv_rows_of(a, q.n) - row0) : 0;
    if (rows <= 0) {                                  // (all CTAs of a cluster)
        if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, (int)DEV_ERR_WAIT_TIMEOUT);
        return;
    }
    const int low = max(q.first + row0 / a.group, -1), high = max(q.first + (row0 + rows - 1) / a.group, -1);      // (below zero: nothing is seen)
    const KvSteps steps(low, high, a.window, a.sinks, STEP);
    const int stride_k = P * W, k0 = rank * W + warp;

    const uint8_t* ring = smem + warp * D * F::STAGE;
    const int pl = c.page_log2, inpage = c.page - 1;
    const bool two = H == 2 && pl == 4;               // a step is on two pages
    // What the table and the scales say of 32 of the warp's steps, one a lane: pages of the step's 16 tokens each (-1: none) and their scales.
    struct Batch {
        int page[H]; float k[H], v[H];
        unsigned there[H];                            // lanes with a page
    };
    auto batch_of = [&](int i) {
        Batch b;
        const int k = k0 + (i + lane) * stride_k, t = k < steps.total ? steps.at(k, STEP) : -1;
#pragma unroll
        for (int z = 0; z < H; ++z) {
            b.page[z] = z == 0 || two ? (int)kv_page(c, q.s, t < 0 || (two && !kv_seen16(t + 16 * z, low, high, a.window, a.sinks)) ? -1 : (t >> pl) + z) : b.page[0];
            b.there[z] = __ballot_sync(0xffffffffu, b.page[z] >= 0);
            const long long at = (long long)max(b.page[z], 0) * c.heads + h;
            b.k[z] = z == 0 || two ? (b.page[z] >= 0 ? c.k_scale[at] : 0.0f) : b.k[0];
            b.v[z] = z == 0 || two ? (b.page[z] >= 0 ? c.v_scale[at] : 0.0f) : b.v[0];
        }
        return b;
    };
    // (when they are needed: as they come they would be waited for)
    auto settle = [&](Batch& b) {
#pragma unroll
        for (int z = 0; z < H; ++z) { b.k[z] = kv_scale(b.k[z]); b.v[z] = kv_scale(b.v[z]); }
    };
    Batch cur = batch_of(0), nxt;
    // Step i of the warp goes into the ring, by its first lane.
    auto issue = [&](int i, int stage, const Batch& b) {
        int page[H];
        page[0] = __shfl_sync(0xffffffffu, b.page[0], i & 31);
        if (H > 1) page[H - 1] = two ? __shfl_sync(0xffffffffu, b.page[H - 1], i & 31) : page[0];
        const int k = k0 + i * stride_k;
        if (lane != 0 || k >= steps.total) return;
        const uint32_t dst = ptx::smem_u32(ring) + stage * F::STAGE, bar = full + 8 * stage;
        if (!two) {                                   // one page: boxes of STEP tokens
            ptx::mbar_arrive_expect_tx(bar, page[0] >= 0 ? F::STAGE : 0);
            if (page[0] >= 0) {
                const int t = steps.at(k, STEP) & inpage, block = page[0] * c.heads + h;
#pragma unroll
                for (int z = 0; z < F::BOXES; ++z) {
                    ptx::tma_load_3d(dst + z * STEP * F::BOX, &k_map, z * F::BOX, t, block, bar);
                    ptx::tma_load_3d(dst + F::HALF + z * STEP * F::BOX, &v_map, z * F::BOX, t, block, bar);
                }
            }
        } else {
            ptx::mbar_arrive_expect_tx(bar, (page[0] >= 0 ? F::STAGE / 2 : 0) + (page[H - 1] >= 0 ? F::STAGE / 2 : 0));
#pragma unroll
            for (int z = 0; z < H; ++z)
                if (page[z] >= 0) {
                    ptx::tma_load_3d(dst + z * 16 * F::BOX, &k_map, 0, 0, page[z] * c.heads + h, bar);
                    ptx::tma_load_3d(dst + F::HALF + z * 16 * F::BOX, &v_map, 0, 0, page[z] * c.heads + h, bar);
                }
        }
    };
#pragma unroll
    for (int i = 0; i < D - 1; ++i) issue(i, i, cur);

    // q: lane's columns of B are row l4 of each 8, dimensions as its chunks of K have them; its columns of X^T are rows 2 c4 and 2 c4 + 1
    // (Warp n turns 8 rows into digits, for all: each warp for itself took as many instructions as two steps.)
    constexpr int BITS = 7 * DIG - 1;                 // the largest value of a row in [2^(BITS - 1), 2^BITS)
    auto dim_of = [&](int j) { return DP == 64 ? c4 * 16 : (j >> 1) * 128 + (2 * c4 + (j & 1)) * 16; };
    if (warp < NT) {
        const int n = warp, r = row0 + 8 * n + l4;
        const bool there = 8 * n + l4 < rows;
        const long long at = (long long)(q.row + (there ? r / a.group : 0)) * a.q_stride + (long long)(h * a.group + (there ? r % a.group : 0)) * c.dim;
        float v[DP / 64][16];
        float top = 0.0f;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            const int d = dim_of(j);
            if (there && d < c.dim) kv_values16(a.q, a.q_type, a.wide_q, at + d, v[j]);
            else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[j][i] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < DP / 64; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) { top = fmaxf(top, fabsf(v[j][i])); odd |= !(fabsf(v[j][i]) < INFINITY); }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        odd = (__ballot_sync(0xffffffffu, odd) >> (lane & 28)) & 15;
        // 2^-e, clamped where it would leave the normal numbers (values below 2^-98 keep fewer bits)
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127 - (BITS - 1), -125), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = odd ? __uint_as_float(0x7fffffffu) : __uint_as_float((uint32_t)(127 + e) << 23);
        if (c4 == 0) row_factor[8 * n + l4] = up * a.scale_log2;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {             // 8 values: a fragment of 4 and 4
                uint32_t digit[DIG][2] = {};
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    int x = odd ? 0 : __float2int_rn(v[j][8 * i + z] * down);
#pragma unroll
                    for (int g = 0; g < DIG; ++g) {   // digits from -64 to 63, the last one what is left (64 at most)
                        const int lowest = g == DIG - 1 ? x : ((x + 64) & 127) - 64;
                        digit[g][z >> 2] |= (uint32_t)(lowest & 255) << (8 * (z & 3));
                        x = (x - lowest) >> 7;
                    }
                }
#pragma unroll
                for (int g = 0; g < DIG; ++g) qs[(((j * 2 + i) * NT + n) * DIG + g) * 32 + lane] = make_uint2(digit[g][0], digit[g][1]);
            }
    }
    __syncthreads();
    uint2 qf[F::Q_SHARED ? 1 : F::QF];
    if (!F::Q_SHARED) {
#pragma unroll
        for (int f = 0; f < F::QF; ++f) qf[F::Q_SHARED ? 0 : f] = qs[f * 32 + lane];
    }
    auto q_at = [&](int f) -> uint2 { return F::Q_SHARED ? qs[f * 32 + lane] : qf[F::Q_SHARED ? 0 : f]; };
    float factor[NT][2];
    int seen_to[NT][2];                               // positions of the lane's two rows
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            factor[n][i] = row_factor[8 * n + 2 * c4 + i];
            seen_to[n][i] = max(q.first + (row0 + min(8 * n + 2 * c4 + i, rows - 1)) / a.group, -1);
        }

    float o[MT][NT][4];
    // A row's M is its largest x + log2(scale of V), as of when that had last grown by 2^6, and o the sum of 2^(x - M + 9) times the scale times codes: in factors 2^(x - m), which l sums, and the scale times
    // `up`, 2^(9 + m - M).  m is the largest x of that time; it only keeps the factors in range.
    float m[NT][2], M[NT][2], l[NT][2], up_top = 0.0f, up_low = INFINITY;       // (the largest and the least up of the lane's rows)
    // (of 32 rows taken anew each time, for the registers' sake)
    constexpr bool KEEP_UP = NT < 4;
    float kept[KEEP_UP ? NT : 1][2];
    auto up_of = [&](int n, int i) { return KEEP_UP ? kept[KEEP_UP ? n : 0][i] : ex2(9.0f + m[n][i] - M[n][i]); };
    auto set_up = [&](int n, int i) {
        const float up = ex2(9.0f + m[n][i] - M[n][i]);
        if (KEEP_UP) kept[KEEP_UP ? n : 0][i] = up;
        up_top = fmaxf(up_top, up);
        up_low = fminf(up_low, up);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = M[n][0] = M[n][1] = kKvNothing;
        l[n][0] = l[n][1] = 0.0f;
        if (KEEP_UP) kept[KEEP_UP ? n : 0][0] = kept[KEEP_UP ? n : 0][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < MT; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
    }

    // the lane's 16 bytes of token l4 (of 8), dimensions dim_of(j); and of V's token 2 c4 (+ 1)
    auto k_at = [&](const uint8_t* st, int group8, int j) {
        if (DP == 64) return st + (group8 * 8 + l4) * 64 + ((c4 ^ (l4 >> 1)) << 4);
        return st + (j >> 1) * STEP * 128 + (group8 * 8 + l4) * 128 + (((2 * c4 + (j & 1)) ^ l4) << 4);
    };
    auto v_at = [&](const uint8_t* st, int group8, int odd_token, int box) {
        const int r = 2 * c4 + odd_token;
        if (DP == 64) return st + (group8 * 8 + r) * 64 + (((l4 >> 1) ^ (r >> 1)) << 4) + (l4 & 1) * 8;
        return st + box * STEP * 128 + (group8 * 8 + r) * 128 + ((l4 ^ r) << 4);
    };
    int stage = 0, ahead = D - 1;
    uint32_t phase = 0;
    for (int k = k0, i = 0; k < steps.total; k += stride_k, ++i) {
        if ((i & 31) == 0) {
            if (i > 0) cur = nxt;
            settle(cur);
            nxt = batch_of(i + 32);
        }
        __syncwarp();                                 // the warp has read the stage that is filled now
        issue(i + D - 1, ahead, (i & 31) + D - 1 < 32 ? cur : nxt);
        float ks[H], vsc[H];
        bool ok[H];
#pragma unroll
        for (int z = 0; z < H; ++z) {
            ks[z] = z == 0 || two ? __shfl_sync(0xffffffffu, cur.k[z], i & 31) : ks[0];
            vsc[z] = z == 0 || two ? __shfl_sync(0xffffffffu, cur.v[z], i & 31) : vsc[0];
            ok[z] = (cur.there[z] >> (i & 31)) & 1u;
        }
        if (!__all_sync(0xffffffffu, (int)blockIdx.x != a.give_up && ptx::mbar_wait(full + 8 * stage, phase, abort_flag))) {
            *abort_flag = 1;
            // given up: the copies on their way land before the ring is something else's (or are given up too)
            for (int z = 0; z < D && k + z * stride_k < steps.total; ++z) {
                volatile int no = 0;
                ptx::mbar_wait(full + 8 * stage, phase, &no);
                if (++stage == D) { stage = 0; phase ^= 1u; }
            }
            break;
        }
        const uint8_t* st = ring + stage * F::STAGE;
        const int t = steps.at(k, STEP);
        // scores
        float x[H][NT][4];
#pragma unroll
        for (int half = 0; half < H; ++half) {
            // (8 or 16 rows at a time, for the registers' sake; K is read again for others)
            constexpr int NG = NT % 2 ? 1 : 2;
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += NG) {
                int sum[NG][DIG][4];
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {
                    const uint4 lo = *reinterpret_cast<const uint4*>(k_at(st, 2 * half, j)), hi = *reinterpret_cast<const uint4*>(k_at(st, 2 * half + 1, j));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t frag[4] = {i ? lo.z : lo.x, i ? hi.z : hi.x, i ? lo.w : lo.y, i ? hi.w : hi.y};
#pragma unroll
                        for (int n = 0; n < NG; ++n)
#pragma unroll
                            for (int g = 0; g < DIG; ++g) mma_i8_16x8(sum[n][g], frag, q_at(((j * 2 + i) * NT + n0 + n) * DIG + g), j == 0 && i == 0);
                    }
                }
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {     // (two digits' sums are below 2^29; the upper two, or the third, count 2^14)
                        const float lower = (float)(sum[n][0][i] + 128 * sum[n][1][i]), upper = (float)(DIG == 4 ? sum[n][2][i] + 128 * sum[n][DIG - 1][i] : sum[n][2][i]);
                        x[half][n0 + n][i] = fmaf(upper, 16384.0f, lower) * (factor[n0 + n][i & 1] * ks[half]);
                    }
            }
        }
        const bool all = ok[0] && ok[H - 1] && t + STEP - 1 <= low && (a.window == 0 || t > high - a.window || t + STEP <= a.sinks);
        if (!all) {
#pragma unroll
            for (int half = 0; half < H; ++half)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = t + half * 16 + (i >> 1) * 8 + l4, p = seen_to[n][i & 1];
                        const bool seen = ok[half] && j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
                        if (!seen) x[half][n][i] = -INFINITY;
                    }
        }
        // the largest x + log2(scale of V) of each row
        float lv[H], va[H];
#pragma unroll
        for (int half = 0; half < H; ++half) {
            va[half] = half == 0 || two ? fmaxf(fabsf(vsc[half]), 0.0f) : va[0];       // (of NaN 0)
            lv[half] = half == 0 || two ? __log2f(va[half]) : lv[0];       // (of 0 minus infinity)
        }
        const float v_top = fmaxf(ok[0] ? va[0] : 0.0f, ok[H - 1] ? va[H - 1] : 0.0f), v_low = fminf(ok[0] ? va[0] : INFINITY, ok[H - 1] ? va[H - 1] : INFINITY);
        // (no factor leaves the numbers: of a row that is not raised x + lv is at most M + 6, and 2^(x - m) at most 2^15 over the other factor, 2^27)
        float to[NT][2];
        bool raise = !(v_top * up_top <= 0x1p110f && v_low * up_low >= 0x1p-12f);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = fmaxf(x[0][n][i], x[0][n][i + 2]) + lv[0];
                if (H > 1) v = fmaxf(v, fmaxf(x[H - 1][n][i], x[H - 1][n][i + 2]) + lv[H - 1]);
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                to[n][i] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                raise |= to[n][i] > M[n][i] + 6.0f;
            }
        bool odd = false;                             // weights below 2^-170 at the most: none
        if (__any_sync(0xffffffffu, raise)) {
            up_top = 0.0f; up_low = INFINITY;
            const float lv_top = __log2f(v_top);
            const bool near = v_top > 0.0f && v_top <= 16.0f * v_low;       // of the step's pages: the largest x is found from x + lv, or 4 more
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float v = to[n][i] - lv_top;
                    if (!near) {
                        v = fmaxf(x[0][n][i], x[0][n][i + 2]);
                        if (H > 1) v = fmaxf(v, fmaxf(x[H - 1][n][i], x[H - 1][n][i + 2]));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                    }
                    const float m_now = fmaxf(m[n][i], v), M_now = fmaxf(fmaxf(M[n][i], to[n][i]), m_now - 104.0f);       // (scales below 2^-104 have no say in M: up is a number)
                    const float f = ex2(M[n][i] - M_now);
                    l[n][i] *= ex2(m[n][i] - m_now);
                    m[n][i] = m_now;
                    M[n][i] = M_now;
                    set_up(n, i);
#pragma unroll
                    for (int j = 0; j < MT; ++j) { o[j][n][i] *= f; o[j][n][i + 2] *= f; }
                }
            // A scale 2^80 above those that a row's M is made of, so that its weights, if any, are below 2^-74 there: m goes down for them, but l stays in range.
            if (__any_sync(0xffffffffu, v_top * up_top > 0x1p100f)) {
                up_top = 0.0f; up_low = INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float m_now = fminf(m[n][i], fmaxf(M[n][i] + 80.0f - lv_top, m[n][i] - 60.0f));
                        l[n][i] *= ex2(m[n][i] - m_now);
                        m[n][i] = m_now;
                        set_up(n, i);
                    }
                odd = __any_sync(0xffffffffu, v_top * up_top > 0x1p126f);
            }
        }
#pragma unroll
        for (int half = 0; half < H; ++half) {
            const float scale = ok[half] ? vsc[half] : 0.0f;
            const bool plain = scale == scale && !odd;       // (a scale of NaN: of all that is seen, also with a weight of nothing)
            uint32_t b[NT][2], d[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float p[4];
                const float factors[2] = {scale * up_of(n, 0), scale * up_of(n, 1)};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = ex2(x[half][n][i] - m[n][i & 1]);
                    l[n][i & 1] += e;
                    p[i] = e * factors[i & 1];
                    if (!plain) p[i] = x[half][n][i] == -INFINITY || factors[i & 1] > 0x1p126f ? 0.0f : p[i];
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
            for (int j = 0; j < F::BOXES; ++j) {
                uint32_t w[4][F::VB / 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t* at = v_at(st + F::HALF, 2 * half + (i >> 1), i & 1, j);
                    if constexpr (F::VB == 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(at);
                        w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(at);
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
        if (++stage == D) { stage = 0; phase ^= 1u; }
        ahead = ahead + 1 == D ? 0 : ahead + 1;
    }
    __syncthreads();                                  // the ring becomes the place of the warps' sums (every copy has been waited for)

    float* sums = reinterpret_cast<float*>(smem);     // [warp][row][dimension]
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
                // (m becomes what l is next to)
                const int e = v > 0.0f && v < INFINITY ? min((int)(__float_as_uint(v) >> 23) - 127, 126) : 0;
                const float u = up_of(n, i), down = __uint_as_float((uint32_t)(127 - e) << 23);
                s[0] = m[n][i] == kKvNothing ? -INFINITY : m[n][i] + (float)e; s[1] = v * down; s[2] = u > 0.0f ? __fdividef(down, u) : 0.0f;
            }
            float* to = sums + (warp * F::ROWS + r) * F::PITCH;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int d = (j / 8) * 128 + l4 * F::VB + 2 * (j % 8);
                *reinterpret_cast<float2*>(to + d) = make_float2(o[j][n][i], o[j][n][i + 2]);
            }
        }
    __syncthreads();
    if (threadIdx.x < F::ROWS) {
        const int r = threadIdx.x;
        float top = -INFINITY, total = 0.0f;
        for (int w = 0; w < W; ++w) top = fmaxf(top, stat[(w * F::ROWS + r) * 3]);
        for (int w = 0; w < W; ++w) {
            float* s = stat + (w * F::ROWS + r) * 3;
            const float f = join_factor(s[0], s[1], top);
            total += times(s[1], f);
            s[2] *= f;
        }
        joined[2 * r] = top; joined[2 * r + 1] = total;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < F::ROWS * (DP / 4); e += blockDim.x) {
        const int r = e / (DP / 4), d = (e % (DP / 4)) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < W; ++w) {
            const float f = stat[(w * F::ROWS + r) * 3 + 2];
            const float4 p = *reinterpret_cast<const float4*>(sums + (w * F::ROWS + r) * F::PITCH + d);
            v.x = fmaf(p.x, f, v.x); v.y = fmaf(p.y, f, v.y); v.z = fmaf(p.z, f, v.z); v.w = fmaf(p.w, f, v.w);
        }
        *reinterpret_cast<float4*>(sums + r * F::PITCH + d) = v;       // (of warp 0's, which only this thread reads)
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, (int)DEV_ERR_WAIT_TIMEOUT);
    if (a.work) {
        __syncthreads();
        float* to = a.work + (size_t)blockIdx.x * (F::ROWS * (DP + 2));
        for (int e = threadIdx.x; e < rows * (DP / 4); e += blockDim.x) {
            const int r = e / (DP / 4), d = (e % (DP / 4)) * 4;
            if (joined[2 * r + 1] != 0.0f) *reinterpret_cast<float4*>(to + r * DP + d) = *reinterpret_cast<const float4*>(sums + r * F::PITCH + d);
        }
        if (threadIdx.x < 2 * rows) to[F::ROWS * DP + threadIdx.x] = joined[threadIdx.x];
        return;
    }
    if (P > 1) {
        __syncwarp();
        ptx::cluster_arrive();
        ptx::cluster_wait();
    } else __syncthreads();
    const uint32_t my_sums = ptx::smem_u32(sums), my_joined = ptx::smem_u32(joined);
    const int quads = c.dim / 4;
    for (int e = rank * (int)blockDim.x + threadIdx.x; e < rows * quads; e += P * (int)blockDim.x) {
        const int r = e / quads, d = (e % quads) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float top = -INFINITY, total = 0.0f;
        if (P == 1) {
            v = *reinterpret_cast<const float4*>(sums + r * F::PITCH + d);
            top = joined[2 * r]; total = joined[2 * r + 1];
        } else {
            for (int p0 = 0; p0 < P; p0 += 2) {       // (P is even; two parts' loads at once)
                float2 ml[2]; float4 part[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    ml[i] = ld_cluster2(ptx::cluster_addr(my_joined + 8 * r, (uint32_t)(p0 + i)));
                    part[i] = ld_cluster4(ptx::cluster_addr(my_sums + 4 * (r * F::PITCH + d), (uint32_t)(p0 + i)));
                }
                const float to = fmaxf(top, fmaxf(ml[0].x, ml[1].x)), f = join_factor(top, total, to);
                total = times(total, f);
                v.x = times(v.x, f); v.y = times(v.y, f); v.z = times(v.z, f); v.w = times(v.w, f);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float fp = join_factor(ml[i].x, ml[i].y, to);
                    total += times(ml[i].y, fp);
                    v.x += times(part[i].x, fp); v.y += times(part[i].y, fp); v.z += times(part[i].z, fp); v.w += times(part[i].w, fp);
                }
                top = to;
            }
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int row = row0 + r;
        const long long token = q.row + row / a.group, head = h * a.group + row % a.group, at = token * a.out_stride + head * c.dim + d;
        kv_store(a.out, a.q_type, at, v.x * inv); kv_store(a.out, a.q_type, at + 1, v.y * inv);
        kv_store(a.out, a.q_type, at + 2, v.z * inv); kv_store(a.out, a.q_type, at + 3, v.w * inv);
        if (a.lse && d == 0) a.lse[token * a.heads + head] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
    }
    if (P > 1) {
        __syncwarp();
        ptx::cluster_arrive();
        ptx::cluster_wait();                          // nobody leaves while its sums are read
    }
}

// The sums of a tile's CTAs in the workspace; a CTA has 4 dimensions of a row each thread.
template <int DP, int NT>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const __grid_constant__ KvAttendArgs a) {
    constexpr int ROWS = 8 * NT, QUADS = DP / 4;
    ptx::grid_start();
    const KvArgs& c = a.c;
    const int h = blockIdx.x % c.heads;
    KvSeq q; int unit;
    if (!kv_locate(c, blockIdx.x / c.heads, a.group, ROWS, 1, q, unit)) return;
    const int row0 = unit * ROWS, rows = min(ROWS, kv_rows_of(a, q.n) - row0);      // (no more than the CTAs that left sums here)
    const int e = blockIdx.y * 256 + threadIdx.x, r = e / QUADS, d = (e % QUADS) * 4;
    if (r >= rows || d >= c.dim) return;
    const float* part = a.work + (size_t)blockIdx.x * a.parts * (ROWS * (DP + 2));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float top = -INFINITY, total = 0.0f;
    constexpr int U = 8;                              // parts whose sums are under way
    for (int p0 = 0; p0 < a.parts; p0 += U) {
        float2 ml[U]; float4 s[U];
        float to = top;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float* from = part + (size_t)(p0 + i) * (ROWS * (DP + 2));
            ml[i] = p0 + i < a.parts ? *reinterpret_cast<const float2*>(from + ROWS * DP + 2 * r) : make_float2(-INFINITY, 0.0f);
            s[i] = ml[i].y != 0.0f ? *reinterpret_cast<const float4*>(from + r * DP + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            to = fmaxf(to, ml[i].x);
        }
        const float f = join_factor(top, total, to);
        total = times(total, f);
        v.x = times(v.x, f); v.y = times(v.y, f); v.z = times(v.z, f); v.w = times(v.w, f);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float fp = join_factor(ml[i].x, ml[i].y, to);
            total += times(ml[i].y, fp);
            v.x += times(s[i].x, fp); v.y += times(s[i].y, fp); v.z += times(s[i].z, fp); v.w += times(s[i].w, fp);
        }
        top = to;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int row = row0 + r;
    const long long token = q.row + row / a.group, head = h * a.group + row % a.group, at = token * a.out_stride + head * c.dim + d;
    kv_store(a.out, a.q_type, at, v.x * inv); kv_store(a.out, a.q_type, at + 1, v.y * inv);
    kv_store(a.out, a.q_type, at + 2, v.z * inv); kv_store(a.out, a.q_type, at + 3, v.w * inv);
    if (a.lse && d == 0) a.lse[token * a.heads + head] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
}

// Bytes of a workspace that a call can use (0: none): few tiles, contexts of 16384 tokens and more.
inline size_t kv_work_bytes(const zant_ctx* ctx, const KvAttendArgs& a) {
    const long long reach = std::min((long long)a.c.width << a.c.page_log2, a.window > 0 ? (long long)a.window + a.sinks : 0x7fffffffffLL);
    if (reach < 16384 || kv_units(a.c, a.group, 32, 1) * a.c.heads * 16 > 3LL * ctx->sm_count) return 0;
    return (size_t)ctx->sm_count * 3 * 32 * ((a.c.dim <= 64 ? 64 : (a.c.dim <= 128 ? 128 : 256)) + 2) * 4;
}

// Codes as boxes of `rows` tokens of a page and head, `box` bytes each, zeros behind the head's end.
inline int32_t encode_kv_map(CUtensorMap* map, const void* p, const KvArgs& c, int box, int rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(ZANT_E_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {(cuuint64_t)c.dim, (cuuint64_t)c.page, (cuuint64_t)c.pages * c.heads}, strides[2] = {(cuuint64_t)c.dim, (cuuint64_t)c.dim * c.page};
    const cuuint32_t sides[3] = {(cuuint32_t)box, (cuuint32_t)rows, 1}, ones[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(p), dims, strides, sides, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              box == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ZANT_OK : fail(ZANT_E_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
}

template <int DP, int NT, bool SPLIT>
inline int32_t launch_kv_attention(zant_ctx* ctx, KvAttendArgs a) {
    using F = KvAttendCfg<DP, NT, SPLIT>;
    long long tiles = kv_units(a.c, a.group, F::ROWS, 1);
    if (a.c.offsets && a.rows_up_to < 0x7fffffff) {       // others take the sequences with more rows: tiles for those with as many as are left
        const int each = (a.rows_up_to + F::ROWS - 1) / F::ROWS;
        if ((long long)each * a.c.seqs < tiles) { a.tiles_each = each; tiles = (long long)each * a.c.seqs; }
    }
    const long long items = tiles * a.c.heads;
    if (items > 0x7fffffffLL / 16) return fail(ZANT_E_TOO_LARGE, "%lld tiles of attention", items);
    // CTAs that share a tile: while they find room side by side and each warp has steps left to take
    const long long reach = std::min((long long)a.c.width << a.c.page_log2, a.window > 0 ? (long long)a.window + a.sinks + 2 * F::STEP : 0x7fffffffffLL);
    const long long steps = (reach + F::STEP - 1) / F::STEP;
    const long long slots = (long long)ctx->sm_count * (F::MOST_WARPS / 4);
    int warps = 4, parts = 1;
    while (parts < 16 && ((items * parts * 2 <= slots && steps > 4LL * parts) || (items * parts * 2 <= 3 * slots && steps >= 64LL * parts))) parts *= 2;
    if (items * parts <= ctx->sm_count && parts < 16 && steps >= (long long)parts * F::MOST_WARPS) warps = F::MOST_WARPS;
    // Few tiles of long contexts: clusters of 16 leave most of the GPU idle (8 of them, one sequence of 131072: 113 us), so as many CTAs as it holds share a tile through the workspace and
    // a second kernel joins them.
    if (a.work) {
        const long long most = std::min({slots / items, steps / (4 * 4), (long long)(a.work_bytes / (items * F::ROWS * (DP + 2) * 4))});
        if (parts == 16 && most >= 24 && !a.tiles_each) { parts = (int)most; warps = 4; }
        else a.work = nullptr;
    }
    a.parts = parts;
    // more CTAs than there is room for at once: the longest sequences first, so that the last ones are short
    a.by_length = !a.c.offsets && !a.tiles_each && a.c.seqs > 1 && a.c.seqs <= 32 * warps && items * parts > slots;
    a.status = ctx->status_word;
    a.give_up = ctx->give_up_cta < 0 ? -1 : (int)(ctx->give_up_cta % (items * parts));
    ctx->give_up_cta = -1;
    alignas(64) CUtensorMap k_map{}, v_map{};
    const int box_rows = std::min(a.c.page, F::STEP);
    ZB_TRY(encode_kv_map(&k_map, a.c.k, a.c, F::BOX, box_rows));
    ZB_TRY(encode_kv_map(&v_map, a.c.v, a.c, F::BOX, box_rows));
    auto kernel = kv_attention_kernel<DP, NT, SPLIT>;
    ZB_SMEM_ATTR(ctx, kernel, F::smem(F::MOST_WARPS));
    static std::atomic<unsigned long long> wide{0ull};
    const unsigned long long bit = 1ull << (ctx->device & 63);
    if (parts > 8 && !a.work && !(wide.load(std::memory_order_acquire) & bit)) {
        ZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        wide.fetch_or(bit, std::memory_order_release);
    }
    launch_cluster(ctx, kernel, dim3((unsigned)(items * parts)), 32 * warps, F::smem(warps), a.work ? 1u : (unsigned)parts, a, k_map, v_map);
    ZB_TRY(check_launch(ctx, "kv_attention_kernel"));
    if (!a.work) return ZANT_OK;
    launch(ctx, kv_attention_join_kernel<DP, NT>, dim3((unsigned)items, (F::ROWS * (DP / 4) + 255) / 256), 256, 0, a);
    return check_launch(ctx, "kv_attention_join_kernel");
}

template <int DP, bool SPLIT>
inline int32_t choose_kv_attention(zant_ctx* ctx, const KvAttendArgs& a) {
    // (where others take the sequences with many rows and these are most, what is left has a token or a few)
    long long rows = ((long long)a.c.rows + a.c.seqs - 1) / a.c.seqs * a.group;
    if (rows > a.rows_up_to) rows = a.group;
    if (rows <= 8) return launch_kv_attention<DP, 1, SPLIT>(ctx, a);
    if constexpr (DP <= 128 && !SPLIT)
        if (rows > 16) return rows <= 24 ? launch_kv_attention<DP, 3, SPLIT>(ctx, a) : launch_kv_attention<DP, 4, SPLIT>(ctx, a);
    return launch_kv_attention<DP, 2, SPLIT>(ctx, a);
}

inline int32_t run_kv_few(zant_ctx* ctx, const KvAttendArgs& a) {
    const bool split = a.q_type == ZANT_F32;
    if (a.c.dim <= 64) return split ? choose_kv_attention<64, true>(ctx, a) : choose_kv_attention<64, false>(ctx, a);
    if (a.c.dim <= 128) return split ? choose_kv_attention<128, true>(ctx, a) : choose_kv_attention<128, false>(ctx, a);
    return split ? choose_kv_attention<256, true>(ctx, a) : choose_kv_attention<256, false>(ctx, a);
}

}  // namespace zb
