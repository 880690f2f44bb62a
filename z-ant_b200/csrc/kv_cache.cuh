// A decoder's key-value cache in 8 bits: pages of tokens, codes [pages, heads, page, dim] with one scale for each page and head.
//
//   writing   s' = max(s, max |x| / 127) over the new values x of a page and head;  codes of new values: nearest integer to x / s', ties to even;
//             codes c that stood in the page: nearest integer to c s / s'  (a page whose first token is written begins anew: s = 0)
//   reading   c * s
//
// Both are bound by memory.  A CTA has one page of one head, keys or values: the new rows are read once for the maximum, which stays in the
// CTA, and their values wait in registers (kKvHold times 16 a thread, all under way at once; what is beyond is read again).  Pages, not tokens, are what the grid
// counts, so that no other CTA writes the page or its scale.  A prompt of 8192 tokens, 8 heads of 128, bf16: written in 15.5 us (3.2 TB/s), read back in 13.6 (3.7); 64 single tokens in a
// graph: written in 3.7, their pages of 32 back in 5.5, the latency of lengths, table and page one after the other.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "context.cuh"
#include "ptx_sm100.cuh"
#include "row_codes.cuh"

namespace zb {

// The cache, and the sequences of a call: `rows` new tokens, those of sequence s are rows offsets[s] to offsets[s + 1] - 1 (without offsets: `per`
// each), the last of the lengths[s] tokens that the sequence has in the cache.
struct KvArgs {
    int8_t* k; int8_t* v; float* k_scale; float* v_scale;
    long long pages; int heads, page, page_log2, dim;
    const int32_t* table; const int32_t* lengths; const int32_t* offsets;
    int seqs, width, rows, per;
};

__device__ __forceinline__ int kv_offset(const KvArgs& a, int s) { return a.offsets ? min(max(a.offsets[s], 0), a.rows) : s * a.per; }

// A sequence of a call: its first row, its new tokens, the position of the first of them (negative: more new tokens than the length says).
struct KvSeq { int s, row, n, first; };
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, int s) {
    KvSeq q;
    q.s = s;
    q.row = kv_offset(a, s);
    q.n = kv_offset(a, s + 1) - q.row;
    const long long room = (long long)a.width << a.page_log2;
    q.first = (int)min((long long)max(a.lengths[s], 0), min(room, 0x7fff0000LL)) - q.n;
    return q;
}

// Work on sequences in units of `size` of a sequence's own count (new tokens times `times`), of which a sequence takes at most
// floor(end / size) - floor(begin / size) + extra: unit w of the whole grid is unit `unit` of sequence s.  The last s whose first unit is not behind w is
// found by the 32 lanes of a warp at once, 32 places in each round.  False where w belongs to no sequence.
__device__ __forceinline__ bool kv_locate(const KvArgs& a, int w, int times, int size, int extra, KvSeq& q, int& unit) {
    if (!a.offsets) {
        const int each = (int)(((long long)a.per * times + size - 1) / size) + extra - 1;
        const int s = w / each;
        if (s >= a.seqs) return false;
        unit = w - s * each;
        q = kv_seq(a, s);
        return true;
    }
    const int lane = threadIdx.x & 31;
    auto base = [&](int s) { return (long long)kv_offset(a, s) * times / size + (long long)extra * s; };
    int lo = 0, n = a.seqs;                           // the answer lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const bool before = at < lo + n && (lane == 0 || base(at) <= w);
        // (in order where offsets are; where they are not, any of the places will do)
        const unsigned hit = __ballot_sync(0xffffffffu, before);
        const int last = 31 - __clz(hit);
        n = min(step, lo + n - (lo + last * step));
        lo += last * step;
    }
    const long long b = base(lo);
    if (b > w) return false;
    unit = (int)(w - b);
    q = kv_seq(a, lo);
    return q.n > 0 && w - b <= (long long)q.n * times / size + 1;
}
// Units that a grid has to have.
inline long long kv_units(const KvArgs& a, int times, int size, int extra) {
    if (!a.offsets) return ((((long long)a.per * times + size - 1) / size) + extra - 1) * a.seqs;
    return (long long)a.rows * times / size + (long long)extra * a.seqs;
}

// Where in the cache page `at` of sequence s lies (its place in the table), -1: nowhere.
__device__ __forceinline__ long long kv_page(const KvArgs& a, int s, int at) {
    if (at < 0 || at >= a.width) return -1;
    const int id = a.table[(long long)s * a.width + at];
    return id >= 0 && id < a.pages ? id : -1;
}

// 16 values each that a thread holds of what it reads.
template <typename T> constexpr int kKvHold = sizeof(T) == 2 ? 4 : 2;

struct KvWriteArgs {
    KvArgs c;
    const void* x[2]; long long stride[2];            // keys, values
    bool wide[2];                                     // rows of whole 16-byte blocks
};

// 16 values of a row, as 16-byte chunks.
template <typename T>
__device__ __forceinline__ void kv_load16(const T* p, bool wide, uint32_t (&w)[sizeof(T) * 4]) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
    }
}

// The largest of the CTA's numbers, for all of its threads.
__device__ __forceinline__ uint32_t kv_block_max(uint32_t m, uint32_t* part) {
    m = __reduce_max_sync(0xffffffffu, m);
    if (blockDim.x == 32) return m;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < blockDim.x / 32 ? part[threadIdx.x & 31] : 0u);
}

// grid: page units, heads, keys | values
template <typename T>
__global__ void __launch_bounds__(256) kv_cache_write_kernel(const __grid_constant__ KvWriteArgs a) {
    using C = RowChunk<T>;
    constexpr int W = sizeof(T) * 4;                  // words of 16 values
    __shared__ uint32_t part[8];
    __shared__ int8_t moved[132];
    ptx::grid_start();
    const KvArgs& c = a.c;
    const int tid = threadIdx.x, threads = blockDim.x, h = blockIdx.y, kv = blockIdx.z;
    KvSeq q; int unit;
    if (!kv_locate(c, blockIdx.x, 1, c.page, 2, q, unit)) return;
    const int at = (max(q.first, 0) >> c.page_log2) + unit, from = max(q.first, at << c.page_log2);
    const int to = min(q.first + q.n, (at + 1) << c.page_log2);
    if (from < 0 || from >= to) return;
    const int begin = from & (c.page - 1), per_row = c.dim >> 4, units = (to - from) * per_row;
    const T* x = static_cast<const T*>(a.x[kv]) + (long long)(q.row + from - q.first) * a.stride[kv] + (long long)h * c.dim;
    const bool wide = a.wide[kv];
    auto load = [&](int u, uint32_t (&w)[W]) { const int t = u / per_row; kv_load16(x + t * a.stride[kv] + (u - t * per_row) * 16, wide, w); };
    constexpr int HOLD = kKvHold<T>;
    uint32_t mine[HOLD][W];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
        if (tid + i * threads < units) load(tid + i * threads, mine[i]);
        else {
#pragma unroll
            for (int z = 0; z < W; ++z) mine[i][z] = 0;
        }
    }
    // (the page is looked up while the rows are on their way)
    const long long page = kv_page(c, q.s, at);
    if (page < 0) return;
    int8_t* codes = (kv ? c.v : c.k) + (page * c.heads + h) * c.page * c.dim;
    float* scale = (kv ? c.v_scale : c.k_scale) + page * c.heads + h;
    const float old = begin == 0 ? 0.0f : *scale;
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
#pragma unroll
        for (int z = 0; z < W; ++z) m = C::top(m, mine[i][z]);
    for (int u = tid + HOLD * threads; u < units; u += threads) {
        uint32_t w[W];
        load(u, w);
#pragma unroll
        for (int z = 0; z < W; ++z) m = C::top(m, w[z]);
    }
    m = kv_block_max(__float_as_uint(C::top_value(m)), part);
    const bool finite = m < 0x7f800000u && old == old;
    const float top = __uint_as_float(m) / 127.0f, s = finite ? fmaxf(old, top) : __uint_as_float(0x7fffffffu);
    const bool tiny = s < 6.7762636e-21f;            // 2^-67: scaled up by 2^80 on the way, see RowScale
    float inv;
    const float big = tiny ? s * 1.2089258e24f : s;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(big));
    const RowScale k(s, big, inv, tiny);
    const bool none = !finite || k.none();
    const bool exactly = tiny || (sizeof(T) == 2 && (__float_as_uint(k.s) & 0xfffu) == 0);
    auto write = [&](int u, const uint32_t (&w)[W]) {
        uint32_t out[4] = {0, 0, 0, 0};
        if (!none) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) codes_of<T>(w + 4 * i, k, exactly, out + i * (4 / (int)sizeof(T)));
        }
        *reinterpret_cast<uint4*>(codes + (long long)begin * c.dim + u * 16) = make_uint4(out[0], out[1], out[2], out[3]);
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
        if (tid + i * threads < units) write(tid + i * threads, mine[i]);
    for (int u = tid + HOLD * threads; u < units; u += threads) {
        uint32_t w[W];
        load(u, w);
        write(u, w);
    }
    if (finite && begin > 0 && s > old) {
        // The quotient of 64 bits is right at every border: 2 c s and (2 t + 1) s' are whole multiples of a unit with 33 bits at most.
        for (int i = tid; i <= 128; i += threads) moved[i] = (int8_t)min(127, (int)rint((double)i * (double)old / (double)s));
        __syncthreads();
        for (int u = tid; u < begin * per_row; u += threads) {
            uint4 v = *reinterpret_cast<const uint4*>(codes + u * 16);
            int8_t* b = reinterpret_cast<int8_t*>(&v);
#pragma unroll
            for (int i = 0; i < 16; ++i) b[i] = b[i] < 0 ? (int8_t)-moved[-b[i]] : moved[b[i]];
            *reinterpret_cast<uint4*>(codes + u * 16) = v;
        }
    }
    __syncthreads();                                  // everyone has the old scale
    if (tid == 0) *scale = s;
}

struct KvReadArgs {
    KvArgs c;
    void* out[2]; long long stride[2];
    bool wide[2];
    int only;                                         // of a grid that is 1 deep: 0 keys, 1 values
};

template <typename T> __device__ __forceinline__ T kv_round(float v);
template <> __device__ __forceinline__ float kv_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half kv_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 kv_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(const __grid_constant__ KvReadArgs a) {
    ptx::grid_start();
    const KvArgs& c = a.c;
    const int tid = threadIdx.x, threads = blockDim.x, h = blockIdx.y, kv = gridDim.z == 1 ? a.only : (int)blockIdx.z;
    KvSeq q; int unit;
    if (!kv_locate(c, blockIdx.x, 1, c.page, 2, q, unit)) return;
    const int at = (q.first >> c.page_log2) + unit;   // (rounds down: positions below zero are on no page)
    const int from = max(q.first, at << c.page_log2), to = min(q.first + q.n, (at + 1) << c.page_log2);
    if (from >= to) return;
    const long long page = kv_page(c, q.s, at);
    const int begin = from & (c.page - 1), per_row = c.dim >> 4, units = (to - from) * per_row;
    const long long block = (page < 0 ? 0 : page) * c.heads + h;
    const int8_t* codes = (kv ? c.v : c.k) + block * c.page * c.dim + (long long)begin * c.dim;
    const float s = page < 0 ? 0.0f : (kv ? c.v_scale : c.k_scale)[block];
    T* out = static_cast<T*>(a.out[kv]) + (long long)(q.row + from - q.first) * a.stride[kv] + (long long)h * c.dim;
    constexpr int HOLD = 4;
    for (int u0 = tid; u0 < units; u0 += HOLD * threads) {
        uint4 v[HOLD];
#pragma unroll
        for (int i = 0; i < HOLD; ++i) v[i] = page >= 0 && u0 + i * threads < units ? *reinterpret_cast<const uint4*>(codes + (u0 + i * threads) * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const int u = u0 + i * threads;
            if (u >= units) break;
            const int8_t* b = reinterpret_cast<const int8_t*>(&v[i]);
            const int t = u / per_row;
            T* to_row = out + t * a.stride[kv] + (u - t * per_row) * 16;
            alignas(16) T y[16];
#pragma unroll
            for (int z = 0; z < 16; ++z) y[z] = kv_round<T>((float)b[z] * s);
            if (a.wide[kv]) {
#pragma unroll
                for (int z = 0; z < (int)sizeof(T); ++z) reinterpret_cast<uint4*>(to_row)[z] = reinterpret_cast<const uint4*>(y)[z];
            } else {
#pragma unroll
                for (int z = 0; z < 16; ++z) to_row[z] = y[z];
            }
        }
    }
}

// Threads for a page's share of the new tokens, 16 values `hold` times each.
inline int kv_threads(const KvArgs& a, int hold) {
    const long long tokens = std::min<long long>(a.page, ((long long)a.rows + a.seqs - 1) / a.seqs), units = (tokens * (a.dim / 16) + hold - 1) / hold;
    return units <= 64 ? 64 : (units <= 128 ? 128 : 256);
}

inline int32_t run_kv_cache_write(zant_ctx* ctx, int32_t dtype, const KvWriteArgs& a) {
    const dim3 grid((unsigned)kv_units(a.c, 1, a.c.page, 2), (unsigned)a.c.heads, 2);
    auto go = [&](auto kernel) { launch(ctx, kernel, grid, kv_threads(a.c, dtype == ZANT_F32 ? 2 : 4), 0, a); return check_launch(ctx, "kv_cache_write_kernel"); };
    if (dtype == ZANT_F32) return go(kv_cache_write_kernel<float>);
    if (dtype == ZANT_F16) return go(kv_cache_write_kernel<__half>);
    return go(kv_cache_write_kernel<__nv_bfloat16>);
}

inline int32_t run_kv_cache_read(zant_ctx* ctx, int32_t dtype, const KvReadArgs& a) {
    const dim3 grid((unsigned)kv_units(a.c, 1, a.c.page, 2), (unsigned)a.c.heads, a.out[0] && a.out[1] ? 2 : 1);
    auto go = [&](auto kernel) { launch(ctx, kernel, grid, kv_threads(a.c, 4), 0, a); return check_launch(ctx, "kv_cache_read_kernel"); };
    if (dtype == ZANT_F32) return go(kv_cache_read_kernel<float>);
    if (dtype == ZANT_F16) return go(kv_cache_read_kernel<__half>);
    return go(kv_cache_read_kernel<__nv_bfloat16>);
}

}  // namespace zb
