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

namespace zb {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

struct QuantizeRowsArgs {
    const void* x; long long x_rows, x_stride; int cols;
    const int32_t* index; long long rows;
    int8_t* q; long long q_stride; float* scale;
};

// 16 bytes of a row: the largest magnitude so far (in the bits of the type, either sign, NaN above all), and the values.
template <typename T> struct RowChunk;
template <> struct RowChunk<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ uint32_t top(uint32_t m, uint32_t w) { asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w)); return m; }
    static __device__ __forceinline__ float top_value(uint32_t m) { return fabsf(__uint_as_float(m)); }
    static __device__ __forceinline__ void values(const uint32_t* w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    }
};
template <> struct RowChunk<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ uint32_t top(uint32_t m, uint32_t w) { asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w)); return m; }
    static __device__ __forceinline__ float top_value(uint32_t m) { return __uint_as_float(max(m & 0x7fffu, (m >> 16) & 0x7fffu) << 16); }
    static __device__ __forceinline__ float2 pair(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ void values(const uint32_t* w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 p = pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
    }
};
template <> struct RowChunk<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ uint32_t top(uint32_t m, uint32_t w) { asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w)); return m; }
    static __device__ __forceinline__ float top_value(uint32_t m) { return __half2float(__ushort_as_half((unsigned short)max(m & 0x7fffu, (m >> 16) & 0x7fffu))); }
    static __device__ __forceinline__ float2 pair(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ void values(const uint32_t* w, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 p = pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
    }
};

// A row's scale, and what turns values into codes.  Rows of tiny values (below 2^-60) are scaled up by 2^80 on the way, which is exact:
// neither the reciprocal nor a remainder leaves the normal numbers then.
struct RowScale {
    float scale, s, inv;
    bool tiny;
    __device__ __forceinline__ RowScale(float scale_, float s_, float inv_, bool tiny_) : scale(scale_), s(s_), inv(inv_), tiny(tiny_) {}
    __device__ __forceinline__ explicit RowScale(float amax) {
        scale = amax / 127.0f;
        tiny = amax < 8.6736174e-19f;
        s = tiny ? scale * 1.2089258e24f : scale;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    }
    __device__ __forceinline__ bool none() const { return !(s > 0.0f); }
    // The nearest integer to the exact quotient v / s: the product with the reciprocal is off by less than one code, and the remainder
    // of the nearest code, v - t s, is exact in fp32 (a multiple of the last place of s or v, and at most about s), so that comparing it
    // with s / 2 decides.
    __device__ __forceinline__ int code(float v) const {
        if (tiny) v *= 1.2089258e24f;
        float t = rintf(v * inv);
        const float rem = fmaf(-t, s, v), half = 0.5f * s;
        const bool odd = (static_cast<int>(t) & 1) != 0;
        if (rem > half || (rem == half && odd)) t += 1.0f;
        if (rem < -half || (rem == -half && odd)) t -= 1.0f;
        return static_cast<int>(fminf(fmaxf(t, -127.0f), 127.0f));
    }
};

template <int N>
__device__ __forceinline__ void pack_codes(const uint32_t* u, uint32_t* out) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        out[i] = __byte_perm(__byte_perm(u[4 * i], u[4 * i + 1], 0x0040), __byte_perm(u[4 * i + 2], u[4 * i + 3], 0x0040), 0x5410);
}

// A chunk's codes one by one.  (Out of line: inlined, it made the kernel wait for instructions half of its time, 56 us where it takes 37.)
template <typename T>
__device__ __noinline__ uint2 codes_again(uint4 w, float scale, float s, float inv, bool tiny) {
    constexpr int N = RowChunk<T>::N;
    const RowScale k{scale, s, inv, tiny};
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
    float f[N];
    RowChunk<T>::values(r, f);
    uint32_t u[N], out[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = (uint32_t)k.code(f[i]);
    pack_codes<N>(u, out);
    return make_uint2(out[0], out[1]);
}

// A chunk's codes, a byte each.
//
// 16-bit values: a quotient next to a border between two codes is common (one of 100: v and the row's maximum are short numbers, and s is one
// rounding away from making it a tie), but it is 2^-25 away or exactly there: 2 v and (2 t + 1) s are multiples of the last place of s.  So
// 1 / s is taken as the sum of its first 12 bits, whose product with v (11 bits at most) and 1/2 add up exactly, and the rest, and everything is
// rounded down: the floor of v / s + 1/2 is the code, in the low bits when 1.5 * 2^23 is added.  Ties proper need an s of at most 11 bits: such rows (and rows of tiny values) go through
// code(), `exactly`.  (With a remainder and a comparison for each value instead: 42 us for 8192 x 8192 bf16, with this 37.)
template <typename T, std::enable_if_t<sizeof(T) == 2, int> = 0>
__device__ __forceinline__ void codes_of(const uint32_t* w, const RowScale& k, bool exactly, uint32_t* out) {
    if (exactly) {
        const uint2 c = codes_again<T>(make_uint4(w[0], w[1], w[2], w[3]), k.scale, k.s, k.inv, k.tiny);
        out[0] = c.x; out[1] = c.y;
        return;
    }
    const float first = __uint_as_float(__float_as_uint(k.inv) & 0xfffff000u), rest = fmaf(-first, k.s, 1.0f) * k.inv;
    const unsigned long long inv = ptx::pack2(first, first), low = ptx::pack2(rest, rest), half = ptx::pack2(0.5f, 0.5f), magic = ptx::pack2(12582912.0f, 12582912.0f);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = RowChunk<T>::pair(w[i]);
        const unsigned long long v = ptx::pack2(p.x, p.y);
        const float2 c = ptx::unpack2(ptx::add2_rm(ptx::fma2_rm(v, low, ptx::fma2_rm(v, inv, half)), magic));
        u[2 * i] = __float_as_uint(c.x);
        u[2 * i + 1] = __float_as_uint(c.y);
    }
    pack_codes<8>(u, out);
}
// f32 values: a remainder of half a step or more (one quotient in 2^17, and ties) sends the chunk through code().
template <typename T, std::enable_if_t<sizeof(T) == 4, int> = 0>
__device__ __forceinline__ void codes_of(const uint32_t* w, const RowScale& k, bool exactly, uint32_t* out) {
    constexpr float MAGIC = 12582912.0f;
    const float half = 0.5f * k.s;
    float most = 0.0f;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = __uint_as_float(w[i]), t = fmaf(v, k.inv, MAGIC);
        u[i] = __float_as_uint(t);
        most = fmaxf(most, fabsf(fmaf(MAGIC - t, k.s, v)));
    }
    pack_codes<4>(u, out);
    if (exactly || most >= half) out[0] = codes_again<T>(make_uint4(w[0], w[1], w[2], w[3]), k.scale, k.s, k.inv, k.tiny).x;
}

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
