// Values of rows as floats, the largest of 16 bytes of them, and int8 codes of values under a scale.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "ptx_sm100.cuh"

namespace zb {

__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

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

}  // namespace zb
