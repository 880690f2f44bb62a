// What the entry points of the language-model operators ask of their arguments.
#pragma once
#include <cstdint>

#include "context.cuh"
#include "status.hpp"

namespace zb {

inline size_t float_size(int32_t dtype) { return dtype == ZANT_F32 ? 4 : (dtype == ZANT_F16 || dtype == ZANT_BF16 ? 2 : 0); }

// Bytes that `rows` rows of `len` elements span, `stride` elements apart (0: dense; the resolved stride is stored).
inline int32_t span_of(const char* what, size_t rows, size_t len, size_t& stride, size_t esz, size_t& bytes) {
    if (stride == 0) stride = len;
    if (stride < len) return fail(ZANT_E_WRONG_STRIDE, "rows of %s are %zu long and %zu apart", what, len, stride);
    size_t n = 0;
    bytes = 0;
    if (rows == 0) return ZANT_OK;
    if (__builtin_mul_overflow(rows - 1, stride, &n) || __builtin_add_overflow(n, len, &n) || __builtin_mul_overflow(n, esz, &bytes) || bytes > (size_t)1 << 62)
        return fail(ZANT_E_TOO_LARGE, "%s spans more than an address can", what);
    return ZANT_OK;
}

inline int32_t check_aligned(const char* what, const void* p, size_t esz) {
    return (reinterpret_cast<uintptr_t>(p) & (esz - 1)) && is_device_ptr(p) ? fail(ZANT_E_INVALID_INPUT, "%s is not aligned to its elements", what) : ZANT_OK;
}

// What the kernels count in an int, with room for the steps of their loops past the end.
inline int32_t check_int(const char* what, size_t v) { return v > 0x7fff0000ULL ? fail(ZANT_E_TOO_LARGE, "%s = %zu", what, v) : ZANT_OK; }

// Nothing of C++ leaves a C entry point.
template <typename F>
inline int32_t c_entry(F&& body) noexcept {
    try { return body(); } catch (...) { return ZANT_E_MEM_ERROR; }
}

}  // namespace zb
