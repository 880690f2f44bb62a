// C entry points of the language-model operators (quantize_rows, qmatmul_scaled, qmatmul_grouped, token_logprobs).
#include <cuda_runtime.h>

#include <cstdint>
#include <new>

#include "../../include/zant_b200.h"
#include "context.cuh"
#include "quantize_rows.cuh"
#include "scaled_gemm_q8.cuh"
#include "status.hpp"
#include "token_logprobs.cuh"

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

inline int32_t scaled_gemm_entry(zant_ctx* ctx, const int8_t* a, size_t rows, size_t k, size_t a_stride, const float* a_scale, const int8_t* w, bool grouped,
                                 size_t groups, size_t n, size_t w_stride, const float* w_scale, const float* bias, const int32_t* offsets, int32_t y_dtype,
                                 void* y, size_t y_stride) {
    const size_t esz = float_size(y_dtype);
    if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "the result of a scaled product is f32, f16 or bf16");
    if (k == 0 || n == 0 || groups == 0) return fail(ZANT_E_INPUT_TENSORS_WRONG_SHAPE, "empty operand");
    if (k > (size_t)kScaledMaxK) return fail(ZANT_E_TOO_LARGE, "k = %zu: int32 sums hold %d products", k, kScaledMaxK);
    if (groups > (size_t)kScaledMaxGroups) return fail(ZANT_E_TOO_LARGE, "%zu groups: %d at most", groups, kScaledMaxGroups);
    ZB_TRY(check_int("rows", rows));
    ZB_TRY(check_int("n", n));
    size_t a_bytes, w_bytes, y_bytes;
    ZB_TRY(span_of("a", rows, k, a_stride, 1, a_bytes));
    ZB_TRY(span_of("w", groups * n, k, w_stride, 1, w_bytes));
    ZB_TRY(span_of("y", rows, n, y_stride, esz, y_bytes));
    if (rows == 0) return ZANT_OK;
    ZB_NEED(a, "a"); ZB_NEED(a_scale, "a_scale"); ZB_NEED(w, "w"); ZB_NEED(w_scale, "w_scale"); ZB_NEED(y, "y");
    if (grouped) ZB_NEED(offsets, "offsets");
    ZB_NEED_CTX(ctx);
    ZB_TRY(check_aligned("a_scale", a_scale, 4));
    ZB_TRY(check_aligned("w_scale", w_scale, 4));
    if (bias) ZB_TRY(check_aligned("bias", bias, 4));
    if (grouped) ZB_TRY(check_aligned("offsets", offsets, 4));
    ZB_TRY(check_aligned("y", y, esz));
    ScaledGemmArgs p{};
    p.a = a; p.a_stride = (long long)a_stride; p.w = w; p.w_stride = (long long)w_stride; p.y_stride = (long long)y_stride;
    p.rows = (int)rows; p.n = (int)n; p.k = (int)k; p.groups = (int)groups;
    p.offsets = offsets;                              // (the choice of the kernel asks whether there are any)
    // Device rows that the TMA cannot read are laid out in the arena, if it holds them as it is (beside what host arrays of the call take) and the
    // call is not captured.
    size_t align_a = scaled_align_bytes(p, false, ctx->sm_count), align_w = scaled_align_bytes(p, true, ctx->sm_count);
    Stager s(ctx);
    const int ia = s.in(a, a_bytes), ias = s.in(a_scale, rows * 4), iw = s.in(w, w_bytes), iws = s.in(w_scale, groups * n * 4), ib = s.in(bias, groups * n * 4);
    const int io = s.in(grouped ? offsets : nullptr, (groups + 1) * 4);
    const int iy = grouped || y_stride != n ? s.inout(y, y_bytes) : s.out(y, y_bytes);
    if ((align_a || align_w) && (!s.holds(align_up(align_a, kArenaAlign) + align_up(align_w, kArenaAlign)) || stream_capturing(ctx) || !is_device_ptr(a) || !is_device_ptr(w)))
        align_a = align_w = 0;
    const int ila = align_a ? s.scratch(align_a) : -1, ilw = align_w ? s.scratch(align_w) : -1;
    ZB_TRY(s.commit());
    p.a = s.ptr<int8_t>(ia); p.a_scale = s.ptr<float>(ias); p.w = s.ptr<int8_t>(iw); p.w_scale = s.ptr<float>(iws);
    p.bias = s.ptr<float>(ib); p.y = s.ptr<void>(iy); p.offsets = s.ptr<int32_t>(io);
    if (ila >= 0) {
        ZB_TRY(run_scaled_align(ctx, p.a, p.a_stride, p.k, (long long)rows, s.ptr<int8_t>(ila)));
        p.a = s.ptr<int8_t>(ila); p.a_stride = (long long)align_up(k, 16);
    }
    if (ilw >= 0) {
        ZB_TRY(run_scaled_align(ctx, p.w, p.w_stride, p.k, (long long)(groups * n), s.ptr<int8_t>(ilw)));
        p.w = s.ptr<int8_t>(ilw); p.w_stride = (long long)align_up(k, 16);
    }
    ZB_TRY(run_scaled_gemm(ctx, y_dtype, p));
    return s.finish();
}

}  // namespace zb

using namespace zb;

extern "C" {

int32_t zant_b200_quantize_rows(zant_ctx* ctx, int32_t x_dtype, const void* x, size_t x_rows, size_t cols, size_t x_stride, const int32_t* index, size_t rows,
                                int8_t* q, size_t q_stride, float* scale) {
    return c_entry([&]() -> int32_t {
        const size_t esz = float_size(x_dtype);
        if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "rows to quantize are f32, f16 or bf16");
        if (cols == 0) return fail(ZANT_E_INPUT_TENSORS_WRONG_SHAPE, "rows without columns");
        if (!index && rows != x_rows) return fail(ZANT_E_INPUT_TENSOR_DIFFERENT_SIZE, "%zu rows of %zu without an index", rows, x_rows);
        ZB_TRY(check_int("rows", rows));
        ZB_TRY(check_int("x_rows", x_rows));
        ZB_TRY(check_int("cols", cols));
        size_t x_bytes, q_bytes;
        ZB_TRY(span_of("x", x_rows, cols, x_stride, esz, x_bytes));
        ZB_TRY(span_of("q", rows, cols, q_stride, 1, q_bytes));
        if (rows == 0) return ZANT_OK;
        if (x_rows) ZB_NEED(x, "x");
        ZB_NEED(q, "q"); ZB_NEED(scale, "scale");
        ZB_NEED_CTX(ctx);
        if (x_rows) ZB_TRY(check_aligned("x", x, esz));
        if (index) ZB_TRY(check_aligned("index", index, 4));
        ZB_TRY(check_aligned("scale", scale, 4));
        Stager s(ctx);
        const int ix = s.in(x_rows ? x : nullptr, x_bytes), ii = s.in(index, rows * 4);
        const int iq = q_stride != cols ? s.inout(q, q_bytes) : s.out(q, q_bytes), is = s.out(scale, rows * 4);
        ZB_TRY(s.commit());
        QuantizeRowsArgs p{};
        p.x = s.ptr<void>(ix); p.x_rows = (long long)x_rows; p.x_stride = (long long)x_stride; p.cols = (int)cols;
        p.index = s.ptr<int32_t>(ii); p.rows = (long long)rows;
        p.q = s.ptr<int8_t>(iq); p.q_stride = (long long)q_stride; p.scale = s.ptr<float>(is);
        ZB_TRY(run_quantize_rows(ctx, x_dtype, p));
        return s.finish();
    });
}

int32_t zant_b200_qmatmul_scaled(zant_ctx* ctx, const int8_t* a, size_t rows, size_t k, size_t a_stride, const float* a_scale, const int8_t* w, size_t n,
                                 size_t w_stride, const float* w_scale, const float* bias, int32_t y_dtype, void* y, size_t y_stride) {
    return c_entry([&] { return scaled_gemm_entry(ctx, a, rows, k, a_stride, a_scale, w, false, 1, n, w_stride, w_scale, bias, nullptr, y_dtype, y, y_stride); });
}

int32_t zant_b200_qmatmul_grouped(zant_ctx* ctx, const int8_t* a, size_t rows, size_t k, size_t a_stride, const float* a_scale, const int8_t* w, size_t groups,
                                  size_t n, size_t w_stride, const float* w_scale, const float* bias, const int32_t* offsets, int32_t y_dtype, void* y,
                                  size_t y_stride) {
    return c_entry([&] { return scaled_gemm_entry(ctx, a, rows, k, a_stride, a_scale, w, true, groups, n, w_stride, w_scale, bias, offsets, y_dtype, y, y_stride); });
}

int32_t zant_b200_token_logprobs(zant_ctx* ctx, int32_t dtype, const void* logits, size_t rows, size_t vocab, size_t stride, const int32_t* tokens,
                                 float* logprob, float* entropy, int32_t top, int32_t* top_ids, float* top_logprobs) {
    return c_entry([&]() -> int32_t {
        const size_t esz = float_size(dtype);
        if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "logits are f32, f16 or bf16");
        if (vocab == 0) return fail(ZANT_E_INPUT_TENSORS_WRONG_SHAPE, "logits of no tokens");
        if (top < 0 || top > kTopMax || (size_t)top > vocab) return fail(ZANT_E_INVALID_INPUT, "top %d of %zu tokens: 0 to %d and at most all", top, vocab, kTopMax);
        ZB_TRY(check_int("rows", rows));
        ZB_TRY(check_int("vocab", vocab));
        size_t bytes;
        ZB_TRY(span_of("logits", rows, vocab, stride, esz, bytes));
        if ((tokens == nullptr) != (logprob == nullptr) && rows) return fail(ZANT_E_NULL_POINTER, "tokens and logprob come together");
        if (rows == 0) return ZANT_OK;
        ZB_NEED(logits, "logits");
        if (top) { ZB_NEED(top_ids, "top_ids"); ZB_NEED(top_logprobs, "top_logprobs"); }
        ZB_NEED_CTX(ctx);
        ZB_TRY(check_aligned("logits", logits, esz));
        if (tokens) { ZB_TRY(check_aligned("tokens", tokens, 4)); ZB_TRY(check_aligned("logprob", logprob, 4)); }
        if (entropy) ZB_TRY(check_aligned("entropy", entropy, 4));
        if (top) { ZB_TRY(check_aligned("top_ids", top_ids, 4)); ZB_TRY(check_aligned("top_logprobs", top_logprobs, 4)); }
        if (!logprob && !entropy && !top) return ZANT_OK;
        Stager s(ctx);
        const int il = s.in(logits, bytes), it = s.in(tokens, rows * 4), ip = s.out(logprob, rows * 4), ie = s.out(entropy, rows * 4);
        const int iti = s.out(top ? top_ids : nullptr, rows * (size_t)top * 4), itp = s.out(top ? top_logprobs : nullptr, rows * (size_t)top * 4);
        ZB_TRY(s.commit());
        TokenLogprobsArgs p{};
        p.x = s.ptr<void>(il); p.rows = (long long)rows; p.stride = (long long)stride; p.vocab = (int)vocab;
        p.tokens = s.ptr<int32_t>(it); p.logprob = s.ptr<float>(ip); p.entropy = s.ptr<float>(ie);
        p.top = top; p.top_ids = s.ptr<int32_t>(iti); p.top_logprobs = s.ptr<float>(itp);
        ZB_TRY(run_token_logprobs(ctx, dtype, p));
        return s.finish();
    });
}

}  // extern "C"
