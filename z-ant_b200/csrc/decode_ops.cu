// C entry points of a decoder's int8 cache (kv_cache_write, kv_cache_read, kv_cache_attention) and of verify_drafts; a unit of its own, compiled beside
// lib.cu.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/zant_b200.h"
#include "context.cuh"
#include "kv_attention.cuh"
#include "kv_cache.cuh"
#include "kv_prompt.cuh"
#include "row_checks.cuh"
#include "status.hpp"
#include "verify_drafts.cuh"

namespace zb {

// The bytes of a cache's codes and scales, and what may be said of it and of a call's sequences before any pointer is looked at.
inline int32_t kv_check(const zant_kv_cache* c, size_t rows, const int32_t* offsets, size_t seqs, size_t width, size_t& code_bytes, size_t& scale_bytes) {
    ZB_NEED(c, "cache");
    if (c->heads == 0 || c->pages == 0) return fail(ZANT_E_INPUT_TENSORS_WRONG_SHAPE, "a cache of %zu pages and %zu heads", c->pages, c->heads);
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1))) return fail(ZANT_E_INVALID_INPUT, "pages of %zu tokens: 16, 32, 64, 128 or 256", c->page);
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) return fail(ZANT_E_UNSUPPORTED_DIMENSION, "heads of %zu dimensions: a multiple of 16, at most 256", c->dim);
    if (c->heads > 65535) return fail(ZANT_E_TOO_LARGE, "%zu heads", c->heads);
    ZB_TRY(check_int("pages", c->pages));
    ZB_TRY(check_int("rows", rows));
    ZB_TRY(check_int("width", width));
    if (seqs > (size_t)1 << 24) return fail(ZANT_E_TOO_LARGE, "%zu sequences", seqs);
    scale_bytes = c->pages * c->heads * 4;
    code_bytes = c->pages * c->heads * c->page * c->dim;       // (below 2^63 by the limits above)
    if (!offsets && rows && (seqs == 0 || rows % seqs)) return fail(ZANT_E_INPUT_TENSOR_DIFFERENT_SIZE, "%zu rows of %zu sequences without offsets", rows, seqs);
    return ZANT_OK;
}

inline int32_t kv_check_pointers(const zant_kv_cache* c, const int32_t* table, size_t width, const int32_t* lengths, const int32_t* offsets) {
    ZB_NEED(c->k, "k codes"); ZB_NEED(c->k_scale, "k scales"); ZB_NEED(c->v, "v codes"); ZB_NEED(c->v_scale, "v scales");
    if (width) ZB_NEED(table, "table");
    ZB_NEED(lengths, "lengths");
    ZB_TRY(check_aligned("k codes", c->k, 16)); ZB_TRY(check_aligned("v codes", c->v, 16));
    ZB_TRY(check_aligned("k scales", c->k_scale, 4)); ZB_TRY(check_aligned("v scales", c->v_scale, 4));
    if (width) ZB_TRY(check_aligned("table", table, 4));
    ZB_TRY(check_aligned("lengths", lengths, 4));
    if (offsets) ZB_TRY(check_aligned("offsets", offsets, 4));
    return ZANT_OK;
}

// The staged places of a cache and a call's sequences.
struct KvSlots {
    int k, ks, v, vs, table, lengths, offsets;
    KvSlots(Stager& s, const zant_kv_cache* c, size_t code_bytes, size_t scale_bytes, const int32_t* t, size_t seqs, size_t width, const int32_t* len, const int32_t* off, bool write) {
        k = write ? s.inout(c->k, code_bytes) : s.in(c->k, code_bytes); ks = write ? s.inout(c->k_scale, scale_bytes) : s.in(c->k_scale, scale_bytes);
        v = write ? s.inout(c->v, code_bytes) : s.in(c->v, code_bytes); vs = write ? s.inout(c->v_scale, scale_bytes) : s.in(c->v_scale, scale_bytes);
        table = s.in(width ? t : nullptr, seqs * width * 4); lengths = s.in(len, seqs * 4); offsets = s.in(off, (seqs + 1) * 4);
    }
    KvArgs args(Stager& s, const zant_kv_cache* c, size_t rows, size_t seqs, size_t width) const {
        KvArgs a{};
        a.k = s.ptr<int8_t>(k); a.k_scale = s.ptr<float>(ks); a.v = s.ptr<int8_t>(v); a.v_scale = s.ptr<float>(vs);
        a.pages = (long long)c->pages; a.heads = (int)c->heads; a.page = (int)c->page; a.dim = (int)c->dim;
        for (a.page_log2 = 4; (1 << a.page_log2) < a.page;) ++a.page_log2;
        a.table = s.ptr<int32_t>(table); a.lengths = s.ptr<int32_t>(lengths); a.offsets = s.ptr<int32_t>(offsets);
        a.seqs = (int)seqs; a.width = (int)width; a.rows = (int)rows; a.per = (int)(rows / seqs);
        return a;
    }
};

inline bool whole_blocks(const void* p, size_t stride, size_t esz) { return ((reinterpret_cast<uintptr_t>(p) | (stride * esz)) & 15) == 0; }

}  // namespace zb

using namespace zb;

extern "C" {

int32_t zant_b200_kv_cache_write(zant_ctx* ctx, const zant_kv_cache* cache, int32_t dtype, const void* k, size_t k_stride, const void* v, size_t v_stride, size_t rows,
                                 const int32_t* table, size_t seqs, size_t width, const int32_t* lengths, const int32_t* offsets) {
    return c_entry([&]() -> int32_t {
        const size_t esz = float_size(dtype);
        if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "keys and values to write are f32, f16 or bf16");
        size_t codes, scales, k_bytes, v_bytes;
        ZB_TRY(kv_check(cache, rows, offsets, seqs, width, codes, scales));
        const size_t len = cache->heads * cache->dim;
        ZB_TRY(span_of("k", rows, len, k_stride, esz, k_bytes));
        ZB_TRY(span_of("v", rows, len, v_stride, esz, v_bytes));
        if (rows == 0 || seqs == 0) return ZANT_OK;
        ZB_NEED(k, "k"); ZB_NEED(v, "v");
        ZB_TRY(kv_check_pointers(cache, table, width, lengths, offsets));
        ZB_NEED_CTX(ctx);
        ZB_TRY(check_aligned("k", k, esz)); ZB_TRY(check_aligned("v", v, esz));
        Stager s(ctx);
        const KvSlots slots(s, cache, codes, scales, table, seqs, width, lengths, offsets, true);
        const int ik = s.in(k, k_bytes), iv = s.in(v, v_bytes);
        ZB_TRY(s.commit());
        KvWriteArgs a{};
        a.c = slots.args(s, cache, rows, seqs, width);
        a.x[0] = s.ptr<void>(ik); a.x[1] = s.ptr<void>(iv);
        a.stride[0] = (long long)k_stride; a.stride[1] = (long long)v_stride;
        a.wide[0] = whole_blocks(a.x[0], k_stride, esz); a.wide[1] = whole_blocks(a.x[1], v_stride, esz);
        ZB_TRY(run_kv_cache_write(ctx, dtype, a));
        return s.finish();
    });
}

int32_t zant_b200_kv_cache_read(zant_ctx* ctx, const zant_kv_cache* cache, int32_t dtype, void* k, size_t k_stride, void* v, size_t v_stride, size_t rows,
                                const int32_t* table, size_t seqs, size_t width, const int32_t* lengths, const int32_t* offsets) {
    return c_entry([&]() -> int32_t {
        const size_t esz = float_size(dtype);
        if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "keys and values are read as f32, f16 or bf16");
        size_t codes, scales, k_bytes, v_bytes;
        ZB_TRY(kv_check(cache, rows, offsets, seqs, width, codes, scales));
        const size_t len = cache->heads * cache->dim;
        ZB_TRY(span_of("k", rows, len, k_stride, esz, k_bytes));
        ZB_TRY(span_of("v", rows, len, v_stride, esz, v_bytes));
        if (rows == 0 || seqs == 0 || (!k && !v)) return ZANT_OK;
        ZB_TRY(kv_check_pointers(cache, table, width, lengths, offsets));
        ZB_NEED_CTX(ctx);
        if (k) ZB_TRY(check_aligned("k", k, esz));
        if (v) ZB_TRY(check_aligned("v", v, esz));
        Stager s(ctx);
        const KvSlots slots(s, cache, codes, scales, table, seqs, width, lengths, offsets, false);
        const int ik = s.inout(k, k_bytes), iv = s.inout(v, v_bytes);
        ZB_TRY(s.commit());
        KvReadArgs a{};
        a.c = slots.args(s, cache, rows, seqs, width);
        a.out[0] = s.ptr<void>(ik); a.out[1] = s.ptr<void>(iv);
        a.stride[0] = (long long)k_stride; a.stride[1] = (long long)v_stride;
        a.wide[0] = whole_blocks(a.out[0], k_stride, esz); a.wide[1] = whole_blocks(a.out[1], v_stride, esz);
        a.only = k ? 0 : 1;
        ZB_TRY(run_kv_cache_read(ctx, dtype, a));
        return s.finish();
    });
}

int32_t zant_b200_kv_cache_attention(zant_ctx* ctx, const zant_kv_cache* cache, int32_t dtype, const void* q, size_t q_stride, size_t rows, size_t heads,
                                     const int32_t* table, size_t seqs, size_t width, const int32_t* lengths, const int32_t* offsets,
                                     float scale, int32_t window, int32_t sinks, void* out, size_t out_stride, float* lse) {
    return c_entry([&]() -> int32_t {
        const size_t esz = float_size(dtype);
        if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "queries and results are f32, f16 or bf16");
        size_t codes, scales, q_bytes, out_bytes;
        ZB_TRY(kv_check(cache, rows, offsets, seqs, width, codes, scales));
        if (heads == 0 || heads % cache->heads) return fail(ZANT_E_INPUT_TENSORS_WRONG_SHAPE, "%zu heads of queries over %zu heads of keys", heads, cache->heads);
        if (heads > 65535) return fail(ZANT_E_TOO_LARGE, "%zu heads", heads);
        ZB_TRY(check_int("pages of all heads", cache->pages * cache->heads));
        if (window < 0 || sinks < 0) return fail(ZANT_E_INVALID_INPUT, "window %d, sinks %d", window, sinks);
        const size_t group = heads / cache->heads, len = heads * cache->dim;
        ZB_TRY(check_int("rows of a key head", rows * group));
        ZB_TRY(span_of("q", rows, len, q_stride, esz, q_bytes));
        ZB_TRY(span_of("out", rows, len, out_stride, esz, out_bytes));
        if (rows == 0 || seqs == 0) return ZANT_OK;
        ZB_NEED(q, "q"); ZB_NEED(out, "out");
        ZB_TRY(kv_check_pointers(cache, table, width, lengths, offsets));
        ZB_NEED_CTX(ctx);
        ZB_TRY(check_aligned("q", q, esz)); ZB_TRY(check_aligned("out", out, esz));
        if (lse) ZB_TRY(check_aligned("lse", lse, 4));
        Stager s(ctx);
        const KvSlots slots(s, cache, codes, scales, table, seqs, width, lengths, offsets, false);
        const int iq = s.in(q, q_bytes), io = s.inout(out, out_bytes), il = s.inout(lse, rows * heads * 4);
        KvAttendArgs a{};
        a.c = slots.args(s, cache, rows, seqs, width);       // (sizes; pointers again when all is in place)
        a.heads = (int)heads; a.group = (int)group; a.q_type = dtype; a.window = window; a.sinks = sinks;
        // a workspace in the arena, unless the call is captured or the arena may not or cannot grow that far
        size_t work = kv_work_bytes(ctx, a);
        if (work && !s.room_for(work)) work = 0;
        const int iw = work ? s.scratch(work) : -1;
        ZB_TRY(s.commit());
        a.c = slots.args(s, cache, rows, seqs, width);
        a.q = s.ptr<void>(iq); a.q_stride = (long long)q_stride;
        a.out = s.ptr<void>(io); a.out_stride = (long long)out_stride; a.lse = s.ptr<float>(il);
        a.scale_log2 = scale * kLog2e;
        a.work = work ? s.ptr<float>(iw) : nullptr; a.work_bytes = work;
        a.wide_q = whole_blocks(a.q, q_stride, esz); a.wide_out = whole_blocks(a.out, out_stride, esz);
        ZB_TRY(run_kv_attention(ctx, a));
        return s.finish();
    });
}

int32_t zant_b200_verify_drafts(zant_ctx* ctx, int32_t dtype, const void* target, size_t target_stride, const void* drafted, size_t drafted_stride, size_t vocab,
                                const int32_t* tokens, size_t drafts, const int32_t* offsets, size_t seqs, const float* accept, const float* sample,
                                int32_t* accepted, int32_t* next) {
    return c_entry([&]() -> int32_t {
        const size_t esz = float_size(dtype);
        if (!esz) return fail(ZANT_E_INPUT_ARRAY_WRONG_TYPE, "probabilities are f32, f16 or bf16");
        if (vocab == 0) return fail(ZANT_E_INPUT_TENSORS_WRONG_SHAPE, "probabilities of no tokens");
        ZB_TRY(check_int("vocab", vocab));
        ZB_TRY(check_int("drafts", drafts));
        if (seqs > (size_t)1 << 24) return fail(ZANT_E_TOO_LARGE, "%zu sequences", seqs);
        size_t t_bytes, d_bytes;
        ZB_TRY(span_of("target", drafts + seqs, vocab, target_stride, esz, t_bytes));
        ZB_TRY(span_of("drafted", drafts, vocab, drafted_stride, esz, d_bytes));
        if (seqs == 0) return ZANT_OK;
        if (!offsets && drafts % seqs) return fail(ZANT_E_INPUT_TENSOR_DIFFERENT_SIZE, "%zu drafts of %zu sequences without offsets", drafts, seqs);
        ZB_NEED(target, "target"); ZB_NEED(sample, "sample"); ZB_NEED(accepted, "accepted"); ZB_NEED(next, "next");
        if (drafts) { ZB_NEED(tokens, "tokens"); ZB_NEED(accept, "accept"); }
        ZB_NEED_CTX(ctx);
        ZB_TRY(check_aligned("target", target, esz));
        if (drafted && drafts) ZB_TRY(check_aligned("drafted", drafted, esz));
        if (drafts) { ZB_TRY(check_aligned("tokens", tokens, 4)); ZB_TRY(check_aligned("accept", accept, 4)); }
        if (offsets) ZB_TRY(check_aligned("offsets", offsets, 4));
        ZB_TRY(check_aligned("sample", sample, 4)); ZB_TRY(check_aligned("accepted", accepted, 4)); ZB_TRY(check_aligned("next", next, 4));
        Stager s(ctx);
        const int it = s.in(target, t_bytes), id = s.in(drafts ? drafted : nullptr, d_bytes), ik = s.in(drafts ? tokens : nullptr, drafts * 4);
        const int io = s.in(offsets, (seqs + 1) * 4), ia = s.in(drafts ? accept : nullptr, drafts * 4), is = s.in(sample, seqs * 4);
        const int ic = s.out(accepted, seqs * 4), in = s.out(next, seqs * 4);
        ZB_TRY(s.commit());
        VerifyArgs a{};
        a.target = s.ptr<void>(it); a.target_stride = (long long)target_stride; a.drafted = s.ptr<void>(id); a.drafted_stride = (long long)drafted_stride;
        a.vocab = (int)vocab; a.tokens = s.ptr<int32_t>(ik); a.offsets = s.ptr<int32_t>(io); a.drafts = (int)drafts; a.seqs = (int)seqs; a.per = (int)(drafts / seqs);
        a.accept = s.ptr<float>(ia); a.sample = s.ptr<float>(is); a.accepted = s.ptr<int32_t>(ic); a.next = s.ptr<int32_t>(in);
        ZB_TRY(run_verify_drafts(ctx, dtype, a));
        return s.finish();
    });
}

}  // extern "C"
