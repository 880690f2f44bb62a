// Drafted tokens against the target's probabilities, with given random numbers.
//
//   draft i of a sequence stands while u_i q_i(d_i) < p_i(d_i); behind the first n that stand comes the token
//   min { v : sum of r_w over w <= v  >  u sum of r },   r = max(p_n - q_n, 0), or p_n where all drafts stand
//
// Probabilities are what the program has made of its logits, so that everything here is exact but sums, which are fp64: products of
// two fp32 numbers and differences fit 53 bits, and the border of a token in the running sum is off by 2^-53 of the whole, 2^29 times less than an fp32 sum's.
//
// Bound by memory: a sequence's own two rows are read once, in segments (16 a CTA, a warp each with 16 loads of a lane under way, up to 8 CTAs a sequence) whose sums every CTA of the
// cluster gets; the CTA that has the segment in which the border lies reads that one again, each thread some neighbouring probabilities.  Rows start at any address (vocabularies are odd), so loads
// are of single ones.  64 sequences of 128001 fp32 probabilities: 23.5 us (2.8 TB/s); 4 of 32000: 6.8 in a graph.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "context.cuh"
#include "ptx_sm100.cuh"
#include "row_codes.cuh"

namespace zb {

struct VerifyArgs {
    const void* target; long long target_stride; const void* drafted; long long drafted_stride; int vocab;
    const int32_t* tokens; const int32_t* offsets; int drafts, seqs, per;
    const float* accept; const float* sample;
    int32_t* accepted; int32_t* next;
    int parts;
};

struct VerifyShared {
    static constexpr int THREADS = 512, SEGS = 16, PARTS = 8;
    double seg[SEGS];                                 // a warp's sums, of this CTA's part of the row
    double all[SEGS * PARTS];
    double warp_sum[SEGS];
    double total, before;
    int n, begin, end, mine, found, last;
};

// A probability; what is none (NaN, negative, infinite) counts as 0.  (One comparison: the others' bits are not below infinity's.)
__device__ __forceinline__ float verify_number(float v) { return __float_as_uint(v) < 0x7f800000u ? v : 0.0f; }

template <typename T>
__global__ void __launch_bounds__(VerifyShared::THREADS) verify_drafts_kernel(const __grid_constant__ VerifyArgs a) {
    using Sh = VerifyShared;
    __shared__ Sh sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, P = a.parts;
    const int part = P > 1 ? (int)ptx::cluster_rank() : 0, s = (int)(blockIdx.x / (unsigned)P);
    ptx::grid_start();
    const T* target = static_cast<const T*>(a.target);
    const T* drafted = static_cast<const T*>(a.drafted);
    if (warp == 0) {
        const int b = a.offsets ? min(max(a.offsets[s], 0), a.drafts) : s * a.per;
        int e = a.offsets ? min(max(a.offsets[s + 1], b), a.drafts) : b + a.per;
        int n = 0;
        for (bool more = true; more && b + n < e;) {
            const int i = b + n + lane;
            int state = 0;                            // 0 stands, 1 does not, 2 no draft
            if (i < e) {
                const int t = a.tokens[i];
                if (t < 0) state = 2;
                else if (t >= a.vocab) state = 1;
                else {
                    const double p = as_float(target[(long long)(i + s) * a.target_stride + t]);
                    const double q = drafted ? (double)as_float(drafted[(long long)i * a.drafted_stride + t]) : 1.0;
                    state = (double)a.accept[i] * q < p ? 0 : 1;
                }
            } else state = 2;
            const unsigned stop = __ballot_sync(0xffffffffu, state != 0);
            if (stop) {
                const int first = __ffs(stop) - 1;
                n += first;
                if (__shfl_sync(0xffffffffu, state, first) == 2) e = b + n;
                more = false;
            } else n += 32;
        }
        if (lane == 0) { sh.n = n; sh.begin = b; sh.end = e; }
    }
    __syncthreads();
    const int n = sh.n, at = sh.begin + n;
    const T* p = target + (long long)(at + s) * a.target_stride;
    bool less = at < sh.end;                          // a draft that did not stand
    const T* q = less && drafted ? drafted + (long long)at * a.drafted_stride : nullptr;
    const int given = less && !drafted ? a.tokens[at] : -1;
    auto mass = [&](int v) -> double {
        const float pv = verify_number(as_float(p[v])), qv = !less ? 0.0f : (q ? verify_number(as_float(q[v])) : (v == given ? 1.0f : 0.0f));
        return pv > qv ? (double)pv - (double)qv : 0.0;
    };
    // segments in order: warp w of part i has the (16 i + w)-th
    const int segs = P * Sh::SEGS;
    auto seg_begin = [&](int i) { return (int)((long long)a.vocab * i / segs); };
    const double u = a.sample[s];
    for (int round = 0; round < 2; ++round) {
        const int v0 = seg_begin(part * Sh::SEGS + warp), v1 = seg_begin(part * Sh::SEGS + warp + 1);
        constexpr int U = 8;
        double sum = 0.0;
        for (int v = v0 + lane; v < v1; v += 32 * U) {
            float pv[U], qv[U];
#pragma unroll
            for (int i = 0; i < U; ++i) pv[i] = v + 32 * i < v1 ? as_float(p[v + 32 * i]) : 0.0f;
            if (less && q) {
#pragma unroll
                for (int i = 0; i < U; ++i) qv[i] = v + 32 * i < v1 ? as_float(q[v + 32 * i]) : 0.0f;
            } else {
#pragma unroll
                for (int i = 0; i < U; ++i) qv[i] = less && v + 32 * i == given ? 1.0f : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                // (compared in fp32, which is exact: comparisons of 64 bits were the busiest instructions)
                const float less_by = verify_number(qv[i]);
                const bool keep = pv[i] > less_by && pv[i] < INFINITY;
                sum += (double)(keep ? pv[i] : 0.0f) - (double)(keep ? less_by : 0.0f);
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) sh.seg[warp] = sum;
        if (tid == 0) { sh.found = 0x7fffffff; sh.last = -1; }
        __syncthreads();
        if (P > 1) {
            ptx::cluster_arrive(); ptx::cluster_wait();
            if (tid < segs) {
                double v;
                asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(ptx::cluster_addr(ptx::smem_u32(&sh.seg[tid % Sh::SEGS]), (uint32_t)(tid / Sh::SEGS))) : "memory");
                sh.all[tid] = v;
            }
            __syncwarp();
            ptx::cluster_arrive(); ptx::cluster_wait();       // nobody leaves, or goes on to its next sums, while its sums are read
        } else if (tid < segs) sh.all[tid] = sh.seg[tid];
        __syncthreads();
        if (warp == 0) {
            // each lane has neighbouring segments: where the running sum passes the border, and the last segment that holds anything
            const int each = (segs + 31) / 32;
            double own = 0.0;
            for (int i = 0; i < each; ++i) own += lane * each + i < segs ? sh.all[lane * each + i] : 0.0;
            double run = own;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const double o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
            const double total = __shfl_sync(0xffffffffu, run, 31), border = u * total;
            double sofar = run - own;
            int mine = 0x7fffffff, filled = -1;
            double mine_before = 0.0, filled_before = 0.0;
            for (int i = 0; i < each && lane * each + i < segs; ++i) {
                const double v = sh.all[lane * each + i];
                if (v > 0.0) { filled = lane * each + i; filled_before = sofar; }
                if (mine == 0x7fffffff && v > 0.0 && sofar + v > border) { mine = lane * each + i; mine_before = sofar; }
                sofar += v;
            }
            int best = mine, most = filled;
#pragma unroll
            for (int d = 16; d; d >>= 1) { best = min(best, __shfl_xor_sync(0xffffffffu, best, d)); most = max(most, __shfl_xor_sync(0xffffffffu, most, d)); }
            if (best != 0x7fffffff ? mine == best : (most >= 0 && filled == most)) { sh.mine = best != 0x7fffffff ? best : most; sh.before = best != 0x7fffffff ? mine_before : filled_before; }
            if (lane == 0) sh.total = total;
        }
        __syncthreads();
        const double total = sh.total, border = u * total;
        if (total == 0.0) {
            if (less && round == 0) { less = false; __syncthreads(); continue; }       // nothing is left of the target's row: the row itself
            if (part == 0 && tid == 0) { a.accepted[s] = n; a.next[s] = -1; }
            return;
        }
        const int mine = sh.mine;
        if (mine / Sh::SEGS != part) return;
        const int w0 = seg_begin(mine), w1 = seg_begin(mine + 1), each = (w1 - w0 + Sh::THREADS - 1) / Sh::THREADS;
        const int from = min(w1, w0 + tid * each), to = min(w1, from + each);
        double own = 0.0;
        for (int v = from; v < to; ++v) own += mass(v);
        double run = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const double o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
        if (lane == 31) sh.warp_sum[warp] = run;
        __syncthreads();
        double sofar = sh.before + (run - own);
        for (int i = 0; i < warp; ++i) sofar += sh.warp_sum[i];
        int found = 0x7fffffff, last = -1;
        for (int v = from; v < to; ++v) {
            const double r = mass(v);
            sofar += r;
            if (r > 0.0) { last = v; if (found == 0x7fffffff && sofar > border) found = v; }
        }
        if (found != 0x7fffffff) atomicMin(&sh.found, found);
        if (last >= 0) atomicMax(&sh.last, last);
        __syncthreads();
        if (tid == 0) { a.accepted[s] = n; a.next[s] = sh.found != 0x7fffffff ? sh.found : sh.last; }
        return;
    }
}

inline int32_t run_verify_drafts(zant_ctx* ctx, int32_t dtype, VerifyArgs a) {
    int parts = 1;
    while (parts < 8 && (long long)a.seqs * parts * 2 <= 4LL * ctx->sm_count && a.vocab / (parts * 2) >= 4096) parts *= 2;
    a.parts = parts;
    auto go = [&](auto kernel) {
        launch_cluster(ctx, kernel, dim3((unsigned)((long long)a.seqs * parts)), VerifyShared::THREADS, 0, (unsigned)parts, a);
        return check_launch(ctx, "verify_drafts_kernel");
    };
    if (dtype == ZANT_F32) return go(verify_drafts_kernel<float>);
    if (dtype == ZANT_F16) return go(verify_drafts_kernel<__half>);
    return go(verify_drafts_kernel<__nv_bfloat16>);
}

}  // namespace zb
