// Attention of many new tokens (prompts, parts of them) over the cache of kv_cache.cuh on tcgen05: the formulas and masks of kv_attention.cuh for results in 16 bits.
//
// A CTA has 256 rows, (new token, head) pairs that share a key head, as two tiles of 128 (with more than 128 dimensions one tile, whose sums take half of tensor memory).  Steps of 128 tokens, whose scores come in halves of 64 with a place each in tensor memory: while a
// row's thread takes the exponentials of one half, the tensor core multiplies V with the other half's weights and takes the next step's scores in its place.  (Whole steps with one
// place: the rows waited 1300 clocks of 4500 for their next scores.)  Codes become f16 (exactly) once for all 256 rows; q is f16 times a power of two for each row, so that its largest value lies in
// [2^14, 2^15) (f16 and bf16 values lose nothing down to 2^-28 of that one).  Scores are 128 x 64 x dim products into tensor memory; each thread has a row of them, finds its maximum, and
// writes the weights back over them as f16, where they are the next product's operand.
//
// A page's scale of K multiplies its columns' scores; its scale of V, over the largest VS of the pages that the CTA sees, goes into the exponent: weights are 2^(x + lv - M + 6) with
// lv = log2(vs / VS) and M a row's own largest x + lv, so that what is rounded to f16 is at most 2^14 (M is raised when one of a warp's rows has grown by 2^8, and then what has been summed is
// rescaled), and what is lost below f16's least numbers is 2^-31 of the row's largest weight times scale, wherever the scales of pages that other rows see lie.  The sum of the weights takes a page's
// factor out again, once for 16 tokens: it is one of 2^(x - M), and in range while scales lie within 2^80 of one another.  CTAs that see others, or a scale of 0, have a form of the rows' code for themselves
// (DEEP) that keeps a second maximum, of x, for it.
//
// A prompt of 8192 tokens, 40 over 8 heads of 128: 814 us (844 TFLOP/s, causal; 52 % of what cuBLAS reaches).  Exponentials and the tensor core are busy 40 % of the time each; a thread's chain of
// loads from tensor memory, exponentials, packing and stores takes 1400 clocks a half step, waits, votes and addresses around it 900.
//
//   warps 0 .. 3, 4 .. 7  q to f16, rows of the first and the second tile      12  TMEM owner, MMA issuer      8 .. 11, 13 .. 15  codes to f16, scales
// Registers: 136 for the rows' threads, 120 for others (setmaxnreg; 128 each at launch).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "context.cuh"
#include "kv_attention.cuh"
#include "kv_cache.cuh"
#include "ptx_sm100.cuh"
#include "row_codes.cuh"

namespace zb {

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
          "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Waits for the thread's loads; the registers of one of them are only read behind it.
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}

// f16 operands, fp32 sums, K-major A; B K-major, or with its N index the contiguous one.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major) {
    return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// One lane of a whole warp (`leader`): D (+)= A B with A in shared memory, or in tensor memory.  Operands in shared memory are rows of 128 bytes in the 128-byte swizzle, 8 rows
// 1024 bytes: K index in the row (K-major), or N index in the row and the next 64 of them `block` bytes further.  Descriptors as halves: the upper one is the same for all.
constexpr uint32_t kKvDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t kv_desc_lo(uint32_t addr, uint32_t block) { return (addr >> 4) | ((block >> 4) << 16); }
__device__ __forceinline__ void mma_f16_ss_if(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, {%6, %6, %6, %6}, p;\n\t}\n"
                 ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(leader), "r"(0u), "r"(kKvDescHi) : "memory");
}
__device__ __forceinline__ void mma_f16_ts_if(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b64 db, {%2, %7};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, {%6, %6, %6, %6}, p;\n\t}\n"
                 ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(leader), "r"(0u), "r"(kKvDescHi) : "memory");
}

// A warpgroup's registers a thread; the shares of all warpgroups add up to what the CTA was launched with.
template <int N> __device__ __forceinline__ void set_registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void set_registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int DP_>
struct KvPromptCfg {
    static constexpr int DP = DP_, TILES = DP > 128 ? 1 : 2, ROWS = 128 * TILES, THREADS = 512;
    // K and V come in units of 128 tokens, of 256 dimensions of 64 (a half of a step); two of each are there
    static constexpr int UNIT = DP > 128 ? 64 : 128, UNITS = 128 / UNIT;
    static constexpr int Q_BLOCK = 128 * 128, BLOCK = UNIT * 128;      // rows of 64 f16 numbers: of a tile's q, of a unit
    static constexpr int Q_OPERAND = Q_BLOCK * (DP / 64), OPERAND = BLOCK * (DP / 64);
    static constexpr int OFF_K = TILES * Q_OPERAND, OFF_V = OFF_K + 2 * OPERAND, OFF_REST = OFF_V + 2 * OPERAND;
    static constexpr int LPR = DP / 16;               // lanes of a row of codes
    static constexpr int TPL = 32 / LPR;              // tokens of a warp's load
    static constexpr int ROWS_REGS = 136, OTHER_REGS = 120;       // 256 x 136 + 256 x 120 = 512 x 128
    static constexpr int INFO = 36, RING = 8;         // words of a step: scales of K, lv, 2^-(lv + 6) of 16 tokens each, which of them there are, which have scales of NaN or far below VS; where they lie
    // factors of rows, info of RING steps, maxima and minima of scales, barriers, address of TMEM, flag
    static constexpr int OFF_INFO = OFF_REST + ROWS * 4, OFF_MAX = OFF_INFO + RING * INFO * 4, OFF_BAR = OFF_MAX + 64, OFF_TMEM = OFF_BAR + 30 * 8, SMEM = OFF_TMEM + 16;
};
struct KvPromptBars {
    uint32_t at;
    __device__ __forceinline__ uint32_t k_full(int s) const { return at + 8 * s; }
    __device__ __forceinline__ uint32_t v_full(int s) const { return at + 16 + 8 * s; }
    __device__ __forceinline__ uint32_t k_empty(int s) const { return at + 32 + 8 * s; }
    __device__ __forceinline__ uint32_t v_empty(int s) const { return at + 48 + 8 * s; }
    __device__ __forceinline__ uint32_t s_full(int x, int b) const { return at + 64 + 16 * x + 8 * b; }
    __device__ __forceinline__ uint32_t p_full(int x, int b) const { return at + 96 + 16 * x + 8 * b; }
    __device__ __forceinline__ uint32_t pv_done(int x) const { return at + 128 + 8 * x; }
    __device__ __forceinline__ uint32_t o_full(int x) const { return at + 144 + 8 * x; }
    __device__ __forceinline__ uint32_t q_full() const { return at + 160; }
    __device__ __forceinline__ uint32_t drained() const { return at + 168; }
    __device__ __forceinline__ uint32_t info_full(int s) const { return at + 176 + 8 * s; }
};

// What all roles know of the CTA's rows.
struct KvPromptTile {
    int s, row, first, row0, rows, h;                 // sequence, its first row, position of its first new token, first of the CTA's rows, how many, key head
    int low0, low1, high0, high1;                     // positions of either tile's first and last row (high < 0: the tile has none, or sees nothing)
    __device__ __forceinline__ int low(int x) const { return x ? low1 : low0; }
    __device__ __forceinline__ int high(int x) const { return x ? high1 : high0; }
    __device__ __forceinline__ int last() const { return max(high0, high1); }
};

// The steps of a tile: those behind the sinks' own from `from` on and before `to` are its (and all of the sinks' before `to`); of these it sees all of the tokens from
// `whole_from` on and before `whole_to`.
struct KvPromptSteps {
    int sink, from, to, whole_from, whole_to;
    __device__ __forceinline__ KvPromptSteps(const KvSteps& s, int low, int high, int window, int sinks) {
        // a step k behind the sinks' begins at 128 (k + add)
        const int add = s.first - s.sink;
        sink = s.sink > 0 ? s.sink : (int)min(((long long)sinks + 127) / 128, (long long)s.total);      // (none of their own: they are in front of `from` all the same)
        to = high < 0 ? 0 : min(s.total, high < 128 * s.first ? min(s.sink, high / 128 + 1) : high / 128 + 1 - add);
        from = window > 0 && low - window + 1 > 0 ? (low - window + 1) / 128 - add : 0;
        whole_to = min(to, low < 127 ? 0 : (low - 127) / 128 + 1 - add);
        whole_from = max(s.sink, window > 0 && high - window + 1 > 0 ? (high - window + 1 + 127) / 128 - add : 0);
    }
    __device__ __forceinline__ bool active(int k) const { return k < to && (k < sink || k >= from); }
    __device__ __forceinline__ bool whole(int k) const { return k >= whole_from && k < whole_to; }
};

// lv of a page whose scale of V is 0: below all others' by more than a weight can make up for.
constexpr float kKvNoScale = -400.0f;
// Pages whose scale is below this part of the largest are far below it.
constexpr float kKvFar = 0x1p-80f;

// The largest of the seven warps' numbers.
__device__ __forceinline__ float kv_prompt_top(const float* part) {
    float v = part[0];
#pragma unroll
    for (int i = 1; i < 7; ++i) v = fmaxf(v, part[i]);
    return v;
}

// A whole warp's wait: polls in turns of 64, one vote and one branch each (mbar_wait's lanes branch by themselves: the waiting warps took a third of all instructions).
__device__ __forceinline__ bool kv_wait(const KvAttendArgs& a, uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    long long t0 = 0;
    while (true) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred P, Q, R;\n\t.reg .u32 n;\n\tmov.u32 n, 0;\n"
                     "KV_WAIT_%=:\n\tmbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\tvote.sync.all.pred Q, P, 0xffffffff;\n\t@Q bra.uni KV_DONE_%=;\n\t"
                     "add.u32 n, n, 1;\n\tsetp.lt.u32 R, n, 64;\n\t@R bra.uni KV_WAIT_%=;\n"
                     "KV_DONE_%=:\n\tselp.u32 %0, 1, 0, Q;\n\t}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        const bool flag = *abort_flag != 0;
        const long long now = clock64();
        if (t0 == 0) t0 = now;
        const bool late = now - t0 > a.wait_budget;
        if (late) *abort_flag = 1;
        if (__any_sync(0xffffffffu, flag || late)) return false;
    }
}

// Codes on their way to f16 operands: warp `warp` of the seven takes every seventh TPL tokens of a unit.
template <typename F>
struct KvConvert {
    static constexpr int WARPS = 7, LPR = F::LPR, GROUPS = F::UNIT / F::TPL, N = (GROUPS + WARPS - 1) / WARPS;
    uint4 w[N];
    // block_of(i): where the i-th 16 tokens lie in the cache, in units of 16 tokens (-1: nowhere); mine: the lane's 16 bytes are dimensions of the head
    template <typename B>
    __device__ __forceinline__ void load(const int8_t* codes, B&& block_of, int warp, int dim, int in_group, int column, bool mine) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int group = i * WARPS + warp, tok = group * F::TPL;
            const int block = GROUPS % WARPS == 0 || group < GROUPS ? block_of(tok >> 4) : -1;
            const int8_t* p = codes + (unsigned long long)(unsigned)block * (unsigned)(16 * dim) + (unsigned)(((tok & 15) + in_group) * dim + column);
            w[i] = make_uint4(0, 0, 0, 0);
            if (mine && block >= 0) w[i] = ptx::ld_global_once(reinterpret_cast<const uint4*>(p));     // (past L1)
        }
    }
    // to: the operand, and the lane's place in row in_group of it
    __device__ __forceinline__ void store(uint8_t* to, int warp, int in_group, int chunk) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int group = i * WARPS + warp, row = group * F::TPL + in_group;
            if (GROUPS % WARPS != 0 && group >= GROUPS) continue;      // (whole warps)
            const uint32_t r[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            uint32_t f[8];
#pragma unroll
            for (int z = 0; z < 4; ++z) { f[2 * z] = codes_f16(r[z]); f[2 * z + 1] = codes_f16(r[z] >> 8); }       // (numbers 0, 2, 1, 3 of each four)
            uint8_t* at = to + row * 128;
            *reinterpret_cast<uint4*>(at + ((chunk ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<uint4*>(at + (((chunk + 1) ^ (row & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
        }
    }
};
__device__ __forceinline__ void kv_written(uint32_t bar) {
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar);
}
// Pages of 16 tokens each of step k: lane i (of 8) has the i-th.
__device__ __forceinline__ int kv_prompt_page(const KvAttendArgs& a, const KvPromptTile& tile, const KvSteps& steps, int k) {
    if (k >= steps.total) return -1;
    const int t = steps.at(k, 128) + 16 * (threadIdx.x & 7);
    return kv_seen16(t, tile.low0, tile.last(), a.window, a.sinks) ? (int)kv_page(a.c, tile.s, t >> a.c.page_log2) : -1;
}
// Where these 16 tokens lie in the cache, in units of 16 tokens (below 2^31: 16 tokens are 256 bytes at least).
__device__ __forceinline__ int kv_prompt_block(const KvArgs& c, const KvPromptTile& tile, const KvSteps& steps, int k, int page) {
    if (page < 0) return -1;
    const int t = steps.at(k, 128) + 16 * (threadIdx.x & 7);
    return (int)((((unsigned)page * (unsigned)c.heads + (unsigned)tile.h) << (c.page_log2 - 4)) + (unsigned)((t & (c.page - 1)) >> 4));
}

// ---- warps 0 .. 7, while the first codes are on their way: q as f16, a power of two for each row.  Says whether the CTA sees scales far below the largest (1, or 0; -1: given up), which it reads before q counts as
// written: the steps' information is not written anew until then.
template <typename F>
__device__ __forceinline__ int kv_prompt_queries(const KvAttendArgs& a, const KvPromptTile& tile, const KvPromptBars& bar, uint8_t* smem, volatile int* abort_flag) {
    constexpr int LPR = F::LPR, TPL = F::TPL;
    const KvArgs& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, which = lane % LPR, in_group = lane / LPR, column = which * 16, chunk = (which & 3) * 2;
    const bool mine = column < c.dim;
    float* row_factor = reinterpret_cast<float*>(smem + F::OFF_REST);
    uint8_t* operand = smem + (which >> 2) * F::Q_BLOCK;
    constexpr int N = F::ROWS / TPL / 8, U = N < 4 ? N : 4;       // a warp's turns; rows that a lane has under way (one at a time: 14800 clocks for all)
#pragma unroll 1
    for (int g0 = 0; g0 < N; g0 += U) {
        uint32_t raw[U][8];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int r = ((g0 + i) * 8 + warp) * TPL + in_group, row = tile.row0 + r;
#pragma unroll
            for (int z = 0; z < 8; ++z) raw[i][z] = 0;
            if (r < tile.rows && mine)
                kv_load16(static_cast<const __half*>(a.q) + (long long)(tile.row + row / a.group) * a.q_stride + (long long)(tile.h * a.group + row % a.group) * c.dim + column, a.wide_q, raw[i]);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int r = ((g0 + i) * 8 + warp) * TPL + in_group;
            float v[16];
            if (a.q_type == ZANT_F16) { RowChunk<__half>::values(raw[i], v); RowChunk<__half>::values(raw[i] + 4, v + 8); }
            else { RowChunk<__nv_bfloat16>::values(raw[i], v); RowChunk<__nv_bfloat16>::values(raw[i] + 4, v + 8); }
            float big = 0.0f;
            bool odd = false;
#pragma unroll
            for (int z = 0; z < 16; ++z) { big = fmaxf(big, fabsf(v[z])); odd |= !(fabsf(v[z]) < INFINITY); }
#pragma unroll
            for (int d = LPR / 2; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
            odd = (__ballot_sync(0xffffffffu, odd) >> (lane / LPR * LPR)) & ((1u << LPR) - 1u);
            const int e = min(max((int)(__float_as_uint(big) >> 23) - 127 - 14, -114), 127);
            // (a negative scale's sign goes into q: scores are multiplied by positive numbers only)
            const float down = odd ? 0.0f : copysignf(__uint_as_float((uint32_t)(127 - e) << 23), a.scale_log2);
            const float up = odd ? __uint_as_float(0x7fffffffu) : __uint_as_float((uint32_t)max(127 + e, 1) << 23);
            if (which == 0) row_factor[r] = up * fabsf(a.scale_log2);
            uint32_t f[8];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                float x[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) x[y] = odd ? 0.0f : v[4 * z + y] * down;
                f[2 * z] = pack_f16(x[0], x[2]);
                f[2 * z + 1] = pack_f16(x[1], x[3]);
            }
            uint8_t* to = operand + (r >> 7) * F::Q_OPERAND + (r & 127) * 128;
            *reinterpret_cast<uint4*>(to + ((chunk ^ (r & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<uint4*>(to + (((chunk + 1) ^ (r & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
        }
    }
    if (!kv_wait(a, bar.info_full(0), 0, abort_flag)) return -1;
    const int any_far = (reinterpret_cast<const volatile int*>(smem + F::OFF_INFO)[25] >> 24) & 1;
    kv_written(bar.q_full());
    return any_far;
}

// ---- warps 8 .. 11 and 13 .. 15: the largest scale of V; K, V and what each step's pages say.  Codes are on their way a step ahead.
template <typename F>
__device__ __forceinline__ void kv_prompt_convert(const KvAttendArgs& a, const KvPromptTile& tile, const KvSteps& steps, const KvPromptBars& bar, uint8_t* smem, volatile int* abort_flag) {
    constexpr int LPR = F::LPR;
    const KvArgs& c = a.c;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - ((threadIdx.x >> 5) < 12 ? 8 : 9), pl = c.page_log2;
    float* info = reinterpret_cast<float*>(smem + F::OFF_INFO);
    float* part = reinterpret_cast<float*>(smem + F::OFF_MAX);
    // the lane's 16 dimensions of a token: their place in its row of codes, and in an operand's
    const int which = lane % LPR, in_group = lane / LPR, column = which * 16, chunk = (which & 3) * 2;
    const bool mine = column < c.dim;
    uint8_t* operand = smem + (which >> 2) * F::BLOCK;
    KvConvert<F> kc, vc;
    // The last warp (it has the fewest tokens) says what a step's pages are like, two steps before the others ask: in the place of step k - 6 then, whose weights have been taken, or
    // step k - 1's K would not have had room.
    int page = -1;
    float ks = 0.0f, vsc = 0.0f;
    auto look = [&](int k) {                          // on their way
        page = kv_prompt_page(a, tile, steps, k);
        ks = page >= 0 ? c.k_scale[(long long)page * c.heads + tile.h] : 0.0f;
        vsc = page >= 0 ? c.v_scale[(long long)page * c.heads + tile.h] : 0.0f;
    };
    auto tell = [&](int k, float vs, bool any_far) {
        float* i = info + (k & (F::RING - 1)) * F::INFO;
        const bool k_nan = !(fabsf(ks) < INFINITY), v_nan = !(fabsf(vsc) < INFINITY);
        const float ratio = page >= 0 && vs > 0.0f && !v_nan ? fabsf(vsc) / vs : 1.0f;
        const bool deep = ratio < kKvFar;             // (where the quotient may be below the least number, the logarithms are not: 2^-277 at the least, and for 0 something less)
        const float lv = deep ? fmaxf(__log2f(fabsf(vsc) * 0x1p64f) - 64.0f - __log2f(vs), kKvNoScale) : fminf(__log2f(ratio), 0.0f);
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0), bad_k = __ballot_sync(0xffffffffu, k_nan), bad_v = __ballot_sync(0xffffffffu, v_nan), far = __ballot_sync(0xffffffffu, deep);
        if (lane < 8) {
            i[lane] = k_nan ? 0.0f : fabsf(ks); i[8 + lane] = lv; i[16 + lane] = deep ? 0.0f : ex2(-lv - 6.0f);
            reinterpret_cast<int*>(i)[28 + lane] = kv_prompt_block(c, tile, steps, k, page);
        }
        if (lane == 0) { reinterpret_cast<int*>(i)[24] = (int)(there & 255u); reinterpret_cast<int*>(i)[25] = (int)((bad_k & 255u) | ((bad_v & 255u) << 8) | ((far & 255u) << 16) | (any_far ? 1u << 24 : 0u)); }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar.info_full(k & (F::RING - 1)));
    };
    auto blocks = [&](int u) { return [=](int i) { return reinterpret_cast<const int*>(info + ((u / F::UNITS) & (F::RING - 1)) * F::INFO)[28 + (u % F::UNITS) * (F::UNIT / 16) + i]; }; };
    // the first unit's codes before anything else
    look(0);
    const int first = kv_prompt_block(c, tile, steps, 0, page);
    auto first_block = [&](int i) { return __shfl_sync(0xffffffffu, first, i & 7); };
    kc.load(c.k, first_block, warp, c.dim, in_group, column, mine);
    vc.load(c.v, first_block, warp, c.dim, in_group, column, mine);

    float top = 0.0f, least = INFINITY;
    if (steps.total > 0) {
        const int low = tile.low0, high = tile.last(), from = a.window > 0 ? max(low - a.window + 1, 0) >> pl : 0, to = (high >> pl) + 1;
        const int sink_pages = a.sinks > 0 ? min(((a.sinks - 1) >> pl) + 1, from) : 0;
#pragma unroll 2
        for (int i = warp * 32 + lane; i < sink_pages + to - from; i += 224) {
            const long long id = kv_page(c, tile.s, i < sink_pages ? i : i - sink_pages + from);
            if (id >= 0) {
                const float scale = fabsf(kv_scale(c.v_scale[id * c.heads + tile.h]));       // (NaN is neither the largest nor the least)
                top = fmaxf(top, scale);
                least = fminf(least, scale);
            }
        }
    }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
    if (lane == 0) { part[warp] = top; part[8 + warp] = -least; }

    __syncwarp();
    ptx::named_barrier_sync(1, 224);                  // (in front of any wait that may be given up)
    const float vs = kv_prompt_top(part);
    const bool any_far = -kv_prompt_top(part + 8) * (1.0f / kKvFar) < vs;
    if (warp == 6) {
        tell(0, vs, any_far);
        look(1);
        tell(1, vs, false);
        look(2);
    }

#pragma unroll 1
    for (int u = 0; u < steps.total * F::UNITS; ++u) {
        const int k = u / F::UNITS;
        const uint32_t free_parity = ((uint32_t)(u >> 1) & 1u) ^ 1u;
        if (!kv_wait(a, bar.info_full((k + 1) & (F::RING - 1)), (uint32_t)((k + 1) / F::RING) & 1u, abort_flag)) return;
        if (!kv_wait(a, bar.k_empty(u & 1), free_parity, abort_flag)) return;
        kc.store(operand + F::OFF_K + (u & 1) * F::OPERAND, warp, in_group, chunk);
        kv_written(bar.k_full(u & 1));
        kc.load(c.k, blocks(u + 1), warp, c.dim, in_group, column, mine);
        if (warp == 6 && u % F::UNITS == 0) {
            tell(k + 2, vs, false);
            look(k + 3);
        }
        if (!kv_wait(a, bar.v_empty(u & 1), free_parity, abort_flag)) return;
        vc.store(operand + F::OFF_V + (u & 1) * F::OPERAND, warp, in_group, chunk);
        kv_written(bar.v_full(u & 1));
        vc.load(c.v, blocks(u + 1), warp, c.dim, in_group, column, mine);
    }
}

// ---- warp 12
template <typename F>
__device__ __forceinline__ void kv_prompt_mma(const KvAttendArgs& a, const KvPromptTile& tile, const KvSteps& steps, const KvPromptBars& bar, uint32_t s0, uint32_t tmem, volatile int* abort_flag) {
    constexpr int DP = F::DP;
    constexpr uint32_t idesc_s = idesc_f16(128, 64, false), idesc_o = idesc_f16(128, DP, true);
    const uint32_t leader = ptx::elect_one() ? 1u : 0u;
    int count[2] = {0, 0};                            // a tile's steps so far
    const KvPromptSteps mine[2] = {KvPromptSteps(steps, tile.low0, tile.high0, a.window, a.sinks), KvPromptSteps(steps, tile.low1, tile.high1, a.window, a.sinks)};
    // where the half of a step lies: a part of its unit, or a unit of its own
    auto unit_at = [&](int k, int b) { return (uint32_t)(F::UNITS == 1 ? (k & 1) * F::OPERAND + b * 64 * 128 : b * F::OPERAND); };
    auto scores = [&](int x, int k, int b) {
        const uint32_t qa = kv_desc_lo(s0 + x * F::Q_OPERAND, 16), kb = kv_desc_lo(s0 + F::OFF_K + unit_at(k, b), 16);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
            mma_f16_ss_if(leader, tmem + x * 128 + b * 64, qa + (((i >> 2) * F::Q_BLOCK + (i & 3) * 32) >> 4), kb + (((i >> 2) * F::BLOCK + (i & 3) * 32) >> 4), idesc_s, i > 0);
        ptx::mma_commit_if(leader, bar.s_full(x, b));
    };
    auto values = [&](int x, int k, int b) {
        const uint32_t vb = kv_desc_lo(s0 + F::OFF_V + unit_at(k, b), F::BLOCK);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_f16_ts_if(leader, tmem + 256 + x * DP, tmem + x * 128 + b * 64 + i * 8, vb + i * (2048 >> 4), idesc_o, (count[x] | b | i) != 0);
        ptx::mma_commit_if(leader, bar.pv_done(x));
        if (b == 1 && k == mine[x].to - 1) ptx::mma_commit_if(leader, bar.o_full(x));      // its last step
    };
    if constexpr (F::UNITS == 2) {
        // one tile; the halves have barriers of their own
        if (steps.total > 0) {
            if (!kv_wait(a, bar.q_full(), 0, abort_flag)) return;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (!kv_wait(a, bar.k_full(b), 0, abort_flag)) return;
                ptx::tc_fence_after();
                if (mine[0].active(0)) scores(0, 0, b);
                ptx::mma_commit_if(leader, bar.k_empty(b));
            }
        }
        for (int k = 0; k < steps.total; ++k) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (!kv_wait(a, bar.v_full(b), (uint32_t)k & 1u, abort_flag)) return;
                if (mine[0].active(k)) {
                    if (!kv_wait(a, bar.p_full(0, b), (uint32_t)count[0] & 1u, abort_flag)) return;
                    ptx::tc_fence_after();
                    values(0, k, b);
                    count[0] += b;
                }
                ptx::mma_commit_if(leader, bar.v_empty(b));
                if (k + 1 < steps.total) {
                    if (!kv_wait(a, bar.k_full(b), (uint32_t)(k + 1) & 1u, abort_flag)) return;
                    ptx::tc_fence_after();
                    if (mine[0].active(k + 1)) scores(0, k + 1, b);
                    ptx::mma_commit_if(leader, bar.k_empty(b));
                }
            }
        }
        return;
    }
    if (steps.total > 0) {
        if (!kv_wait(a, bar.q_full(), 0, abort_flag) || !kv_wait(a, bar.k_full(0), 0, abort_flag)) return;
        ptx::tc_fence_after();
#pragma unroll
        for (int i = 0; i < 4; ++i) if (mine[i & 1].active(0)) scores(i & 1, 0, i >> 1);
        ptx::mma_commit_if(leader, bar.k_empty(0));
    }
    for (int k = 0; k < steps.total; ++k) {
        const uint32_t parity = (uint32_t)(k >> 1) & 1u, next_parity = (uint32_t)((k + 1) >> 1) & 1u;
        if (!kv_wait(a, bar.v_full(k & 1), parity, abort_flag)) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                 // the first half of either tile, the second
            const int x = i & 1, b = i >> 1;
            if (mine[x].active(k)) {
                if (!kv_wait(a, bar.p_full(x, b), (uint32_t)count[x] & 1u, abort_flag)) return;
                ptx::tc_fence_after();
                values(x, k, b);
                count[x] += b;
            }
            if (i == 3) ptx::mma_commit_if(leader, bar.v_empty(k & 1));
            if (k + 1 < steps.total) {
                if (i == 0 && !kv_wait(a, bar.k_full((k + 1) & 1), next_parity, abort_flag)) return;
                ptx::tc_fence_after();
                if (mine[x].active(k + 1)) scores(x, k + 1, b);
            }
        }
        if (k + 1 < steps.total) ptx::mma_commit_if(leader, bar.k_empty((k + 1) & 1));
    }
}

// What scores are multiplied with: not 0, so that minus infinity stays what it is.
__device__ __forceinline__ float kv_prompt_factor(float f) { return f == 0.0f ? 1e-38f : f; }

// Weights of a row's 64 scores in tensor memory at `ts` (minus infinity: not seen), in pairs, under the base `base` (log2): p, their sum with each page's factor taken out (without pages far below VS, whose
// factor is none), and the largest exponents over the base, with the pages' scales (the result) and, of DEEP, without (`top_x`).
template <bool DEEP>
__device__ __forceinline__ float kv_prompt_weights(uint32_t ts, const float* info, float factor, float base, uint32_t (&p)[32], float& sum, float& top_x) {
    uint32_t v[64];
    float top = -INFINITY, plain = -INFINITY;
    sum = 0.0f;
    ptx::tmem_ld32(ts, v);
    ptx::tmem_ld32(ts + 32, v + 32);
    ptx::tmem_wait_ld32(v);
    ptx::tmem_wait_ld32(v + 32);
#pragma unroll
    for (int g = 0; g < 4; ++g) {                     // 16 tokens, which are on one page
        const float f = kv_prompt_factor(factor * info[g]);
        const float lv = info[8 + g], b = lv + 6.0f - base;
        const unsigned long long f2 = ptx::pack2(f, f), b2 = ptx::pack2(b, b);
        unsigned long long s2 = 0;
        float most = -INFINITY;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const float2 e = ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(v[16 * g + 2 * y]), __uint_as_float(v[16 * g + 2 * y + 1])), f2, b2));
            most = fmaxf(most, fmaxf(e.x, e.y));
            const float2 w = make_float2(ex2(e.x), ex2(e.y));
            s2 = ptx::add2(s2, ptx::pack2(w.x, w.y));
            p[8 * g + y] = pack_f16(w.x, w.y);
        }
        top = fmaxf(top, most);
        if (DEEP) plain = fmaxf(plain, most - lv);
        const float2 s1 = ptx::unpack2(s2);
        sum = fmaf(s1.x + s1.y, info[16 + g], sum);
    }
    top_x = plain - 6.0f;
    return top - 6.0f;
}
// The first n of 32 columns.
__device__ __forceinline__ uint32_t first_columns(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

// ---- warps 0 .. 7, a row each thread
//
// The base of the exponents is the maximum of earlier steps: one pass over the scores gives weights and their maximum, and only where that has grown by 2^8 (a row's first step, and few
// others) it is taken again.  (A pass for the maximum in front: twice the time.)  Steps that a row sees in part have minus infinity written over the other scores first, so that there is one
// form of the pass, which is what the instruction cache has to hold (with a second form for such steps beside it: 7000 clocks a step where this one takes 3300).  Pages with a scale of NaN count as
// zeros, and so do rows of q with one; the rows that see such a page, or anything, are noted and get their NaN at the end.
template <typename F, bool DEEP>
__device__ __forceinline__ void kv_prompt_rows(const KvAttendArgs& a, const KvPromptTile& tile, const KvSteps& steps, const KvPromptBars& bar, uint8_t* smem, uint32_t tmem, volatile int* abort_flag) {
    constexpr int DP = F::DP;
    const KvArgs& c = a.c;
    const int x = threadIdx.x >> 7, r = threadIdx.x & 127, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = x * 128 + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, to = tmem + 256 + x * DP + lanes;
    const float* all_info = reinterpret_cast<const float*>(smem + F::OFF_INFO);
    const int row = tile.row0 + min(mine, tile.rows - 1), pos = max(tile.first + row / a.group, -1);
    float factor = 0.0f, M = -INFINITY, l = 0.0f;       // l: the sum of 2^(x - M), of DEEP of 2^(x - m)
    float m = -INFINITY;
    const KvPromptSteps own(steps, tile.low(x), tile.high(x), a.window, a.sinks);
    int count = 0, spoilt = 0;                        // halves so far; 1: by a page's scale of K, or by q, 2: of V
    if (own.to > 0) {
        if (!kv_wait(a, bar.q_full(), 0, abort_flag)) return;
        factor = reinterpret_cast<const float*>(smem + F::OFF_REST)[mine];
        if (!(factor < INFINITY)) { factor = 0.0f; spoilt = 1; }
    }
    for (int j = 0; j < 2 * own.to; ++j) {            // halves of steps
        const int k = j >> 1, b = j & 1;
        if (!own.active(k)) continue;
        const uint32_t ts = tmem + x * 128 + b * 64 + lanes;
        if (!kv_wait(a, bar.s_full(x, b), (uint32_t)(count >> 1) & 1u, abort_flag)) return;
        ptx::tc_fence_after();
        // (what the step's pages say was said before its K was there)
        const float* info = all_info + (k & (F::RING - 1)) * F::INFO;
        const int2 pages = *reinterpret_cast<const int2*>(info + 24);
        if (pages.x != 255 || (pages.y & 0xffff) != 0 || !own.whole(k)) {
            const int there = pages.x >> (4 * b), k_nan = pages.y >> (4 * b), v_nan = pages.y >> (8 + 4 * b);       // of the half's four 16 tokens
            const int t = steps.at(k, 128) + 64 * b, upto = pos - t, behind = (a.window == 0 ? -1 : max(pos - a.window, -1)) - t, sunk = a.sinks - t;       // columns seen: <= upto, and > behind or < sunk
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
                uint32_t seen = first_columns(upto + 1 - 32 * g) & (~first_columns(behind + 1 - 32 * g) | first_columns(sunk - 32 * g));
                seen &= ((there >> (2 * g)) & 1 ? 0xffffu : 0u) | ((there >> (2 * g + 1)) & 1 ? 0xffff0000u : 0u);
                if (((seen & 0xffffu) && ((k_nan >> (2 * g)) & 1)) || ((seen >> 16) && ((k_nan >> (2 * g + 1)) & 1))) spoilt |= 1;
                if (((seen & 0xffffu) && ((v_nan >> (2 * g)) & 1)) || ((seen >> 16) && ((v_nan >> (2 * g + 1)) & 1))) spoilt |= 2;
                if (__all_sync(0xffffffffu, seen == 0xffffffffu)) continue;
                uint32_t v[32];
                ptx::tmem_ld32(ts + 32 * g, v);
                ptx::tmem_wait_ld32(v);
#pragma unroll
                for (int y = 0; y < 32; ++y) v[y] = (seen >> y) & 1u ? v[y] : 0xff800000u;
                tmem_st16(ts + 32 * g, v);
                tmem_st16(ts + 32 * g + 16, v + 16);
            }
            tmem_wait_st();
        }
        uint32_t p[32];
        float sum;
#pragma unroll 1
        for (int again = 0; again < 2; ++again) {
            float top_x;
            const float base = M == -INFINITY ? 0.0f : M, top = kv_prompt_weights<DEEP>(ts, info + 4 * b, factor, base, p, sum, top_x);
            const bool raise = M == -INFINITY ? top > -INFINITY : (top > 8.0f || (DEEP && base + top_x > m + 60.0f));       // (m only keeps the sum in range)
            if (again || !__any_sync(0xffffffffu, raise)) break;
            // rows that have grown at all go along
            const float M_now = fmaxf(M, base + top), f = M_now == M ? 1.0f : ex2(M - M_now);
            M = M_now;
            if (DEEP) {
                const float m_now = fmaxf(m, base + top_x);
                l *= m_now == m ? 1.0f : ex2(m - m_now);
                m = m_now;
            } else l *= f;
            if (count > 0) {
                // the half before is in the sums (the one before that was, or this one's scores would not have had room)
                if (!kv_wait(a, bar.pv_done(x), (uint32_t)(count - 1) & 1u, abort_flag)) return;
                ptx::tc_fence_after();
#pragma unroll 1
                for (int g = 0; g < DP / 16; ++g) {
                    uint32_t v[16];
                    ptx::tmem_ld16(to + g * 16, v);
                    tmem_wait_ld16(v);
#pragma unroll
                    for (int y = 0; y < 16; ++y) v[y] = __float_as_uint(__uint_as_float(v[y]) * f);
                    tmem_st16(to + g * 16, v);
                }
            }
        }
        if (!DEEP) l += sum;
        else {
            const float over = M == -INFINITY ? 1.0f : ex2(0.5f * (M - m)), bx = m == -INFINITY ? 0.0f : m;       // (its square may be too small where the product is not)
            l = fmaf(sum * over, over, l);
            int far = (reinterpret_cast<const volatile int*>(info)[25] >> (16 + 4 * b)) & 15;       // (the same for all rows) pages far below VS: their weights by themselves
#pragma unroll 1
            for (int g = 0; far != 0; ++g, far >>= 1) {
                if (!(far & 1)) continue;
                uint32_t v[16];
                ptx::tmem_ld16(ts + g * 16, v);
                tmem_wait_ld16(v);
                const float f = kv_prompt_factor(factor * info[4 * b + g]);
#pragma unroll
                for (int y = 0; y < 16; ++y) l += ex2(fmaf(__uint_as_float(v[y]), f, -bx));
            }
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) tmem_st16(ts + g * 16, p + 16 * g);
        tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar.p_full(x, b));
        ++count;
    }
    if (count > 0) {
        if (!kv_wait(a, bar.o_full(x), 0, abort_flag)) return;
        ptx::tc_fence_after();
    }
    const float* part = reinterpret_cast<const float*>(smem + F::OFF_MAX);
    const float vs = count > 0 ? kv_prompt_top(part) : 0.0f;
    const bool mine_there = mine < tile.rows;
    if (l == 0.0f) spoilt = 0;                        // (sees nothing)
    if (spoilt & 1) l = __uint_as_float(0x7fffffffu);
    float out_scale = l == 0.0f ? 0.0f : vs * (1.0f / 64.0f) / l;
    if (DEEP) {                                       // VS 2^(M - m) is a scale that the row has seen, or more than a weight below one: the power in four factors, none of which is too small
        const float quarter = l == 0.0f ? 0.0f : ex2(0.25f * (M - m));
        out_scale = out_scale * quarter * quarter * quarter * quarter;
    }
    if (spoilt) out_scale = __uint_as_float(0x7fffffffu);
    const long long token = tile.row + row / a.group, head = tile.h * a.group + row % a.group, at = token * a.out_stride + head * c.dim;
#pragma unroll
    for (int g = 0; g < DP / 16; ++g) {
        uint32_t v[16];
        __syncwarp();                                 // (lanes that have stored and lanes without a row load together)
        if (count > 0) {                              // (the same for the whole warp)
            ptx::tmem_ld16(to + g * 16, v);
            tmem_wait_ld16(v);
        } else {
#pragma unroll
            for (int y = 0; y < 16; ++y) v[y] = 0;
        }
        if (mine_there && g * 16 < c.dim) {
            uint32_t w[8];
#pragma unroll
            for (int y = 0; y < 4; ++y) {             // numbers 0, 2, 1, 3 of each four
                const float d0 = __uint_as_float(v[4 * y]) * out_scale, d2 = __uint_as_float(v[4 * y + 1]) * out_scale, d1 = __uint_as_float(v[4 * y + 2]) * out_scale,
                            d3 = __uint_as_float(v[4 * y + 3]) * out_scale;
                if (a.q_type == ZANT_F16) { w[2 * y] = pack_f16(d0, d1); w[2 * y + 1] = pack_f16(d2, d3); }
                else {
                    const __nv_bfloat162 b0 = __floats2bfloat162_rn(d0, d1), b1 = __floats2bfloat162_rn(d2, d3);
                    w[2 * y] = *reinterpret_cast<const uint32_t*>(&b0); w[2 * y + 1] = *reinterpret_cast<const uint32_t*>(&b1);
                }
            }
            uint16_t* o = static_cast<uint16_t*>(a.out) + at + g * 16;
            if (a.wide_out) {
                reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
#pragma unroll
                for (int y = 0; y < 16; ++y) o[y] = (uint16_t)(w[y >> 1] >> (16 * (y & 1)));
            }
        }
    }
    if (a.lse && mine_there) a.lse[token * a.heads + head] = l == 0.0f ? -INFINITY : ((DEEP ? m : M) + log2f(l)) * kLn2;
}

template <int DP>
__global__ void __launch_bounds__(KvPromptCfg<DP>::THREADS, 1) kv_prompt_kernel(const __grid_constant__ KvAttendArgs a) {
    using F = KvPromptCfg<DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const KvArgs& c = a.c;
    const int warp = threadIdx.x >> 5;
    const uint32_t s0 = ptx::smem_u32(smem);
    const KvPromptBars bar{s0 + F::OFF_BAR};
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + F::OFF_TMEM + 8);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(bar.k_full(i), 7); ptx::mbar_init(bar.v_full(i), 7);
            ptx::mbar_init(bar.k_empty(i), 1); ptx::mbar_init(bar.v_empty(i), 1);
            for (int b = 0; b < 2; ++b) { ptx::mbar_init(bar.s_full(i, b), 1); ptx::mbar_init(bar.p_full(i, b), 4); }
            ptx::mbar_init(bar.pv_done(i), 1); ptx::mbar_init(bar.o_full(i), 1);
        }
        for (int i = 0; i < F::RING; ++i) ptx::mbar_init(bar.info_full(i), 1);
        ptx::mbar_init(bar.q_full(), 8); ptx::mbar_init(bar.drained(), 1);
        ptx::mbar_fence_init();
        *abort_flag = (int)blockIdx.x == a.give_up ? 1 : 0;
    }
    if (warp == 12) {
        ptx::tmem_alloc(s0 + F::OFF_TMEM, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + F::OFF_TMEM);
    ptx::grid_start();

    // late tiles see the most tokens: they go first
    const int units = (int)(gridDim.x / (unsigned)c.heads), work = units - 1 - (int)(blockIdx.x / (unsigned)c.heads);
    KvPromptTile tile;
    KvSeq q; int unit;
    const bool any = kv_locate(c, work, a.group, F::ROWS, 1, q, unit);
    tile.h = (int)(blockIdx.x % (unsigned)c.heads);
    tile.row0 = unit * F::ROWS;
    tile.rows = any && q.n * a.group > a.more_rows_than ? min(F::ROWS, q.n * a.group - tile.row0) : 0;
    if (tile.rows > 0) {                              // (the same for the whole CTA)
        tile.s = q.s; tile.row = q.row; tile.first = q.first;
        tile.low0 = max(q.first + tile.row0 / a.group, -1);
        tile.high0 = max(q.first + (tile.row0 + min(tile.rows, 128) - 1) / a.group, -1);      // (of 256 dimensions all of them)
        tile.low1 = max(q.first + (tile.row0 + 128) / a.group, -1);
        tile.high1 = tile.rows <= 128 ? -1 : max(q.first + (tile.row0 + tile.rows - 1) / a.group, -1);
        const KvSteps steps(tile.low0, tile.last(), a.window, a.sinks, 128);
        if (warp < 8) {
            set_registers_up<F::ROWS_REGS>();
            const int far = kv_prompt_queries<F>(a, tile, bar, smem, abort_flag);
            if (far == 0) kv_prompt_rows<F, false>(a, tile, steps, bar, smem, tmem, abort_flag);
            else if (far == 1) kv_prompt_rows<F, true>(a, tile, steps, bar, smem, tmem, abort_flag);
        } else {
            set_registers_down<F::OTHER_REGS>();
            if (warp != 12) kv_prompt_convert<F>(a, tile, steps, bar, smem, abort_flag);
            else {
                kv_prompt_mma<F>(a, tile, steps, bar, s0, tmem, abort_flag);
                // what the tensor core still does ends before its operands' memory is another kernel's, also where a wait was given up
                const uint32_t leader = ptx::elect_one() ? 1u : 0u;
                ptx::mma_commit_if(leader, bar.drained());
                volatile int no = 0;
                ptx::mbar_wait(bar.drained(), 0, &no);
            }
        }
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, (int)DEV_ERR_WAIT_TIMEOUT);
}

template <int DP>
inline int32_t launch_kv_prompt(zant_ctx* ctx, KvAttendArgs a) {
    using F = KvPromptCfg<DP>;
    const long long grid = kv_units(a.c, a.group, F::ROWS, 1) * a.c.heads;
    if (grid > 0x7fffffffLL) return fail(ZANT_E_TOO_LARGE, "%lld tiles of attention", grid);
    a.status = ctx->status_word;
    a.give_up = ctx->give_up_cta < 0 ? -1 : (int)(ctx->give_up_cta % grid);
    ctx->give_up_cta = -1;
    a.wait_budget = a.give_up < 0 ? ptx::kWaitBudgetCycles : 4000000;
    ZB_SMEM_ATTR(ctx, kv_prompt_kernel<DP>, F::SMEM);
    launch(ctx, kv_prompt_kernel<DP>, dim3((unsigned)grid), F::THREADS, F::SMEM, a);
    return check_launch(ctx, "kv_prompt_kernel");
}

// A sequence with more rows of a key head than this is a prompt.  Where prompts' tiles fill half of the SMs, 30 rows take as long here as in kv_attention_kernel (16 x 6 tokens of 5 heads
// over 6000: 164 us both; 12 tokens 168, 282 there; 3 tokens 164, 82); fewer tiles leave SMs idle that kv_attention_kernel's clusters use (2 x 6 over 6000: 125 us here, 55
// there; 2 x 48 140, 127; over 500 2 x 12 25 both).
inline int kv_prompt_from(const zant_ctx* ctx, const KvAttendArgs& a) {
    const long long tiles = kv_units(a.c, a.group, a.c.dim > 128 ? 128 : 256, 1) * a.c.heads;
    const long long reach = std::min((long long)a.c.width << a.c.page_log2, a.window > 0 ? (long long)a.window + a.sinks : 0x7fffffffffLL);
    return tiles * 2 >= ctx->sm_count ? 28 : (reach >= 2048 ? 192 : 64);
}

inline int32_t run_kv_attention(zant_ctx* ctx, KvAttendArgs a) {
    a.more_rows_than = 0; a.rows_up_to = 0x7fffffff;
    if (a.q_type == ZANT_F32) return run_kv_few(ctx, a);
    // Which sequences have many rows is known on the device only, unless all have the same number: both kernels run then, and each takes its own.
    const bool uniform = !a.c.offsets;
    const long long most = uniform ? (long long)a.c.per * a.group : (long long)a.c.rows * a.group;
    const int from = kv_prompt_from(ctx, a);
    if (most > from) {
        KvAttendArgs p = a;
        p.more_rows_than = from;
        ZB_TRY(a.c.dim <= 64 ? launch_kv_prompt<64>(ctx, p) : (a.c.dim <= 128 ? launch_kv_prompt<128>(ctx, p) : launch_kv_prompt<256>(ctx, p)));
        if (uniform) return ZANT_OK;
        a.rows_up_to = from;
    }
    return run_kv_few(ctx, a);
}

}  // namespace zb
