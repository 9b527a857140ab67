// Attention for prompt portions on the 5th-generation tensor cores (bfloat16, heads of up to 256 elements in steps of 16), over
// pages of 128 positions: what read_kv_fp8_spans makes of an 8-bit cache.  Heads of up to 128 elements here, longer ones below
// (prefill_wide_kernel).
//
// A row is a (token, query head) pair; the rows of a tile are the query heads of one kv head for consecutive tokens of a
// request, so that a block of keys and values that has been brought in serves all of them, and a portion of few tokens fills
// its tiles with its heads (the kernel of attention_prefill_tc.cu has a head's tokens for rows: a portion of 300 tokens takes
// tiles of 256 and 44 there, of 2,100 rows here where 7 heads share their keys).  One CTA takes two sub-tiles of up to 128 rows
// and walks the request's keys in blocks of 128:
//
//   S_t = Q_t K_j^T    tcgen05.mma 128 x 128 x head_dim, Q by TMA ([token][head][64 elements] boxes), S_t in tensor memory
//   P_t = 2^(S_t - m)  a thread a row: cap, mask by absolute position, running maximum and sum in 32 bits, P in bfloat16 over S_t
//   O_t += P_t V_j     tcgen05.mma, A from tensor memory, V as an N-major B operand; its first half as soon as half of P_t is
//                      written
//
// Warps: 0 brings keys and values (TMA, two places each), 1 the queries and issues the products in the order PV_0(i), S_0(i + 1),
// PV_1(i), S_1(i + 1), which keeps the sub-tiles half a block apart: one's products run under the other's softmax.  4 - 7 and 8 -
// 11 are the sub-tiles' rows; they hold a row's 128 scores in registers, which the first four warps have left to them.
//
// What bounds it, in clocks of a pair of blocks, of which the four products are 2,056: a sub-tile's chain of waits.  Scores read and
// their maximum found 500, asked whether it is to be raised 190, weights 1,540 (their 2^x alone 1,024), the rest of PV and the next
// S 1,330.  B200: 3,600 clocks a pair with few blocks running, 2.39 us with all (966 TFLOP/s for 4,096 tokens behind 28,672; 28 heads of 128 on 4).  Six
// portions of 300 tokens behind up to 3,800, the pages' reading back included: 86 us; a prompt of 2,048 of 16 heads with their own
// keys 49.5 (by the kernel of attention_prefill_tc.cu 65); with capped scores 129 and 70, and 152 and 83 where
// scores come near the cap (there 280 and 139).  Tried: scores read twice instead of held, P in one piece 2.91 us a pair; a
// thread of its own for each sub-tile's products, softmaxes in turns 2.56, without turns 2.89 (both then do the same at the same
// time); a quarter of the 2^x by polynomial 2.64; rolled loops around the products 2.71.  Converting the 8-bit pages in this
// kernel, by seven more warps, cost the softmax threads a third of their registers and the tile its pace (162 us and 86 us where
// reading back first then took 124 and 67).
//
// A row of the cache that is not finite arrives as a key of NaN and a value of 0 (read_kv_fp8_spans): the scores against it are
// NaN where a query sees it and masked away where none does, and 0 times the value is 0.  What lies behind a request's last
// position in its last page is 0.
//
// Weights are rounded to bfloat16 (at most 2^-8 of the weight) for the second product, whose other operand is bfloat16; the denominator
// adds them up unrounded.  Adding up what the product has, as the general forms of attention_prefill_tc.cu do, is an instruction a score more:
// the portions 89 us instead of 86, capped 140 instead of 129, for results off by 2.05e-3 of their size instead of 2.16e-3, and where all
// values lie around 1 by 0.0083 at most instead of 0.0134.
//
// Registers: 168 a thread at the launch, of which the first four warps give their share away.  The forms for heads of 128 spill 60 bytes a
// thread, those for 64 20, the wide ones none.
//
// The running maximum is raised only when it grows by more than 2^8; O is then scaled in tensor memory.  Every wait is bounded
// (status 3).  Tiles with many key blocks may be cut into runs, which a second kernel adds up in their order (items: as the plan of
// the kernel above, with tokens for rows and kv heads for heads).
#include "tc_common.cuh"
#include "api.h"

namespace {
using namespace fxtc;

constexpr int BQ = 128, BK = 128, NTHREADS = 384, TMEM_COLS = 512, ITEM_INTS = 8, N_BARS = 19;
constexpr int REGS_FEW = 88, REGS_MANY = 208;   // a thread of the first four warps, of the softmax: together what the block is launched with
constexpr float RAISE_MAX_BY = 8.f;   // in powers of two
constexpr float CAP_SMALL = 0.8f, CAP_LARGE = 0.66f;      // (tanh(CAP_SMALL) = 0.664)

struct Args {
    const int* block_table; int table_width, n_pages;       // [entries][blocks of 128 positions]
    const int* items;
    bf16* out; long ldo;
    float *part_o, *part_ml;
    int n_kv_heads, group, per_sub, head_dim, window;     // per_sub: tokens of a sub-tile
    float scale_log2e, cap_in;                            // scores in powers of two: q.k scale_log2e, capped scale_log2e tanh(q.k cap_in)
    int* status;
};

template <int D> struct Smem {
    static constexpr int HALVES = D / 64, SUB = 128 * 128, TILE = HALVES * SUB;         // a [128 rows][128 bytes] piece; a tile
    static constexpr int K_OFF = 2 * TILE, V_OFF = 4 * TILE, TOTAL = 6 * TILE + 1024;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                   "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two 32-bit numbers in a register pair.
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t both(float x) { return pair_of(__float_as_uint(x), __float_as_uint(x)); }
__device__ __forceinline__ float2 parts_of(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
// mbar_wait whose first answer is mostly yes.
__device__ __forceinline__ bool met(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
    return mbar_wait(bar, parity, abort_flag);
}
// Capped scores: a warp's of a block become tanh(k s).  Where none that counts is beyond |k s| = 0.8 (mostly so: caps are several times what
// scores come to), the odd polynomial x + x z p(z), z = x^2, p fitted by a linear program for the smallest largest relative error (4.3e-8; in
// 32 bits 1.4e-7 of each score).  Else 1 - 2 / (e^2x + 1), which is off by some 3e-7 of the cap however small the score: at most 5e-7 of the
// largest score that the warp's rows have met.  Two scores an instruction, for what a cap costs is instructions.  A block behind one with a
// score that large is not looked at first (`look`).  B200, the portions of 300 tokens and the prompt of 2,048 named above, scores of up to
// some 20: 129 and 70 us under caps of 30 and more, 152 and 83 under one of 15, 151 and 80 under one of 4; with the second form alone 150 and
// 80; always looking 159 and 85 under the cap of 4; the polynomial up to 1/2 only, of a term less, 120 and 65 under a cap of 50, 164 and 87
// under one of 15; one rational function for every size 173 and 87.
// Hidden scores are no numbers while they are looked at, which fmaxf passes over, and rows that do not exist have no say: which form is taken
// hangs on the request's own scores.
__device__ __forceinline__ uint64_t tanh_small(uint64_t x) {
    const uint64_t z = pair_mul(x, x);
    const uint64_t p = pair_fma(pair_fma(pair_fma(pair_fma(both(-4.390075137e-03f), z, both(1.916173016e-02f)), z, both(-5.316196404e-02f)), z,
                                         both(1.332244125e-01f)), z, both(-3.333283229e-01f));
    return pair_fma(pair_mul(x, z), p, x);
}
__device__ __forceinline__ uint64_t tanh_any(uint64_t x2log2e) {
    const float2 x = parts_of(x2log2e);
    const float2 d = parts_of(pair_add(pair_of(__float_as_uint(exp2_fast(x.x)), __float_as_uint(exp2_fast(x.y))), both(1.f)));
    return pair_fma(pair_of(__float_as_uint(reciprocal_fast(d.x)), __float_as_uint(reciprocal_fast(d.y))), both(-2.f), both(1.f));
}
template <typename F> __device__ __forceinline__ void each_pair(uint32_t (&c)[32], float k, F&& f) {
    const uint64_t k2 = both(k);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float2 y = parts_of(f(pair_mul(pair_of(c[i], c[i + 1]), k2)));
        c[i] = __float_as_uint(y.x); c[i + 1] = __float_as_uint(y.y);
    }
}
// A row's scores into registers, capped (then what they are multiplied with, scale_log2e, is the cap) and masked, and the largest of them.
template <bool CAPPED>
__device__ __forceinline__ float scores_of(uint32_t (&c)[4][32], uint32_t ts, const Args& a, bool interior, int kb, int lo_r, int p_r, bool row_ok, bool& look) {
    auto hide = [&](uint32_t as) {
        if (__builtin_expect(interior, 1)) return;       // (out of the way of what most blocks run through)
#pragma unroll
        for (int k = 0; k < BK; ++k)
            if (kb + k > p_r || kb + k < lo_r) c[k / 32][k % 32] = as;
    };
    bool small = !CAPPED;
    if (!CAPPED || look) {
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_ld32(ts + 32 * i, c[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_ld_wait_for(c[i]);
        if constexpr (CAPPED) {
            hide(0x7fffffffu);                           // no number
            float size[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < BK; i += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    size[e] = fmaxf(fmaxf(size[e], fabsf(__uint_as_float(c[i / 32][i % 32 + e]))), fabsf(__uint_as_float(c[i / 32][i % 32 + 4 + e])));
            small = __all_sync(0xffffffffu, !row_ok || fmaxf(fmaxf(size[0], size[1]), fmaxf(size[2], size[3])) * a.cap_in <= CAP_SMALL);
            if (small) {
#pragma unroll
                for (int i = 0; i < 4; ++i) each_pair(c[i], a.cap_in, tanh_small);
            }
        }
    }
    if (!small) {                                        // (read again where they have been looked at: no copy of what is still on its way)
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_ld32(ts + 32 * i, c[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tc_ld_wait_for(c[i]);
            each_pair(c[i], a.cap_in * 2.8853900817779268f, tanh_any);      // 2 log2(e)
        }
    }
    hide(0xff800000u);                                   // -infinity
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < BK; k += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            mx[e] = fmaxf(fmaxf(mx[e], __uint_as_float(c[k / 32][k % 32 + e])), __uint_as_float(c[k / 32][k % 32 + 4 + e]));
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    if constexpr (CAPPED) look = !__any_sync(0xffffffffu, row_ok && top > CAP_LARGE);
    return top;
}
// 32 scores' weights in bfloat16 pairs into 16 columns of tensor memory, their sums (before they are rounded) onto sum2.
__device__ __forceinline__ void weights_of(const uint32_t* c, uint32_t at, uint64_t scale2, uint64_t ref2, uint64_t* sum2) {
    uint32_t out[16];
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
        float2 e = parts_of(pair_fma(pair_of(c[k], c[k + 1]), scale2, ref2));
        e.x = exp2_fast(e.x); e.y = exp2_fast(e.y);
        sum2[k / 2 % 2] = pair_add(sum2[k / 2 % 2], pair_of(__float_as_uint(e.x), __float_as_uint(e.y)));
        __nv_bfloat162 pr = __floats2bfloat162_rn(e.x, e.y);
        out[k >> 1] = *reinterpret_cast<uint32_t*>(&pr);
    }
    tc_st16(at, out);
}
template <int D> __device__ __forceinline__ void shrink(uint32_t to, float alpha) {
#pragma unroll 1
    for (int col = 0; col < D; col += 16) {
        uint32_t o[16];
        tc_ld16(to + col, o);
        tc_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
        tc_st16(to + col, o);
    }
}
// A row's result, or its part of a tile that was cut (slot: among the parts' rows).  has: it has seen keys.
template <int D>
__device__ __forceinline__ void put_row(uint32_t to, const Args& a, bool row_ok, bool has, float m, float l, int part, long slot, bf16* dst) {
    if (part >= 0 && row_ok) { a.part_ml[slot * 2] = has ? m * a.scale_log2e : -INFINITY; a.part_ml[slot * 2 + 1] = has ? l : 0.f; }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (!has && part >= 0) return;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        uint32_t ob[32];
        __syncwarp();
        if (has) { tc_ld32(to + c * 32, ob); tc_ld_wait(); }
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
            if (!row_ok || c * 32 + k >= a.head_dim) continue;
            if (part >= 0) {
                float* o = a.part_o + slot * D + c * 32 + k;
                *reinterpret_cast<uint4*>(o) = make_uint4(ob[k], ob[k + 1], ob[k + 2], ob[k + 3]);
                *reinterpret_cast<uint4*>(o + 4) = make_uint4(ob[k + 4], ob[k + 5], ob[k + 6], ob[k + 7]);
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = l == 0.f ? 0.f : __uint_as_float(ob[k + e]) * inv;
                Pack<bf16>::store(dst + c * 32 + k, x);
            }
        }
    }
}
template <int D, bool CAPPED>
__global__ void __launch_bounds__(NTHREADS, 1) prefill_grouped_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                      const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a)
{
    using L = Smem<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag_s;
    __shared__ uint32_t tmem_base_s;
    __shared__ __align__(8) uint64_t bars_s[N_BARS];
    volatile int* abort_flag = &abort_flag_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    auto bar = [&](int i) { return smem_u32(&bars_s[i]); };
    auto q_full = [&](int t) { return bar(t); };
    auto s_full = [&](int t) { return bar(2 + t); };
    auto p_half = [&](int t) { return bar(4 + t); };
    auto p_full = [&](int t) { return bar(6 + t); };
    auto k_empty = [&](int b) { return bar(8 + b); };
    auto v_empty = [&](int b) { return bar(10 + b); };
    auto o_done = [&](int t) { return bar(12 + t); };
    auto k_full = [&](int b) { return bar(14 + b); };
    auto v_full = [&](int b) { return bar(16 + b); };
    const uint32_t drained = bar(18);

    if (threadIdx.x == 0) {
        abort_flag_s = 0;
        for (int i = 0; i < N_BARS; ++i) mbar_init(bar(i), i >= 4 && i < 8 ? 4 : 1);      // (p_half, p_full: four warps)
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_base_s)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    fx_pdl_wait();   // set up while the kernel before this one drains; its results (and the lists, which may be new) from here on

    const int* item = a.items + (long)blockIdx.y * ITEM_INTS;
    const int tok0 = item[0], n_tok = item[1], entry = item[2], pos0 = item[3], kb_begin = item[4], kb_end = item[5], part = item[6];
    const int kvh = blockIdx.x, per = a.per_sub, nt = n_tok > per ? 2 : 1;
    auto tokens_of = [&](int t) { return min(per, n_tok - t * per); };
    auto lo_of = [&](int t) { return max(fx_first_key(pos0 + t * per, a.window, 0) / BK, kb_begin); };
    auto hi_of = [&](int t) { return min((pos0 + t * per + tokens_of(t) - 1) / BK, kb_end - 1); };
    const int lo0 = lo_of(0), hi0 = hi_of(0), lo1 = nt > 1 ? lo_of(1) : 1, hi1 = nt > 1 ? hi_of(1) : 0;      // (none: lo > hi)
    const bool act0 = lo0 <= hi0, act1 = lo1 <= hi1;
    const int first_blk = act0 && act1 ? min(lo0, lo1) : act0 ? lo0 : lo1, last_blk = act0 && act1 ? max(hi0, hi1) : act0 ? hi0 : hi1;
    const int n_walk = max(0, last_blk - first_blk + 1);
    auto active = [&](int t, int i) { const int j = first_blk + i; return t < nt && i < n_walk && j >= (t ? lo1 : lo0) && j <= (t ? hi1 : hi0); };
    auto last_of = [&](int t) { return (t ? act1 : act0) ? (t ? hi1 : hi0) - first_blk : -1; };
    auto tmem_s = [&](int t) { return tmem + 128u * t; };            // S_t, and P_t over its first 64 columns
    auto tmem_o = [&](int t) { return tmem + 256u + 128u * t; };

    int k_asked = 0, v_asked = 0;                                    // blocks under way or there
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
        if (warp == 1) {
            // ---------------- queries; products: S_0(0), S_1(0), then PV_0(i), S_0(i + 1), PV_1(i), S_1(i + 1) ----------------
            if (lane == 0) {
                for (int t = 0; t < nt; ++t) {
                    mbar_expect_tx(q_full(t), (uint32_t)(L::HALVES * per * a.group * 128));
                    for (int h = 0; h < L::HALVES; ++h) tma_load_4d(base + t * L::TILE + h * L::SUB, &map_q, h * 64, 0, kvh, tok0 + t * per, q_full(t));
                }
                constexpr uint32_t idesc_s = instr_desc_ex(BQ, BK, 0), idesc_o = instr_desc_ex(BQ, D, 1);
                uint32_t n_p[2] = {0, 0};
                auto issue_s = [&](int t, int b) {
                    tc_fence_after();
#pragma unroll
                    for (int h = 0; h < L::HALVES; ++h) {
                        const uint64_t dq = smem_desc(base + t * L::TILE + h * L::SUB), dk = smem_desc(base + L::K_OFF + b * L::TILE + h * L::SUB);
#pragma unroll
                        for (int k = 0; k < 4; ++k) tc_mma(tmem_s(t), dq + 2u * k, dk + 2u * k, idesc_s, (h | k) != 0);
                    }
                    tc_commit(s_full(t));
                };
                auto k_there = [&](int i) { return i >= n_walk || met(k_full(i & 1), (uint32_t)(i >> 1) & 1u, abort_flag); };
                bool ok = k_there(0);
                for (int t = 0; t < nt && ok; ++t) {
                    ok = met(q_full(t), 0, abort_flag);
                    if (ok && active(t, 0)) issue_s(t, 0);
                }
                if (ok && n_walk > 0) tc_commit(k_empty(0));
                ok = ok && (n_walk == 0 || met(v_full(0), 0, abort_flag)) && k_there(1);
                for (int i = 0; i < n_walk && ok; ++i) {
                    const int b = i & 1;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (t >= nt || !ok) continue;
                        if (active(t, i)) {
                            auto issue_o = [&](int ks0) {
                                tc_fence_after();
#pragma unroll
                                for (int k = 0; k < BK / 32; ++k)
                                    tc_mma_ts(tmem_o(t), tmem_s(t) + 8u * (ks0 + k), smem_desc_lbo_sbo(base + L::V_OFF + b * L::TILE + (ks0 + k) * 2048, L::SUB, 1024),
                                              idesc_o, (n_p[t] | (ks0 + k)) != 0);
                            };
                            ok = met(p_half(t), n_p[t] & 1u, abort_flag);
                            if (!ok) continue;
                            issue_o(0);
                            ok = met(p_full(t), n_p[t] & 1u, abort_flag);
                            if (!ok) continue;
                            issue_o(BK / 32);
                            ++n_p[t];
                        }
                        if (active(t, i + 1)) issue_s(t, b ^ 1);
                        else if (i == last_of(t)) tc_commit(o_done(t));
                    }
                    if (!ok) break;
                    tc_commit(v_empty(b));                          // every product that reads these has been issued
                    if (i + 1 < n_walk) {
                        tc_commit(k_empty(b ^ 1));
                        ok = met(v_full(b ^ 1), (uint32_t)((i + 1) >> 1) & 1u, abort_flag) && k_there(i + 2);      // (while the weights are made)
                    }
                }
                if (*abort_flag) {                                  // given up: no product may outlive tensor memory
                    tc_commit(drained);
                    for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try_wait(drained, 0); ++i) { }
                }
            }
            __syncwarp();
        } else if (warp == 0) {
            // ---------------- keys and values: a block is a page ----------------
            if (lane == 0) {
                const int* table = a.block_table + (long)entry * a.table_width;
                for (int i = 0; i < n_walk; ++i) {
                    const int b = i & 1, j = first_blk + i, found = j < a.table_width ? table[j] : -1, page = found < 0 ? a.n_pages : found;   // (none: zeros)
                    if (!met(k_empty(b), (uint32_t)((i >> 1) & 1) ^ 1u, abort_flag)) break;
                    mbar_expect_tx(k_full(b), (uint32_t)L::TILE);
                    for (int h = 0; h < L::HALVES; ++h) tma_load_4d(base + L::K_OFF + b * L::TILE + h * L::SUB, &map_k, h * 64, 0, kvh, page, k_full(b));
                    ++k_asked;
                    if (!met(v_empty(b), (uint32_t)((i >> 1) & 1) ^ 1u, abort_flag)) break;
                    mbar_expect_tx(v_full(b), (uint32_t)L::TILE);
                    for (int h = 0; h < L::HALVES; ++h) tma_load_4d(base + L::V_OFF + b * L::TILE + h * L::SUB, &map_v, h * 64, 0, kvh, page, v_full(b));
                    ++v_asked;
                }
            }
            __syncwarp();
        }
    } else {
        // ---------------- softmax: a row a thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
        const int t = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;      // (tensor memory: a warp may touch lanes 32 (warp % 4) ..)
        if (t < nt) {
            const int rows_t = tokens_of(t) * a.group, tok = r / a.group, pos_t = pos0 + t * per, p_r = pos_t + tok;
            const int lo_r = fx_first_key(p_r, a.window, 0), lo_last = fx_first_key(pos_t + tokens_of(t) - 1, a.window, 0);
            const uint32_t lane_off = (uint32_t)(quad * 32) << 16, ts = tmem_s(t) + lane_off, to = tmem_o(t) + lane_off;
            float m = -INFINITY, l = 0.f;
            bool ok = true, look = true;
            int cnt = 0;
            for (int i = 0; i < n_walk; ++i) {
                if (!active(t, i)) continue;
                ok = __all_sync(0xffffffffu, met(s_full(t), (uint32_t)cnt & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
                if (__builtin_expect(quad * 32 >= rows_t, 0)) {               // none of the warp's rows exists: what its rows of P hold reaches no others
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(p_half(t)); mbar_arrive(p_full(t)); }
                    ++cnt;
                    continue;
                }
                const int kb = (first_blk + i) * BK;
                const bool interior = kb + BK - 1 <= pos_t && kb >= lo_last;   // every row sees all of the block: no masking (most blocks)
                uint32_t c[4][32];
                const float mn = fmaxf(m, scores_of<CAPPED>(c, ts, a, interior, kb, lo_r, p_r, r < rows_t, look));
                const bool raise = r < rows_t && mn > m && (m == -INFINITY || (mn - m) * a.scale_log2e > RAISE_MAX_BY);
                if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
                    const float alpha = m == -INFINITY ? 0.f : exp2_fast((m - mn) * a.scale_log2e);
                    l *= alpha;
                    m = mn;
                    if (cnt > 0) shrink<D>(to, alpha);
                }
                // weights in bfloat16 pairs over the first 64 columns of S, all of which has been read
                const float ref = m == -INFINITY ? 0.f : m * a.scale_log2e;
                const uint64_t scale2 = both(a.scale_log2e), ref2 = both(-ref);
                uint64_t sum2[2] = {0, 0};
                auto weigh = [&](int chunk) { weights_of(c[chunk], ts + chunk * 16, scale2, ref2, sum2); };
                weigh(0);
                weigh(1);
                tc_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half(t));
                weigh(2);
                weigh(3);
                tc_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(t));
                const float2 sum = parts_of(pair_add(sum2[0], sum2[1]));
                l += sum.x + sum.y;
                ++cnt;
            }
            const bool has = last_of(t) >= 0;
            if (ok && has) ok = __all_sync(0xffffffffu, met(o_done(t), 0, abort_flag));
            if (ok) {
                tc_fence_after();
                const long slot = ((long)max(part, 0) * a.n_kv_heads + kvh) * (2 * BQ) + t * BQ + r;
                put_row<D>(to, a, r < rows_t, has, m, l, part, slot,
                           a.out + (long)(tok0 + t * per + tok) * a.ldo + ((long)kvh * a.group + r % a.group) * a.head_dim);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0 && abort_flag_s) {
        // given up: the copies under way still land
        auto settle = [](uint32_t at, uint32_t parity) { for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try_wait(at, parity); ++i) { } };
        for (int t = 0; t < nt; ++t) settle(q_full(t), 0);
        for (int i = max(0, k_asked - 2); i < k_asked; ++i) settle(k_full(i & 1), (uint32_t)(i >> 1) & 1u);
        for (int i = max(0, v_asked - 2); i < v_asked; ++i) settle(v_full(i & 1), (uint32_t)(i >> 1) & 1u);
        if (a.status) atomicExch(a.status, STATUS_TC_TIMEOUT);
    }
}

// Heads of 129 to 256 elements: one tile of up to 128 rows a CTA, whose O takes 256 columns.  S has two places, so that S(i + 1) is
// made while P(i) is, and PV(i) runs under the softmax of block i + 1; keys and values have one place each, keys given back when S has
// read them.  B200, reading back included: 2,048 tokens of 8 heads of 256 with their own keys 40 us (by attention_prefill.cu 250), 25
// portions of up to 499 tokens behind up to 1,000, 8 heads on 1, 99 (621).
constexpr int WIDE_THREADS = 256, WIDE_D = 256, WIDE_BARS = 13;
struct WideSmem { static constexpr int SUB = 128 * 128, TILE = 4 * SUB, K_OFF = TILE, V_OFF = 2 * TILE, TOTAL = 3 * TILE + 1024; };

template <bool CAPPED>
__global__ void __launch_bounds__(WIDE_THREADS, 1) prefill_wide_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a)
{
    using L = WideSmem;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag_s;
    __shared__ uint32_t tmem_base_s;
    __shared__ __align__(8) uint64_t bars_s[WIDE_BARS];
    volatile int* abort_flag = &abort_flag_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    auto bar = [&](int i) { return smem_u32(&bars_s[i]); };
    auto s_full = [&](int b) { return bar(b); };
    auto p_half = [&](int b) { return bar(2 + b); };                     // (of either place: a warp may be a block ahead of another)
    auto p_full = [&](int b) { return bar(4 + b); };
    const uint32_t q_full = bar(6), k_full = bar(7), v_full = bar(8), k_empty = bar(9), v_empty = bar(10), o_done = bar(11), drained = bar(12);
    if (threadIdx.x == 0) {
        abort_flag_s = 0;
        for (int i = 0; i < WIDE_BARS; ++i) mbar_init(bar(i), i >= 2 && i < 6 ? 4 : 1);      // (p_half, p_full: four warps)
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_base_s)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s, tmem_o = tmem + 256u;
    fx_pdl_wait();

    const int* item = a.items + (long)blockIdx.y * ITEM_INTS;
    const int tok0 = item[0], n_tok = item[1], entry = item[2], pos0 = item[3], kb_begin = item[4], kb_end = item[5], part = item[6];
    const int kvh = blockIdx.x, first_blk = max(fx_first_key(pos0, a.window, 0) / BK, kb_begin), last_blk = min((pos0 + n_tok - 1) / BK, kb_end - 1);
    const int n = max(0, last_blk - first_blk + 1);
    const int* table = a.block_table + (long)entry * a.table_width;
    auto page_of = [&](int i) {                                          // (none: behind the last, zeros)
        const int j = first_blk + i, found = j < a.table_width ? table[j] : -1;
        return found < 0 ? a.n_pages : found;
    };

    int asked = 0;                                                       // of this thread's copies: keys', values'
    if (warp == 0 || warp == 2) {
        // ---------------- keys, values ----------------
        if (lane == 0) {
            const bool keys = warp == 0;
            const uint32_t full = keys ? k_full : v_full, empty = keys ? k_empty : v_empty, at = base + (keys ? L::K_OFF : L::V_OFF);
            for (int i = 0; i < n; ++i, ++asked) {
                const int page = page_of(i);
                if (!met(empty, ((uint32_t)i & 1u) ^ 1u, abort_flag)) break;
                mbar_expect_tx(full, (uint32_t)L::TILE);
                for (int h = 0; h < 4; ++h) tma_load_4d(at + h * L::SUB, keys ? &map_k : &map_v, h * 64, 0, kvh, page, full);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- the queries; products: S(0), then S(i + 1), PV(i) ----------------
        if (lane == 0) {
            mbar_expect_tx(q_full, (uint32_t)(4 * a.per_sub * a.group * 128));
            for (int h = 0; h < 4; ++h) tma_load_4d(base + h * L::SUB, &map_q, h * 64, 0, kvh, tok0, q_full);
            constexpr uint32_t idesc_s = instr_desc_ex(BQ, BK, 0), idesc_o = instr_desc_ex(BQ, WIDE_D, 1);
            bool ok = met(q_full, 0, abort_flag);
            auto issue_s = [&](int i) {
                if (!met(k_full, (uint32_t)i & 1u, abort_flag)) return false;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint64_t dq = smem_desc(base + h * L::SUB), dk = smem_desc(base + L::K_OFF + h * L::SUB);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma(tmem + 128u * (i & 1), dq + 2u * k, dk + 2u * k, idesc_s, (h | k) != 0);
                }
                tc_commit(s_full(i & 1));
                tc_commit(k_empty);
                return true;
            };
            ok = ok && (n == 0 || issue_s(0));
            for (int i = 0; i < n && ok; ++i) {
                if (i + 1 < n) ok = issue_s(i + 1);
                ok = ok && met(v_full, (uint32_t)i & 1u, abort_flag) && met(p_half(i & 1), (uint32_t)(i >> 1) & 1u, abort_flag);
                auto issue_o = [&](int ks0) {
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k)
                        tc_mma_ts(tmem_o, tmem + 128u * (i & 1) + 8u * (ks0 + k), smem_desc_lbo_sbo(base + L::V_OFF + (ks0 + k) * 2048, L::SUB, 1024), idesc_o,
                                  (i | (ks0 + k)) != 0);
                };
                if (!ok) break;
                issue_o(0);
                ok = met(p_full(i & 1), (uint32_t)(i >> 1) & 1u, abort_flag);
                if (!ok) break;
                issue_o(BK / 32);
                tc_commit(o_done);
                tc_commit(v_empty);
            }
            if (*abort_flag) {                                           // given up: no product may outlive tensor memory
                tc_commit(drained);
                for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try_wait(drained, 0); ++i) { }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------- softmax: a row a thread ----------------
        const int quad = warp & 3, r = quad * 32 + lane, rows = n_tok * a.group, tok = r / a.group, p_r = pos0 + tok;
        const int lo_r = fx_first_key(p_r, a.window, 0), lo_last = fx_first_key(pos0 + n_tok - 1, a.window, 0);
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16, to = tmem_o + lane_off;
        float m = -INFINITY, l = 0.f;
        bool ok = true, look = true;
        for (int i = 0; i < n; ++i) {
            ok = __all_sync(0xffffffffu, met(s_full(i & 1), (uint32_t)(i >> 1) & 1u, abort_flag));
            if (!ok) break;
            tc_fence_after();
            if (__builtin_expect(quad * 32 >= rows, 0)) {                // none of the warp's rows exists
                tc_fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(p_half(i & 1)); mbar_arrive(p_full(i & 1)); }
                continue;
            }
            const int kb = (first_blk + i) * BK;
            const bool interior = kb + BK - 1 <= pos0 && kb >= lo_last;
            const uint32_t ts = tmem + 128u * (i & 1) + lane_off;
            uint32_t c[4][32];
            const float mn = fmaxf(m, scores_of<CAPPED>(c, ts, a, interior, kb, lo_r, p_r, r < rows, look));
            const bool raise = r < rows && mn > m && (m == -INFINITY || (mn - m) * a.scale_log2e > RAISE_MAX_BY);
            if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
                const float alpha = m == -INFINITY ? 0.f : exp2_fast((m - mn) * a.scale_log2e);
                l *= alpha;
                m = mn;
                if (i > 0) {                                             // (S(i) was made behind PV(i - 2) and ahead of PV(i - 1))
                    ok = __all_sync(0xffffffffu, met(o_done, (uint32_t)(i - 1) & 1u, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    shrink<WIDE_D>(to, alpha);
                }
            }
            const float ref = m == -INFINITY ? 0.f : m * a.scale_log2e;
            const uint64_t scale2 = both(a.scale_log2e), ref2 = both(-ref);
            uint64_t sum2[2] = {0, 0};
            weights_of(c[0], ts, scale2, ref2, sum2);
            weights_of(c[1], ts + 16, scale2, ref2, sum2);
            tc_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_half(i & 1));
            weights_of(c[2], ts + 32, scale2, ref2, sum2);
            weights_of(c[3], ts + 48, scale2, ref2, sum2);
            tc_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(i & 1));
            const float2 sum = parts_of(pair_add(sum2[0], sum2[1]));
            l += sum.x + sum.y;
        }
        // (what S(n - 1) says is that PV(n - 3) has ended: a phase at a time from there)
        if (ok && n > 1) ok = __all_sync(0xffffffffu, met(o_done, (uint32_t)(n - 2) & 1u, abort_flag));
        if (ok && n > 0) ok = __all_sync(0xffffffffu, met(o_done, (uint32_t)(n - 1) & 1u, abort_flag));
        if (ok) {
            tc_fence_after();
            put_row<WIDE_D>(to, a, r < rows, n > 0, m, l, part, ((long)max(part, 0) * a.n_kv_heads + kvh) * BQ + r,
                            a.out + (long)(tok0 + tok) * a.ldo + ((long)kvh * a.group + r % a.group) * a.head_dim);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM_COLS) : "memory");
    }
    if (abort_flag_s && lane == 0 && warp < 3) {
        // given up: this thread's copies under way still land
        auto settle = [](uint32_t at, uint32_t parity) { for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try_wait(at, parity); ++i) { } };
        if (warp == 1) settle(q_full, 0);
        else if (asked > 0) settle(warp == 0 ? k_full : v_full, (uint32_t)(asked - 1) & 1u);
        if (a.status) atomicExch(a.status, STATUS_TC_TIMEOUT);
    }
}

// The runs of a tile that was cut: merges int32 [n][4] = (first token, tokens, first part, runs); a warp a row.
template <int D> __global__ void __launch_bounds__(128) prefill_grouped_merge_kernel(const int* __restrict__ merges, const __grid_constant__ Args a)
{
    fx_pdl_wait();
    const int* mg = merges + (long)blockIdx.x * 4;
    const int tok0 = mg[0], n_tok = mg[1], part0 = mg[2], runs = mg[3], kvh = blockIdx.y;
    constexpr int ROWS = D > 128 ? BQ : 2 * BQ;
    const int lane = threadIdx.x & 31, row = blockIdx.z * 4 + (threadIdx.x >> 5), t = row / BQ, r = row % BQ;
    if (r >= min(a.per_sub, n_tok - t * a.per_sub) * a.group) return;      // (a whole warp)
    constexpr int PER = D / 32;
    const long slot0 = ((long)part0 * a.n_kv_heads + kvh) * ROWS + row, step = (long)a.n_kv_heads * ROWS;
    float m = -INFINITY, l = 0.f;                                            // lane c: run c's (at most 32)
    if (lane < runs) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (slot0 + lane * step) * 2);
        m = ml.x; l = ml.y;
    }
    const float top = warp_max(m), w = l == 0.f ? 0.f : exp2f(m - top), sum = warp_sum(l * w);
    float acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (int c = 0; c < runs; ++c) {
        const float wc = __shfl_sync(0xffffffffu, w, c);
        if (wc == 0.f) continue;                                             // (a run without keys for this row has written no sums)
        const float* src = a.part_o + (slot0 + c * step) * D + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = fmaf(src[i], wc, acc[i]);
    }
    bf16* dst = a.out + (long)(tok0 + t * a.per_sub + r / a.group) * a.ldo + ((long)kvh * a.group + r % a.group) * a.head_dim + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane * PER + i < a.head_dim) dst[i] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc[i] / sum);
}

template <int D, bool CAPPED>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int n_items, const int* merges, int n_merges, cudaStream_t s)
{
    auto kern = prefill_grouped_kernel<D, CAPPED>;
    // what the softmax threads ask for has to be there: the block's registers at its launch
    static int regs = 0;                                 // (found once; a call that could not be answered is asked again)
    if (!regs) {
        cudaFuncAttributes at;
        if (const cudaError_t e = cudaFuncGetAttributes(&at, kern)) return (int)e;
        regs = at.numRegs;
    }
    if (regs * 3 < REGS_FEW + 2 * REGS_MANY) return FX_ERR_REGISTERS;
    // of the current device: asked for each time
    if (const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::TOTAL)) return (int)e;
    fx_launch_pdl(kern, dim3(a.n_kv_heads, n_items), NTHREADS, Smem<D>::TOTAL, s, mq, mk, mv, a);
    if (n_merges > 0) fx_launch_pdl(prefill_grouped_merge_kernel<D>, dim3(n_merges, a.n_kv_heads, 2 * BQ / 4), 128, 0, s, merges, a);
    return fx_launch_status();
}

template <bool CAPPED>
int launch_wide(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int n_items, const int* merges, int n_merges, cudaStream_t s)
{
    auto kern = prefill_wide_kernel<CAPPED>;
    // of the current device: asked for each time
    if (const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WideSmem::TOTAL)) return (int)e;
    fx_launch_pdl(kern, dim3(a.n_kv_heads, n_items), WIDE_THREADS, WideSmem::TOTAL, s, mq, mk, mv, a);
    if (n_merges > 0) fx_launch_pdl(prefill_grouped_merge_kernel<WIDE_D>, dim3(n_merges, a.n_kv_heads, BQ / 4), 128, 0, s, merges, a);
    return fx_launch_status();
}

bool encode(CUtensorMap* map, const void* ptr, cuuint64_t d0, cuuint64_t d1, cuuint64_t d2, cuuint64_t d3, cuuint64_t s1, cuuint64_t s2, cuuint64_t s3,
            cuuint32_t b1, cuuint32_t b3)
{
    EncodeTiledFn fn = encode_fn();
    const cuuint64_t dims[4] = {d0, d1, d2, d3}, strides[3] = {s1 * 2, s2 * 2, s3 * 2};
    const cuuint32_t box[4] = {64, b1, 1, b3}, ones[4] = {1, 1, 1, 1};
    return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

// Keys and values: pages [n_pages][kv heads][128][head_dim], block_table [entries][table_width] names those of an entry's positions
// 128 j .. 128 j + 127.  items: int32 [n_items][8] = (first flat token, tokens, entry, position of the first token, first key block, end
// of the key blocks, part or -1, 0); a tile holds up to 2 * (128 / group) tokens (128 / group of heads above 128 elements), group = n_heads
// / n_kv_heads <= 128.  part_o [parts][kv heads][256][64 or 128] ([128][256]), part_ml [parts][kv heads][256 (128)][2].
extern "C" int fx_prefill_attention_grouped(const void* q, long ldq, int n_tokens, const void* k_pages, const void* v_pages, int n_pages,
                                            const int* block_table, int table_width, const int* items, int n_items, void* out, long ldo,
                                            int n_heads, int n_kv_heads, int head_dim, int window, float scale, float softcap, float* part_o, float* part_ml,
                                            const int* merges, int n_merges, int* status, void* stream)
{
    if (n_items <= 0 || n_tokens <= 0) return FX_OK;
    if (head_dim <= 0 || head_dim > WIDE_D || head_dim % 16 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > BQ ||
        n_pages <= 0 || table_width <= 0 || window < 0 || !(scale > 0.f) || !(softcap >= 0.f) || n_items > 65535 || n_kv_heads > 65535 ||
        (n_merges > 0 && (!part_o || !part_ml || !merges))) return FX_ERR_SIZE;
    if (ldq % 8 || ldo % 8 || (uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)k_pages % 16 || (uintptr_t)v_pages % 16 || (uintptr_t)part_o % 16)
        return FX_ERR_ALIGN;
    const int group = n_heads / n_kv_heads, per = BQ / group;
    constexpr float LOG2E = 1.4426950408889634f;
    const bool capped = softcap > 0.f;
    const Args a = {block_table, table_width, n_pages, items, (bf16*)out, ldo, part_o, part_ml, n_kv_heads, group, per, head_dim, window,
                    (capped ? softcap : scale) * LOG2E, capped ? scale / softcap : 0.f, status};
    CUtensorMap mq, mk, mv;
    const cuuint64_t W = head_dim, G = n_kv_heads;
    if (!encode(&mq, q, W, group, G, n_tokens, W, W * group, ldq, group, per) || !encode(&mk, k_pages, W, BK, G, n_pages, W, BK * W, G * BK * W, BK, 1) ||
        !encode(&mv, v_pages, W, BK, G, n_pages, W, BK * W, G * BK * W, BK, 1)) return FX_ERR_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    if (head_dim > 128) return capped ? launch_wide<true>(mq, mk, mv, a, n_items, merges, n_merges, s) : launch_wide<false>(mq, mk, mv, a, n_items, merges, n_merges, s);
    if (capped) return head_dim <= 64 ? launch<64, true>(mq, mk, mv, a, n_items, merges, n_merges, s) : launch<128, true>(mq, mk, mv, a, n_items, merges, n_merges, s);
    return head_dim <= 64 ? launch<64, false>(mq, mk, mv, a, n_items, merges, n_merges, s) : launch<128, false>(mq, mk, mv, a, n_items, merges, n_merges, s);
}
