// Attention of few tokens a request over 8-bit cache pages (the form: fp8.cuh) on the 5th-generation tensor cores, which take
// the pages' bytes as they are: nothing converts a cached element.
//
//   grid = (token, kv head x block of HB = 4 or 8 query heads, run of keys); a tile is 128 positions.
//
//   S^T = K Q^T     tcgen05.mma kind::f8f6f4, 128 keys x (heads x parts) x head_dim.  K as TMA lays it down ([key][128 bytes],
//                   128-byte swizzle).  A query is e4m3 in PARTS_Q parts: with q' = q 2^-x (its largest element between 128 and
//                   256), part 1 is q' rounded to e4m3, part n + 1 what is left times 16 rounded again, each part a column of
//                   its own; two parts hold a bfloat16 element exactly (4 + 4 bits), six a 32-bit one.
//   softmax         a thread owns a key: it adds up its heads' parts in 32 bits, multiplies by the key's 2^K, caps and masks,
//                   and makes p = 2^(s - ref) for the denominator and w = p 2^V / 2^refw for the second product.
//   O^T += V^T W^T  tcgen05.mma, 128 elements x (heads x parts) x 128 keys.  V as TMA lays it down is its transpose with the
//                   elements side by side (M-major A); W in three parts of e4m3 (six in 32 bits), written [key][32 bytes] with
//                   the 32-byte swizzle (N-major B).
//
// Why parts: e4m3 keeps 4 bits, and products of e4m3 are added up in 32 bits (measured: beside a sum of 2^16 in the same
// instruction a product of 2^-9 is kept, in the next one of 2^-7), so that the sum over the parts is the product of the wider
// number.  Weights are first rounded to 16-bit floating numbers (2^-12 of the weight) for 16-bit rows; the third part ends at
// 2^-13 of a weight and at 2^-18 of 1 where the largest weight lies between 2^5 and 2^8, six parts at 2^-24 and 2^-30.
// What it costs is columns, of which the instruction has more than 8 heads need.
//
// The references ref and refw are whole powers of two, for each head, the same in all threads of a group: ref for the sum of
// weights, refw for the weights times 2^V (a cached value's scale belongs to its key, and with it the weight may be of any size).
// They are raised when a score passes ref by 6 or a weighted scale refw by 8; then O in tensor memory is multiplied by the power
// of two between the old and the new one.  After the first tile that is rare.
//
// Warp 0 asks for tiles (TMA, a ring of 3 stages; a stage of heads up to 128 elements is 32 KB, two blocks an SM), warp 1 issues
// the products S(j) as their keys land, warps 2 - 5 and 6 - 9 are two groups of softmax threads: a group takes every other tile,
// with references, W and O of its own, and its first thread issues its O(j).  While one group waits for its product the other
// works.  The two are added up at the end.  Every wait is bounded (status 3).
//
// What bounds it, B200.  74 requests of 16,384 positions stream 6.88 TB/s, their second half 7.35 (1.25 GB a step and three steps' caches in
// turn: none of it from the L2; torch's sum reads 4 GiB at 6.8, a copy moves 6.55, reads and writes together), and a launch
// costs 8 to 11 us beside that, the last blocks of a round among them: 64 requests of up to 4,096 positions, 28 heads on 4 of 128,
// 39.6 us of which the bytes are 27.4; one request of 131,072 in 33.0 of 20.6 (its 74 runs a kv head: 2.2 us to add them up); one of 37 in 5.4, a
// chain of waits (lookups 0.9 us, boxes asked 1.6, all met 2.0, keys landed 2.3, S 2.6, W 3.1, O 3.5, written 4.2).
// Measured beside it: one group of softmax threads 57 us for the 64 requests; two groups that share a place for W 40.5; rings of
// their own for keys and values 41.3; blocks in order of their lengths 39.8 (and requests with a window 29.1 -> 30.5).
//
// Positions outside the run or without a page: their boxes are asked for behind the last page, where TMA fills in zeros without
// reading, or hold what is in the page beside the run's own; their weights are 0, and their values are made 0, so that bytes that
// nobody has written reach nothing.  A position whose row is not finite has E = 255: its scale is NaN, and so is the result of the
// queries that see it.
//
// Runs of a token's keys leave (sum of weighted values over the sum of weights, ref, sum of weights) and a second kernel adds them
// up in their order.
#include "fp8.cuh"
#include "tc_common.cuh"
#include "api.h"

namespace {
using namespace fxtc;

constexpr int TK = 128, NSOFT = 128, NTHREADS = 64 + 2 * NSOFT, STAGES = 3, S_PLACES = 3, SLAB = TK * 128, W_ROW = 32, W_BYTES = TK * W_ROW;
constexpr float NO_REF = -1e30f;                                 // no score yet
constexpr float RAISE = 6.f, RAISE_W = 8.f, ROOM = 2.f, ROOM_W = 5.f;

struct Args {
    const void* q; long ldq;
    const uint8_t *k_exp, *v_exp;
    const int* block_table; int n_slots, table_width, page_size, n_pages, box;
    const int *positions, *token_seq, *seq_slot, *tokens;
    void* out; long ldo;
    float *part_o, *part_ml;
    int n_entries, n_heads, n_kv_heads, head_dim, window, n_splits;
    float q_scale, cap;                                          // cap 0: scores in powers of two; else scale / cap, and cap in powers of two
    int* status;
};

// The keys [k_begin, k_end) of run `split`: whole tiles of the token's visible ones, as even as they go.
__device__ __forceinline__ void run_of(int pos, int lo, int split, int n_splits, int& k_begin, int& k_end)
{
    const int first = lo / TK, n = pos / TK - first + 1, per = (n + n_splits - 1) / n_splits;
    k_begin = max(lo, (first + split * per) * TK);
    k_end = min(pos + 1, (first + min((split + 1) * per, n)) * TK);
    if (split * per >= n || pos < 0) k_end = k_begin;
}

template <typename T, int HB, int SLABS> struct Lay {
    static constexpr int PARTS_Q = sizeof(T) == 2 ? 2 : 6, PARTS_W = sizeof(T) == 2 ? 3 : 6;
    static constexpr int NS = (HB * PARTS_Q + 15) / 16 * 16, NO = (HB * PARTS_W + 15) / 16 * 16;      // columns (M = 128: in steps of 16)
    static constexpr int COLS_O = S_PLACES * NS, COLS = COLS_O + 2 * SLABS * NO;                      // (O of either group)
    static constexpr int TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int STAGE = 2 * SLABS * SLAB;                                                    // K slabs, V slabs
    static constexpr int Q_OFF = STAGES * STAGE, W_OFF = Q_OFF + SLABS * NS * 128, TOTAL = W_OFF + 2 * W_BYTES + 1024;
    static_assert(NO <= W_ROW && COLS <= (SLABS == 1 ? 256 : 512), "a key's weights are a row of 32 bytes; two blocks share the SM's tensor memory");
};

__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// Instruction descriptor: e4m3 operands, 32-bit sums; a_mn, b_mn: the operand's M (N) extent is the contiguous one.
__host__ __device__ constexpr uint32_t idesc8(int m, int n, int a_mn, int b_mn) {
    return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// 32-byte swizzle: rows of 32 bytes, 8-row groups 256 bytes apart
__device__ __forceinline__ uint64_t desc32(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(W_BYTES >> 4) << 16) | ((uint64_t)(256 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)6 << 61);
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
__device__ __forceinline__ float warp_max_f32(float v) {         // (numbers that are none have no say unless there is no other)
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {            // 2^x to 2 steps; 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Barriers of a group's 128 threads: one that asks all of them, and one that only the group's first warp waits at.
__device__ __forceinline__ bool any_of_group(int g, bool x) {
    uint32_t r;
    asm volatile("{.reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, %2, %3, p; selp.u32 %0, 1, 0, q;}"
                 : "=r"(r) : "r"((uint32_t)x), "r"(1 + g), "n"(NSOFT) : "memory");
    return r != 0;
}
__device__ __forceinline__ void group_written(int g, bool waits) {
    if (waits) asm volatile("bar.sync %0, %1;" ::"r"(3 + g), "n"(NSOFT) : "memory");
    else asm volatile("bar.arrive %0, %1;" ::"r"(3 + g), "n"(NSOFT) : "memory");
}
__device__ __forceinline__ bool any_of_soft(bool x) {            // of both groups
    uint32_t r;
    asm volatile("{.reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 5, %2, p; selp.u32 %0, 1, 0, q;}"
                 : "=r"(r) : "r"((uint32_t)x), "n"(2 * NSOFT) : "memory");
    return r != 0;
}
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(uint32_t v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(v));
    return r;
}
// A wait that does not give up when another role has (bounded all the same).
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try_wait(bar, parity); ++i) { }
}
// 16 (x - y), two 16-bit floating numbers, exact here
__device__ __forceinline__ uint32_t rest_f16x2(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("{.reg .b32 d; sub.f16x2 d, %1, %2; mul.f16x2 %0, d, %3;}" : "=r"(r) : "r"(x), "r"(y), "r"(0x4c004c00u));
    return r;
}

template <typename T, int HB, int SLABS>
__global__ void __launch_bounds__(NTHREADS, SLABS == 1 ? 2 : 1) decode_fp8_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                                 const __grid_constant__ CUtensorMap map_v,
                                                                                 const __grid_constant__ Args a)
{
    using L = Lay<T, HB, SLABS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag_s;
    __shared__ uint32_t tmem_base_s;
    __shared__ __align__(8) uint64_t bars_s[2 * STAGES + 2 * S_PLACES + 5];
    __shared__ __align__(16) float c_s[HB];                              // what a head's raw score is multiplied with
    // of a group: references of its heads, 2^(ref - refw); while they are raised: maxima of its warps, what sums and O shrink by
    __shared__ __align__(16) float ref_s[2][HB], refw_s[2][HB], ratio_s[2][HB], shrink_s[2][HB], shrink_o_s[2][16], most_s[2][2][4][HB];
    __shared__ float sum_s[2][4][HB];
    volatile int* abort_flag = &abort_flag_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - smem_u32(smem_raw));
    auto full = [&](int s) { return smem_u32(&bars_s[s]); };
    auto empty = [&](int s) { return smem_u32(&bars_s[STAGES + s]); };
    auto s_full = [&](int b) { return smem_u32(&bars_s[2 * STAGES + b]); };
    auto s_empty = [&](int b) { return smem_u32(&bars_s[2 * STAGES + S_PLACES + b]); };
    auto o_done = [&](int i) { return smem_u32(&bars_s[2 * STAGES + 2 * S_PLACES + i]); };         // of a group, a phase for each of its tiles
    auto drained = [&](int i) { return smem_u32(&bars_s[2 * STAGES + 2 * S_PLACES + 2 + i]); };

    if (threadIdx.x == 0) {
        abort_flag_s = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < S_PLACES; ++b) { mbar_init(s_full(b), 1); mbar_init(s_empty(b), 4); }
        for (int i = 0; i < 2; ++i) mbar_init(o_done(i), 1);
        for (int i = 0; i < 3; ++i) mbar_init(drained(i), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    fx_pdl_wait_only();
    const int group = a.n_heads / a.n_kv_heads, blocks_g = (group + HB - 1) / HB;
    const int kvh = blockIdx.y / blocks_g, h0 = kvh * group + blockIdx.y % blocks_g * HB, nh = min(HB, kvh * group + group - h0);
    const int tkn = a.tokens ? a.tokens[blockIdx.x] : blockIdx.x, split = blockIdx.z, D = a.head_dim;
    // (a decode step's token t is mostly its entry t: the slot that would be its is asked for beside the answer)
    const int likely = a.seq_slot[min(tkn, a.n_entries - 1)], seq = a.token_seq[tkn], pos = a.positions[tkn];
    const int slot = seq == tkn ? likely : a.seq_slot[seq];
    int k_begin, k_end;
    run_of(pos, fx_first_key(pos, a.window, 0), split, a.n_splits, k_begin, k_end);
    if (slot < 0 || slot >= a.n_slots) k_end = k_begin;
    if (k_begin >= k_end) {                       // (the whole block) no key: zeros, or a run that the merge counts for nothing
        for (int i = threadIdx.x; i < nh * D; i += NTHREADS) {
            if (a.n_splits == 1) reinterpret_cast<T*>(a.out)[(long)tkn * a.ldo + (long)h0 * D + i] = from_f32<T>(0.f);
            else if (i < nh) {
                const long at = ((long)blockIdx.x * a.n_heads + h0 + i) * a.n_splits + split;
                a.part_ml[2 * at] = NO_REF; a.part_ml[2 * at + 1] = 0.f;
            }
        }
        return;
    }
    const int* table = a.block_table + (long)slot * a.table_width;
    const int first_tile = k_begin / TK, n_tiles = (k_end - 1) / TK - first_tile + 1;

    // The producer's warp: lane b asks for a tile's box b of a.box keys.  The first tiles are asked for before the block meets.
    const int n_boxes = TK / a.box;
    int page_next = -1, asked = min(STAGES, n_tiles);
    auto page_of = [&](int j) {                                          // of this lane's box in tile j; behind the pool: zeros
        const int key = (first_tile + j) * TK + lane * a.box;
        if (lane >= n_boxes || j >= n_tiles || key >= k_end || key + a.box <= k_begin) return -1;
        return fx_page_of(table, a.table_width, a.n_pages, key, a.page_size);
    };
    auto ask_box = [&](int j, int b, int found, int off) {
        const int s = j % STAGES, page = found < 0 ? a.n_pages : found;
        const uint32_t dst = base + s * L::STAGE + b * a.box * 128;
#pragma unroll
        for (int sl = 0; sl < SLABS; ++sl) {
            tma_load_4d(dst + sl * SLAB, &map_k, sl * 128, off, kvh, page, full(s));
            tma_load_4d(dst + (SLABS + sl) * SLAB, &map_v, sl * 128, off, kvh, page, full(s));
        }
    };
    auto ask = [&](int j, int found) {
        if (lane == 0) mbar_expect_tx(full(j % STAGES), (uint32_t)L::STAGE);
        __syncwarp();
        if (lane < n_boxes) ask_box(j, lane, found, found < 0 ? 0 : ((first_tile + j) * TK + lane * a.box) % a.page_size);
        __syncwarp();
    };
    if (warp == 0) {
        // the first tiles' boxes, a lane each
        const int j = lane / n_boxes, b = lane - j * n_boxes, key = (first_tile + j) * TK + b * a.box;
        const bool mine = j < asked;
        int page = -1;
        if (mine && key < k_end && key + a.box > k_begin) page = fx_page_of(table, a.table_width, a.n_pages, key, a.page_size);
        if (lane < asked) mbar_expect_tx(full(lane), (uint32_t)L::STAGE);
        __syncwarp();
        if (mine) ask_box(j, b, page, page < 0 ? 0 : key % a.page_size);
        __syncwarp();
        page_next = page_of(STAGES);
    }

    // The softmax threads: a key a thread; group g takes the tiles g, g + 2, ...
    const int g = (warp - 2) >> 2, sw = (warp - 2) & 3, st = threadIdx.x - 64;
    const int quad = warp & 3, r = quad * 32 + lane;                     // (tensor memory: a warp may touch lanes 32 (warp % 4) ..)
    // Where this thread's keys lie: entry `at` of the table and position `off` of a page, moved on by two tiles at a time.
    // A key's page is looked up two of the group's tiles ahead, its exponents one ahead (-1: the key does not count).
    const int hop = 2 * TK / a.page_size, hop_off = 2 * TK % a.page_size;
    int key_p = (first_tile + g) * TK + r, at_p = key_p / a.page_size, off_p = key_p - at_p * a.page_size;
    int off_e = off_p;
    auto next_page = [&]() {
        int page = -1;
        if (key_p >= k_begin && key_p < k_end && at_p < a.table_width) {
            page = table[at_p];
            if (page >= a.n_pages) page = -1;
        }
        key_p += 2 * TK; at_p += hop; off_p += hop_off;
        if (off_p >= a.page_size) { off_p -= a.page_size; ++at_p; }
        return page;
    };
    auto next_exps = [&](int page) {
        int e = -1;
        if (page >= 0) {
            const long at = ((long)page * a.n_kv_heads + kvh) * a.page_size + off_e;
            e = (int)a.k_exp[at] | (int)a.v_exp[at] << 8;
        }
        off_e += hop_off;
        if (off_e >= a.page_size) off_e -= a.page_size;
        return e;
    };
    int exps_next = -1;
    if (warp >= 2) {
        // the queries in parts: a warp a head; rows of the columns that no head has are zeros
        const int h = warp - 2;
        const T* row = reinterpret_cast<const T*>(a.q) + (long)tkn * a.ldq + (long)(h0 + min(h, nh - 1)) * D;
        float x[SLABS * 4];
#pragma unroll
        for (int i = 0; i < SLABS * 4; ++i) x[i] = lane + 32 * i < D && h < nh ? to_f32(row[lane + 32 * i]) : 0.f;
        page_next = next_page();
        for (int i = st; i < SLABS * L::NS * 8; i += 2 * NSOFT) reinterpret_cast<uint4*>(sm + L::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
        if (st < 2 * HB) { (&ref_s[0][0])[st] = NO_REF; (&refw_s[0][0])[st] = NO_REF; (&ratio_s[0][0])[st] = 1.f; }
        any_of_soft(false);
        if (h < HB) {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < SLABS * 4; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
            most = __reduce_max_sync(0xffffffffu, most);
            // q 2^-x in [128, 256): the exponent field of its largest element, less 7 (at least 2^-119; an element that is no
            // finite number makes the head's factor none)
            const int field = max((int)(most >> 23), 8);
            const float inv = __uint_as_float((uint32_t)(254 - field + 7) << 23);
            if (lane == 0) c_s[h] = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.q_scale / inv;
#pragma unroll
            for (int i = 0; i < SLABS * 4; ++i) {
                const int e = lane + 32 * i;
                if (e >= D || h >= nh || most >= 0x7f800000u) continue;
                float v = x[i] * inv;
#pragma unroll
                for (int p = 0; p < L::PARTS_Q; ++p) {
                    const uint32_t b = fx_fp8_pack2(v, 0.f);
                    const int n = p * HB + h, c = e & 127;
                    sm[L::Q_OFF + (e >> 7) * L::NS * 128 + n * 128 + (((c >> 4) ^ (n & 7)) << 4) + (c & 15)] = (uint8_t)b;
                    v = (v - fx_fp8_float2(b).x) * 16.f;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        exps_next = next_exps(page_next);
        page_next = next_page();
    }

    // Tensor memory is taken behind the wait for the kernel before and ahead of the leave for the kernel behind to be set up:
    // neither can hold it while waiting for this one.
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_base_s)), "r"((uint32_t)L::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    fx_pdl_trigger();
    const uint32_t tmem = tmem_base_s;

    if (warp == 0) {
        // ---------------- producer: the other tiles, each when its stage is free ----------------
        for (int j = STAGES; j < n_tiles; ++j, ++asked) {
            const bool ok = mbar_wait(empty(j % STAGES), (uint32_t)(j / STAGES - 1) & 1u, abort_flag);
            if (__any_sync(0xffffffffu, !ok)) break;
            ask(j, page_next);
            page_next = page_of(j + 1);
        }
    } else if (warp == 1) {
        // ---------------- scores: S(j) as soon as its keys and a place for it are there ----------------
        if (lane == 0) {
            constexpr uint32_t idesc_s = idesc8(TK, L::NS, 0, 0);
            const int steps = (D + 31) / 32;                             // of 32 elements
            bool ok = true;
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int s = j % STAGES, b = j % S_PLACES;
                ok = mbar_wait(full(s), (uint32_t)(j / STAGES) & 1u, abort_flag);
                if (ok && j >= S_PLACES) ok = mbar_wait(s_empty(b), (uint32_t)(j / S_PLACES - 1) & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t k = base + s * L::STAGE, q = base + L::Q_OFF;
#pragma unroll
                for (int ks = 0; ks < 4 * SLABS; ++ks)
                    if (ks < steps)
                        mma8(tmem + b * L::NS, smem_desc(k + ks / 4 * SLAB + ks % 4 * 32), smem_desc(q + ks / 4 * L::NS * 128 + ks % 4 * 32),
                             idesc_s, ks != 0);
                tc_commit(s_full(b));
            }
            if (*abort_flag) { tc_commit(drained(2)); settle(drained(2), 0); }   // given up: no product may outlive tensor memory
        }
        __syncwarp();
    } else {
        // ---------------- softmax ----------------
        constexpr uint32_t idesc_o = idesc8(128, L::NO, 1, 1);
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), col_o = L::COLS_O + g * SLABS * L::NO;
        float l[HB];
#pragma unroll
        for (int h = 0; h < HB; ++h) l[h] = 0.f;
        bool fine = true;

        for (int j = g; j < n_tiles; j += 2) {
            const int exps = exps_next, b = j % S_PLACES;
            exps_next = next_exps(page_next);
            page_next = next_page();
            const bool live = exps >= 0;
            const float k_scale = fx_fp8_scale(exps & 255), v_scale = live ? fx_fp8_scale(exps >> 8 & 255) : 0.f;
            // What lies where nobody has written may be no number, and 0 times it is none: such values become zeros, while the scores
            // are made.  (The tile is there: the scores' product waits for the same barrier.)
            if (!live && mbar_wait(full(j % STAGES), (uint32_t)(j / STAGES) & 1u, abort_flag)) {
                uint8_t* v = sm + j % STAGES * L::STAGE + SLABS * SLAB + r * 128;
#pragma unroll
                for (int i = 0; i < SLABS * 8; ++i) *reinterpret_cast<uint4*>(v + i / 8 * SLAB + ((i ^ r) & 7) * 16) = make_uint4(0, 0, 0, 0);   // (rows side by side: other banks)
            }
            __syncwarp();
            bool ok = mbar_wait(s_full(b), (uint32_t)(j / S_PLACES) & 1u, abort_flag);
            tc_fence_after();
            float s[HB], p[HB], w[HB];
            {
                uint32_t raw[L::NS];
#pragma unroll
                for (int c = 0; c < L::NS; c += 16) tc_ld16(lanes + b * L::NS + c, raw + c);
                tc_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty(b));
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    float x = __uint_as_float(raw[(L::PARTS_Q - 1) * HB + h]);
#pragma unroll
                    for (int n = L::PARTS_Q - 2; n >= 0; --n) x = fmaf(x, 0.0625f, __uint_as_float(raw[n * HB + h]));
                    s[h] = x * (k_scale * c_s[h]);
                }
            }
            if (a.cap > 0.f) {
#pragma unroll
                for (int h = 0; h < HB; ++h) s[h] = a.cap * tanhf(s[h]);
            }
            if (!__all_sync(0xffffffffu, live)) {
#pragma unroll
                for (int h = 0; h < HB; ++h) s[h] = live ? s[h] : -INFINITY;
            }
            float over = -INFINITY, over_w = 0.f;                        // how far a score passes its reference; the largest weight
            auto weigh = [&]() {
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    const float x = s[h] - ref_s[g][h];
                    p[h] = exp2_fast(x);
                    w[h] = p[h] * v_scale * ratio_s[g][h];
                    over = fmaxf(over, x);
                    over_w = fmaxf(over_w, w[h]);
                }
            };
            const bool first = j == g;                                   // (no reference yet)
            if (!first) weigh();
            if (first || any_of_group(g, over > RAISE || over_w > 256.f || !ok)) {
                const float v_log = (float)((exps >> 8 & 255) - 127);
                const int h = lane % HB;
                const float ref = ref_s[g][h], refw = refw_s[g][h];
#pragma unroll
                for (int i = 0; i < HB; ++i) {
                    const float m = warp_max_f32(s[i]), mw = warp_max_f32(s[i] + v_log);
                    if (lane == 0) { most_s[g][0][sw][i] = m; most_s[g][1][sw][i] = mw; }
                }
                if (!first && !mbar_wait(o_done(g), (uint32_t)((j >> 1) - 1) & 1u, abort_flag)) ok = false;      // O as it stands, and nobody adds to it
                if (any_of_group(g, !ok)) { fine = false; break; }
                tc_fence_after();
                {   // every warp the same, a lane a head (the values before were read ahead of the barrier)
                    const float m = fmaxf(fmaxf(most_s[g][0][0][h], most_s[g][0][1][h]), fmaxf(most_s[g][0][2][h], most_s[g][0][3][h]));
                    const float mw = fmaxf(fmaxf(most_s[g][1][0][h], most_s[g][1][1][h]), fmaxf(most_s[g][1][2][h], most_s[g][1][3][h]));
                    const float now = m - ref > RAISE ? ceilf(m) - ROOM : ref, now_w = mw - refw > RAISE_W ? ceilf(mw) - ROOM_W : refw;
                    shrink_s[g][h] = exp2_fast(ref - now);
                    shrink_o_s[g][lane % 16] = exp2_fast(refw - now_w);   // (columns repeat their heads)
                    ratio_s[g][h] = exp2_fast(now - now_w);
                    ref_s[g][h] = now; refw_s[g][h] = now_w;
                }
                __syncwarp();
                if (!first) {
#pragma unroll
                    for (int i = 0; i < HB; ++i) l[i] *= shrink_s[g][i];
#pragma unroll 1
                    for (int c = 0; c < SLABS * L::NO; c += 16) {
                        uint32_t o[16];
                        tc_ld16(lanes + col_o + c, o);
                        tc_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink_o_s[g][i]);
                        tc_st16(lanes + col_o + c, o);
                    }
                    tc_st_wait();
                }
                weigh();
            } else {
                ok = mbar_wait(o_done(g), (uint32_t)((j >> 1) - 1) & 1u, abort_flag);        // the group's W before this one: its place is free
            }
            uint32_t word[L::NO / 4];
#pragma unroll
            for (int i = 0; i < L::NO / 4; ++i) word[i] = 0u;
#pragma unroll
            for (int h = 0; h < HB; h += 4) {
                uint32_t x[2];
                float y[4] = {w[h], w[h + 1], w[h + 2], w[h + 3]};
                if (sizeof(T) == 2) { x[0] = f16x2_of(y[0], y[1]); x[1] = f16x2_of(y[2], y[3]); }
#pragma unroll
                for (int i = 0; i < 4; ++i) l[h + i] += p[h + i];
#pragma unroll
                for (int n = 0; n < L::PARTS_W; ++n) {
                    uint32_t lo, hi;
                    if constexpr (sizeof(T) == 2) {
                        lo = pack_f16x2(x[0]); hi = pack_f16x2(x[1]);
                        if (n + 1 < L::PARTS_W) { x[0] = rest_f16x2(x[0], fx_fp8_unpack2(lo)); x[1] = rest_f16x2(x[1], fx_fp8_unpack2(hi)); }
                    } else {
                        lo = fx_fp8_pack2(y[0], y[1]); hi = fx_fp8_pack2(y[2], y[3]);
                        const float2 f = fx_fp8_float2(lo), f2 = fx_fp8_float2(hi);
                        y[0] = (y[0] - f.x) * 16.f; y[1] = (y[1] - f.y) * 16.f; y[2] = (y[2] - f2.x) * 16.f; y[3] = (y[3] - f2.y) * 16.f;
                    }
                    word[(n * HB + h) / 4] = __byte_perm(lo, hi, 0x5410);
                }
            }
            uint8_t* row = sm + L::W_OFF + g * W_BYTES + r * W_ROW;
#pragma unroll
            for (int c = 0; c < L::NO / 16; ++c)
                *reinterpret_cast<uint4*>(row + ((c ^ (r >> 2 & 1)) << 4)) = make_uint4(word[4 * c], word[4 * c + 1], word[4 * c + 2], word[4 * c + 3]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before();
            // O += V^T W^T, by the group's first thread when all its keys' weights are written
            group_written(g, sw == 0);
            if (sw == 0 && lane == 0) {
                tc_fence_after();
                const uint32_t v = base + j % STAGES * L::STAGE + SLABS * SLAB, wt = base + L::W_OFF + g * W_BYTES;
#pragma unroll
                for (int sl = 0; sl < SLABS; ++sl)
#pragma unroll
                    for (int ks = 0; ks < TK / 32; ++ks)                 // 32 keys: four 8-key groups, 1024 bytes apart in V, 256 in W
                        mma8(tmem + col_o + sl * L::NO, smem_desc_lbo_sbo(v + sl * SLAB + ks * 4096, SLAB, 1024), desc32(wt + ks * 32 * W_ROW), idesc_o,
                             j > 1 || ks > 0);
                tc_commit(empty(j % STAGES));
                tc_commit(o_done(g));
            }
            __syncwarp();
            if (!ok) fine = false;                                       // (seen by all at the next barrier, or behind the loop)
        }

        if (!fine && sw == 0 && lane == 0) { tc_commit(drained(g)); settle(drained(g), 0); }

        // ---- the run's result: this thread has element r of every slab, its group half of the heads, over both groups' tiles ----
        const int own = (n_tiles - g + 1) / 2;                           // the group's tiles
        const bool ok = fine && (own == 0 || mbar_wait(o_done(g), (uint32_t)(own - 1) & 1u, abort_flag));
        // HB sums over 32 lanes: half of what a lane has goes to its partner, until each has one head's; the rest as ever
#pragma unroll
        for (int n = HB / 2, o = 16; n > 0; n >>= 1, o >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int h = 0; h < n; ++h) {
                const float give = up ? l[h] : l[h + n], keep = up ? l[h + n] : l[h];
                l[h] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        }
#pragma unroll
        for (int o = 16 / HB; o > 0; o >>= 1) l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        // (lane's bits from the highest on choose the upper or lower half: they are the head's)
        if (lane % (32 / HB) == 0) sum_s[g][sw][lane / (32 / HB)] = l[0];
        if (!any_of_soft(!ok)) {
            tc_fence_after();
            // what a head's O of either group is multiplied with: 2^(refw - ref) over all weights' sum; a lane a head
            const bool two = n_tiles > 1;
            float factor[2], all;
            {
                const int h = lane % HB;
                const float ref = two ? fmaxf(ref_s[0][h], ref_s[1][h]) : ref_s[0][h];
                const float s0 = (sum_s[0][0][h] + sum_s[0][1][h]) + (sum_s[0][2][h] + sum_s[0][3][h]);
                const float s1 = (sum_s[1][0][h] + sum_s[1][1][h]) + (sum_s[1][2][h] + sum_s[1][3][h]);
                all = s0 * exp2_fast(ref_s[0][h] - ref);
                if (two) all = fmaf(s1, exp2_fast(ref_s[1][h] - ref), all);
                const float over = all == 0.f ? 0.f : 1.f / all;
                factor[0] = exp2_fast(refw_s[0][h] - ref) * over;
                factor[1] = two ? exp2_fast(refw_s[1][h] - ref) * over : 0.f;
                if (a.n_splits > 1 && warp == 2 && lane < nh) {
                    const long at = ((long)blockIdx.x * a.n_heads + h0 + h) * a.n_splits + split;
                    a.part_ml[2 * at] = ref; a.part_ml[2 * at + 1] = all;
                }
            }
#pragma unroll
            for (int sl = 0; sl < SLABS; ++sl) {
                const int e = sl * 128 + r;
                uint32_t o[2][L::NO];
#pragma unroll
                for (int c = 0; c < L::NO; c += 16) tc_ld16(lanes + L::COLS_O + sl * L::NO + c, o[0] + c);
                if (two) {
#pragma unroll
                    for (int c = 0; c < L::NO; c += 16) tc_ld16(lanes + L::COLS_O + (SLABS + sl) * L::NO + c, o[1] + c);
                }
                tc_ld_wait();
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    if (h / (HB / 2) != g) continue;                     // (a group takes half of the heads)
                    float v = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float f = __shfl_sync(0xffffffffu, factor[i], h);
                        if (i == 1 && !two) continue;
                        float x = __uint_as_float(o[i][(L::PARTS_W - 1) * HB + h]);
#pragma unroll
                        for (int n = L::PARTS_W - 2; n >= 0; --n) x = fmaf(x, 0.0625f, __uint_as_float(o[i][n * HB + h]));
                        v = fmaf(x, f, v);
                    }
                    if (h >= nh || e >= D) continue;
                    if (a.n_splits == 1) reinterpret_cast<T*>(a.out)[(long)tkn * a.ldo + (long)(h0 + h) * D + e] = from_f32<T>(v);
                    else a.part_o[(((long)blockIdx.x * a.n_heads + h0 + h) * a.n_splits + split) * D + e] = v;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::TMEM));
    if (threadIdx.x == 0 && abort_flag_s) {
        for (int j = max(0, asked - STAGES); j < asked; ++j) settle(full(j % STAGES), (uint32_t)(j / STAGES) & 1u);   // (copies still under way land first)
        if (a.status) atomicExch(a.status, STATUS_TC_TIMEOUT);
    }
}

// The runs of a (token, head): sum_s l_s 2^(m_s - m) mean_s / sum_s l_s 2^(m_s - m).  A warp takes every eighth run, a lane four
// elements at a time, and the warps' sums are added up in their order.  Bound by latency: with a thread an element that walks all
// runs the 74 of one long request took longer to add up than an eighth of the attention itself.
constexpr int MERGE_WARPS = 8, MAX_RUNS = 128, MERGE_DIM = 256;

template <typename T> __global__ void __launch_bounds__(MERGE_WARPS * 32) decode_fp8_merge_kernel(const __grid_constant__ Args a)
{
    __shared__ float w_s[MAX_RUNS], top_s[MERGE_WARPS], sum_s[MERGE_WARPS];
    __shared__ __align__(16) float acc_s[MERGE_WARPS][MERGE_DIM];
    fx_pdl_wait();
    const int n = a.n_splits, D = a.head_dim, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tkn = a.tokens ? a.tokens[blockIdx.x] : blockIdx.x;
    const long at = ((long)blockIdx.x * a.n_heads + h) * n;
    const bool mine = (int)threadIdx.x < n;
    const float m = mine ? a.part_ml[2 * (at + threadIdx.x)] : NO_REF, l = mine ? a.part_ml[2 * (at + threadIdx.x) + 1] : 0.f;
    const float top = warp_max(m);
    if (lane == 0) top_s[warp] = top;
    __syncthreads();
    float ref = top_s[0];
#pragma unroll
    for (int i = 1; i < MERGE_WARPS; ++i) ref = fmaxf(ref, top_s[i]);
    const float w = l == 0.f ? 0.f : l * exp2f(m - ref), part = warp_sum(w);
    if (mine) w_s[threadIdx.x] = w;
    if (lane == 0) sum_s[warp] = part;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < MERGE_WARPS; ++i) sum += sum_s[i];
    for (int e = 4 * lane; e < D; e += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = warp; i < n; i += MERGE_WARPS) {
            const float wi = w_s[i];
            if (wi == 0.f) continue;                                     // (a run without keys has written no values)
            const float4 o = *reinterpret_cast<const float4*>(a.part_o + (at + i) * D + e);
            acc.x = fmaf(wi, o.x, acc.x); acc.y = fmaf(wi, o.y, acc.y); acc.z = fmaf(wi, o.z, acc.z); acc.w = fmaf(wi, o.w, acc.w);
        }
        *reinterpret_cast<float4*>(&acc_s[warp][e]) = acc;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += MERGE_WARPS * 32) {
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < MERGE_WARPS; ++i) acc += acc_s[i][e];
        reinterpret_cast<T*>(a.out)[(long)tkn * a.ldo + (long)h * D + e] = from_f32<T>(sum == 0.f ? 0.f : acc / sum);
    }
}

template <typename T, int HB, int SLABS> int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, dim3 grid, cudaStream_t s)
{
    auto kern = decode_fp8_kernel<T, HB, SLABS>;
    // of the current device: asked for each time
    if (const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<T, HB, SLABS>::TOTAL)) return (int)e;
    fx_launch_pdl(kern, grid, NTHREADS, Lay<T, HB, SLABS>::TOTAL, s, mk, mv, a);
    return fx_launch_status();
}

bool encode(CUtensorMap* map, const void* ptr, const Args& a)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t D = a.head_dim, P = a.page_size, G = a.n_kv_heads;
    const cuuint64_t dims[4] = {D, P, G, (cuuint64_t)a.n_pages}, strides[3] = {D, P * D, G * P * D};
    const cuuint32_t box[4] = {128, (cuuint32_t)a.box, 1, 1}, ones[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T> int run(const CUtensorMap& mk, const CUtensorMap& mv, Args& a, int n_tokens, cudaStream_t s)
{
    // heads a block takes: 4, or 8, whose columns and registers leave two blocks an SM (32 bits, with six parts: 4); more heads of
    // a kv head: blocks side by side
    const int group = a.n_heads / a.n_kv_heads, hb = group <= 4 || sizeof(T) == 4 ? 4 : 8;
    const dim3 grid(n_tokens, a.n_kv_heads * ((group + hb - 1) / hb), a.n_splits);
    if (grid.y > 65535u) return FX_ERR_SIZE;
    int rc;
    if constexpr (sizeof(T) == 2) {
        if (hb == 8) rc = a.head_dim <= 128 ? launch<T, 8, 1>(mk, mv, a, grid, s) : launch<T, 8, 2>(mk, mv, a, grid, s);
    }
    if (hb == 4) rc = a.head_dim <= 128 ? launch<T, 4, 1>(mk, mv, a, grid, s) : launch<T, 4, 2>(mk, mv, a, grid, s);
    if (rc || a.n_splits == 1) return rc;
    fx_launch_pdl(decode_fp8_merge_kernel<T>, dim3(n_tokens, a.n_heads), MERGE_WARPS * 32, 0, s, a);
    return fx_launch_status();
}

}  // namespace

extern "C" int fx_decode_attention_fp8(const void* q, long ldq, int dtype, const void* k_pages, const void* v_pages, const void* k_exp,
                                       const void* v_exp, const int* block_table, int n_slots, int table_width, int page_size, int n_pages,
                                       const int* positions, const int* token_seq, const int* seq_slot, int n_entries, const int* tokens,
                                       int n_tokens, void* out, long ldo, int n_heads, int n_kv_heads, int head_dim, int window, float scale, float softcap,
                                       int n_splits, float* part_o, float* part_ml, int* status, void* stream)
{
    if (n_tokens <= 0) return FX_OK;
    if (head_dim <= 0 || head_dim > 256 || head_dim % 16 || page_size <= 0 || page_size % 16 || n_pages <= 0 || n_slots <= 0 || table_width <= 0 ||
        n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads > 65535 || n_entries <= 0 || window < 0 || softcap < 0.f || n_splits < 1 ||
        n_splits > MAX_RUNS || (n_splits > 1 && (!part_o || !part_ml))) return FX_ERR_SIZE;
    if ((uintptr_t)k_pages % 16 || (uintptr_t)v_pages % 16) return FX_ERR_ALIGN;
    int box = TK;                                                        // keys a TMA box: the largest that stays in a page
    while (page_size % box) box /= 2;
    constexpr float LOG2E = 1.4426950408889634f;
    Args a = {q, ldq, (const uint8_t*)k_exp, (const uint8_t*)v_exp, block_table, n_slots, table_width, page_size, n_pages, box, positions, token_seq,
              seq_slot, tokens, out, ldo, part_o, part_ml, n_entries, n_heads, n_kv_heads, head_dim, window, n_splits,
              softcap > 0.f ? scale / softcap : scale * LOG2E, softcap * LOG2E, status};
    CUtensorMap mk, mv;
    if (!encode(&mk, k_pages, a) || !encode(&mv, v_pages, a)) return FX_ERR_SIZE;
    if (dtype == FX_F32) return run<float>(mk, mv, a, n_tokens, (cudaStream_t)stream);
    if (dtype == FX_BF16) return run<bf16>(mk, mv, a, n_tokens, (cudaStream_t)stream);
    return FX_ERR_DTYPE;
}
