// Keys and values into 8-bit cache pages, and back (the form: fp8.cuh).
//
// Pages: bytes [page][kv head][position in the page][head_dim], exponents [page][kv head][position in the page].
//
// Writing.  A warp takes a head's row of one token: loads it, rotates it where it is a query or a key (the arithmetic and the
// pairing of the rotary kernel in elementwise.cu; queries and keys are also put back into the row, as that kernel does),
// finds the largest |x| with one warp-wide maximum over the bits, which are ordered as the numbers are and put everything
// that is no finite number on top, and stores head_dim bytes and the exponent.  Keys are quantised from the values as they
// are rounded to the row's type, so that what the cache holds does not depend on which kernel rotated them.
//
// Reading back.  Rows of a step by (position, token) lists, or whole stretches of requests into pages of another type of the
// same shape, which the attention kernels for 16- and 32-bit pages take as they are.
//
// Both move bytes and do nothing else of note: the bound is memory bandwidth, at few tokens the launch.
#include "fp8.cuh"
#include "api.h"

namespace {

struct WriteArgs {
    void* qkv; long ld;
    const int *positions, *token_seq, *seq_slot;
    const float *inv_freq, *cos_sin;
    int rotary_dim, pairing;
    uint8_t *k_pages, *v_pages, *k_exp, *v_exp;
    const int* block_table; int n_slots, table_width, page_size, n_pages;
    int n_tokens, n_heads, n_kv_heads, head_dim, first_head, write_cache;
    int* status;
};

constexpr int WRITE_WARPS = 4, MAX_DIM = 256;

// Where token t's position lies; -1: nowhere.
__device__ __forceinline__ int page_of_token(const int* positions, const int* token_seq, const int* seq_slot, const int* block_table, int n_slots,
                                             int table_width, int n_pages, int page_size, int t, int pos)
{
    const int slot = seq_slot[token_seq[t]];
    return slot >= 0 && slot < n_slots ? fx_page_of(block_table + (long)slot * table_width, table_width, n_pages, pos, page_size) : -1;
}

// An element of pair i behind its rotation: its own value p, its partner's q.
__device__ __forceinline__ float turned(const WriteArgs& a, int t, int pos, float p, float q, int i, bool second)
{
    float s, c;
    if (a.cos_sin) {
        const float2 cs = *reinterpret_cast<const float2*>(a.cos_sin + ((long)t * (a.rotary_dim >> 1) + i) * 2);
        c = cs.x; s = cs.y;
    } else sincosf((float)pos * a.inv_freq[i], &s, &c);
    return second ? q * s + p * c : p * c - q * s;
}

// Rows of LANES lanes with 16 bytes each (or 32 lanes with 32 bytes), a rotation of the whole head in halves or none.  A block
// takes a token's rows, or a share of them (blockIdx.y); a lane loads R rows' parts before it works on the first.  What bounds
// it is how many bytes are under way: the place of a token's position is four loads that hang on one another, beside which its
// rows arrive.  B200, 2,709 tokens with 16 heads of 128 for keys and for values, written and read back: one row a warp 34.4 us,
// four rows a lane 20.5 (each of the two launches moves 33 MB, 5.1 us of the memory); 32 tokens of 4 heads 4.5, which are the launches.
template <typename T, int DIM, int R>
__global__ void __launch_bounds__(WRITE_WARPS * 32) write_rows_kernel(WriteArgs a)
{
    constexpr int NE = DIM * (int)sizeof(T) / 16 > 32 ? DIM / 32 : 16 / (int)sizeof(T), LANES = DIM / NE, PER = 32 / LANES * WRITE_WARPS;
    fx_pdl_wait();
    const int t = blockIdx.x, sub = threadIdx.x % LANES, heads = a.n_heads + 2 * a.n_kv_heads;
    const int h_first = a.first_head + blockIdx.y * PER * R + threadIdx.x / LANES;
    const int pos = a.positions[t];
    T* rows = reinterpret_cast<T*>(a.qkv) + (long)t * a.ld + sub * NE;
    float x[R][NE];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int h = h_first + u * PER;
#pragma unroll
        for (int i = 0; i < NE; i += Pack<T>::N) {
            if (h < heads) Pack<T>::load(rows + (long)h * DIM + i, x[u] + i);
            else
#pragma unroll
                for (int e = 0; e < Pack<T>::N; ++e) x[u][i + e] = 0.f;
        }
    }
    int page = -1;
    if (a.write_cache) {
        page = page_of_token(a.positions, a.token_seq, a.seq_slot, a.block_table, a.n_slots, a.table_width, a.n_pages, a.page_size, t, pos);
        if (page < 0 && threadIdx.x == 0 && a.status) atomicExch(a.status, 2);
    }
    const long at0 = (long)page * a.n_kv_heads * a.page_size + pos % a.page_size;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int h = h_first + u * PER;                                   // (the lanes of a row agree on it, a warp's may not)
        float* y = x[u];
        if (a.inv_freq) {
            const bool rotated = h < a.n_heads + a.n_kv_heads;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float other = __shfl_xor_sync(0xffffffffu, y[i], LANES / 2);
                if (rotated) y[i] = to_f32(from_f32<T>(turned(a, t, pos, y[i], other, (sub % (LANES / 2)) * NE + i, sub >= LANES / 2)));
            }
            if (rotated)
#pragma unroll
                for (int i = 0; i < NE; i += Pack<T>::N) Pack<T>::store(rows + (long)h * DIM + i, y + i);
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) most = max(most, __float_as_uint(y[i]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (page < 0 || h < a.n_heads || h >= heads) continue;
        const int exponent = fx_fp8_exponent(most);
        const bool none = exponent == FX_FP8_NAN, is_v = h >= a.n_heads + a.n_kv_heads;
        if (exponent == FX_FP8_MAX_BYTE)
#pragma unroll
            for (int i = 0; i < NE; ++i) y[i] = fminf(fmaxf(y[i], -FX_FP8_MOST), FX_FP8_MOST);
        const float inv = none ? 0.f : fx_fp8_inverse(exponent);
        const long at = at0 + (long)(h - a.n_heads - (is_v ? a.n_kv_heads : 0)) * a.page_size;
        uint32_t w[NE / 4];
#pragma unroll
        for (int i = 0; i < NE; i += 4)
            w[i / 4] = none ? 0u : fx_fp8_pack2(y[i] * inv, y[i + 1] * inv) | fx_fp8_pack2(y[i + 2] * inv, y[i + 3] * inv) << 16;
        uint8_t* dst = (is_v ? a.v_pages : a.k_pages) + at * DIM + sub * NE;
        if constexpr (NE == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
        else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
        if (sub == 0) (is_v ? a.v_exp : a.k_exp)[at] = (uint8_t)exponent;
    }
}

// Any other row of up to MAX_DIM elements, a warp a row: a lane has the elements lane, lane + 32, ...
template <typename T>
__global__ void __launch_bounds__(WRITE_WARPS * 32) write_any_kernel(WriteArgs a)
{
    constexpr int NE = MAX_DIM / 32;
    __shared__ float row_s[WRITE_WARPS][MAX_DIM];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.head_dim;
    const int heads = a.n_heads + 2 * a.n_kv_heads - a.first_head;         // rows of a token that are looked at
    fx_pdl_wait();
    const long item = (long)blockIdx.x * WRITE_WARPS + warp;
    if (item >= (long)a.n_tokens * heads) return;
    const int t = (int)(item / heads), h = a.first_head + (int)(item - (long)t * heads);
    const bool rotated = a.inv_freq && h < a.n_heads + a.n_kv_heads;
    const int pos = a.positions[t];
    T* row = reinterpret_cast<T*>(a.qkv) + (long)t * a.ld + (long)h * D;
    float x[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) x[i] = lane + 32 * i < D ? to_f32(row[lane + 32 * i]) : 0.f;
    int page = -1;
    if (a.write_cache && h >= a.n_heads) {
        page = page_of_token(a.positions, a.token_seq, a.seq_slot, a.block_table, a.n_slots, a.table_width, a.n_pages, a.page_size, t, pos);
        if (page < 0 && lane == 0 && a.status) atomicExch(a.status, 2);
    }
    if (rotated) {
        const int half = a.rotary_dim >> 1;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (lane + 32 * i < D) row_s[warp][lane + 32 * i] = x[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = lane + 32 * i;
            if (e >= a.rotary_dim) continue;
            const bool second = a.pairing ? e & 1 : e >= half;
            const T y = from_f32<T>(turned(a, t, pos, x[i], row_s[warp][a.pairing ? e ^ 1 : second ? e - half : e + half],
                                           a.pairing ? e >> 1 : second ? e - half : e, second));
            x[i] = to_f32(y);
            row[e] = y;
        }
    }
    if (page < 0) return;                                                  // (a whole warp)
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
    const int exponent = fx_fp8_exponent(__reduce_max_sync(0xffffffffu, most));
    if (exponent == FX_FP8_MAX_BYTE)
#pragma unroll
        for (int i = 0; i < NE; ++i) x[i] = fminf(fmaxf(x[i], -FX_FP8_MOST), FX_FP8_MOST);
    const bool none = exponent == FX_FP8_NAN, is_v = h >= a.n_heads + a.n_kv_heads;
    const float inv = none ? 0.f : fx_fp8_inverse(exponent);
    const long at = ((long)page * a.n_kv_heads + (h - a.n_heads - (is_v ? a.n_kv_heads : 0))) * a.page_size + pos % a.page_size;
    uint8_t* dst = (is_v ? a.v_pages : a.k_pages) + at * D;
    if (lane == 0) (is_v ? a.v_exp : a.k_exp)[at] = (uint8_t)exponent;
#pragma unroll
    for (int i = 0; i < NE; ++i)
        if (lane + 32 * i < D) dst[lane + 32 * i] = none ? 0 : (uint8_t)fx_fp8_pack2(x[i] * inv, 0.f);
}

struct ReadArgs {
    const uint8_t *k_pages, *v_pages, *k_exp, *v_exp;
    const int* block_table; int n_slots, table_width, page_size, n_pages;
    const int *positions, *token_seq, *seq_slot;
    const int* spans; int n_spans, n_rows, out_page, attend;
    void *k_out, *v_out;
    int n_kv_heads, head_dim;
};

// 16 values of a row.
template <typename T> __device__ __forceinline__ void put16(T* dst, uint4 w, float scale)
{
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = fx_fp8_float2(v[i] & 0xffffu), q = fx_fp8_float2(v[i] >> 16);
        f[4 * i] = p.x * scale; f[4 * i + 1] = p.y * scale; f[4 * i + 2] = q.x * scale; f[4 * i + 3] = q.y * scale;
    }
#pragma unroll
    for (int i = 0; i < 16; i += Pack<T>::N) Pack<T>::store(dst + i, f + i);
}

// The rows of a step: k_out, v_out [tokens][kv heads][head_dim].  A block takes a token's rows, or a share of them
// (blockIdx.y); a thread READ_AHEAD times VEC elements, all asked for before the first is written.
constexpr int READ_THREADS = 128, READ_AHEAD = 4;

template <typename T, int VEC>
__global__ void __launch_bounds__(READ_THREADS) read_rows_kernel(ReadArgs a)
{
    fx_pdl_wait();
    const int D = a.head_dim, per_row = D / VEC, n = 2 * a.n_kv_heads * per_row, t = blockIdx.x, pos = a.positions[t];
    const int slot = a.seq_slot[a.token_seq[t]];
    const int page = slot >= 0 && slot < a.n_slots ? fx_page_of(a.block_table + (long)slot * a.table_width, a.table_width, a.n_pages, pos, a.page_size) : -1;
    const long at0 = page < 0 ? 0 : (long)page * a.n_kv_heads * a.page_size + pos % a.page_size;
    uint4 w[READ_AHEAD];
    int e[READ_AHEAD];
#pragma unroll
    for (int u = 0; u < READ_AHEAD; ++u) {
        const int i = (blockIdx.y * READ_AHEAD + u) * READ_THREADS + threadIdx.x, row = i / per_row, h = row % a.n_kv_heads;
        w[u] = make_uint4(0, 0, 0, 0);
        e[u] = 0;
        if (i >= n || page < 0) continue;
        const bool is_v = row >= a.n_kv_heads;
        const long at = at0 + (long)h * a.page_size;
        const uint8_t* src = (is_v ? a.v_pages : a.k_pages) + at * D + (i - row * per_row) * VEC;
        if constexpr (VEC == 16) w[u] = *reinterpret_cast<const uint4*>(src);
        else w[u].x = *src;
        e[u] = (is_v ? a.v_exp : a.k_exp)[at];
    }
#pragma unroll
    for (int u = 0; u < READ_AHEAD; ++u) {
        const int i = (blockIdx.y * READ_AHEAD + u) * READ_THREADS + threadIdx.x, row = i / per_row, h = row % a.n_kv_heads;
        if (i >= n) continue;
        T* dst = reinterpret_cast<T*>(row >= a.n_kv_heads ? a.v_out : a.k_out) + ((long)t * a.n_kv_heads + h) * D + (i - row * per_row) * VEC;
        const float scale = fx_fp8_scale(e[u]);
        if constexpr (VEC == 16) put16(dst, w[u], scale);
        else *dst = from_f32<T>(fx_fp8_float2(w[u].x).x * scale);
    }
}

// Stretches of requests (spans: entry, first position, end, first row; each in pages of its own, in order) into pages
// [page of the rows][kv head][position][head_dim] of out_page positions, which need not be the cache's.  A block takes a page of
// a head, keys or values, or a share of it (blockIdx.z); what lies before a stretch in its first page and behind its end in its last is 0.  For attention: a position of which the key or
// the value is not finite becomes a key of NaN and a value of 0, so that it makes those queries' results NaN that see it, and no
// other's (a weight of 0 times NaN is none).
// What bounds it is again the bytes under way: a row's place is looked up once (once for all rows where they are a page of the
// cache's own) and all of a thread's bytes are asked for before the first is written.  B200, 4 requests of up to 32,768
// positions, 4 heads of 128, into bfloat16: 44 us, 5.3 TB/s (with places looked up by every thread 45.7).
template <typename T, int VEC>
__global__ void __launch_bounds__(READ_THREADS) read_spans_kernel(ReadArgs a)
{
    __shared__ int place_s[READ_THREADS * READ_AHEAD];                      // of a row among the cache's positions; -1: nowhere
    fx_pdl_wait();
    const int D = a.head_dim, P = a.out_page, row0 = blockIdx.x * P, per_row = D / VEC;
    int before = 0;                                                         // stretches that begin at this page or before it
    for (int i = 0; i < a.n_spans; i += 32) {
        const int k = i + (threadIdx.x & 31);
        before += __popc(__ballot_sync(0xffffffffu, k < a.n_spans && a.spans[4 * k + 3] - row0 < P));
    }
    const int4 span = *reinterpret_cast<const int4*>(a.spans + 4 * max(before - 1, 0));
    const int pos0 = span.y + row0 - span.w, skip = span.w - row0, live = min(P, span.z - pos0);
    const int slot = a.seq_slot[span.x], h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1, known = slot >= 0 && slot < a.n_slots;
    const int* table = a.block_table + (long)(known ? slot : 0) * a.table_width;
    // this block's elements: the pieces from `first` on, of the page's rows from row_a on
    const long first = (long)blockIdx.z * (READ_AHEAD * READ_THREADS), n = (long)P * per_row;
    const int row_a = (int)(first / per_row), row_b = (int)min((long)P, (first + READ_AHEAD * READ_THREADS - 1) / per_row + 1);
    const bool whole = P == a.page_size && pos0 % P == 0;                   // (the block's rows are a page of the cache)
    int place0 = -1;
    if (whole) {
        const int page = known ? fx_page_of(table, a.table_width, a.n_pages, pos0, P) : -1;
        if (page >= 0) place0 = (page * a.n_kv_heads + h) * P;
    } else {
        for (int r = row_a + threadIdx.x; r < row_b; r += READ_THREADS) {
            const int page = r >= skip && r < live && known ? fx_page_of(table, a.table_width, a.n_pages, pos0 + r, a.page_size) : -1;
            place_s[r - row_a] = page < 0 ? -1 : (page * a.n_kv_heads + h) * a.page_size + (pos0 + r) % a.page_size;
        }
        __syncthreads();
    }
    const uint8_t *pages = is_v ? a.v_pages : a.k_pages, *own = is_v ? a.v_exp : a.k_exp, *other = is_v ? a.k_exp : a.v_exp;
    T* dst = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + ((long)blockIdx.x * a.n_kv_heads + h) * P * D;
    uint4 w[READ_AHEAD];
    int e[READ_AHEAD], e2[READ_AHEAD];
#pragma unroll
    for (int u = 0; u < READ_AHEAD; ++u) {
        const long i = first + u * READ_THREADS + threadIdx.x;
        const int r = (int)(i / per_row), at = i >= n ? -1 : !whole ? place_s[r - row_a] : r >= skip && r < live && place0 >= 0 ? place0 + r : -1;
        w[u] = make_uint4(0, 0, 0, 0);
        e[u] = e2[u] = 0;
        if (at < 0) continue;
        const uint8_t* src = pages + (long)at * D + (i - (long)r * per_row) * VEC;
        if constexpr (VEC == 16) w[u] = *reinterpret_cast<const uint4*>(src);
        else w[u].x = *src;
        e[u] = own[at];
        if (a.attend) e2[u] = other[at];
    }
#pragma unroll
    for (int u = 0; u < READ_AHEAD; ++u) {
        const long i = first + u * READ_THREADS + threadIdx.x;
        if (i >= n) continue;
        float scale = fx_fp8_scale(e[u]);
        if (a.attend && (e[u] == FX_FP8_NAN || e2[u] == FX_FP8_NAN)) scale = is_v ? 0.f : __uint_as_float(0x7fc00000u);
        if constexpr (VEC == 16) put16(dst + i * 16, w[u], scale);
        else dst[i] = from_f32<T>(fx_fp8_float2(w[u].x).x * scale);
    }
}

template <typename T, int DIM> void launch_rows(const WriteArgs& a, cudaStream_t s)
{
    constexpr int NE = DIM * (int)sizeof(T) / 16 > 32 ? DIM / 32 : 16 / (int)sizeof(T), PER = 32 / (DIM / NE) * WRITE_WARPS;
    const int heads = a.n_heads + 2 * a.n_kv_heads - a.first_head;
    // (few tokens: every row a block of its own fills the machine sooner)
    if ((long)a.n_tokens * fx_cdiv(heads, PER) >= 8L * fx_sm_count())
        fx_launch_pdl(write_rows_kernel<T, DIM, 4>, dim3(a.n_tokens, (unsigned)fx_cdiv(heads, 4 * PER)), WRITE_WARPS * 32, 0, s, a);
    else
        fx_launch_pdl(write_rows_kernel<T, DIM, 1>, dim3(a.n_tokens, (unsigned)fx_cdiv(heads, PER)), WRITE_WARPS * 32, 0, s, a);
}
template <typename T> void launch_write(const WriteArgs& a, bool whole, cudaStream_t s)
{
    if (whole && a.head_dim == 64) return launch_rows<T, 64>(a, s);
    if (whole && a.head_dim == 128) return launch_rows<T, 128>(a, s);
    if (whole && a.head_dim == 256) return launch_rows<T, 256>(a, s);
    const long rows = (long)a.n_tokens * (a.n_heads + 2 * a.n_kv_heads - a.first_head);
    fx_launch_pdl(write_any_kernel<T>, (unsigned)fx_cdiv(rows, WRITE_WARPS), WRITE_WARPS * 32, 0, s, a);
}

}  // namespace

extern "C" int fx_rope_kv_write_fp8(void* qkv, int dtype, long ld, const int* positions, const int* token_seq, const int* seq_slot,
                                    const float* inv_freq, const float* cos_sin, int rotary_dim, int pairing, void* k_pages,
                                    void* v_pages, void* k_exp, void* v_exp, const int* block_table, int n_slots, int table_width,
                                    int page_size, int n_pages, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                    int write_cache, int* status, void* stream)
{
    if (n_tokens <= 0 || n_kv_heads <= 0) return FX_OK;
    if (head_dim <= 0 || head_dim > MAX_DIM || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim || page_size <= 0 || n_heads < 0 ||
        pairing < 0 || pairing > 1 || n_pages <= 0 || n_slots <= 0 || table_width <= 0) return FX_ERR_SIZE;
    if (rotary_dim == 0) inv_freq = nullptr;
    if (!inv_freq && !write_cache) return FX_OK;
    const WriteArgs a = {qkv, ld, positions, token_seq, seq_slot, inv_freq, cos_sin, rotary_dim, pairing, (uint8_t*)k_pages, (uint8_t*)v_pages,
                         (uint8_t*)k_exp, (uint8_t*)v_exp, block_table, n_slots, table_width, page_size, n_pages, n_tokens, n_heads, n_kv_heads,
                         head_dim, inv_freq ? 0 : n_heads, write_cache, status};
    if ((long)n_tokens * (n_heads + 2 * n_kv_heads) > 0x7fffffffL || n_heads + 2 * n_kv_heads > 65535) return FX_ERR_SIZE;
    if (inv_freq && (uintptr_t)cos_sin % 8) return FX_ERR_ALIGN;
    const int es = dtype == FX_F32 ? 4 : 2;
    const bool whole = (!inv_freq || (rotary_dim == head_dim && pairing == 0)) && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
                       ld * es % 16 == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)k_pages % 8 == 0 && (uintptr_t)v_pages % 8 == 0;
    if (dtype == FX_F32) launch_write<float>(a, whole, (cudaStream_t)stream);
    else if (dtype == FX_BF16) launch_write<bf16>(a, whole, (cudaStream_t)stream);
    else return FX_ERR_DTYPE;
    return fx_launch_status();
}

// spans null: the rows of the lists positions, token_seq; else n_spans stretches of n_rows rows together.
extern "C" int fx_read_kv_fp8(const void* k_pages, const void* v_pages, const void* k_exp, const void* v_exp, const int* block_table,
                              int n_slots, int table_width, int page_size, int n_pages, const int* positions, const int* token_seq,
                              const int* seq_slot, const int* spans, int n_spans, int n_rows, int out_page, int attend, void* k_out, void* v_out, int dtype,
                              int n_kv_heads, int head_dim, void* stream)
{
    if (n_rows <= 0 || n_kv_heads <= 0) return FX_OK;
    if (head_dim <= 0 || page_size <= 0 || n_pages <= 0 || n_slots <= 0 || table_width <= 0 || n_kv_heads > 32767 ||
        (long)n_pages * n_kv_heads * page_size > 0x7fffffffL) return FX_ERR_SIZE;
    if (dtype != FX_F32 && dtype != FX_BF16) return FX_ERR_DTYPE;
    const ReadArgs a = {(const uint8_t*)k_pages, (const uint8_t*)v_pages, (const uint8_t*)k_exp, (const uint8_t*)v_exp, block_table, n_slots,
                        table_width, page_size, n_pages, positions, token_seq, seq_slot, spans, n_spans, n_rows, out_page, attend, k_out, v_out, n_kv_heads, head_dim};
    const bool vec = head_dim % 16 == 0 && (uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0;
    if ((uintptr_t)spans % 16) return FX_ERR_ALIGN;
    cudaStream_t s = (cudaStream_t)stream;
    if (spans) {
        if (n_spans <= 0 || out_page <= 0 || n_rows % out_page || (long)out_page * head_dim > (1L << 30)) return FX_ERR_SIZE;
        const long pieces = fx_cdiv((long)out_page * (head_dim / (vec ? 16 : 1)), READ_THREADS * READ_AHEAD);
        if (pieces > 65535) return FX_ERR_SIZE;
        const dim3 grid(n_rows / out_page, 2 * n_kv_heads, (unsigned)pieces);
        if (dtype == FX_F32) vec ? fx_launch_pdl(read_spans_kernel<float, 16>, grid, READ_THREADS, 0, s, a) : fx_launch_pdl(read_spans_kernel<float, 1>, grid, READ_THREADS, 0, s, a);
        else vec ? fx_launch_pdl(read_spans_kernel<bf16, 16>, grid, READ_THREADS, 0, s, a) : fx_launch_pdl(read_spans_kernel<bf16, 1>, grid, READ_THREADS, 0, s, a);
        return fx_launch_status();
    }
    const dim3 blocks(n_rows, (unsigned)fx_cdiv(2L * n_kv_heads * (head_dim / (vec ? 16 : 1)), READ_THREADS * READ_AHEAD));
    if (blocks.y > 65535u) return FX_ERR_SIZE;
    if (dtype == FX_F32) vec ? fx_launch_pdl(read_rows_kernel<float, 16>, blocks, READ_THREADS, 0, s, a) : fx_launch_pdl(read_rows_kernel<float, 1>, blocks, READ_THREADS, 0, s, a);
    else vec ? fx_launch_pdl(read_rows_kernel<bf16, 16>, blocks, READ_THREADS, 0, s, a) : fx_launch_pdl(read_rows_kernel<bf16, 1>, blocks, READ_THREADS, 0, s, a);
    return fx_launch_status();
}
