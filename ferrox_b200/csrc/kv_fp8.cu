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

// Elements a lane holds: NE neighbours from lane * NE on (WHOLE: rows of 32 NE elements on the vectors' grid, a rotation of
// the whole head in halves or none), else lane, lane + 32, ...
template <typename T, int NE, bool WHOLE>
__global__ void __launch_bounds__(WRITE_WARPS * 32) write_kernel(WriteArgs a)
{
    __shared__ float row_s[WHOLE ? 1 : WRITE_WARPS][WHOLE ? 1 : MAX_DIM];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.head_dim;
    const int heads = a.n_heads + 2 * a.n_kv_heads - a.first_head;         // rows of a token that are looked at
    fx_pdl_wait();
    const long item = (long)blockIdx.x * WRITE_WARPS + warp;
    if (item >= (long)a.n_tokens * heads) return;
    const int t = (int)(item / heads), h = a.first_head + (int)(item - (long)t * heads);
    const bool rotated = a.inv_freq && h < a.n_heads + a.n_kv_heads, cached = a.write_cache && h >= a.n_heads;
    const int pos = a.positions[t];
    T* row = reinterpret_cast<T*>(a.qkv) + (long)t * a.ld + (long)h * D;
    float x[NE];
    if (WHOLE) {
        if constexpr (NE * sizeof(T) >= 16) {
#pragma unroll
            for (int i = 0; i < NE; i += Pack<T>::N) Pack<T>::load(row + lane * NE + i, x + i);
        } else if constexpr (NE * sizeof(T) == 8 && sizeof(T) == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(row + lane * NE);
            x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u);
            x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i) x[i] = to_f32(row[lane * NE + i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NE; ++i) x[i] = lane + 32 * i < D ? to_f32(row[lane + 32 * i]) : 0.f;
    }
    int page = -1, slot = 0;
    if (cached) {
        slot = a.seq_slot[a.token_seq[t]];
        if (slot >= 0 && slot < a.n_slots)
            page = fx_page_of(a.block_table + (long)slot * a.table_width, a.table_width, a.n_pages, pos, a.page_size);
        if (page < 0 && lane == 0 && a.status) atomicExch(a.status, 2);
    }
    if (rotated) {
        const int half = a.rotary_dim >> 1;
        auto turn = [&](float p, float q, int i, bool second) {            // element of pair i: its own value p, its partner's q
            float s, c;
            if (a.cos_sin) {
                const float2 cs = *reinterpret_cast<const float2*>(a.cos_sin + ((long)t * half + i) * 2);
                c = cs.x; s = cs.y;
            } else sincosf((float)pos * a.inv_freq[i], &s, &c);
            return second ? q * s + p * c : p * c - q * s;
        };
        if (WHOLE) {
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float other = __shfl_xor_sync(0xffffffffu, x[i], 16);
                x[i] = turn(x[i], other, (lane & 15) * NE + i, lane >= 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (lane + 32 * i < D) row_s[warp][lane + 32 * i] = x[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int e = lane + 32 * i;
                if (e >= a.rotary_dim) continue;
                const bool second = a.pairing ? e & 1 : e >= half;
                x[i] = turn(x[i], row_s[warp][a.pairing ? e ^ 1 : second ? e - half : e + half], a.pairing ? e >> 1 : second ? e - half : e, second);
            }
        }
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const T y = from_f32<T>(x[i]);
            x[i] = to_f32(y);
            const int e = WHOLE ? lane * NE + i : lane + 32 * i;
            if (WHOLE || e < a.rotary_dim) row[e] = y;
        }
    }
    if (page < 0) return;                                                  // (a whole warp)
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
    most = __reduce_max_sync(0xffffffffu, most);
    const int exponent = fx_fp8_exponent(most);
    if (exponent == FX_FP8_MAX_BYTE)
#pragma unroll
        for (int i = 0; i < NE; ++i) x[i] = fminf(fmaxf(x[i], -FX_FP8_MOST), FX_FP8_MOST);
    const float inv = exponent == FX_FP8_NAN ? 0.f : fx_fp8_inverse(exponent);
    const bool is_v = h >= a.n_heads + a.n_kv_heads;
    const long at = ((long)page * a.n_kv_heads + (h - a.n_heads - (is_v ? a.n_kv_heads : 0))) * a.page_size + pos % a.page_size;
    uint8_t* dst = (is_v ? a.v_pages : a.k_pages) + at * D;
    if (lane == 0) (is_v ? a.v_exp : a.k_exp)[at] = (uint8_t)exponent;
    auto byte2 = [&](float p, float q) { return exponent == FX_FP8_NAN ? 0u : fx_fp8_pack2(p * inv, q * inv); };
    if (WHOLE) {
        if constexpr (NE == 2) {
            *reinterpret_cast<uint16_t*>(dst + lane * 2) = (uint16_t)byte2(x[0], x[1]);
        } else {
#pragma unroll
            for (int i = 0; i < NE; i += 4)
                *reinterpret_cast<uint32_t*>(dst + lane * NE + i) = byte2(x[i], x[i + 1]) | byte2(x[i + 2], x[i + 3]) << 16;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (lane + 32 * i < D) dst[lane + 32 * i] = (uint8_t)byte2(x[i], 0.f);
    }
}

struct ReadArgs {
    const uint8_t *k_pages, *v_pages, *k_exp, *v_exp;
    const int* block_table; int n_slots, table_width, page_size, n_pages;
    const int *positions, *token_seq, *seq_slot;
    const int* spans; int n_spans, n_rows;
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

// The rows of a step: k_out, v_out [tokens][kv heads][head_dim].  VEC elements a thread.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) read_rows_kernel(ReadArgs a)
{
    fx_pdl_wait();
    const int D = a.head_dim, per_row = D / VEC;
    const long n = (long)a.n_rows * a.n_kv_heads * per_row * 2;
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
        const int c = (int)(i % per_row);
        const long rest = i / per_row;
        const bool is_v = rest & 1;
        const int h = (int)((rest >> 1) % a.n_kv_heads), t = (int)((rest >> 1) / a.n_kv_heads);
        const int slot = a.seq_slot[a.token_seq[t]], pos = a.positions[t];
        const int page = slot >= 0 && slot < a.n_slots ? fx_page_of(a.block_table + (long)slot * a.table_width, a.table_width, a.n_pages, pos, a.page_size) : -1;
        T* dst = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + ((long)t * a.n_kv_heads + h) * D + c * VEC;
        const long at = ((long)max(page, 0) * a.n_kv_heads + h) * a.page_size + (page < 0 ? 0 : pos % a.page_size);
        const uint8_t* src = (is_v ? a.v_pages : a.k_pages) + at * D + c * VEC;
        const float scale = page < 0 ? 0.f : fx_fp8_scale((is_v ? a.v_exp : a.k_exp)[at]);
        if constexpr (VEC == 16) put16(dst, page < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(src), scale);
        else *dst = from_f32<T>(page < 0 ? 0.f : fx_fp8_float2(*src).x * scale);
    }
}

// Stretches of requests (spans: entry, first position, end, first row; first position and row at a page's start, rows in
// order) into pages [page of the rows][kv head][position][head_dim].  A block takes a page of a head, keys or values; what
// lies behind a stretch's end in its last page is 0.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) read_spans_kernel(ReadArgs a)
{
    fx_pdl_wait();
    const int D = a.head_dim, P = a.page_size, row0 = blockIdx.x * P, per_row = D / VEC;
    int lo = 0, hi = a.n_spans - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.spans[4 * mid + 3] <= row0) lo = mid;
        else hi = mid - 1;
    }
    const int* span = a.spans + 4 * lo;
    const int pos0 = span[1] + row0 - span[3], live = min(P, span[2] - pos0);
    const int slot = a.seq_slot[span[0]], h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const int page = live > 0 && slot >= 0 && slot < a.n_slots
        ? fx_page_of(a.block_table + (long)slot * a.table_width, a.table_width, a.n_pages, pos0, P) : -1;
    const long at = ((long)max(page, 0) * a.n_kv_heads + h) * P;
    const uint8_t* src = (is_v ? a.v_pages : a.k_pages) + at * D;
    const uint8_t* exps = (is_v ? a.v_exp : a.k_exp) + at;
    T* dst = reinterpret_cast<T*>(is_v ? a.v_out : a.k_out) + ((long)blockIdx.x * a.n_kv_heads + h) * P * D;
    for (int i = threadIdx.x; i < P * per_row; i += blockDim.x) {
        const int r = i / per_row;
        const bool there = page >= 0 && r < live;
        const float scale = there ? fx_fp8_scale(exps[r]) : 0.f;
        if constexpr (VEC == 16) put16(dst + i * 16, there ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0), scale);
        else dst[i] = from_f32<T>(there ? fx_fp8_float2(src[i]).x * scale : 0.f);
    }
}

template <typename T> void launch_write(const WriteArgs& a, unsigned blocks, bool whole, cudaStream_t s)
{
    const int n = WRITE_WARPS * 32;
    if (whole && a.head_dim == 64) return fx_launch_pdl(write_kernel<T, 2, true>, blocks, n, 0, s, a);
    if (whole && a.head_dim == 128) return fx_launch_pdl(write_kernel<T, 4, true>, blocks, n, 0, s, a);
    if (whole && a.head_dim == 256) return fx_launch_pdl(write_kernel<T, 8, true>, blocks, n, 0, s, a);
    if (a.head_dim <= 64) return fx_launch_pdl(write_kernel<T, 2, false>, blocks, n, 0, s, a);
    if (a.head_dim <= 128) return fx_launch_pdl(write_kernel<T, 4, false>, blocks, n, 0, s, a);
    return fx_launch_pdl(write_kernel<T, 8, false>, blocks, n, 0, s, a);
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
    const long blocks = fx_cdiv((long)n_tokens * (n_heads + 2 * n_kv_heads - a.first_head), WRITE_WARPS);
    if (blocks > 0x7fffffffL) return FX_ERR_SIZE;
    const int es = dtype == FX_F32 ? 4 : 2;
    const bool whole = (!inv_freq || (rotary_dim == head_dim && pairing == 0)) && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
                       ld * es % 16 == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)k_pages % 4 == 0 && (uintptr_t)v_pages % 4 == 0;
    if (dtype == FX_F32) launch_write<float>(a, (unsigned)blocks, whole, (cudaStream_t)stream);
    else if (dtype == FX_BF16) launch_write<bf16>(a, (unsigned)blocks, whole, (cudaStream_t)stream);
    else return FX_ERR_DTYPE;
    return fx_launch_status();
}

// spans null: the rows of the lists positions, token_seq; else n_spans stretches of n_rows rows together.
extern "C" int fx_read_kv_fp8(const void* k_pages, const void* v_pages, const void* k_exp, const void* v_exp, const int* block_table,
                              int n_slots, int table_width, int page_size, int n_pages, const int* positions, const int* token_seq,
                              const int* seq_slot, const int* spans, int n_spans, int n_rows, void* k_out, void* v_out, int dtype,
                              int n_kv_heads, int head_dim, void* stream)
{
    if (n_rows <= 0 || n_kv_heads <= 0) return FX_OK;
    if (head_dim <= 0 || page_size <= 0 || n_pages <= 0 || n_slots <= 0 || table_width <= 0 || n_kv_heads > 32767) return FX_ERR_SIZE;
    if (dtype != FX_F32 && dtype != FX_BF16) return FX_ERR_DTYPE;
    const ReadArgs a = {(const uint8_t*)k_pages, (const uint8_t*)v_pages, (const uint8_t*)k_exp, (const uint8_t*)v_exp, block_table, n_slots,
                        table_width, page_size, n_pages, positions, token_seq, seq_slot, spans, n_spans, n_rows, k_out, v_out, n_kv_heads, head_dim};
    const bool vec = head_dim % 16 == 0 && (uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (spans) {
        if (n_spans <= 0 || n_rows % page_size || (long)page_size * head_dim > (1L << 30)) return FX_ERR_SIZE;
        const dim3 grid(n_rows / page_size, 2 * n_kv_heads);
        if (dtype == FX_F32) vec ? fx_launch_pdl(read_spans_kernel<float, 16>, grid, 256, 0, s, a) : fx_launch_pdl(read_spans_kernel<float, 1>, grid, 256, 0, s, a);
        else vec ? fx_launch_pdl(read_spans_kernel<bf16, 16>, grid, 256, 0, s, a) : fx_launch_pdl(read_spans_kernel<bf16, 1>, grid, 256, 0, s, a);
        return fx_launch_status();
    }
    const long n = (long)n_rows * n_kv_heads * 2 * (head_dim / (vec ? 16 : 1));
    const long most = fx_sm_count() * 8L;
    const unsigned blocks = (unsigned)(fx_cdiv(n, 256) < most ? fx_cdiv(n, 256) : most);
    if (dtype == FX_F32) vec ? fx_launch_pdl(read_rows_kernel<float, 16>, blocks, 256, 0, s, a) : fx_launch_pdl(read_rows_kernel<float, 1>, blocks, 256, 0, s, a);
    else vec ? fx_launch_pdl(read_rows_kernel<bf16, 16>, blocks, 256, 0, s, a) : fx_launch_pdl(read_rows_kernel<bf16, 1>, blocks, 256, 0, s, a);
    return fx_launch_status();
}
