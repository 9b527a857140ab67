// Attention of query tokens over 8-bit cache pages (the form: fp8.cuh) on the CUDA cores: any head size up to 256, any page
// size.  The tensor-core kernel of attention_decode_fp8.cu takes head sizes and pages of a multiple of 16.
//
//   s_j = scale * 2^(K_j - 127) * (q . e4m3(k_j)),  capped c tanh(s / c);  p_j = exp(s_j - m);  acc += p_j 2^(V_j - 127) e4m3(v_j)
//
// One block per (token, head).  Keys are taken in blocks of 32 aligned to absolute positions, which the warps take in turns, lane j
// scoring key j; the block's maximum and sum update the warp's running (m, l), and the lanes then share out the head for the sum of
// p V.  The warps' results are added up in their order.  A position without a page is skipped.  All arithmetic is 32-bit.
//
// What bounds it: the latency of narrow loads (four bytes of a key, one of a value) and their conversion, far from what the memory
// could deliver.  B200, 16 heads of 20 elements on 4: one request of 4,000 positions 167 us, 64 of up to 4,096 384 (a warp a
// (token, head) with a byte at a time: 1,166 and 1,231); 16 of 128 on 4 in pages of 5, 64 of up to 4,096, 813 (4,935).
#include "fp8.cuh"
#include "api.h"

namespace {

constexpr int WARPS = 8, MAX_DIM = 256, NV = MAX_DIM / 32;

struct Args {
    const void* q; long ldq;
    const uint8_t *k_pages, *v_pages, *k_exp, *v_exp;
    const int* block_table; int n_slots, table_width, page_size, n_pages;
    const int *positions, *token_seq, *seq_slot, *tokens;
    void* out; long ldo;
    int n_heads, n_kv_heads, head_dim, window;
    float scale, softcap;
};

// VEC: bytes of a key that are loaded at once.
template <typename T, int VEC> __global__ void __launch_bounds__(WARPS * 32) attention_fp8_kernel(Args a)
{
    __shared__ float q_s[MAX_DIM], m_s[WARPS], l_s[WARPS], acc_s[WARPS][MAX_DIM];
    fx_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.head_dim, h = blockIdx.y;
    const int t = a.tokens ? a.tokens[blockIdx.x] : blockIdx.x;
    const int kvh = h / (a.n_heads / a.n_kv_heads), pos = a.positions[t], slot = a.seq_slot[a.token_seq[t]];
    const bool slot_ok = slot >= 0 && slot < a.n_slots;
    const int* table = a.block_table + (long)(slot_ok ? slot : 0) * a.table_width;
    const T* qh = reinterpret_cast<const T*>(a.q) + (long)t * a.ldq + (long)h * D;
    for (int i = threadIdx.x; i < D; i += WARPS * 32) q_s[i] = to_f32(qh[i]);
    __syncthreads();

    const int lo = fx_first_key(pos, a.window, 0);
    float m = -INFINITY, l = 0.f, acc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.f;
    for (int kb = (lo & ~31) + 32 * warp; slot_ok && kb <= pos; kb += 32 * WARPS) {
        const int key = kb + lane;
        const int page = key >= lo && key <= pos ? fx_page_of(table, a.table_width, a.n_pages, key, a.page_size) : -1;
        long place = -1;
        float s = -INFINITY, v_scale = 0.f;
        if (page >= 0) {
            place = ((long)page * a.n_kv_heads + kvh) * a.page_size + key % a.page_size;
            const uint8_t* kr = a.k_pages + place * D;
            float dot = 0.f;
#pragma unroll 4
            for (int i = 0; i < D; i += VEC) {
                if constexpr (VEC == 4) {
                    const uint32_t b = *reinterpret_cast<const uint32_t*>(kr + i);
                    const float2 x = fx_fp8_float2(b & 0xffffu), y = fx_fp8_float2(b >> 16);
                    dot = fmaf(q_s[i + 3], y.y, fmaf(q_s[i + 2], y.x, fmaf(q_s[i + 1], x.y, fmaf(q_s[i], x.x, dot))));
                } else dot = fmaf(q_s[i], fx_fp8_float2(kr[i]).x, dot);
            }
            s = dot * fx_fp8_scale(a.k_exp[place]) * a.scale;
            if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
            v_scale = fx_fp8_scale(a.v_exp[place]);
        }
        const float m_new = fmaxf(m, warp_max(s));
        // (a score that is no number has no say in the maximum and makes its row's sums none)
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float p = page >= 0 ? expf(s - ref) : 0.f, alpha = m == -INFINITY ? 1.f : expf(m - ref), w = p * v_scale;
        l = l * alpha + warp_sum(p);
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] *= alpha;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const float wj = __shfl_sync(0xffffffffu, w, j);
            const long at = __shfl_sync(0xffffffffu, place, j);
            const uint8_t* vr = a.v_pages + at * D;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at >= 0 && lane + 32 * i < D) acc[i] = fmaf(wj, fx_fp8_float2(vr[lane + 32 * i]).x, acc[i]);
        }
        m = m_new;
    }
    if (lane == 0) { m_s[warp] = m; l_s[warp] = l; }
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (lane + 32 * i < D) acc_s[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float top = m_s[0], sum = 0.f, factor[WARPS];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, m_s[w]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        factor[w] = m_s[w] == -INFINITY ? 0.f : expf(m_s[w] - top);
        sum += l_s[w] * factor[w];
    }
    for (int e = threadIdx.x; e < D; e += WARPS * 32) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) x += acc_s[w][e] * factor[w];
        reinterpret_cast<T*>(a.out)[(long)t * a.ldo + (long)h * D + e] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
    }
}

}  // namespace

extern "C" int fx_attention_fp8(const void* q, long ldq, int dtype, const void* k_pages, const void* v_pages, const void* k_exp,
                                const void* v_exp, const int* block_table, int n_slots, int table_width, int page_size, int n_pages,
                                const int* positions, const int* token_seq, const int* seq_slot, const int* tokens, int n_tokens,
                                void* out, long ldo, int n_heads, int n_kv_heads, int head_dim, int window, float scale, float softcap,
                                void* stream)
{
    if (n_tokens <= 0 || n_heads <= 0) return FX_OK;
    if (head_dim <= 0 || head_dim > MAX_DIM || n_kv_heads <= 0 || n_heads % n_kv_heads || page_size <= 0 || n_pages <= 0 || n_slots <= 0 ||
        table_width <= 0 || window < 0 || n_heads > 65535) return FX_ERR_SIZE;
    const Args a = {q, ldq, (const uint8_t*)k_pages, (const uint8_t*)v_pages, (const uint8_t*)k_exp, (const uint8_t*)v_exp, block_table, n_slots,
                    table_width, page_size, n_pages, positions, token_seq, seq_slot, tokens, out, ldo, n_heads, n_kv_heads, head_dim, window,
                    scale, softcap};
    const dim3 grid(n_tokens, n_heads);
    const bool wide = head_dim % 4 == 0 && (uintptr_t)k_pages % 4 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == FX_F32) fx_launch_pdl(wide ? attention_fp8_kernel<float, 4> : attention_fp8_kernel<float, 1>, grid, WARPS * 32, 0, st, a);
    else if (dtype == FX_BF16) fx_launch_pdl(wide ? attention_fp8_kernel<bf16, 4> : attention_fp8_kernel<bf16, 1>, grid, WARPS * 32, 0, st, a);
    else return FX_ERR_DTYPE;
    return fx_launch_status();
}
