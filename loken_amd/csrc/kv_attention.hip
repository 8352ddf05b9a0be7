// Attention over the paged 8-bit cache (lk_kv_attention_q8).

#include <math.h>

#include "kv_cache.h"

namespace {

struct Attend {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    KvPool pool;
    const int32_t *table, *lens, *starts;
    int64_t table_stride;
    int table_cols, rows, heads, group, window;
    float scale;
};

// One wave to a row and head: sixty-four positions at a time, a lane to a position for the scores, a lane to
// a column for the sums.
template <typename T, int D>
__global__ __launch_bounds__(64) void kv_attention_row_kernel(Attend a, int seqs) {
    constexpr int PER = D / 64;
    __shared__ float q_lds[D], p_lds[64];
    const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kv = head / a.group;
    int seq = -1;
    for (int i = lane; i < seqs; i += 64)
        if (a.starts[i] <= row && row < a.starts[i + 1]) seq = i;
    for (int o = 32; o; o >>= 1) seq = max(seq, __shfl_xor(seq, o));
    if (seq < 0) return;
    const int shift = a.pool.page_shift, P = 1 << shift;
    const int64_t pos = (int64_t)a.lens[seq] - (a.starts[seq + 1] - row);
    const int64_t last = min(pos, ((int64_t)a.table_cols << shift) - 1);
    const int64_t first = a.window > 0 ? max((int64_t)0, pos - a.window + 1) : 0;
    for (int i = 0; i < PER; ++i) q_lds[lane + 64 * i] = to_f32(((const T*)a.q)[row * a.q_stride + head * D + lane + 64 * i]) * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[PER] = {};
    for (int64_t j0 = first & ~(int64_t)63; j0 <= last; j0 += 64) {
        const int64_t j = j0 + lane;
        const int64_t page = j >= first && j <= last ? a.table[seq * a.table_stride + (j >> shift)] : -1;
        const bool seen = page >= 0 && page < a.pool.pages;
        const int64_t at = (seen ? page : 0) * a.pool.heads + kv;
        float s = -INFINITY;
        if (seen) {
            const int8_t* k = a.pool.k + ((at << shift) + (j & (P - 1))) * D;
            float dot = 0.f;
            for (int d = 0; d < D; ++d) dot += q_lds[d] * (float)k[d];
            s = dot * a.pool.k_scales[at];
        }
        float top = s;
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float m_new = fmaxf(m, top), keep = m_new == -INFINITY ? 1.f : expf(m - m_new);
        const float p = seen ? expf(s - m_new) : 0.f;
        l = l * keep + wave_sum(p);
        m = m_new;
        for (int i = 0; i < PER; ++i) acc[i] *= keep;
        p_lds[lane] = seen ? p * a.pool.v_scales[at] : 0.f;
        __syncthreads();
        for (int b = 0; b < 4; ++b) {
            const int64_t jb = min(j0 + 16 * b, last);
            int64_t vp = a.table[seq * a.table_stride + (jb >> shift)];
            if (vp < 0 || vp >= a.pool.pages) vp = 0;
            const int8_t* v = a.pool.v + ((vp * a.pool.heads + kv) << shift) * D + ((jb & (P - 1)) >> 4) * D * 16;
            for (int t = 0; t < 16; ++t)
                for (int i = 0; i < PER; ++i) acc[i] += p_lds[16 * b + t] * (float)v[(lane + 64 * i) * 16 + t];
        }
        __syncthreads();
    }
    for (int i = 0; i < PER; ++i)
        ((T*)a.out)[row * a.out_stride + head * D + lane + 64 * i] = from_f32<T>(l == 0.f ? 0.f : acc[i] / l);
}

template <typename T>
static void launch(const Attend& a, int seqs, int head_dim, hipStream_t s) {
    const dim3 grid(a.rows, a.heads);
    if (head_dim == 64) hipLaunchKernelGGL((kv_attention_row_kernel<T, 64>), grid, dim3(64), 0, s, a, seqs);
    else if (head_dim == 128) hipLaunchKernelGGL((kv_attention_row_kernel<T, 128>), grid, dim3(64), 0, s, a, seqs);
    else hipLaunchKernelGGL((kv_attention_row_kernel<T, 256>), grid, dim3(64), 0, s, a, seqs);
}

}  // namespace

extern "C" int lk_kv_attention_q8(const void* q, int type, int64_t q_stride, void* out, int64_t out_stride, const void* k_codes,
                                  const void* v_codes, const float* k_scales, const float* v_scales, int pages, int page_tokens,
                                  const int32_t* table, int64_t table_stride, int table_cols, const int32_t* lens, const int32_t* starts,
                                  int seqs, int rows, int max_fresh, int max_len, int heads, int kv_heads, int head_dim, float scale,
                                  int window, void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    if (!kv_pool_ok(k_codes, v_codes, k_scales, v_scales, pages, kv_heads, head_dim, page_tokens)) return LK_ERR_ARG;
    if (seqs < 0 || rows < 0 || max_fresh < 0 || max_len < 0 || table_cols < 0 || table_stride < table_cols || window < 0 ||
        !(scale > 0.0f && scale <= 3.402823466e38f) || heads <= 0 || heads > 65535 || heads % kv_heads != 0)
        return LK_ERR_ARG;
    if (seqs == 0 || rows == 0) return LK_OK;
    const int64_t row = (int64_t)heads * head_dim;
    if (!q || !out || !lens || !starts || (table_cols > 0 && !table) || (((uintptr_t)q | (uintptr_t)out) & (size - 1)) || q_stride < row ||
        out_stride < row)
        return LK_ERR_ARG;
    const Attend a{q, out, q_stride, out_stride, {(int8_t*)k_codes, (int8_t*)v_codes, (float*)k_scales, (float*)v_scales, pages, kv_heads, kv_log2(page_tokens)},
                   table, lens, starts, table_stride, table_cols, rows, heads, heads / kv_heads, window, scale};
    if (type == LK_TYPE_F32) launch<float>(a, seqs, head_dim, (hipStream_t)stream);
    else if (type == LK_TYPE_F16) launch<__half>(a, seqs, head_dim, (hipStream_t)stream);
    else launch<__hip_bfloat16>(a, seqs, head_dim, (hipStream_t)stream);
    return lk_launch_status();
}
