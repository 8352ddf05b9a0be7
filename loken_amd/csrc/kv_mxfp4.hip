// Rows into and out of the paged 4-bit cache (lk_kv_write_mxfp4, lk_kv_read_mxfp4).
//
// A lane takes eight values, four lanes a block: their largest value through two lane exchanges, its power from the exponent's bits, codes by
// comparison with the seven borders (x / 2^E is exact, so there is no rounding to get wrong). A few rows are bound by one launch's chain of slot, row and stores: one row of
// 8 + 8 heads of 128 written 2.6 us, 64 in f32 3.2; many by the vector instructions of the comparisons beside the rows' bytes: 2048 in bf16 7.3, 4096 12.0, 1.8 TB/s. (Kernel trace.)

#include "kv_mxfp4.h"

namespace {

constexpr int WG = 256;

template <typename T, int D>
__global__ __launch_bounds__(WG) void mx_write_kernel(const T* k, const T* v, int64_t k_stride, int64_t v_stride, const int64_t* slots, int64_t eights, MxPool pool) {
    constexpr int PER = D / 8;
    const int64_t at = (int64_t)blockIdx.x * WG + threadIdx.x;
    const int64_t item = at < eights ? at : eights - 1;   // (a whole wave comes to the lane exchanges)
    const int d0 = (int)(item % PER) * 8;
    const int64_t rest = item / PER;
    const int head = (int)(rest % pool.heads);
    const int64_t tok = rest / pool.heads, slot = slots[tok];
    const bool value = blockIdx.y;
    const T* row = value ? v + tok * v_stride : k + tok * k_stride;
    const MxEight<T> raw = *(const MxEight<T>*)(row + head * D + d0);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32(raw.v[e]);
    const bool present = at < eights && slot >= 0 && slot >> pool.page_shift < pool.pages;
    const int64_t page = (slot >> pool.page_shift) * pool.heads + head;
    mx_store_eight<D>(pool, value, page, (int)(slot & ((1 << pool.page_shift) - 1)), d0, x, present);
}

template <typename T, int D>
__global__ __launch_bounds__(WG) void mx_read_kernel(const int64_t* slots, int64_t eights, MxPool pool, T* k_out, T* v_out) {
    constexpr int PER = D / 8;
    const int64_t item = (int64_t)blockIdx.x * WG + threadIdx.x;
    if (item >= eights) return;
    const int d0 = (int)(item % PER) * 8;
    const int64_t rest = item / PER;
    const int head = (int)(rest % pool.heads);
    const int64_t slot = slots[rest / pool.heads];
    const bool value = blockIdx.y;
    MxEight<T> out;
    if (slot >= 0 && slot >> pool.page_shift < pool.pages) {
        const int64_t page = (slot >> pool.page_shift) * pool.heads + head;
        const int tok = (int)(slot & ((1 << pool.page_shift) - 1));
        const uint32_t codes = MxPlace<D>::load(pool, value, page, tok, d0);
        const int power = *MxPlace<D>::power(pool, value, page, tok, d0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t c = codes >> (4 * e) & 7;
            // 2 x code: 0 1 2 3 4 6 8 12
            const float twice = (float)(0xC8643210u >> (4 * c) & 15);
            const float m = power == 255 ? NAN : ldexpf(twice, power - 128);
            out.v[e] = from_f32<T>(codes >> (4 * e) & 8 ? -m : m);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) out.v[e] = from_f32<T>(0.f);
    }
    *(MxEight<T>*)((value ? v_out : k_out) + item * 8) = out;
}

template <class F>
static int by_type_and_dim(int type, int head_dim, F f) {
    auto dim = [&](auto t) {
        if (head_dim == 64) f(t, std::integral_constant<int, 64>{});
        else if (head_dim == 128) f(t, std::integral_constant<int, 128>{});
        else f(t, std::integral_constant<int, 256>{});
    };
    if (type == LK_TYPE_F32) dim(0.f);
    else if (type == LK_TYPE_F16) dim(__half{});
    else dim(__hip_bfloat16{});
    return lk_launch_status();
}

}  // namespace

extern "C" int lk_kv_write_mxfp4(const void* k, const void* v, int type, int64_t k_stride, int64_t v_stride, const int64_t* slots, int tokens,
                                 int kv_heads, int head_dim, int page_tokens, int pages, void* k_codes, void* v_codes, void* k_powers,
                                 void* v_powers, void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    if (!mx_pool_ok(k_codes, v_codes, k_powers, v_powers, pages, kv_heads, head_dim, page_tokens) || tokens < 0) return LK_ERR_ARG;
    if (tokens == 0) return LK_OK;
    const int64_t row = (int64_t)kv_heads * head_dim;
    if (!k || !v || !slots || ((uintptr_t)slots & 7) || (((uintptr_t)k | (uintptr_t)v) & (size - 1)) || k_stride < row || v_stride < row) return LK_ERR_ARG;
    const int64_t eights = (int64_t)tokens * row / 8, blocks = (eights + WG - 1) / WG;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    const MxPool pool{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_powers, (uint8_t*)v_powers, pages, kv_heads, kv_log2(page_tokens)};
    return by_type_and_dim(type, head_dim, [&](auto t, auto d) {
        using T = decltype(t);
        hipLaunchKernelGGL((mx_write_kernel<T, d.value>), dim3((unsigned)blocks, 2), dim3(WG), 0, (hipStream_t)stream, (const T*)k, (const T*)v, k_stride, v_stride,
                           slots, eights, pool);
    });
}

extern "C" int lk_kv_read_mxfp4(const int64_t* slots, int tokens, int kv_heads, int head_dim, int page_tokens, int pages, const void* k_codes,
                                const void* v_codes, const void* k_powers, const void* v_powers, void* k_out, void* v_out, int type,
                                void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    if (!mx_pool_ok(k_codes, v_codes, k_powers, v_powers, pages, kv_heads, head_dim, page_tokens) || tokens < 0) return LK_ERR_ARG;
    if (tokens == 0) return LK_OK;
    if (!k_out || !v_out || !slots || ((uintptr_t)slots & 7) || (((uintptr_t)k_out | (uintptr_t)v_out) & (size - 1))) return LK_ERR_ARG;
    const int64_t eights = (int64_t)tokens * kv_heads * head_dim / 8, blocks = (eights + WG - 1) / WG;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    const MxPool pool{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_powers, (uint8_t*)v_powers, pages, kv_heads, kv_log2(page_tokens)};
    return by_type_and_dim(type, head_dim, [&](auto t, auto d) {
        using T = decltype(t);
        hipLaunchKernelGGL((mx_read_kernel<T, d.value>), dim3((unsigned)blocks, 2), dim3(WG), 0, (hipStream_t)stream, slots, eights, pool, (T*)k_out, (T*)v_out);
    });
}
