// The steps around the paged 8-bit cache that move little and are bound by latency: which pages a batch's
// sequences get and where each new token goes (lk_kv_plan), the new tokens' rows into the cache (lk_kv_write_q8)
// and rows of the cache as values (lk_kv_read_q8).

#include "kv_cache.h"

#pragma clang fp contract(off)

namespace {

// ---------------------------------------------------------------------------------------------
// The plan: need_i = ceil((past_i + fresh_i) / P) - ceil(past_i / P) pages for sequence i, taken from the free list in
// the order of the sequences; starts = exclusive sums of fresh; row t of sequence i stands at position
// past_i + t - starts_i, whose slot is page * P + position % P.
//
// One launch: every workgroup sums all lengths itself (8 bytes a sequence, from L2) and finds the sequence of its
// rows by bisection in LDS, so nothing waits for a launch that only adds up lengths.
// ---------------------------------------------------------------------------------------------
constexpr int PLAN_WG = 256, PLAN_ROWS = 4 * PLAN_WG;   // rows of a workgroup

static __device__ __forceinline__ int clamp_i32(int64_t v) { return v > 0x7FFFFFFF ? 0x7FFFFFFF : (int)v; }

// Exclusive sums over the workgroup's threads of `a` and `b`, and their totals.
static __device__ __forceinline__ void wg_scan2(int64_t& a, int64_t& b, int64_t (*meet)[2], int64_t& total_a, int64_t& total_b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t sa = a, sb = b;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t ua = __shfl_up(sa, o), ub = __shfl_up(sb, o);
        if (lane >= o) { sa += ua; sb += ub; }
    }
    if (lane == 63) { meet[wave][0] = sa; meet[wave][1] = sb; }
    __syncthreads();
    int64_t before_a = 0, before_b = 0;
    total_a = total_b = 0;
    for (int w = 0; w < PLAN_WG / 64; ++w) {
        if (w < wave) { before_a += meet[w][0]; before_b += meet[w][1]; }
        total_a += meet[w][0];
        total_b += meet[w][1];
    }
    a = before_a + sa - a;
    b = before_b + sb - b;
}

// The last of first[0 .. n - 1] (rising) that is not above `v`, first[0] = 0 <= v.
static __device__ __forceinline__ int last_not_above(const int* first, int n, int v) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ __launch_bounds__(PLAN_WG) void kv_plan_kernel(const int32_t* __restrict__ past, const int32_t* __restrict__ fresh, int seqs,
                                                          int page_shift, const int32_t* __restrict__ free_pages, int n_free,
                                                          const int32_t* __restrict__ taken_in, int32_t* table, int64_t table_stride,
                                                          int table_cols, int32_t* __restrict__ lens, int32_t* __restrict__ starts,
                                                          int64_t* __restrict__ slots, int32_t* __restrict__ positions, int rows,
                                                          int32_t* __restrict__ taken_out) {
    extern __shared__ int plan_lds[];   // [seqs] first row, [seqs] first new page
    __shared__ int64_t meet[PLAN_WG / 64][2];
    int *row0 = plan_lds, *page0 = plan_lds + seqs;
    const int t = threadIdx.x, P = 1 << page_shift;
    const bool writes = blockIdx.x == 0;
    const int per = (seqs + PLAN_WG - 1) / PLAN_WG, i0 = t * per, i1 = min(i0 + per, seqs);
    int64_t tokens = 0, pages = 0;
    for (int i = i0; i < i1; ++i) {
        const int64_t p = max(past[i], 0), f = max(fresh[i], 0);
        tokens += f;
        pages += ((p + f + P - 1) >> page_shift) - ((p + P - 1) >> page_shift);
    }
    int64_t all_tokens, all_pages;
    wg_scan2(tokens, pages, meet, all_tokens, all_pages);
    for (int i = i0; i < i1; ++i) {
        const int64_t p = max(past[i], 0), f = max(fresh[i], 0);
        row0[i] = clamp_i32(tokens);
        page0[i] = clamp_i32(pages);
        if (writes) {
            starts[i] = clamp_i32(tokens);
            lens[i] = clamp_i32(p + f);
        }
        tokens += f;
        pages += ((p + f + P - 1) >> page_shift) - ((p + P - 1) >> page_shift);
    }
    const int64_t taken = taken_in ? max(*taken_in, 0) : 0;
    if (writes && t == 0) {
        starts[seqs] = clamp_i32(all_tokens);
        *taken_out = clamp_i32(taken + all_pages);
    }
    __syncthreads();
    auto page_of = [&](int64_t nth) { return taken + nth < n_free ? free_pages[taken + nth] : -1; };
    // the tables' new entries
    const int n_pages = clamp_i32(all_pages), n_rows = clamp_i32(all_tokens);
    for (int64_t j = (int64_t)blockIdx.x * PLAN_WG + t; j < n_pages; j += (int64_t)gridDim.x * PLAN_WG) {
        const int i = last_not_above(page0, seqs, (int)j);
        const int64_t col = (((int64_t)max(past[i], 0) + P - 1) >> page_shift) + j - page0[i];
        if (col < table_cols) table[i * table_stride + col] = page_of(j);
    }
    // the rows; a new page's number comes from the free list, where no workgroup waits for another's store
    for (int64_t r = (int64_t)blockIdx.x * PLAN_ROWS + t; r < min((int64_t)rows, ((int64_t)blockIdx.x + 1) * PLAN_ROWS); r += PLAN_WG) {
        int64_t slot = -1, at = 0;
        if (r < n_rows) {
            const int i = last_not_above(row0, seqs, (int)r);
            const int64_t p = max(past[i], 0);
            at = p + r - row0[i];
            const int64_t col = at >> page_shift, have = (p + P - 1) >> page_shift;
            if (col < table_cols) {
                const int64_t page = col < have ? table[i * table_stride + col] : page_of(page0[i] + col - have);
                if (page >= 0) slot = (page << page_shift) + (at & (P - 1));
            }
        }
        slots[r] = slot;
        positions[r] = clamp_i32(at);
    }
}

// ---------------------------------------------------------------------------------------------
// New rows into the cache. The rows of a call that belong to one page, with no row of another between them, are a run; the wave that
// finds a run's first row writes the run. With s_old the page's scale (0 where the run holds the page's first
// token, which starts the page anew):
//     s = max(s_old, max |x| / 127),   old codes c -> round(c s_old / s),   new codes round(x / s)
// quotients exact, halves away from zero. A product with 1 / s gives the quotient's whole part q or its neighbour; the
// remainder x - q s is exact in one fused multiply-add (for q > 0 both are multiples of s's last place, and what is left is
// below 2 s), and at least half of s where the code is one more.
// ---------------------------------------------------------------------------------------------
static __device__ __forceinline__ float wave_most(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

static __device__ __forceinline__ int code_of(float x, float s, float inv) {
    const float a = fabsf(x);
    const float q = fminf(floorf(a * inv), 127.0f);   // or a neighbour of the quotient's whole part; the remainder below then says so
    const int c = min((int)q + (fmaf(-q, s, a) >= 0.5f * s ? 1 : 0), 127);
    return x != x || inv == 0.0f ? 0 : x < 0.0f ? -c : c;
}

// An old code at the new scale; 64 bits hold c s_old and q s exactly.
static __device__ __forceinline__ int rescaled(int c, float ratio, double s_old, double s) {
    const int a = abs(c);
    int q = (int)floorf(fmaf((float)a, ratio, 0.5f));
    const double r = fma(-(double)q, s, (double)a * s_old);
    q += r >= 0.5 * s ? 1 : r < -0.5 * s ? -1 : 0;
    return c < 0 ? -q : q;
}

template <typename T, int D>
__global__ __launch_bounds__(128) void kv_write_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t k_stride, int64_t v_stride,
                                                       const int64_t* __restrict__ slots, int tokens, KvPool pool, int window) {
    constexpr int PER = D / 64;
    const int lane = threadIdx.x & 63, head = blockIdx.y;
    const bool values = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) != 0;   // wave 0: keys, wave 1: values
    const int P = 1 << pool.page_shift, shift = pool.page_shift;
    auto page_at = [&](int t) -> int64_t {
        if (t < 0 || t >= tokens) return -1;
        const int64_t s = slots[t];
        return s < 0 || (s >> shift) >= pool.pages ? -1 : s >> shift;
    };
    const T* rows = (values ? v : k) + (int64_t)head * D + lane;
    const int64_t stride = values ? v_stride : k_stride;
    const int first = blockIdx.x * window;
    const int64_t mine = lane < window ? page_at(first + lane) : -1;
    uint64_t leaders = __ballot(mine >= 0 && mine != page_at(first + lane - 1));
    while (leaders) {
        const int t0 = first + __ffsll((unsigned long long)leaders) - 1;
        leaders &= leaders - 1;
        const int64_t page = page_at(t0);
        // absent rows do not end a run: the last row before them may be of the same page
        bool inside = false;
        for (int t = t0; t > 0; t -= 64) {
            const int64_t before = page_at(t - 1 - lane);
            const uint64_t there = __ballot(before >= 0);
            if (!there) continue;
            inside = (__ballot(before == page) >> (__ffsll((unsigned long long)there) - 1)) & 1;
            break;
        }
        if (inside) continue;
        // the run's length, and whether it holds the page's first token
        int n = 0;
        bool anew = false;
        for (;;) {
            const int t = t0 + n + lane;
            const int64_t here = page_at(t);
            const uint64_t ends = __ballot(t >= tokens || (here >= 0 && here != page));
            const uint64_t zero = __ballot(here == page && (slots[t] & (P - 1)) == 0);
            const int more = ends ? __ffsll((unsigned long long)ends) - 1 : 64;
            anew = anew || (zero & (more == 64 ? ~0ull : (1ull << more) - 1)) != 0;
            n += more;
            if (more < 64) break;
        }
        float most = 0.0f;
        for (int j = 0; j < n; ++j) {
            if (page_at(t0 + j) != page) continue;   // an absent row
            const T* row = rows + (int64_t)(t0 + j) * stride;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float a = fabsf(to_f32(row[64 * i]));
                most = fmaxf(most, a <= 3.402823466e38f ? a : 0.0f);   // the scale is that of the finite values
            }
        }
        most = wave_most(most);
        float* scale_at = (values ? pool.v_scales : pool.k_scales) + page * pool.heads + head;
        const float stored = *scale_at;
        const float s_old = !anew && stored <= 3.402823466e38f && stored > 0.0f ? stored : 0.0f;
        float s = fmaxf(s_old, most / 127.0f);
        if (s < 1.17549435e-38f) s = 0.0f;   // a scale with no normal 1 / s: the page holds zeros
        int8_t* codes = (values ? pool.v : pool.k) + ((page * pool.heads + head) << shift) * D;
        if (anew || s != s_old) {
            const float ratio = s > 0.0f ? s_old / s : 0.0f;
            for (int at = lane * 16; at < (D << shift); at += 64 * 16) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (s_old > 0.0f) {
                    w = *(const uint4*)(codes + at);
                    uint32_t* u = (uint32_t*)&w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t r = 0;
#pragma unroll
                        for (int b = 0; b < 4; ++b) r |= (uint32_t)(rescaled((int8_t)(u[i] >> (8 * b)), ratio, s_old, s) & 0xFF) << (8 * b);
                        u[i] = r;
                    }
                }
                *(uint4*)(codes + at) = w;
            }
            if (lane == 0) *scale_at = s;
            __threadfence();   // the new codes below are stored after these, which other lanes wrote
        }
        const float inv = s > 0.0f ? 1.0f / s : 0.0f;
        for (int j = 0; j < n;) {
            const int t = t0 + j;
            if (page_at(t) != page) { ++j; continue; }
            const int off = (int)(slots[t] & (P - 1));
            const T* row = rows + (int64_t)t * stride;
            // a whole run of sixteen values of a column is one store
            if (values && (off & 15) == 0 && j + 16 <= n && __ballot(lane < 16 && slots[t + min(lane, 15)] != slots[t] + lane) == 0) {
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int b = 0; b < 16; ++b)
                        w[b / 4] |= (uint32_t)(code_of(to_f32(row[b * stride + 64 * i]), s, inv) & 0xFF) << (8 * (b % 4));
                    *(uint4*)(codes + ((off >> 4) * D + lane + 64 * i) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                j += 16;
                continue;
            }
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int d = lane + 64 * i, c = code_of(to_f32(row[64 * i]), s, inv);
                codes[values ? ((off >> 4) * D + d) * 16 + (off & 15) : off * D + d] = (int8_t)c;
            }
            ++j;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Rows of the cache as values: one wave to sixteen rows of a head and side.
// ---------------------------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(128) void kv_read_kernel(const int64_t* __restrict__ slots, int tokens, KvPool pool, T* __restrict__ k_out,
                                                      T* __restrict__ v_out) {
    constexpr int PER = D / 64;
    const int lane = threadIdx.x & 63, head = blockIdx.y;
    const bool values = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) != 0;
    const int shift = pool.page_shift, mask = (1 << shift) - 1;
    T* out = values ? v_out : k_out;
    for (int t = blockIdx.x * 16; t < min(tokens, (int)blockIdx.x * 16 + 16); ++t) {
        const int64_t slot = slots[t], page = slot >> shift;
        const bool held = slot >= 0 && page < pool.pages;
        const int off = (int)(slot & mask);
        const int8_t* codes = (values ? pool.v : pool.k) + (((held ? page : 0) * pool.heads + head) << shift) * D;
        const float s = (values ? pool.v_scales : pool.k_scales)[(held ? page : 0) * pool.heads + head];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int d = lane + 64 * i;
            const int8_t c = codes[values ? ((off >> 4) * D + d) * 16 + (off & 15) : off * D + d];
            out[((int64_t)t * pool.heads + head) * D + d] = from_f32<T>(held ? (float)c * s : 0.0f);
        }
    }
}

template <template <typename, int> class Launch, class... A>
static int by_type_and_dim(int type, int head_dim, A... a) {
    auto dims = [&](auto tag) {
        using T = decltype(tag);
        if (head_dim == 64) Launch<T, 64>::run(a...);
        else if (head_dim == 128) Launch<T, 128>::run(a...);
        else Launch<T, 256>::run(a...);
        return lk_launch_status();
    };
    if (type == LK_TYPE_F32) return dims(float{});
    if (type == LK_TYPE_F16) return dims(__half{});
    return dims(__hip_bfloat16{});
}

template <typename T, int D>
struct Write {
    static void run(const void* k, const void* v, int64_t ks, int64_t vs, const int64_t* slots, int tokens, KvPool pool, int window, hipStream_t s) {
        hipLaunchKernelGGL((kv_write_kernel<T, D>), dim3((tokens + window - 1) / window, pool.heads), dim3(128), 0, s, (const T*)k, (const T*)v,
                           ks, vs, slots, tokens, pool, window);
    }
};
template <typename T, int D>
struct Read {
    static void run(const int64_t* slots, int tokens, KvPool pool, void* k, void* v, hipStream_t s) {
        hipLaunchKernelGGL((kv_read_kernel<T, D>), dim3((tokens + 15) / 16, pool.heads), dim3(128), 0, s, slots, tokens, pool, (T*)k, (T*)v);
    }
};

}  // namespace

extern "C" int lk_kv_plan(const int32_t* past, const int32_t* fresh, int seqs, int page_tokens, const int32_t* free_pages, int n_free,
                          const int32_t* taken, int32_t* table, int64_t table_stride, int table_cols, int32_t* lens, int32_t* starts,
                          int64_t* slots, int32_t* positions, int rows, int32_t* taken_out, void* stream) {
    if (seqs < 0 || rows < 0 || n_free < 0 || !kv_page_tokens_ok(page_tokens) || table_cols < 0 || table_stride < table_cols) return LK_ERR_ARG;
    if (!starts || !taken_out || taken == taken_out || (seqs > 0 && (!past || !fresh || !lens || (table_cols > 0 && !table))) ||
        (rows > 0 && (!slots || !positions)) || (n_free > 0 && !free_pages) || ((uintptr_t)slots & 7))
        return LK_ERR_ARG;
    if (seqs > LK_KV_PLAN_SEQS) return LK_ERR_SIZE;
    // a kernel gets 64 KB of LDS unless the runtime is told otherwise
    if (seqs * 8 > 60 * 1024 &&
        hipFuncSetAttribute((const void*)kv_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, seqs * 8) != hipSuccess) {
        (void)hipGetLastError();
        return LK_ERR_LAUNCH;
    }
    const int blocks = rows > 0 ? (rows + PLAN_ROWS - 1) / PLAN_ROWS : 1;
    hipLaunchKernelGGL(kv_plan_kernel, dim3(blocks), dim3(PLAN_WG), seqs * 8, (hipStream_t)stream, past, fresh, seqs, kv_log2(page_tokens),
                       free_pages, n_free, taken, table, table_stride, table_cols, lens, starts, slots, positions, rows, taken_out);
    return lk_launch_status();
}

extern "C" int lk_kv_write_q8(const void* k, const void* v, int type, int64_t k_stride, int64_t v_stride, const int64_t* slots, int tokens,
                              int kv_heads, int head_dim, int page_tokens, int pages, void* k_codes, void* v_codes, float* k_scales,
                              float* v_scales, void* stream) {
    if (!kv_type_size(type)) return LK_ERR_TYPE;
    if (tokens < 0 || !kv_pool_ok(k_codes, v_codes, k_scales, v_scales, pages, kv_heads, head_dim, page_tokens)) return LK_ERR_ARG;
    if (tokens == 0) return LK_OK;
    const int64_t row = (int64_t)kv_heads * head_dim;
    if (!k || !v || !slots || ((uintptr_t)slots & 7) || (((uintptr_t)k | (uintptr_t)v) & (kv_type_size(type) - 1)) || k_stride < row ||
        v_stride < row)
        return LK_ERR_ARG;
    const KvPool pool{(int8_t*)k_codes, (int8_t*)v_codes, k_scales, v_scales, pages, kv_heads, kv_log2(page_tokens)};
    const int window = tokens <= 512 ? 1 : 16;
    return by_type_and_dim<Write>(type, head_dim, k, v, k_stride, v_stride, slots, tokens, pool, window, (hipStream_t)stream);
}

extern "C" int lk_kv_read_q8(const int64_t* slots, int tokens, int kv_heads, int head_dim, int page_tokens, int pages, const void* k_codes,
                             const void* v_codes, const float* k_scales, const float* v_scales, void* k_out, void* v_out, int type,
                             void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    if (tokens < 0 || !kv_pool_ok(k_codes, v_codes, k_scales, v_scales, pages, kv_heads, head_dim, page_tokens)) return LK_ERR_ARG;
    if (tokens == 0) return LK_OK;
    if (!slots || !k_out || !v_out || ((uintptr_t)slots & 7) || (((uintptr_t)k_out | (uintptr_t)v_out) & (size - 1))) return LK_ERR_ARG;
    const KvPool pool{(int8_t*)k_codes, (int8_t*)v_codes, (float*)k_scales, (float*)v_scales, pages, kv_heads, kv_log2(page_tokens)};
    return by_type_and_dim<Read>(type, head_dim, slots, tokens, pool, k_out, v_out, (hipStream_t)stream);
}
