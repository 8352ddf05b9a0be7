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
    extern __shared__ int plan_lds[];   // [seqs] first row, [seqs] first new page, [seqs] past
    __shared__ int64_t meet[PLAN_WG / 64][2];
    int *row0 = plan_lds, *page0 = plan_lds + seqs, *had = plan_lds + 2 * seqs;
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
        had[i] = (int)p;
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
        const int64_t col = (((int64_t)had[i] + P - 1) >> page_shift) + j - page0[i];
        if (col < table_cols) table[i * table_stride + col] = page_of(j);
    }
    // the rows; a new page's number comes from the free list, where no workgroup waits for another's store
    for (int64_t r = (int64_t)blockIdx.x * PLAN_ROWS + t; r < min((int64_t)rows, ((int64_t)blockIdx.x + 1) * PLAN_ROWS); r += PLAN_WG) {
        int64_t slot = -1, at = 0;
        if (r < n_rows) {
            const int i = last_not_above(row0, seqs, (int)r);
            const int64_t p = had[i];
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
// New rows into the cache. The rows of a call that belong to one page, with no row of another between them, are a run; the workgroup that
// finds a run's first row writes the run: a workgroup for its keys, one for its values, of as many waves as hold a page. With s_old the page's scale (0 where the run
// holds the page's first token, which starts the page anew):
//     s = max(s_old, max |x| / 127),   old codes c -> round(c s_old / s),   new codes round(x / s)
// quotients exact, halves away from zero. A product with 1 / s gives the quotient's whole part q or its neighbour; the
// remainder x - q s is exact in one fused multiply-add (for q > 0 both are multiples of s's last place, and what is left is
// below 2 s), and at least half of s where the code is one more.
//
// What it costs is latency: slots, then rows and scale, then (where a scale grows) the page. A lane holds four columns of eight
// consecutive rows, whose loads are all in flight together: four codes of a key row are one store, eight of a value column another.
// 64 single tokens of 8 heads of 128 in f32: 6 us; 1504 rows of a prompt in bf16, 16 tokens a page: 8 us. (With slots looked up row by
// row and a fence before the new codes the single tokens took 12.)
// ---------------------------------------------------------------------------------------------
constexpr int ROWS_HELD = 8, WRITE_WAVES = 8;

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

static __device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 0xFF) | (uint32_t)(b & 0xFF) << 8 | (uint32_t)(c & 0xFF) << 16 | (uint32_t)(d & 0xFF) << 24;
}

template <typename T, int D>
__global__ __launch_bounds__(64 * WRITE_WAVES) void kv_write_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t k_stride, int64_t v_stride,
                                                       bool aligned, const int64_t* __restrict__ slots, int tokens, KvPool pool, int window) {
    constexpr int LANES = D / 4;                       // of a row
    constexpr int OF_WAVE = ROWS_HELD * (64 / LANES);  // rows that a wave holds
    __shared__ uint32_t tables[64];
    __shared__ float meet[WRITE_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int head = blockIdx.y, side = blockIdx.z;    // keys, values
    const int batch = OF_WAVE * waves, d0 = 4 * (lane % LANES), row0 = OF_WAVE * wave + ROWS_HELD * (lane / LANES);
    const int P = 1 << pool.page_shift, shift = pool.page_shift;
    auto page_of = [&](int64_t slot) -> int64_t { return slot < 0 || (slot >> shift) >= pool.pages ? -1 : slot >> shift; };
    auto slot_at = [&](int t) -> int64_t { return t < 0 || t >= tokens ? -1 : slots[t]; };
    const T* rows = (side ? v : k) + (int64_t)head * D + d0;
    const int64_t stride = side ? v_stride : k_stride;
    // the window's rows, the one before them and what fits behind
    const int first = blockIdx.x * window, base = first - 1;
    const int64_t my_slot = slot_at(base + lane), my_page = page_of(my_slot);
    const int64_t page_before = __shfl_up((long long)my_page, 1);   // (by all lanes: one that is left out has nothing to give)
    uint64_t leaders = __ballot(my_page >= 0 && my_page != page_before) & ((1ull << window) - 1) << 1;
    while (leaders) {
        const int at = __ffsll((unsigned long long)leaders) - 1, t0 = base + at;
        leaders &= leaders - 1;
        const int64_t page = __shfl((long long)my_page, at), slot0 = __shfl((long long)my_slot, at);
        // absent rows do not end a run: the last row before them may be of the same page
        bool inside = false;
        if (t0 > 0 && __shfl((long long)my_page, at - 1) < 0)
            for (int t = t0; t > 0; t -= 64) {
                const int64_t before = page_of(slot_at(t - 1 - lane));
                const uint64_t there = __ballot(before >= 0);
                if (!there) continue;
                inside = (__ballot(before == page) >> (__ffsll((unsigned long long)there) - 1)) & 1;
                break;
            }
        if (inside) continue;
        // The run's rows, up to the last present one (a batch's padding may follow); whether it holds the page's first token; whether its
        // rows are the page's tokens in their order.
        int n = 0, rows_there = 0;
        bool anew = false, straight = true;
        for (int skip = at, t_here = base;; skip = 0, t_here += 64) {
            const int t = t_here + lane;
            const int64_t slot = t_here == base ? my_slot : slot_at(t), here = page_of(slot);
            const uint64_t from = ~0ull << skip;
            const uint64_t ends = __ballot(t >= tokens || (here >= 0 && here != page)) & from;
            const int stop = ends ? __ffsll((unsigned long long)ends) - 1 : 64;
            const uint64_t there = __ballot(here == page) & from & (stop == 64 ? ~0ull : (1ull << stop) - 1);
            anew = anew || (__ballot((slot & (P - 1)) == 0) & there) != 0;
            straight = straight && (__ballot(slot != slot0 + (t - t0)) & there) == 0;
            rows_there += __popcll(there);
            if (there) n = t_here + 64 - __clzll((long long)there) - t0;
            if (stop < 64) break;
        }
        straight = straight && rows_there == n;
        const bool whole = straight && n == P;   // (then it starts with the first)
        float x[ROWS_HELD][4];
        int64_t off[ROWS_HELD];   // the token's place in the page; -1: not the page's
        auto load = [&](int j0) {
#pragma unroll
            for (int i = 0; i < ROWS_HELD; ++i) {
                const int j = j0 + row0 + i;
                off[i] = -1;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
                if (j < n) {
                    const T* row = rows + (int64_t)(t0 + j) * stride;
                    if (aligned) {
                        const float4 f = Load4<T>::at(row);
                        x[i][0] = f.x; x[i][1] = f.y; x[i][2] = f.z; x[i][3] = f.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[i][e] = to_f32(row[e]);
                    }
                    const int64_t slot = straight ? slot0 + j : slots[t0 + j];
                    off[i] = page_of(slot) == page ? slot & (P - 1) : -1;
                }
            }
        };
        float* scale_at = (side ? pool.v_scales : pool.k_scales) + page * pool.heads + head;
        const float stored = *scale_at;
        float most = 0.0f;
        for (int j0 = 0; j0 < n; j0 += batch) {
            load(j0);
#pragma unroll
            for (int i = 0; i < ROWS_HELD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = fabsf(x[i][e]);
                    most = fmaxf(most, off[i] >= 0 && a <= 3.402823466e38f ? a : 0.0f);   // the scale is that of the finite values
                }
        }
        most = wave_most(most);
        if (waves > 1) {
            __syncthreads();   // the last run's reads
            if (lane == 0) meet[wave] = most;
            __syncthreads();
            for (int w = 0; w < waves; ++w) most = fmaxf(most, meet[w]);
        }
        const float s_old = !anew && stored <= 3.402823466e38f && stored > 0.0f ? stored : 0.0f;
        float s = fmaxf(s_old, most / 127.0f);
        if (s < 1.17549435e-38f) s = 0.0f;   // a scale with no normal 1 / s: the page holds zeros
        int8_t* codes = (side ? pool.v : pool.k) + ((page * pool.heads + head) << shift) * D;
        if ((anew || s != s_old) && threadIdx.x == 0) *scale_at = s;
        if ((anew && !whole) || (!anew && s != s_old)) {
            const float ratio = s > 0.0f ? s_old / s : 0.0f;
            // what each byte becomes: four of them a lane
            uint8_t* table = (uint8_t*)tables;
            if (s_old > 0.0f) {
                if (wave == 0) tables[lane] = pack4(rescaled((int8_t)(4 * lane), ratio, s_old, s), rescaled((int8_t)(4 * lane + 1), ratio, s_old, s),
                                           rescaled((int8_t)(4 * lane + 2), ratio, s_old, s), rescaled((int8_t)(4 * lane + 3), ratio, s_old, s));
                __syncthreads();
            }
            for (int p = threadIdx.x * 16; p < (D << shift); p += blockDim.x * 16) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (s_old > 0.0f) {
                    w = *(const uint4*)(codes + p);
                    uint32_t* u = (uint32_t*)&w;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        u[i] = (uint32_t)table[u[i] & 0xFF] | (uint32_t)table[u[i] >> 8 & 0xFF] << 8 | (uint32_t)table[u[i] >> 16 & 0xFF] << 16 |
                               (uint32_t)table[u[i] >> 24] << 24;
                }
                *(uint4*)(codes + p) = w;
            }
            // the new codes below go where other threads have just stored: stores that have been waited for are in front of them
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        const float inv = s > 0.0f ? 1.0f / s : 0.0f;
        for (int j0 = 0; straight && j0 < n; j0 += batch) {
            if (n > batch) load(j0);
            int c[ROWS_HELD][4];
#pragma unroll
            for (int i = 0; i < ROWS_HELD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[i][e] = code_of(x[i][e], s, inv);
            if (side == 0) {
#pragma unroll
                for (int i = 0; i < ROWS_HELD; ++i)
                    if (off[i] >= 0) *(uint32_t*)(codes + off[i] * D + d0) = pack4(c[i][0], c[i][1], c[i][2], c[i][3]);
            } else if (off[ROWS_HELD - 1] >= 0 && (off[0] & 7) == 0) {
#pragma unroll
                for (int h = 0; h < ROWS_HELD; h += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *(uint2*)(codes + ((off[h] >> 4) * D + d0 + e) * 16 + (off[h] & 8)) =
                            make_uint2(pack4(c[h][e], c[h + 1][e], c[h + 2][e], c[h + 3][e]), pack4(c[h + 4][e], c[h + 5][e], c[h + 6][e], c[h + 7][e]));
            } else {
#pragma unroll
                for (int i = 0; i < ROWS_HELD; ++i)
                    if (off[i] >= 0)
#pragma unroll
                        for (int e = 0; e < 4; ++e) codes[((off[i] >> 4) * D + d0 + e) * 16 + (off[i] & 15)] = (int8_t)c[i][e];
            }
        }
        // Other runs may name a token twice, and the last row stays: one row after the other, a column always the same lane's.
        for (int j = 0; !straight && wave == 0 && j < n; ++j) {
            const int64_t slot = slots[t0 + j];
            if (page_of(slot) != page || lane >= LANES) continue;
            const T* row = rows + (int64_t)(t0 + j) * stride;
            const int place = (int)(slot & (P - 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = code_of(to_f32(row[e]), s, inv);
                codes[side ? ((place >> 4) * D + d0 + e) * 16 + (place & 15) : place * D + d0 + e] = (int8_t)c;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Rows of the cache as values: a wave to sixteen rows of a head and side. Sixteen rows that are a run of the cache (sixteen tokens
// in their order) are one load a column of the values.
// ---------------------------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(128) void kv_read_kernel(const int64_t* __restrict__ slots, int tokens, KvPool pool, T* __restrict__ k_out,
                                                      T* __restrict__ v_out) {
    constexpr int PER = D / 64;
    const int lane = threadIdx.x & 63, head = blockIdx.y, t0 = blockIdx.x * 16, n = min(tokens - t0, 16);
    const bool values = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) != 0;
    const int shift = pool.page_shift, mask = (1 << shift) - 1;
    const int8_t* codes = values ? pool.v : pool.k;
    const float* scales = values ? pool.v_scales : pool.k_scales;
    T* out = (values ? v_out : k_out) + ((int64_t)t0 * pool.heads + head) * D + lane;
    const int64_t row = (int64_t)pool.heads * D;
    // lanes 0 .. 15: a row's slot, where its codes start, and its scale
    const int64_t slot = (lane & 15) < n ? slots[t0 + (lane & 15)] : -1, page = slot >> shift;
    const bool held = slot >= 0 && page < pool.pages;
    const int64_t at_page = (held ? page : 0) * pool.heads + head;
    const int64_t start = (at_page << shift) * D;
    const float s = held ? scales[at_page] : 0.0f;
    const int off = held ? (int)(slot & mask) : 0;
    const int64_t slot0 = __shfl((long long)slot, 0);
    if (values && __ballot(!held || slot != slot0 + (lane & 15) || (slot0 & 15) != 0) == 0) {
        const float s0 = __shfl(s, 0);
        const int8_t* from = codes + __shfl((long long)start, 0) + ((int64_t)(__shfl(off, 0) >> 4) * D + lane) * 16;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint4 w = *(const uint4*)(from + 64 * 16 * i);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 16; ++j) out[j * row + 64 * i] = from_f32<T>((float)(int8_t)(u[j / 4] >> (8 * (j % 4))) * s0);
        }
        return;
    }
    int8_t c[16][PER];   // all loads before the first store
#pragma unroll
    for (int j = 0; j < 16; ++j) {   // (a row that is absent or none: of page 0, and not used)
        const int offj = __shfl(off, j);
        const int8_t* from = codes + __shfl((long long)start, j);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int d = lane + 64 * i;
            c[j][i] = from[values ? ((offj >> 4) * D + d) * 16 + (offj & 15) : offj * D + d];
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float sj = __shfl(s, j);   // 0 where the row is absent
        const bool is = __shfl((int)held, j) != 0;
        if (j < n)
#pragma unroll
            for (int i = 0; i < PER; ++i) out[j * row + 64 * i] = from_f32<T>(is ? (float)c[j][i] * sj : 0.0f);
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
        const int four = 4 * sizeof(T) - 1;
        const bool aligned = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(ks * sizeof(T)) | (uintptr_t)(vs * sizeof(T))) & four) == 0;
        const int of_wave = ROWS_HELD * 256 / D, waves = min(WRITE_WAVES, ((1 << pool.page_shift) + of_wave - 1) / of_wave);
        hipLaunchKernelGGL((kv_write_kernel<T, D>), dim3((tokens + window - 1) / window, pool.heads, 2), dim3(64 * waves), 0, s, (const T*)k,
                           (const T*)v, ks, vs, aligned, slots, tokens, pool, window);
    }
};
template <typename T, int D>
struct Read {
    static void run(const int64_t* slots, int tokens, KvPool pool, void* k, void* v, hipStream_t s) {
        hipLaunchKernelGGL((kv_read_kernel<T, D>), dim3((tokens + 15) / 16, pool.heads), dim3(128), 0, s, slots, tokens, pool, (T*)k, (T*)v);
    }
};

}  // namespace

// Whether any two of the arrays, the first `inputs` of which are only read, share memory that one of them is written to.
struct Bytes {
    const void* at;
    int64_t size;
};
static bool written_together(const Bytes* a, int inputs, int all) {
    for (int j = inputs; j < all; ++j)
        for (int i = 0; i < j; ++i) {
            const uintptr_t p = (uintptr_t)a[i].at, q = (uintptr_t)a[j].at;
            if (a[i].size > 0 && a[j].size > 0 && (p < q ? q - p < (uint64_t)a[i].size : p - q < (uint64_t)a[j].size)) return true;
        }
    return false;
}

extern "C" int lk_kv_plan(const int32_t* past, const int32_t* fresh, int seqs, int page_tokens, const int32_t* free_pages, int n_free,
                          const int32_t* taken, int32_t* table, int64_t table_stride, int table_cols, int32_t* lens, int32_t* starts,
                          int64_t* slots, int32_t* positions, int rows, int32_t* taken_out, void* stream) {
    if (seqs < 0 || rows < 0 || n_free < 0 || !kv_page_tokens_ok(page_tokens) || table_cols < 0 || table_stride < table_cols) return LK_ERR_ARG;
    if (!starts || !taken_out || taken == taken_out || (seqs > 0 && (!past || !fresh || !lens || (table_cols > 0 && !table))) ||
        (rows > 0 && (!slots || !positions)) || (n_free > 0 && !free_pages) || ((uintptr_t)slots & 7))
        return LK_ERR_ARG;
    if (seqs > LK_KV_PLAN_SEQS) return LK_ERR_SIZE;
    // every workgroup reads all lengths while the first one writes its sums
    const Bytes arrays[] = {{past, 4 * (int64_t)seqs}, {fresh, 4 * (int64_t)seqs}, {free_pages, 4 * (int64_t)n_free}, {taken, taken ? 4 : 0},
                            {table, seqs > 0 && table_cols > 0 ? 4 * ((seqs - 1) * table_stride + table_cols) : 0}, {lens, 4 * (int64_t)seqs},
                            {starts, 4 * ((int64_t)seqs + 1)}, {slots, 8 * (int64_t)rows}, {positions, 4 * (int64_t)rows}, {taken_out, 4}};
    if (written_together(arrays, 4, 10)) return LK_ERR_ARG;
    // a kernel gets 64 KB of LDS unless the runtime is told otherwise
    if (seqs * 12 > 60 * 1024 &&
        hipFuncSetAttribute((const void*)kv_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, seqs * 12) != hipSuccess) {
        (void)hipGetLastError();
        return LK_ERR_LAUNCH;
    }
    const int blocks = rows > 0 ? (rows + PLAN_ROWS - 1) / PLAN_ROWS : 1;
    hipLaunchKernelGGL(kv_plan_kernel, dim3(blocks), dim3(PLAN_WG), seqs * 12, (hipStream_t)stream, past, fresh, seqs, kv_log2(page_tokens),
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
    // Rows of which a workgroup writes the runs that start there, one after the other: single tokens' runs are a row each, a prompt's a
    // page, and a workgroup that finds none costs 3 ns. 1504 rows of a prompt in bf16, 16 and 32 rows to a workgroup: 7.7 and 11.3 us
    // with pages of 16 tokens, 9.2 and 7.7 of 32, 10.1 and 8.3 of 64, 16.2 and 9.9 of 128.
    const int window = tokens <= 128 ? 1 : tokens <= 1024 ? 4 : page_tokens < 32 ? page_tokens : 32;
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
