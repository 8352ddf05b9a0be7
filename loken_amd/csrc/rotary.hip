// Norms of the query and key heads and their rotation in one pass (lk_qk_norm_rope), and the same with keys and values going straight into the
// 4-bit cache (lk_qk_norm_rope_kv_mxfp4).
//
// A head's values x become y = x / sqrt(mean x^2 + eps) * w, and of y the pairs (a, b) become (a cos - b sin, a sin + b cos), the angle of pair i
// being position * frequency[i]. A pair's angle is the same for all heads of a token: a workgroup makes the angles of its tokens once, in
// LDS, in 64 bits (a far position's angle in 32 bits is off by position * 2^-24), and its waves take heads in turn.
//
// A lane holds four neighbouring pairs of a head (a, b apart by `pairs`, or side by side), so a pair never leaves its lane; what is not rotated
// goes the same way, by pairs that stay as they are. Queries are computed in 32 bits and rounded once. Keys that go to the cache are computed in 64: a value next
// to the border of two codes would else come out as the other one. They pass through LDS, where a block's 32 values come together.
//
// Bound by the rows' bytes: 4096 tokens of 32 + 8 heads of 128, bf16, three axes of positions 17.4 us, 4.8 TB/s in and out. Into the cache by the 64-bit norms and
// rotations too: 2048 tokens of 32 + 8 + 8 heads, bf16, 14.6 us without norms, 18.3 with them; a few tokens by the chain position, angle, rows: one token 3.1 us. (Kernel trace.)

#include <type_traits>

#include "kv_mxfp4.h"

namespace {

constexpr int WAVES = 4, WG = 64 * WAVES;
constexpr int VEC = 4;   // pairs of a lane

struct Rotate {
    const void *q, *k, *v;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    int rows, heads, kv_heads;
    const float *q_weight, *k_weight;
    float eps;
    const int32_t* positions;
    int64_t axis_stride;
    int axes;
    const float* frequencies;
    const uint8_t* axis;
    int pairs;
    float factor;
    const int64_t* slots;
    MxPool pool;
};

template <typename T>
struct __attribute__((aligned(sizeof(T)))) Four { T v[VEC]; };

// Where a lane's pairs u0 .. u0 + 3 of a head stand: two runs of four values, which are the pairs' first and second values or, of neighbours, the
// first and the last two pairs.
struct Runs {
    int lo, hi;
    __device__ __forceinline__ Runs(int u0, int pairs, bool neighbours) {
        const bool apart = !neighbours && u0 < pairs;
        lo = apart ? u0 : 2 * u0;
        hi = apart ? u0 + pairs : 2 * u0 + VEC;
    }
};

// A lane's four pairs, normed, and turned if they are of the rotation.
template <typename F, typename T, int D, bool NEIGHBOURS>
static __device__ __forceinline__ void turn(const T* x, const float* weight, float eps, const Runs& at, bool turned, const F (&cosine)[VEC], const F (&sine)[VEC],
                                            F (&y)[2 * VEC]) {
    const Four<T> lo = *(const Four<T>*)(x + at.lo), hi = *(const Four<T>*)(x + at.hi);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        y[j] = (F)to_f32(lo.v[j]);
        y[VEC + j] = (F)to_f32(hi.v[j]);
    }
    if (weight) {
        const Four<float> wl = *(const Four<float>*)(weight + at.lo), wh = *(const Four<float>*)(weight + at.hi);
        F sum = 0;
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) sum += y[j] * y[j];
#pragma unroll
        for (int o = 1; o < D / 2 / VEC; o <<= 1) sum += __shfl_xor(sum, o);
        const F by = (F)1 / sqrt(sum * (F)(1.0 / D) + (F)eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            y[j] = y[j] * by * (F)wl.v[j];
            y[VEC + j] = y[VEC + j] * by * (F)wh.v[j];
        }
    }
    if (!turned) return;   // (not by an angle of 0: beside an infinity that would leave no number)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int a = NEIGHBOURS ? 2 * j : j, b = NEIGHBOURS ? 2 * j + 1 : VEC + j;
        const F first = y[a], second = y[b];
        y[a] = first * cosine[j] - second * sine[j];
        y[b] = first * sine[j] + second * cosine[j];
    }
}

// `tokens` to a workgroup: one whose heads the waves share, or, into the cache, WAVES of them, one a wave.
template <typename T, int D, bool NEIGHBOURS, bool CACHE>
__global__ __launch_bounds__(WG) void rotate_kernel(Rotate r, int tokens_of) {
    const int tokens = CACHE ? tokens_of : 1;
    constexpr int LANES = D / 2 / VEC, AT_ONCE = 64 / LANES;   // lanes of a head, heads of a wave
    using K = typename std::conditional<CACHE, double, float>::type;
    struct Angle { K c, s; };
    __shared__ Angle angles[(CACHE ? WAVES : 1) * D / 2];
    __shared__ K meet[CACHE ? WAVES : 1][CACHE ? AT_ONCE * D : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = blockIdx.x * tokens;
    for (int i = threadIdx.x; i < min(tokens, r.rows - row0) * r.pairs; i += WG) {
        const int tok = i / r.pairs, pair = i - tok * r.pairs;
        const int axis = r.axis ? min((int)r.axis[pair], r.axes - 1) : 0;
        double s, c;
        sincos((double)r.positions[axis * r.axis_stride + row0 + tok] * (double)r.frequencies[pair], &s, &c);
        angles[i] = Angle{(K)(c * (double)r.factor), (K)(s * (double)r.factor)};
    }
    __syncthreads();
    const int tok = tokens == 1 ? 0 : wave, row = row0 + tok;
    if (row >= r.rows) return;
    const int u0 = lane % LANES * VEC, sub = lane / LANES;
    const Runs at(u0, r.pairs, NEIGHBOURS);
    K ck[VEC], sk[VEC];
    float cq[VEC], sq[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const Angle a = u0 < r.pairs ? angles[tok * r.pairs + u0 + j] : Angle{0, 0};
        ck[j] = a.c;
        sk[j] = a.s;
        cq[j] = (float)a.c;
        sq[j] = (float)a.s;
    }
    int64_t slot = 0, page = 0;
    bool present = false;
    if (CACHE) {
        slot = r.slots[row];
        present = slot >= 0 && slot >> r.pool.page_shift < r.pool.pages;
        page = (slot >> r.pool.page_shift) * r.pool.heads;
    }
    const int place = (int)(slot & ((1 << r.pool.page_shift) - 1)), d0 = lane % LANES * 8;
    const int of_q = (r.heads + AT_ONCE - 1) / AT_ONCE, of_k = (r.kv_heads + AT_ONCE - 1) / AT_ONCE;
    for (int item = tokens == 1 ? wave : 0; item < of_q + (CACHE ? 2 : 1) * of_k; item += tokens == 1 ? WAVES : 1) {
        if (item < of_q) {
            const int head = item * AT_ONCE + sub, from = min(head, r.heads - 1);   // (a whole wave comes to the lane exchanges)
            float y[2 * VEC];
            turn<float, T, D, NEIGHBOURS>((const T*)r.q + row * r.q_stride + from * D, r.q_weight, r.eps, at, u0 < r.pairs, cq, sq, y);
            if (head < r.heads) {
                Four<T> lo, hi;
#pragma unroll
                for (int j = 0; j < VEC; ++j) { lo.v[j] = from_f32<T>(y[j]); hi.v[j] = from_f32<T>(y[VEC + j]); }
                T* out = (T*)r.q_out + row * r.q_out_stride + head * D;
                *(Four<T>*)(out + at.lo) = lo;
                *(Four<T>*)(out + at.hi) = hi;
            }
        } else if (item < of_q + of_k) {
            const int head = (item - of_q) * AT_ONCE + sub, from = min(head, r.kv_heads - 1);
            K y[2 * VEC];
            turn<K, T, D, NEIGHBOURS>((const T*)r.k + row * r.k_stride + from * D, r.k_weight, r.eps, at, u0 < r.pairs, ck, sk, y);
            if constexpr (CACHE) {
                K* mine = meet[wave] + sub * D;
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < VEC; ++j) { mine[at.lo + j] = y[j]; mine[at.hi + j] = y[VEC + j]; }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                K x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = mine[d0 + e];
                mx_store_eight<D>(r.pool, false, page + from, place, d0, x, present && head < r.kv_heads);
            } else if (head < r.kv_heads) {
                Four<T> lo, hi;
#pragma unroll
                for (int j = 0; j < VEC; ++j) { lo.v[j] = from_f32<T>((float)y[j]); hi.v[j] = from_f32<T>((float)y[VEC + j]); }
                T* out = (T*)r.k_out + row * r.k_out_stride + head * D;
                *(Four<T>*)(out + at.lo) = lo;
                *(Four<T>*)(out + at.hi) = hi;
            }
        } else if constexpr (CACHE) {
            const int head = (item - of_q - of_k) * AT_ONCE + sub, from = min(head, r.kv_heads - 1);
            const MxEight<T> raw = *(const MxEight<T>*)((const T*)r.v + row * r.v_stride + from * D + d0);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = to_f32(raw.v[e]);
            mx_store_eight<D>(r.pool, true, page + from, place, d0, x, present && head < r.kv_heads);
        }
    }
}

template <typename T, int D, bool CACHE>
static int launch_of(const Rotate& r, bool neighbours, hipStream_t s) {
    // A token's heads over four waves, but into the cache, whose angles in 64 bits take long, a token a wave once each CU has more than eight tokens: their
    // angles are made side by side. 32 + 8 heads of 128 with norms, bf16, kernel trace: 4096 tokens into the cache 30.6 us in fours of waves, 26.9 a token a wave, 2048
    // 18.8 and 19.6, 1024 11.0 and 17.0; without the cache (calls) 4096 16.7 and 17.5, 1024 7.6 and 11.5.
    const int tokens = CACHE && r.rows > 8 * lk_device().cus ? WAVES : 1;
    const dim3 grid((unsigned)((r.rows + tokens - 1) / tokens)), threads(WG);
    if (neighbours) hipLaunchKernelGGL((rotate_kernel<T, D, true, CACHE>), grid, threads, 0, s, r, tokens);
    else hipLaunchKernelGGL((rotate_kernel<T, D, false, CACHE>), grid, threads, 0, s, r, tokens);
    return lk_launch_status();
}
template <typename T, bool CACHE>
static int launch_dim(const Rotate& r, int head_dim, bool neighbours, hipStream_t s) {
    return head_dim == 64 ? launch_of<T, 64, CACHE>(r, neighbours, s) : head_dim == 128 ? launch_of<T, 128, CACHE>(r, neighbours, s) : launch_of<T, 256, CACHE>(r, neighbours, s);
}
template <bool CACHE>
static int launch(const Rotate& r, int type, int head_dim, bool neighbours, hipStream_t s) {
    if (type == LK_TYPE_F32) return launch_dim<float, CACHE>(r, head_dim, neighbours, s);
    if (type == LK_TYPE_F16) return launch_dim<__half, CACHE>(r, head_dim, neighbours, s);
    return launch_dim<__hip_bfloat16, CACHE>(r, head_dim, neighbours, s);
}

// What both entry points ask of their arguments.
static int check(const Rotate& r, int size, int head_dim) {
    if (r.rows < 0 || r.heads <= 0 || r.heads > 65535 || r.kv_heads <= 0 || r.kv_heads > 65535 || !kv_head_dim_ok(head_dim) || r.pairs < 0 || r.pairs % VEC ||
        2 * r.pairs > head_dim || r.axes <= 0 || r.axes > LK_ROTARY_AXES || r.axis_stride < r.rows || !(r.eps >= 0.0f && r.eps <= 3.402823466e38f) ||
        !(fabsf(r.factor) <= 3.402823466e38f))
        return LK_ERR_ARG;
    if (r.rows == 0) return LK_OK;
    const int64_t of_q = (int64_t)r.heads * head_dim, of_k = (int64_t)r.kv_heads * head_dim;
    if (!r.q || !r.k || !r.q_out || (r.pairs && (!r.positions || !r.frequencies)) || r.q_stride < of_q || r.q_out_stride < of_q || r.k_stride < of_k ||
        (((uintptr_t)r.q | (uintptr_t)r.k | (uintptr_t)r.q_out) & (size - 1)))
        return LK_ERR_ARG;
    return LK_OK;
}

}  // namespace

extern "C" int lk_qk_norm_rope(const void* q, const void* k, int type, int64_t q_stride, int64_t k_stride, void* q_out, void* k_out,
                               int64_t q_out_stride, int64_t k_out_stride, int rows, int heads, int kv_heads, int head_dim,
                               const float* q_weight, const float* k_weight, float eps, const int32_t* positions, int64_t axis_stride,
                               int axes, const float* frequencies, const uint8_t* axis, int pairs, int neighbours, float factor,
                               void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    const Rotate r{q, k, nullptr, q_out, k_out, q_stride, k_stride, 0, q_out_stride, k_out_stride, rows, heads, kv_heads, q_weight, k_weight, eps, positions,
                   axis_stride, axes, frequencies, axis, pairs, factor, nullptr, MxPool{}};
    const int status = check(r, size, head_dim);
    if (status != LK_OK || rows == 0) return status;
    if (!k_out || ((uintptr_t)k_out & (size - 1)) || k_out_stride < (int64_t)kv_heads * head_dim) return LK_ERR_ARG;
    return launch<false>(r, type, head_dim, neighbours != 0, (hipStream_t)stream);
}

extern "C" int lk_qk_norm_rope_kv_mxfp4(const void* q, const void* k, const void* v, int type, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                        void* q_out, int64_t q_out_stride, const int64_t* slots, int rows, int heads, int kv_heads,
                                        int head_dim, const float* q_weight, const float* k_weight, float eps, const int32_t* positions,
                                        int64_t axis_stride, int axes, const float* frequencies, const uint8_t* axis, int pairs,
                                        int neighbours, float factor, int page_tokens, int pages, void* k_codes, void* v_codes,
                                        void* k_powers, void* v_powers, void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    if (!mx_pool_ok(k_codes, v_codes, k_powers, v_powers, pages, kv_heads, head_dim, page_tokens)) return LK_ERR_ARG;
    const Rotate r{q, k, v, q_out, nullptr, q_stride, k_stride, v_stride, q_out_stride, 0, rows, heads, kv_heads, q_weight, k_weight, eps, positions,
                   axis_stride, axes, frequencies, axis, pairs, factor, slots,
                   {(uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_powers, (uint8_t*)v_powers, pages, kv_heads, kv_log2(page_tokens)}};
    const int status = check(r, size, head_dim);
    if (status != LK_OK || rows == 0) return status;
    if (!v || !slots || ((uintptr_t)v & (size - 1)) || ((uintptr_t)slots & 7) || v_stride < (int64_t)kv_heads * head_dim) return LK_ERR_ARG;
    return launch<true>(r, type, head_dim, neighbours != 0, (hipStream_t)stream);
}
