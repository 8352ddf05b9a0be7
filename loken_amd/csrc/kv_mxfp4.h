// The paged key / value cache in 4 bits (MXFP4): layout and what its kernels share.
//
// 32 neighbouring values of a token and head are a block: a power of two 2^(byte - 127) and 32 codes e2m1 (a sign and one of 0, 1/2, 1,
// 3/2, 2, 3, 4, 6), two to a byte, the first in its low half. A page holds `P` consecutive positions of one sequence, P = 16, 32, .. 256:
//   keys           [pages][heads][P][D / 2]            a token's row together: sixteen tokens' rows are the matrix instruction's operand
//   their powers   [pages][heads][P][D / 32]
//   values         [pages][heads][P / 4][16][4][D / 32]   of four tokens a sixteenth of the row each, together: what a lane takes of them
//   their powers   [pages][heads][D / 32][P]           of four tokens one word
// A token's bytes are its own, so rows are written in any order and by any workgroup.
#pragma once
#include "kv_cache.h"

struct MxPool {
    uint8_t *k, *v, *k_powers, *v_powers;
    int pages, heads, page_shift;   // page_shift: log2 of P
};

// The pool's own arguments: every entry point of the cache asks the same of them.
static inline bool mx_pool_ok(const void* k, const void* v, const void* kp, const void* vp, int pages, int heads, int head_dim, int page_tokens) {
    return k && v && kp && vp && pages > 0 && heads > 0 && heads <= 65535 && kv_head_dim_ok(head_dim) && kv_page_tokens_ok(page_tokens) &&
           (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (((uintptr_t)kp | (uintptr_t)vp) & 15) == 0;
}

// Powers that are written: 2^-96 .. 2^125. Every value is then a normal number of f32 and bf16, and so is its product with a softmax weight's last
// piece: what the matrix unit makes of smaller ones is not relied on.
constexpr int MX_LEAST = -96, MX_MOST = 125;

// E of a block whose largest finite value is `most` >= 0: the least with most < 7 * 2^E. (6 is the largest code; 7 lies as far from it as from the
// next power's 4 * 2.) As bits: a quarter more in the mantissa carries into the exponent from 1.75 on.
static __device__ __forceinline__ int mx_power(float most) {
    const int e = (int)((__float_as_uint(most) + 0x00200000u) >> 23) - 129;
    return min(max(e, MX_LEAST), MX_MOST);
}
static __device__ __forceinline__ int mx_power(double most) {
    const int e = (int)(((uint64_t)__double_as_longlong(most) + 0x0004000000000000ull) >> 52) - 1025;
    return min(max(e, MX_LEAST), MX_MOST);
}
static __device__ __forceinline__ float mx_inverse(int e, float) { return __uint_as_float((uint32_t)(127 - e) << 23); }
static __device__ __forceinline__ double mx_inverse(int e, double) { return __longlong_as_double((long long)(1023 - e) << 52); }

// The code of x / 2^E: the nearest, halves to the even code, 6 above it; the sign of what is below zero in bit 3; 0 for what is no number.
template <typename F>
static __device__ __forceinline__ uint32_t mx_code(F y) {
    const F m = y < 0 ? -y : y;
    const uint32_t code = (uint32_t)(m > (F)0.25) + (m >= (F)0.75) + (m > (F)1.25) + (m >= (F)1.75) + (m > (F)2.5) + (m >= (F)3.5) + (m > (F)5.0);
    return code | (y < 0 ? 8u : 0u);
}

// Where eight neighbouring values from d0 (a multiple of 8) of a token go.
template <int D>
struct MxPlace {
    static constexpr int PART = D / 32;   // bytes of a token in a piece of four tokens
    // `page`: page * heads + head; `at`: the token's place in its page
    static __device__ __forceinline__ void store(const MxPool& p, bool value, int64_t page, int at, int d0, uint32_t codes) {
        if (!value) {
            *(uint32_t*)(p.k + ((page << p.page_shift) + at) * (D / 2) + d0 / 2) = codes;
            return;
        }
        uint8_t* of_page = p.v + (page << p.page_shift) * (D / 2);
        if (D == 64) {   // a sixteenth of the row is four values
            uint8_t* to = of_page + (((at >> 2) * 16 + d0 / 4) * 4 + (at & 3)) * PART;
            *(uint16_t*)to = (uint16_t)codes;
            *(uint16_t*)(to + 4 * PART) = (uint16_t)(codes >> 16);
        } else {
            *(uint32_t*)(of_page + (((at >> 2) * 16 + d0 / (D / 16)) * 4 + (at & 3)) * PART + d0 % (D / 16) / 2) = codes;
        }
    }
    static __device__ __forceinline__ uint32_t load(const MxPool& p, bool value, int64_t page, int at, int d0) {
        if (!value) return *(const uint32_t*)(p.k + ((page << p.page_shift) + at) * (D / 2) + d0 / 2);
        const uint8_t* of_page = p.v + (page << p.page_shift) * (D / 2);
        if (D == 64) {
            const uint8_t* from = of_page + (((at >> 2) * 16 + d0 / 4) * 4 + (at & 3)) * PART;
            return *(const uint16_t*)from | (uint32_t)*(const uint16_t*)(from + 4 * PART) << 16;
        }
        return *(const uint32_t*)(of_page + (((at >> 2) * 16 + d0 / (D / 16)) * 4 + (at & 3)) * PART + d0 % (D / 16) / 2);
    }
    static __device__ __forceinline__ uint8_t* power(const MxPool& p, bool value, int64_t page, int at, int d0) {
        const int64_t of_page = (page << p.page_shift) * PART;
        return value ? p.v_powers + of_page + ((int64_t)(d0 / 32) << p.page_shift) + at : p.k_powers + of_page + at * PART + d0 / 32;
    }
};

// Eight neighbouring values of a token and head as codes, into their place; the four lanes of an aligned group hold a block's 32 and come together.
template <int D, typename F>
static __device__ __forceinline__ void mx_store_eight(const MxPool& p, bool value, int64_t page, int at, int d0, const F (&x)[8], bool store) {
    F most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const F m = x[e] < 0 ? -x[e] : x[e];
        most = m <= (F)3.4028234663852886e38 && m > most ? m : most;   // (past f32's end, infinite or no number: does not count)
    }
    F other = __shfl_xor(most, 1);
    most = other > most ? other : most;
    other = __shfl_xor(most, 2);
    most = other > most ? other : most;
    if (!store) return;
    const int e2 = mx_power(most);
    const F by = mx_inverse(e2, (F)0);
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) codes |= mx_code(x[e] * by) << (4 * e);
    MxPlace<D>::store(p, value, page, at, d0, codes);
    if ((d0 & 31) == 0) *MxPlace<D>::power(p, value, page, at, d0) = (uint8_t)(e2 + 127);
}

// Eight neighbouring values of a row that starts on any value of its type.
template <typename T>
struct __attribute__((aligned(sizeof(T)))) MxEight { T v[8]; };
