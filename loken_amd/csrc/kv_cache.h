// The paged key / value cache in 8 bits: layout and what its kernels share.
//
// A page holds `P` consecutive positions of one sequence for every key / value head, P = 16, 32, .. 256. With
// B = P / 16 runs of sixteen tokens:
//   keys    int8 [pages][heads][P][D]          a token's row together: the matrix instruction's operand takes 16 bytes of it a lane
//   values  int8 [pages][heads][B][D][16]      sixteen tokens of a column together, which is what that operand takes of the values
//   scales  f32  [pages][heads], one array for either side; a value is code * scale, codes -127 .. 127
#pragma once
#include "lk_common.h"

constexpr int KV_RUN = 16;   // tokens of a run

struct KvPool {
    int8_t *k, *v;
    float *k_scales, *v_scales;
    int pages, heads, page_shift;   // page_shift: log2 of P
};

static inline bool kv_page_tokens_ok(int p) { return p >= 16 && p <= 256 && (p & (p - 1)) == 0; }
static inline bool kv_head_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }
static inline int kv_log2(int p) { return __builtin_ctz((unsigned)p); }
// The pools' own arguments: every entry point of the cache asks the same of them.
static inline bool kv_pool_ok(const void* k, const void* v, const void* ks, const void* vs, int pages, int heads, int head_dim, int page_tokens) {
    return k && v && ks && vs && pages > 0 && heads > 0 && heads <= 65535 && kv_head_dim_ok(head_dim) && kv_page_tokens_ok(page_tokens) &&
           (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (((uintptr_t)ks | (uintptr_t)vs) & 3) == 0;
}
static inline int kv_type_size(int type) { return type == LK_TYPE_F32 ? 4 : type == LK_TYPE_F16 || type == LK_TYPE_BF16 ? 2 : 0; }
