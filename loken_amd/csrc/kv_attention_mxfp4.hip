// Attention over the paged 4-bit cache (lk_kv_attention_mxfp4): how contexts are cut into parts, and the launches.

#include "kv_attention_mxfp4.h"
#include "stream_scratch.h"

namespace {

constexpr int MOST_PARTS = 1024;

// Parts of a context of `tiles` steps for `groups` workgroups of one part each: until there are `want` workgroups, of at
// least `least` steps.
static void cut(Attend& a, int64_t groups, int tiles, int want, int least) {
    int64_t parts = (want + groups - 1) / groups;
    parts = parts < (tiles + least - 1) / least ? parts : (tiles + least - 1) / least;
    a.splits = parts < 1 ? 1 : parts < MOST_PARTS ? (int)parts : MOST_PARTS;
    a.least_tiles = tiles > a.splits ? (tiles + a.splits - 1) / a.splits : 1;
}

}  // namespace

extern "C" int lk_kv_attention_mxfp4(const void* q, int type, int64_t q_stride, void* out, int64_t out_stride, const void* k_codes,
                                     const void* v_codes, const void* k_powers, const void* v_powers, int pages, int page_tokens,
                                     const int32_t* table, int64_t table_stride, int table_cols, const int32_t* lens,
                                     const int32_t* starts, int seqs, int rows, int max_fresh, int max_len, int heads, int kv_heads,
                                     int head_dim, float scale, int window, float cap, void* stream) {
    const int size = kv_type_size(type);
    if (!size) return LK_ERR_TYPE;
    if (!mx_pool_ok(k_codes, v_codes, k_powers, v_powers, pages, kv_heads, head_dim, page_tokens)) return LK_ERR_ARG;
    if (seqs < 0 || rows < 0 || max_fresh < 0 || max_len < 0 || table_cols < 0 || table_stride < table_cols || window < 0 ||
        !(scale > 0.0f && scale <= 3.402823466e38f) || !(cap >= 0.0f && cap <= 3.402823466e38f) || heads <= 0 || heads > 65535 || heads % kv_heads != 0)
        return LK_ERR_ARG;
    if (seqs == 0 || rows == 0) return LK_OK;
    const int64_t row = (int64_t)heads * head_dim;
    if (!q || !out || !lens || !starts || (table_cols > 0 && !table) || (((uintptr_t)q | (uintptr_t)out) & (size - 1)) || q_stride < row ||
        out_stride < row)
        return LK_ERR_ARG;
    if ((int64_t)table_cols * page_tokens > 0x7FFFFC00 || (int64_t)rows * (heads / kv_heads) > 0x7FFFFFFF) return LK_ERR_SIZE;   // positions and what is added to them fit 32 bits
    hipStream_t s = (hipStream_t)stream;
    const int group = heads / kv_heads;
    int group_shift = 31;
    while ((1 << (group_shift - 31)) < group) ++group_shift;
    const KvPool sizes{nullptr, nullptr, nullptr, nullptr, pages, kv_heads, kv_log2(page_tokens)};
    AttendMx a{{q, out, q_stride, out_stride, sizes, table, lens, starts, table_stride, table_cols, seqs, rows, heads, group, window, scale, false, 1, 1, 0,
                nullptr, nullptr, 0, 0x7FFFFFFF, (uint32_t)(((1ull << group_shift) + group - 1) / group), group_shift},
               {(uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_powers, (uint8_t*)v_powers, pages, kv_heads, kv_log2(page_tokens)},
               cap};
    // What the caller says of the sizes chooses launches; whatever the sequences are, the kernel takes each.
    const int tokens = max_fresh < 1 ? 1 : max_fresh < rows ? max_fresh : rows;
    const int64_t most_rows = (int64_t)tokens * group;
    const int max_rows = most_rows < 0x7FFFFFFF ? (int)most_rows : 0x7FFFFFFF;
    const int64_t table_tokens = (int64_t)table_cols * page_tokens;
    const int64_t seen = window > 0 && window < max_len ? (int64_t)window + tokens : max_len;
    const int tiles = (int)((min(seen, table_tokens) + KV_TILE - 1) / KV_TILE);
    const int per = mx_few_rows(type == LK_TYPE_F32, head_dim, max_rows), cus = lk_device().cus;
    const int64_t groups = (int64_t)seqs * kv_heads * ((max_rows - 1) / per + 1);
    const int slots = cus * mx_few_on_simd(type == LK_TYPE_F32, head_dim, per);   // workgroups that run at once
    const int64_t most_steps = (int64_t)seqs * ((table_tokens + KV_TILE - 1) / KV_TILE + 1);
    if (seqs > 1 && max_rows <= per && groups <= 4 * cus && groups * tiles > 16 * cus && most_steps < 0x7FFFFFFF) {
        a.chunks = (slots + kv_heads - 1) / kv_heads;
        a.least_tiles = 4;
    } else {
        cut(a, groups, tiles, slots, tiles <= 16 ? 16 : 4);
        a.part_seq = tokens;
    }
    const int64_t part_rows = a.chunks ? (int64_t)kv_heads * a.chunks * 2 * per : a.splits > 1 ? (int64_t)seqs * a.part_seq * heads * a.splits : 0;
    LkScratch scratch(s);
    if (part_rows) {
        float* mem = (float*)scratch.get(LK_SCRATCH_ATTENTION, (size_t)part_rows * (head_dim + 2) * 4);
        if (!mem) return LK_ERR_NOMEM;
        a.part_ml = (float2*)mem;
        a.part_o = mem + 2 * part_rows;
    }
    int status = kv_attention_mxfp4_few(a, type, head_dim, max_rows, s);
    if (status == LK_OK && part_rows) status = kv_attention_join(a, type, head_dim, per, true, tokens, s);
    return status;
}
