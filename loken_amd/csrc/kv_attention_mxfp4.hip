// Attention over the paged 4-bit cache (lk_kv_attention_mxfp4): how contexts are cut into parts, and the launches.

#include "kv_attention_mxfp4.h"
#include "stream_scratch.h"

namespace {

constexpr int MOST_PARTS = 1024;

// Whether what a product is multiplied by, mx_unit or mx_under, is a normal number: an infinite one makes none of a product of 0, a subnormal one has lost bits.
static bool factor_ok(float scale, float cap) {
    if (!(scale >= 0x1p-126f && scale <= 0x1p127f) || !(cap == 0.0f || (cap >= 0x1p-64f && cap <= 0x1p64f))) return false;
    const double of_cap = cap > 0.0f ? (double)scale / cap : 1.0;
    return of_cap >= 0x1p-124 && of_cap <= 0x1p125;
}

// Parts of a context of `tiles` steps for `groups` workgroups of one part each: until there are `want` workgroups, of at
// least `least` steps.
static void cut(Attend& a, int64_t groups, int tiles, int want, int least) {
    int64_t parts = (want + groups - 1) / groups;
    parts = parts < (tiles + least - 1) / least ? parts : (tiles + least - 1) / least;
    a.splits = parts < 1 ? 1 : parts < MOST_PARTS ? (int)parts : MOST_PARTS;
    a.least_tiles = tiles > a.splits ? (tiles + a.splits - 1) / a.splits : 1;
}

// Parts of the many-rows kernel's contexts, of `tiles` steps for `groups` row tiles and heads, `layer` workgroups being one wave for every SIMD and
// `on_simd` of them there at once: those that take the least time where a workgroup takes 5 us to start and `step` us a step, waves that fill a SIMD
// that much each and those that do not 0.7 of a step more, and each row and head's part 0.35 ns to be stored and joined, 4 us in all beside.
static void cut_many(Attend& a, int64_t groups, int tiles, int64_t layer, int on_simd, double step) {
    const double rows = (double)a.rows * a.heads;
    double least = 1e30;
    for (int parts = 1, of = 0; parts <= 64 && parts <= tiles / 2 + 1; ++parts) {
        const int per = (tiles + parts - 1) / parts;
        if (per == of) continue;
        of = per;
        const int64_t full = groups * parts / (layer * on_simd), rest = (groups * parts - full * layer * on_simd + layer - 1) / layer;
        const double most = on_simd > 1 ? on_simd : 1.5, last = rest ? rest + 0.7 : 0.0;
        const double waves = full * most + (last < most ? last : most);
        const double time = waves * per * step + 5.0 * (full + (rest > 0)) + (parts > 1 ? 4.0 + rows * parts * 0.35e-3 : 0.0);
        if (time < least) {
            least = time;
            a.splits = parts;
            a.least_tiles = per > 1 ? per : 1;
        }
    }
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
        !factor_ok(scale, cap) || heads <= 0 || heads > 65535 || heads % kv_heads != 0)
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
    // What the caller says of the sizes chooses launches; whatever the sequences are, one of the kernels takes each.
    const bool f32 = type == LK_TYPE_F32, f16 = type == LK_TYPE_F16;
    const int tokens = max_fresh < 1 ? 1 : max_fresh < rows ? max_fresh : rows;
    const int64_t most_rows = (int64_t)tokens * group;
    const int max_rows = most_rows < 0x7FFFFFFF ? (int)most_rows : 0x7FFFFFFF;
    const bool many = max_rows > MX_FEW_ROWS, few = group <= MX_FEW_ROWS && (!many || seqs > 1);
    const int64_t table_tokens = (int64_t)table_cols * page_tokens;
    const int64_t seen = window > 0 && window < max_len ? (int64_t)window + tokens : max_len;
    const int tiles = (int)((min(seen, table_tokens) + KV_TILE - 1) / KV_TILE), cus = lk_device().cus;
    AttendMx af = a, am = a;
    // Beside a sequence of many rows the few-rows kernel takes what one of its workgroups holds for a token's rows.
    const int few_max = many ? mx_few_rows(f32, group) : max_rows, per = mx_few_rows(f32, few_max);
    const int few_tokens = many ? few_max / group : tokens;
    if (few) {
        af.few_rows = many ? few_max : 0x7FFFFFFF;
        const int64_t groups = (int64_t)seqs * kv_heads * ((few_max - 1) / per + 1);
        const int slots = cus * mx_few_on_simd(f32, f16, head_dim, per);   // workgroups that run at once
        const int64_t most_steps = (int64_t)seqs * ((table_tokens + KV_TILE - 1) / KV_TILE + 1);
        // Pieces of equal lengths, across sequences, where those are long: a piece has to find its sequence and begins anew at each, some 10 us in all,
        // which ragged lengths win back from 96 steps a CU on, or 224 where sequences are many beside their steps. 8 sequences up to 32768 tokens, 8 heads of
        // 128, bf16: 45 us by sequence, 38 in pieces; 64 up to 8192 71, 65; 32 up to 8192 45, 51; 64 up to 2000 28, 40 (calls).
        const bool long_ones = tiles > seqs && groups * tiles >= (int64_t)(tiles >= 8 * (int64_t)seqs ? 96 : 224) * cus;
        if (seqs > 1 && few_max <= per && groups <= 4 * cus && long_ones && most_steps < 0x7FFFFFFF) {
            af.chunks = (slots + kv_heads - 1) / kv_heads;
            af.least_tiles = 4;
        } else {
            cut(af, groups, tiles, slots < 2 * cus ? slots : 2 * cus, tiles <= 16 ? 16 : 4);   // (three to a CU: 131072 tokens 2 us longer, more to join)
            af.part_seq = few_tokens;
        }
    }
    const int64_t part_rows_f = !few ? 0 : af.chunks ? (int64_t)kv_heads * af.chunks * 2 * per : af.splits > 1 ? (int64_t)seqs * af.part_seq * heads * af.splits : 0;
    int64_t part_rows_m = 0;
    const int many_rows = mx_many_rows(f32, head_dim);
    if (many) {
        am.few_rows = few ? few_max : 0;
        // as many sequences as fill the batch with the most rows that one has
        const int64_t filled = (rows + (int64_t)tokens / 2) / tokens, long_seqs = filled < seqs ? filled : seqs;
        cut_many(am, long_seqs * ((max_rows - 1) / many_rows + 1) * kv_heads, tiles, 2 * cus, mx_many_on_simd(f32, f16, head_dim),
                 (f32 ? 1.1 : f16 ? 0.8 : 0.6) * head_dim / 128);
        if (am.splits > 1) part_rows_m = (int64_t)rows * heads * am.splits;
    }
    LkScratch scratch(s);
    if (part_rows_f + part_rows_m) {
        float* mem = (float*)scratch.get(LK_SCRATCH_ATTENTION, (size_t)(part_rows_f + part_rows_m) * (head_dim + 2) * 4);
        if (!mem) return LK_ERR_NOMEM;
        af.part_ml = (float2*)mem;
        am.part_ml = af.part_ml + part_rows_f;
        af.part_o = mem + 2 * (part_rows_f + part_rows_m);
        am.part_o = af.part_o + part_rows_f * head_dim;
    }
    int status = LK_OK;
    if (many) status = kv_attention_mxfp4_many(am, type, head_dim, s);
    if (status == LK_OK && few) status = kv_attention_mxfp4_few(af, type, head_dim, few_max, s);
    if (status == LK_OK && part_rows_m) status = kv_attention_join(am, type, head_dim, many_rows, false, tokens, s);
    if (status == LK_OK && part_rows_f) status = kv_attention_join(af, type, head_dim, per, true, few_tokens, s);
    return status;
}
