// Attention over the paged 8-bit cache (lk_kv_attention_q8): which kernel takes a sequence, how contexts are cut into parts,
// and the launch that joins the parts.

#include "kv_attention.h"
#include "stream_scratch.h"

namespace {

constexpr int MOST_PARTS = 1024, JOIN_WAVES = 4;

// Where the parts of a row and head are.
struct PartsOf {
    int parts;
    int64_t base, step, first;
    __device__ __forceinline__ void set(const Attend& a, const KvSeq& s, int seq, int tok, int head, int per) {
        const unsigned group = a.group, all_rows = (unsigned)s.tokens() * group, r = (unsigned)tok * group + (head - a.token_of(head) * group);   // below 2^31
        if (a.chunks) {
            parts = 1;
            base = step = first = 0;
            if ((int)all_rows > per) return;
            const KvPieces pieces(a, per);
            const int at = KvPieces::first_of(a, per, seq), steps = kv_steps_of(a, seq, per);
            const int c0 = min(at / pieces.length, a.chunks - 1), c1 = min((at + steps - 1) / pieces.length, a.chunks - 1);
            parts = c1 - c0 + 1;
            // the piece that the sequence starts in has it second, the others first
            base = ((int64_t)a.token_of(head) * a.chunks + c0) * 2 * per + r;
            step = 2 * per;
            first = per;
            return;
        }
        const unsigned r0 = r / per * per, r1 = min(r0 + per, all_rows) - 1;
        parts = KvSpan(a, s, s.first + a.token_of(r0), s.first + a.token_of(r1)).parts;
        base = (a.part_row(seq, s, s.first + tok) * a.heads + head) * a.splits;
        step = 1;
        first = 0;
    }
    __device__ __forceinline__ int64_t at(int p) const { return base + p * step + (p == 0 ? first : 0); }
};

// The parts of a row's context: sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p. A workgroup to a row and head (rows of a workgroup of
// the launch before, `per` of them, have the same parts), its waves taking parts in turn, eight parts' loads in flight: with one after
// the other 128 parts of one row took 88 us.
template <typename T, int D>
__global__ __launch_bounds__(64 * JOIN_WAVES) void kv_join_kernel(Attend a, int per, bool few, int tokens) {
    constexpr int PER = D / 64, AHEAD = 8;
    __shared__ float share[MOST_PARTS], sums[JOIN_WAVES][D], meet[JOIN_WAVES][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.heads, seq = blockIdx.x / a.heads / tokens;
    const KvSeq s(a, seq);
    const int64_t all_rows = (int64_t)s.tokens() * a.group;
    if ((all_rows <= a.few_rows) != few) return;
    for (int tok = blockIdx.x / a.heads % tokens; tok < s.tokens(); tok += tokens) {
        PartsOf of;
        of.set(a, s, seq, tok, head, per);
        const int parts = of.parts;   // at most MOST_PARTS
        if (parts == 1) continue;
        float m = -INFINITY;
        for (int p = threadIdx.x; p < parts; p += 64 * JOIN_WAVES) m = fmaxf(m, a.part_ml[of.at(p)].x);
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (lane == 0) meet[wave][0] = m;
        __syncthreads();
        m = fmaxf(fmaxf(meet[0][0], meet[1][0]), fmaxf(meet[2][0], meet[3][0]));
        float l = 0.f;
        for (int p = threadIdx.x; p < parts; p += 64 * JOIN_WAVES) {
            const float2 ml = a.part_ml[of.at(p)];
            // (a part whose scores are no numbers has no maximum and a sum that is none)
            const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);
            l += ml.x == -INFINITY ? ml.y : ml.y * f;
            share[p] = f;
        }
        l = wave_sum(l);
        if (lane == 0) meet[wave][1] = l;
        __syncthreads();
        l = (meet[0][1] + meet[1][1]) + (meet[2][1] + meet[3][1]);
        float acc[PER] = {};
        for (int p0 = wave; p0 < parts; p0 += AHEAD * JOIN_WAVES) {
            float x[AHEAD][PER];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int i = 0; i < PER; ++i) x[j][i] = a.part_o[of.at(min(p0 + j * JOIN_WAVES, parts - 1)) * D + lane + 64 * i];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (p0 + j * JOIN_WAVES < parts) {
                    const float f = share[p0 + j * JOIN_WAVES];
#pragma unroll
                    for (int i = 0; i < PER; ++i) acc[i] = fmaf(x[j][i], f, acc[i]);
                }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) sums[wave][lane + 64 * i] = acc[i];
        __syncthreads();
        T* out = (T*)a.out + (int64_t)(s.first + tok) * a.out_stride + (int64_t)head * D;
        for (int d = threadIdx.x; d < D; d += 64 * JOIN_WAVES) {
            const float total = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
            out[d] = from_f32<T>(l == 0.f ? 0.f : total / l);
        }
        __syncthreads();
    }
}

// The same for a few parts: a wave to a row and AT heads, whose loads are in flight together. `few`: items are (sequence, one of
// `tokens`, head); else (row of the batch, heads AT at a time).
template <typename T, int D, int AT>
__global__ __launch_bounds__(64 * JOIN_WAVES) void kv_join_few_parts_kernel(Attend a, int per, bool few, int tokens, int64_t items) {
    constexpr int PER = D / 64, AHEAD = AT == 1 ? 8 : 4;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * JOIN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= items) return;
    const int of_row = (a.heads + AT - 1) / AT, head0 = AT * (int)(item % of_row);
    int seq = (int)(item / of_row / tokens), tok = (int)(item / of_row % tokens);
    if (!few) {   // the last sequence that starts at or before the row
        const int row = (int)(item / of_row);
        seq = 0;
        for (int n = a.seqs; n > 1;) {
            const int step = (n + 63) / 64;
            const bool is = lane * step < n && a.starts[seq + lane * step] <= row;
            const int back = max(__popcll(__ballot(is)) - 1, 0) * step;
            seq += back;
            n = min(step, n - back);
        }
        tok = row - max(a.starts[seq], 0);
    }
    const KvSeq s(a, seq);
    if (((int64_t)s.tokens() * a.group <= a.few_rows) != few || tok < 0) return;
    for (; tok < s.tokens(); tok += few ? tokens : 0x40000000) {
        int parts[AT], most = 0;
        PartsOf of[AT];
#pragma unroll
        for (int h = 0; h < AT; ++h) {
            of[h].set(a, s, seq, tok, min(head0 + h, a.heads - 1), per);
            parts[h] = head0 + h < a.heads ? __builtin_amdgcn_readfirstlane(of[h].parts) : 0;
            most = max(most, parts[h]);
        }
        if (most < 2) continue;
        float m[AT], l[AT], acc[AT][PER] = {};
#pragma unroll
        for (int h = 0; h < AT; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
        }
        // sums relative to the largest maximum so far
        for (int p0 = 0; p0 < most; p0 += AHEAD) {
            float x[AT][AHEAD][PER];
            float2 ml[AT][AHEAD];
#pragma unroll
            for (int h = 0; h < AT; ++h)
#pragma unroll
                for (int j = 0; j < AHEAD; ++j)
                    if (p0 + j < parts[h]) {
                        const int64_t from = of[h].at(p0 + j);
                        ml[h][j] = a.part_ml[from];
#pragma unroll
                        for (int i = 0; i < PER; ++i) x[h][j][i] = a.part_o[from * D + lane + 64 * i];
                    }
#pragma unroll
            for (int h = 0; h < AT; ++h) {
                float now = m[h];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) now = p0 + j < parts[h] ? fmaxf(now, ml[h][j].x) : now;
                const float back = m[h] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[h] - now);   // (what has no maximum is zeros, or no number)
                l[h] *= back;
#pragma unroll
                for (int i = 0; i < PER; ++i) acc[h][i] *= back;
                m[h] = now;
#pragma unroll
                for (int j = 0; j < AHEAD; ++j)
                    if (p0 + j < parts[h]) {
                        const float f = ml[h][j].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[h][j].x - now);
                        l[h] += ml[h][j].x == -INFINITY ? ml[h][j].y : ml[h][j].y * f;
#pragma unroll
                        for (int i = 0; i < PER; ++i) acc[h][i] = fmaf(x[h][j][i], f, acc[h][i]);
                    }
            }
        }
        T* out = (T*)a.out + (int64_t)(s.first + tok) * a.out_stride + (int64_t)head0 * D + lane;
#pragma unroll
        for (int h = 0; h < AT; ++h)
            if (parts[h] > 1)
#pragma unroll
                for (int i = 0; i < PER; ++i) out[h * D + 64 * i] = from_f32<T>(l[h] == 0.f ? 0.f : acc[h][i] / l[h]);
    }
}

template <typename T, int D>
static int join_of(const Attend& a, int per, bool few, int tokens, hipStream_t s) {
    // Heads of a row together where there are more rows and heads than waves run at once: 700 rows of 32 heads in three parts 15 us, 18
    // one by one; 64 rows behind 4096 tokens
    // (32 us in all) four longer that way
    constexpr int AT = 4;
    const bool together = !few && (int64_t)a.rows * a.heads > 32 * lk_device().cus;
    const int64_t items = few ? (int64_t)a.seqs * tokens * a.heads : (int64_t)a.rows * (together ? (a.heads + AT - 1) / AT : a.heads);
    const bool wide = few && (a.chunks ? a.chunks > 8 * a.seqs : a.splits > 8);   // four waves to a row from nine parts on
    const int64_t blocks = wide ? items : (items + JOIN_WAVES - 1) / JOIN_WAVES;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    const dim3 grid((unsigned)blocks), threads(64 * JOIN_WAVES);
    if (wide) hipLaunchKernelGGL((kv_join_kernel<T, D>), grid, threads, 0, s, a, per, few, tokens);
    else if (!together) hipLaunchKernelGGL((kv_join_few_parts_kernel<T, D, 1>), grid, threads, 0, s, a, per, few, tokens, items);
    else hipLaunchKernelGGL((kv_join_few_parts_kernel<T, D, AT>), grid, threads, 0, s, a, per, few, tokens, items);
    return lk_launch_status();
}

template <typename T>
static int join(const Attend& a, int head_dim, int per, bool few, int tokens, hipStream_t s) {
    return head_dim == 64 ? join_of<T, 64>(a, per, few, tokens, s) : head_dim == 128 ? join_of<T, 128>(a, per, few, tokens, s) : join_of<T, 256>(a, per, few, tokens, s);
}

}  // namespace

int kv_attention_join(const Attend& a, int type, int head_dim, int per, bool few, int tokens, hipStream_t s) {
    if (type == LK_TYPE_F32) return join<float>(a, head_dim, per, few, tokens, s);
    if (type == LK_TYPE_F16) return join<__half>(a, head_dim, per, few, tokens, s);
    return join<__hip_bfloat16>(a, head_dim, per, few, tokens, s);
}

namespace {

// Sequences of up to this many rows (token, head of a group) are the few-rows kernel's.
constexpr int FEW_ROWS = 16;

// Parts of a context of `tiles` steps for `groups` workgroups of one part each: until there are `want` workgroups, of at
// least `least` steps.
static void cut(Attend& a, int64_t groups, int tiles, int want, int least) {
    int64_t parts = (want + groups - 1) / groups;
    parts = parts < (tiles + least - 1) / least ? parts : (tiles + least - 1) / least;
    a.splits = parts < 1 ? 1 : parts < MOST_PARTS ? (int)parts : MOST_PARTS;
    a.least_tiles = tiles > a.splits ? (tiles + a.splits - 1) / a.splits : 1;
}

// Parts of the many-rows kernel's contexts, of `tiles` steps for `groups` row tiles and heads: those that take the least time where
// a workgroup takes 6 us to start and `step` us a step, as many at once as the CUs hold, and each row and head's part 0.35 ns to be stored
// and joined, 4 us in all beside. In bf16 (us measured, and by this rule's sum): 64 rows behind 4096 tokens 5 / 9 / 17 parts 32 / 29 / 38
// (30 / 26 / 38); 200 behind 4096 5 / 9 parts 59 / 52 (62 / 55), both more than one round; four sequences of 500 behind 1000 whole / in two
// 79 / 144 (73 / 134).
static void cut_many(Attend& a, int64_t groups, int tiles, bool f32, int head_dim, int cus) {
    const int64_t slots = (int64_t)cus * (f32 && head_dim < 256 ? 2 : 1);
    const double rows = (double)a.rows * a.heads;
    double least = 1e30;
    for (int parts = 1, of = 0; parts <= 64 && parts <= tiles / 2 + 1; ++parts) {
        const int per = (tiles + parts - 1) / parts;
        if (per == of) continue;
        of = per;
        const int64_t rounds = (groups * parts + slots - 1) / slots;
        // f32 of up to 128 columns: two workgroups to a CU, each slower for it
        const double step = head_dim == 256 ? (f32 ? 8.0 : 4.8) : (!f32 ? 1.28 : groups * parts <= cus ? 2.8 : 3.6) * head_dim / 128;
        const double time = (double)rounds * (per * step + 6.0) + (parts > 1 ? 4.0 + rows * parts * 0.35e-3 : 0.0);
        if (time < least) {
            least = time;
            a.splits = parts;
            a.least_tiles = per > 1 ? per : 1;
        }
    }
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
    if ((int64_t)table_cols * page_tokens > 0x7FFFFC00 || (int64_t)rows * (heads / kv_heads) > 0x7FFFFFFF) return LK_ERR_SIZE;   // positions and what is added to them fit 32 bits
    hipStream_t s = (hipStream_t)stream;
    const int group = heads / kv_heads;
    int group_shift = 31;
    while ((1 << (group_shift - 31)) < group) ++group_shift;
    const Attend a{q, out, q_stride, out_stride, {(int8_t*)k_codes, (int8_t*)v_codes, (float*)k_scales, (float*)v_scales, pages, kv_heads, kv_log2(page_tokens)},
                   table, lens, starts, table_stride, table_cols, seqs, rows, heads, group, window, scale, (((uintptr_t)q | (uintptr_t)(q_stride * size)) & 15) == 0, 1, 1, 0, nullptr, nullptr, 0, 0,
                   (uint32_t)(((1ull << group_shift) + group - 1) / group), group_shift};
    // What the caller says of the sizes chooses launches; whatever the sequences are, one of the kernels takes each.
    const int tokens = max_fresh < 1 ? 1 : max_fresh < rows ? max_fresh : rows;
    const int64_t most_rows = (int64_t)tokens * group;
    const int max_rows = most_rows < 0x7FFFFFFF ? (int)most_rows : 0x7FFFFFFF;
    const bool many = max_rows > FEW_ROWS, few = group <= FEW_ROWS && (!many || seqs > 1);
    const int64_t table_tokens = (int64_t)table_cols * page_tokens;
    const int64_t seen = window > 0 && window < max_len ? (int64_t)window + tokens : max_len;
    const int tiles = (int)((min(seen, table_tokens) + KV_TILE - 1) / KV_TILE);
    Attend af = a, am = a;
    const bool f32 = type == LK_TYPE_F32;
    // Beside a sequence of many rows the few-rows kernel takes what one of its workgroups holds, if that is a token's.
    const int one_wg = kv_few_rows(f32, head_dim, FEW_ROWS), few_limit = group <= one_wg ? one_wg : FEW_ROWS;
    const int few_max = many ? few_limit : max_rows, few_per = kv_few_rows(f32, head_dim, few_max);
    const int cus = lk_device().cus;
    // Workgroups of the few-rows kernel that run at once: one to a CU where its registers leave a SIMD one wave. 64 sequences of 4000
    // tokens, 32 heads over 4 of 128 f32 values, in pieces or parts for one / two to a CU: 55 / 71 us; eight of them 18 / 26.
    const int few_slots = head_dim == 256 || (head_dim == 128 && few_per > kv_few_rows(f32, head_dim, 1)) ? cus : 2 * cus;
    if (few) {
        af.few_rows = many ? few_limit : 0x7FFFFFFF;
        const int64_t groups = (int64_t)seqs * kv_heads * ((few_max + few_per - 1) / few_per);
        // Long contexts of several sequences whose rows fit a workgroup each: pieces of equal length, as many as run at
        // once. 64 sequences of 1 to 8010 tokens, 32 heads over 8 of 128 f32 values: 116 us against 139 with parts per sequence; all of
        // 4096 104 against 107. With more than four heads and sequences to a CU parts per sequence balance by themselves (256 of 1024
        // tokens: 108 us, 121 in pieces, whose every sequence costs a start of 3 us).
        const int64_t most_steps = (int64_t)seqs * ((table_tokens + KV_TILE - 1) / KV_TILE + 1);
        if (seqs > 1 && few_max <= few_per && groups <= 4 * cus && groups * tiles > 16 * cus && most_steps < 0x7FFFFFFF) {
            af.chunks = (few_slots + kv_heads - 1) / kv_heads;
            af.least_tiles = 4;
        } else {
            // A context of up to 1024 positions stays in one launch; a longer one in parts of at least a step for each wave. One sequence
            // of 1024 / 2048 / 8192 tokens: 12.1 / 13.6 / 13.9 us a call, with parts of 16 steps 12.0 / 16.7 / 17.9, of 4 steps from
            // the start 13.8 / 13.6 / 13.9.
            cut(af, groups, tiles, few_slots, tiles <= 16 ? 16 : 4);
            af.part_seq = many ? few_limit / group : tokens;
        }
    }
    const int64_t part_rows_f = !few ? 0 : af.chunks ? (int64_t)kv_heads * af.chunks * 2 * few_per : af.splits > 1 ? (int64_t)seqs * af.part_seq * heads * af.splits : 0;
    int64_t part_rows_m = 0;
    if (many) {
        am.few_rows = few ? few_limit : 0;
        // as many sequences as fill the batch with the most rows that one has
        const int64_t long_seqs = min((int64_t)seqs, (rows + (int64_t)tokens / 2) / tokens);
        cut_many(am, long_seqs * ((max_rows - 1) / KV_MANY_ROWS + 1) * kv_heads, tiles, f32, head_dim, cus);
        if (am.splits > 1) part_rows_m = (int64_t)rows * heads * am.splits;
    }
    LkScratch scratch(s);
    if (part_rows_f + part_rows_m) {
        const size_t floats = (size_t)(part_rows_f + part_rows_m) * (head_dim + 2);
        float* mem = (float*)scratch.get(LK_SCRATCH_ATTENTION, floats * 4);
        if (!mem) return LK_ERR_NOMEM;
        af.part_ml = (float2*)mem;
        am.part_ml = af.part_ml + part_rows_f;
        af.part_o = mem + 2 * (part_rows_f + part_rows_m);
        am.part_o = af.part_o + part_rows_f * head_dim;
    }
    int status = LK_OK;
    if (many) status = kv_attention_many(am, type, head_dim, max_rows, s);
    if (status == LK_OK && few) status = kv_attention_few(af, type, head_dim, few_max, s);
    if (status == LK_OK && part_rows_m) status = kv_attention_join(am, type, head_dim, KV_MANY_ROWS, false, tokens, s);
    if (status == LK_OK && part_rows_f) status = kv_attention_join(af, type, head_dim, few_per, true, many ? few_limit / group : tokens, s);
    return status;
}
