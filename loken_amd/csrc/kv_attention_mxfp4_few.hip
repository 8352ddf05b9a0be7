// Attention over the 4-bit cache for a few rows of a sequence: single tokens, and the handful a draft brings.
//
// Both products run on v_mfma_f32_16x16x32_bf16: a code times its block's power of two is a bf16 exactly, two codes an instruction, and so are
// queries and softmax weights as sums of bf16 pieces (bf16 queries one, f16 two, f32 three; weights two, f32 three). Products are then exact but for
// weights of 16 bits, sums are f32. Up to four rows (f32; eight else) leave room for the pieces in the operand of sixteen columns: a slot of a row takes
// one piece, and a product is one instruction; a row's slots, two or four neighbouring lanes, add up what they have. More rows take a column each and an instruction a piece.
//
// One wave takes a step: 64 positions as four tiles of sixteen. Scores come as (16 positions) x (16 columns): a lane holds column l % 16 and four positions
// of each tile, which are, two tiles together, what the second product wants of the weights in that lane: nothing crosses lanes but maxima and the slots' sums.
// The values' operand is (16 columns) x (32 positions): the cache has the values of four tokens that a lane takes in one piece; codes of one token
// become bf16 by its block's power, and halves of words change places to bring a column's positions together.
// Sums come as (16 columns) x (16 rows): a lane's row again, so maxima and corrections are the lane's own.
//
// The next step's loads are in flight through a step, the pages of the one behind it too. Four waves take steps in turn and meet in LDS; long contexts
// are cut into parts, which a second launch joins.
//
// Bound by the cache's bytes where they are many: 64 sequences of up to 8192 tokens, 8 heads of 128, 287 MB in 73 to 75 us, 3.9 TB/s of the 4.9 that a copy
// reaches; 131072 tokens of one sequence 30.9 us, 4.6 TB/s. Else by the chain table, codes, scores, sums: 517 tokens 11.4 us. (Kernel trace.)

#include "kv_attention_mxfp4.h"

namespace {

constexpr int WAVES = 4;

static __device__ __forceinline__ float sum_over_groups(float v) { return swap_add32(swap_add16(v)); }

template <typename T, int D, int SLOTS>
struct Few {
    static constexpr int PIECES = sizeof(T) == 4 ? 3 : std::is_same<T, __half>::value ? 2 : 1;   // of a query value
    static constexpr int SHARES = sizeof(T) == 4 ? 3 : 2;                                         // of a weight
    static constexpr int QP = SLOTS == 1 ? PIECES : 1, SP = SLOTS == 1 ? SHARES : 1;              // operands of them
    static constexpr int ROWS = 16 / SLOTS, KS = D / 32, NB = D / 16, W = D / 32, PART = D / 32;
    static constexpr int ON_SIMD = mx_few_on_simd(sizeof(T) == 4, std::is_same<T, __half>::value, D, ROWS);
    // One buffer of codes, where that puts one more wave on a SIMD.
    static constexpr bool ONE = ON_SIMD > (D == 128 && SLOTS > 1 ? 2 : 1) && D > 64;
};

// What the slots of a row have together.
template <int SLOTS>
static __device__ __forceinline__ float sum_of_slots(float v) {
    if (SLOTS >= 2) v += dpp_f32<0xB1>(v);   // lanes 1, 0, 3, 2
    if (SLOTS >= 4) v += dpp_f32<0x4E>(v);   // lanes 2, 3, 0, 1
    return v;
}

// CAP: whether and how scores are capped (as a branch at run time the compiler takes the tanh always, and the result where it is asked for)
template <typename T, int D, int SLOTS, int CAP>
__global__ __launch_bounds__(64 * WAVES, (Few<T, D, SLOTS>::ON_SIMD)) void mx_few_kernel(AttendMx a, int row_tiles) {
    using F = Few<T, D, SLOTS>;
    __shared__ float sums[WAVES][F::ROWS][D + 4];
    __shared__ float tops[WAVES][F::ROWS], weights[WAVES][F::ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int slot = i % SLOTS;
    const float second = slot >= 1 ? 1.f : 0.f, third = slot >= 2 ? 1.f : 0.f;   // whether the slot's piece is behind the first, the second
    const int shift = a.mx.page_shift;
    // The workgroup's place: (part, row tile, head, sequence), the part fastest; or (head, piece), a piece being of one or
    // several sequences.
    int kv, seq, seq_end, tile0 = 0, part = 0;
    int first_step = 0, at_step = 0, end_step = 0, length = 1;   // the first step of `seq`, the piece's steps, and how many a piece has
    if (a.chunks) {
        kv = blockIdx.x % a.mx.heads;
        part = blockIdx.x / a.mx.heads;
        const KvPieces pieces(a, F::ROWS);
        length = pieces.length;
        if ((int64_t)part * length >= pieces.total) return;
        at_step = part * length;
        end_step = (int)min((int64_t)at_step + length, (int64_t)pieces.total);
        seq = __builtin_amdgcn_readfirstlane(KvPieces::sequence_at(a, F::ROWS, at_step, first_step));
        first_step = __builtin_amdgcn_readfirstlane(first_step);
        seq_end = a.seqs;
        row_tiles = 1;
    } else {
        unsigned at = blockIdx.x;
        part = at % a.splits;
        at /= a.splits;
        tile0 = at % row_tiles;
        at /= row_tiles;
        kv = at % a.mx.heads;
        seq = at / a.mx.heads;
        seq_end = seq + 1;
    }
    for (int steps = 0; seq < seq_end && (a.chunks == 0 || first_step < end_step); ++seq, first_step += steps) {
      const KvSeq s(a, seq);
      const int64_t rows_of_all = (int64_t)s.tokens() * a.group;
      steps = 0;
      if (rows_of_all == 0 || rows_of_all > a.few_rows) continue;
      const int all_rows = (int)rows_of_all;
      for (int tile = tile0; tile * F::ROWS < all_rows; tile += row_tiles) {
        const int r0 = tile * F::ROWS, r1 = min(r0 + F::ROWS, all_rows) - 1;
        const KvSpan span(a, s, s.first + a.token_of(r0), s.first + a.token_of(r1));
        int t_begin = 0, t_end = span.tiles;
        int64_t to = -1;   // the first row of the sums' place among the parts; -1: they are not a part
        if (a.chunks) {
            steps = all_rows > F::ROWS ? 1 : max(1, span.tiles);   // as kv_steps_of
            if (all_rows <= F::ROWS) {
                t_begin = max(at_step - first_step, 0);
                t_end = min(end_step - first_step, span.tiles);
                if (first_step < at_step || first_step + steps > end_step)
                    to = (((int64_t)kv * a.chunks + part) * 2 + (first_step / length == part ? 1 : 0)) * F::ROWS;
            }
        } else {
            if (part >= span.parts) continue;
            t_begin = part * span.per_part;
            t_end = min(span.tiles, t_begin + span.per_part);
            if (span.parts > 1) to = 0;
        }
        t_begin = __builtin_amdgcn_readfirstlane(t_begin);
        t_end = __builtin_amdgcn_readfirstlane(t_end);
        const int lo = __builtin_amdgcn_readfirstlane(span.lo), hi = __builtin_amdgcn_readfirstlane(span.hi);
        // positions that some row of the tile sees: [seen_from, hi)
        const int seen_from = a.window > 0 ? (int)max((int64_t)0, s.pos_of_0 + s.first + a.token_of(r0) - a.window + 1) : 0;

        // (as memory that nobody writes, which scalar loads read: what a wave's vector loads wait for stays theirs)
        const auto* entries = (const __attribute__((address_space(4))) int32_t*)(uint64_t)(a.table + seq * a.table_stride);
        // A step's tile, from its first position; past the end the last one again, which is in the cache (a load that is left out at times
        // would be waited for at the next use of any).
        const int last_tile = (min(hi, lo + t_end * KV_TILE) - 1) & ~15;
        auto at_tile = [&](int t, int b) { return min(lo + t * KV_TILE + 16 * b, last_tile); };
        auto page_of = [&](int t, int b) { return entries[at_tile(t, b) >> shift]; };
        // (a page's address is the wave's own, a lane's place in a tile always the same)
        const uint32_t key_at = i * (D / 2) + g * (D / 8), key_power_at = i * F::PART + (D == 256 ? 2 * g : D == 64 ? g >> 1 : g);
        const uint32_t value_at = (g * 16 + i) * (D / 8), value_power_at = ((i * F::PART / 16) << shift) + 4 * g;
        // A step's codes and powers. Where registers hold two of them the next step's are loaded while this one's are at work, else its keys once this
        // one's scores are there and its values behind this one's products.
        struct Loaded {
            MxWords<F::W> k[4], v[4];
            uint32_t kp[4], vp[4];   // powers: of the lane's block or two of a key; of four tokens' values
        } loaded[F::ONE ? 1 : 2];
        const uint8_t *keys = a.mx.k + key_at, *key_powers = a.mx.k_powers + key_power_at, *values = a.mx.v + value_at, *value_powers = a.mx.v_powers + value_power_at;
        // a page's tokens among all: rows of either side are as long
        auto tokens_before = [&](int page) { return ((int64_t)((unsigned)page < (unsigned)a.mx.pages ? page : 0) * a.mx.heads + kv) << shift; };
        auto load_keys = [&](Loaded& into, int t, const int (&pages)[4]) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int64_t tok = tokens_before(pages[b]) + (at_tile(t, b) & ((1 << shift) - 1));
                into.k[b] = *(const MxWords<F::W>*)(keys + tok * (D / 2));
                if (D == 256) into.kp[b] = *(const uint16_t*)(key_powers + tok * F::PART);
                else into.kp[b] = key_powers[tok * F::PART];
            }
        };
        auto load_values = [&](Loaded& into, int t, const int (&pages)[4]) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int64_t page = tokens_before(pages[b]), tok = page + (at_tile(t, b) & ((1 << shift) - 1));
                into.v[b] = *(const MxWords<F::W>*)(values + tok * (D / 2));
                into.vp[b] = *(const uint32_t*)(value_powers + page * (F::PART - 1) + tok);
            }
        };
        int t = t_begin + wave;
        int pages[4] = {}, next[4] = {};   // of this step and of the wave's next one
        if (t < t_end) {
#pragma unroll
            for (int b = 0; b < 4; ++b) pages[b] = page_of(t, b);
#pragma unroll
            for (int b = 0; b < 4; ++b) next[b] = page_of(t + WAVES, b);
            load_keys(loaded[0], t, pages);
            load_values(loaded[0], t, pages);
        }

        const float under = mx_under<CAP>(a.scale, a.cap);
        // the rows' pieces, and what a product, or its tanh, is in powers of two
        mx_b8 q[F::KS][F::QP];
        const int r = r0 + i / SLOTS;
        const int of_seq = a.token_of(min(r, r1)), tok = s.first + of_seq, head = kv * a.group + min(r, r1) - of_seq * a.group;
        const int pos = r <= r1 ? (int)max(s.pos_of_0 + tok, (int64_t)-1) : -1;
        const T* row = (const T*)a.q + tok * a.q_stride + (int64_t)head * D + g * (D / 4);
        bool finite = true;
#pragma unroll
        for (int ks = 0; ks < F::KS; ++ks) {
            const MxEight<T> raw = *(const MxEight<T>*)(row + 8 * ks);
            uint32_t w[F::PIECES][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = to_f32(raw.v[2 * e]), y = to_f32(raw.v[2 * e + 1]);
                finite = finite && fabsf(x) < INFINITY && fabsf(y) < INFINITY;
                uint32_t both[F::PIECES];
                mx_cut<F::PIECES>(x, y, both);
#pragma unroll
                for (int p = 0; p < F::PIECES; ++p) w[p][e] = both[p];
            }
            if (SLOTS > 1) {   // the slot's piece alone
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t mine = slot == 0 ? w[0][e] : 0;
#pragma unroll
                    for (int p = 1; p < F::PIECES; ++p) mine = slot == p ? w[p][e] : mine;
                    w[0][e] = mine;
                }
            }
#pragma unroll
            for (int p = 0; p < F::QP; ++p) q[ks][p] = __builtin_bit_cast(mx_b8, make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]));
        }
        const uint64_t odd = __ballot(!finite);
        finite = (odd >> i & 0x0001000100010001ull) == 0;
        const float unit = finite ? mx_unit<CAP>(a.scale, a.cap) : NAN;
        int pos_least = r <= r1 ? pos : 0x7FFFFFFF, pos_most = pos;
        for (int o = 1; o < 16; o <<= 1) {
            pos_least = min(pos_least, __shfl_xor(pos_least, o));
            pos_most = max(pos_most, __shfl_xor(pos_most, o));
        }

        float m = -INFINITY, base = 0.f, l = 0.f;   // the largest product or tanh, that as a score, and the sum of weights relative to it
        v4f acc[F::NB];
#pragma unroll
        for (int b = 0; b < F::NB; ++b) acc[b] = (v4f){0.f, 0.f, 0.f, 0.f};

        auto step = [&](Loaded& now, Loaded& then) {
            const int p0 = lo + t * KV_TILE;
            int behind[4], absent = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                behind[b] = page_of(t + 2 * WAVES, b);
                absent |= (unsigned)pages[b] < (unsigned)a.mx.pages && p0 + 16 * b < hi ? 0 : 1 << b;   // (behind the table's end: the last tile again)
            }
            if (!F::ONE) {
                load_keys(then, t + WAVES, next);
                load_values(then, t + WAVES, next);
            }
            // whether every row sees every position of the step
            const bool whole = p0 + KV_TILE - 1 <= pos_least && (a.window == 0 || p0 > pos_most - a.window) && absent == 0;
            v4f sc[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                sc[b] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < F::KS; ++ks) {
                    const float power = D == 256 && ks >= F::KS / 2 ? mx_power_of<1>(now.kp[b]) : mx_power_of<0>(now.kp[b]);
                    const mx_b8 op = mx_eight(now.k[b].w[ks], power);
#pragma unroll
                    for (int p = 0; p < F::QP; ++p) sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op, q[ks][p], sc[b], 0, 0, 0);
                }
            }
            if (F::ONE) load_keys(then, t + WAVES, next);
            uint32_t share[F::SP][4][2];   // weights: of a tile's four positions
            float x[16], top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = sum_of_slots<SLOTS>(sc[e >> 2][e & 3]);
            if (CAP) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = mx_tanh<CAP>(x[e], under);
            }
            if (!whole) {
                asm volatile("");   // (stays a branch: the looks at sixteen positions would else be made in every step)
                const int last = pos - p0 - 4 * g, first = a.window > 0 ? last - a.window : -0x40000000;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 16 * (e >> 2) + (e & 3);
                    if (at > last || at <= first || (absent >> (e >> 2) & 1)) x[e] = -INFINITY;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, x[e]);
            top = mx_max_over_groups(top);
            if (__ballot(top > m)) {
                const float most = fmaxf(m, top), to = most == -INFINITY ? 0.f : most * unit;
                const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(base - to);
                l *= keep;
#pragma unroll
                for (int b = 0; b < F::NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[b][e] *= keep;
                m = most;
                base = to;
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(fmaf(x[4 * b + e], unit, -base));
                    l += p[e];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (SLOTS > 1) {
                        uint32_t piece = mx_pack(p[2 * h], p[2 * h + 1]);
#pragma unroll
                        for (int j = 1; j < F::SHARES; ++j) {
                            const float less = j == 1 ? second : third;
                            p[2 * h] = fmaf(__uint_as_float(piece << 16), -less, p[2 * h]);
                            p[2 * h + 1] = fmaf(__uint_as_float(piece & 0xFFFF0000u), -less, p[2 * h + 1]);
                            piece = mx_pack(p[2 * h], p[2 * h + 1]);
                        }
                        share[0][b][h] = piece;
                    } else {
                        uint32_t both[F::SHARES];
                        mx_pieces<F::SHARES>(p[2 * h], p[2 * h + 1], both);
#pragma unroll
                        for (int j = 0; j < F::SP; ++j) share[j][b][h] = both[j];
                    }
                }
            }
            if (!whole) {
                // what no row sees may hold anything: its values count as zeros
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t seen = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int at = p0 + 16 * b + 4 * g + j;
                        if (at >= seen_from && at < hi && !(absent >> b & 1)) seen |= 0xFFu << (8 * j);
                    }
                    now.vp[b] &= seen;
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int b0 = 2 * half;
                float power[8];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    power[4 * b] = mx_power_of<0>(now.vp[b0 + b]);
                    power[4 * b + 1] = mx_power_of<1>(now.vp[b0 + b]);
                    power[4 * b + 2] = mx_power_of<2>(now.vp[b0 + b]);
                    power[4 * b + 3] = mx_power_of<3>(now.vp[b0 + b]);
                }
                mx_b8 w[F::SP];
#pragma unroll
                for (int j = 0; j < F::SP; ++j)
                    w[j] = __builtin_bit_cast(mx_b8, make_uint4(share[j][b0][0], share[j][b0][1], share[j][b0 + 1][0], share[j][b0 + 1][1]));
#pragma unroll
                for (int byte = 0; byte < F::PART; ++byte) {   // columns 2 byte and 2 byte + 1 of the lane's sixteenth
                    uint32_t c[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int at = (j & 3) * F::PART + byte;
                        const uint32_t word = now.v[b0 + (j >> 2)].w[at >> 2];
                        const int sel = at & 3;
                        c[j] = sel == 0 ? mx_two<0>(word, power[j]) : sel == 1 ? mx_two<1>(word, power[j]) : sel == 2 ? mx_two<2>(word, power[j]) : mx_two<3>(word, power[j]);
                    }
                    uint32_t even[4], odd[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        even[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x05040100u);
                        odd[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x07060302u);
                    }
                    const mx_b8 op0 = __builtin_bit_cast(mx_b8, make_uint4(even[0], even[1], even[2], even[3]));
                    const mx_b8 op1 = __builtin_bit_cast(mx_b8, make_uint4(odd[0], odd[1], odd[2], odd[3]));
#pragma unroll
                    for (int j = 0; j < F::SP; ++j) {
                        acc[2 * byte] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op0, w[j], acc[2 * byte], 0, 0, 0);
                        acc[2 * byte + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op1, w[j], acc[2 * byte + 1], 0, 0, 0);
                    }
                }
            }
            if (F::ONE) load_values(then, t + WAVES, next);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                pages[b] = next[b];
                next[b] = behind[b];
            }
            t += WAVES;
        };
        while (t < t_end) {
            step(loaded[0], loaded[F::ONE ? 0 : 1]);
            if (!F::ONE && t < t_end) step(loaded[F::ONE ? 0 : 1], loaded[0]);
        }

        // the slots' sums, and the four waves' relative to their common maximum, an operand's rows at a time
        l = sum_over_groups(l);
        m = m == -INFINITY ? m : base;
        if (g == 0 && slot == 0) tops[wave][i / SLOTS] = m;
        if (SLOTS > 1) {
#pragma unroll
            for (int b = 0; b < F::NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[b][e] = sum_of_slots<SLOTS>(slot < F::SHARES ? acc[b][e] : 0.f);
        }
        __syncthreads();
        const int column = i / SLOTS;
        const float top = fmaxf(fmaxf(tops[0][column], tops[1][column]), fmaxf(tops[2][column], tops[3][column]));
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        // column of the sums: the lane's rows 4 g + e of the operand are sixteenths of the head
        if (slot == 0) {
            // (a part whose scores are no numbers has a sum that is none, and may have no maximum)
            if (g == 0) weights[wave][column] = m == -INFINITY ? l : l * f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int b = 0; b < F::NB; ++b) sums[wave][column][(4 * g + e) * (D / 16) + b] = acc[b][e] * f;
        }
        __syncthreads();
        for (int at = threadIdx.x; at < min(r1 - r0 + 1, F::ROWS) * D; at += 64 * WAVES) {
            const int rr = at / D, d = at % D;
            float total = 0.f, lw = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                total += sums[w][rr][d];
                lw += weights[w][rr];
            }
            const int of_seq = a.token_of(r0 + rr), head = kv * a.group + r0 + rr - of_seq * a.group;
            const int64_t row = s.first + of_seq;
            if (to < 0) {
                ((T*)a.out)[row * a.out_stride + (int64_t)head * D + d] = from_f32<T>(lw == 0.f ? 0.f : total / lw);
            } else {
                const int64_t place = a.chunks ? to + rr : (a.part_row(seq, s, (int)row) * a.heads + head) * a.splits + part;
                a.part_o[place * D + d] = total;
                if (d == 0) a.part_ml[place] = make_float2(fmaxf(fmaxf(tops[0][rr], tops[1][rr]), fmaxf(tops[2][rr], tops[3][rr])), lw);
            }
        }
        __syncthreads();
      }
    }
}

template <typename T, int D, int CAP>
static int launch(const AttendMx& a, int max_rows, hipStream_t s) {
    constexpr int SLOTS = sizeof(T) == 4 ? 4 : 2;
    const int per = mx_few_rows(sizeof(T) == 4, max_rows), row_tiles = max_rows < 1 ? 1 : (max_rows - 1) / per + 1;
    const int64_t blocks = a.chunks ? (int64_t)a.chunks * a.mx.heads : (int64_t)a.seqs * a.mx.heads * row_tiles * a.splits;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    const dim3 grid((unsigned)blocks), threads(64 * WAVES);
    if (per == 16 / SLOTS) hipLaunchKernelGGL((mx_few_kernel<T, D, SLOTS, CAP>), grid, threads, 0, s, a, row_tiles);
    else hipLaunchKernelGGL((mx_few_kernel<T, D, 1, CAP>), grid, threads, 0, s, a, row_tiles);
    return lk_launch_status();
}

template <typename T, int D>
static int by_cap(const AttendMx& a, int max_rows, hipStream_t s) {
    const int cap = mx_cap_of(a.cap, sizeof(T) == 4);
    if constexpr (sizeof(T) == 2)
        if (cap == MX_NEAR) return launch<T, D, MX_NEAR>(a, max_rows, s);
    return cap == MX_FAR ? launch<T, D, MX_FAR>(a, max_rows, s) : launch<T, D, MX_NONE>(a, max_rows, s);
}

template <typename T>
static int by_dim(const AttendMx& a, int head_dim, int max_rows, hipStream_t s) {
    return head_dim == 64 ? by_cap<T, 64>(a, max_rows, s) : head_dim == 128 ? by_cap<T, 128>(a, max_rows, s) : by_cap<T, 256>(a, max_rows, s);
}

}  // namespace

int kv_attention_mxfp4_few(const AttendMx& a, int type, int head_dim, int max_rows, hipStream_t s) {
    if (type == LK_TYPE_F32) return by_dim<float>(a, head_dim, max_rows, s);
    if (type == LK_TYPE_F16) return by_dim<__half>(a, head_dim, max_rows, s);
    return by_dim<__hip_bfloat16>(a, head_dim, max_rows, s);
}
