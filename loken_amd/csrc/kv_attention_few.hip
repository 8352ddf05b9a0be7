// Attention over the 8-bit cache for a few rows of a sequence: single tokens, and the handful a draft brings.
//
// The cache's codes go to the int8 matrix unit as they lie in memory: nothing converts them. The other operands, queries
// and softmax weights, are numbers of many bits and are written in base 256 with digits -128 .. 127, each digit a row of
// its own in a 16-row operand that a few rows would leave mostly empty: three digits for f32 (24 bits with the sign), two for f16
// and bf16 (a key's code holds 7 bits of its page's largest value, the query's two digits 15 of its row's). So
//     q . k = s_q s_k sum_i 256^i (digit_i . code),    sum_j p_j v_j = (v_max / F) sum_i 256^i (digit_i(p_j F s_v,j / v_max) . code_j)
// where every product in parentheses is exact in int32, over the head dimension or over a step of 64 positions, and v_max is the largest value
// scale that the row sees in the step. Weights are taken relative to the step's own maximum before they are cut into digits, so a step far
// below the row's maximum loses no bits.
//
// One wave takes a step: 64 positions as four runs of sixteen. v_mfma_i32_16x16x64_i8 gives the scores as (16 positions) x
// (16 slots); the positions of its operand are chosen so that lane group g ends with the sixteen of run g, which is how the second
// product wants its weights, in the same lanes. A lane's run lies in one page: one pair of scales a lane and step. Loads of the
// next step's keys go out once the scores have been taken, its values' once the sums have been: both are in flight through the other
// half of the step, without registers of their own.
//
// Four waves take steps in turn and meet in LDS; long contexts are cut into parts, which a second launch joins.

#include "kv_attention.h"

namespace {

constexpr int WAVES = 4;

template <typename T, int D, int NT>
struct Few {
    static constexpr int DIGITS = sizeof(T) == 4 ? 3 : 2;
    static constexpr int SLOTS = DIGITS == 3 ? 4 : 2;   // slots of a row in the 16-row operand
    static constexpr int RPT = 16 / SLOTS;              // rows of an operand
    static constexpr int ROWS = NT * RPT;               // rows of a workgroup
    static constexpr int KK = D / 64, NB = D / 16;
    static constexpr int PER = DIGITS == 3 ? 1 : 2;     // rows whose sums a lane holds, per operand
    // The largest numbers the digits are made of. They hold 127 * (65536 + 256 + 1) and 127 * (256 + 1); the first leaves room for a last place of f32.
    static constexpr float Q_MAX = DIGITS == 3 ? 127.f * 65536 : 127.f * 256 + 127;
    static constexpr int Q_BITS = DIGITS == 3 ? 23 : 15;   // Q_MAX is just below 2^Q_BITS
    static constexpr float Q_ROUND = 1 << Q_BITS;
    static constexpr float P_MAX = DIGITS == 3 ? 63.f * 65536 + 127 * 256 + 127 : 127.f * 256 + 127;   // below 2^22: see cut()
    // Whole numbers of weights are brought to size before a scale comes in: with the scale alone a small one's quotient would be subnormal.
    static constexpr float P_UNIT = DIGITS == 3 ? 0x1p-22f : 0x1p-15f, P_LEFT = 1.f / (P_MAX * P_UNIT);   // just above 1
    static constexpr int BALANCE = DIGITS == 3 ? 0x808080 : 0x8080;
};

static __device__ __forceinline__ v4i mfma(uint4 a, uint4 b, v4i c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8((v4i){(int)a.x, (int)a.y, (int)a.z, (int)a.w}, (v4i){(int)b.x, (int)b.y, (int)b.z, (int)b.w}, c, 0, 0, 0);
}

// The maximum over the four lanes l, l + 16, l + 32, l + 48.
static __device__ __forceinline__ float max_over_groups(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
static __device__ __forceinline__ float sum_over_groups(float v) { return swap_add32(swap_add16(v)); }

// Byte `digit` of four numbers as one word; selectors of v_perm, two bytes each.
static __device__ __forceinline__ uint32_t four_digits(int t0, int t1, int t2, int t3, uint32_t pick) {
    const uint32_t a = __builtin_amdgcn_perm((uint32_t)t1, (uint32_t)t0, pick), b = __builtin_amdgcn_perm((uint32_t)t3, (uint32_t)t2, pick);
    return __builtin_amdgcn_perm(b, a, 0x05040100u);
}

template <typename T, int D, int NT>
__global__ __launch_bounds__(64 * WAVES, D < 256 && !(D == 128 && NT == 2) ? 2 : 1) void kv_attention_few_kernel(Attend a, int row_tiles) {
    using F = Few<T, D, NT>;
    __shared__ float sums[WAVES][F::ROWS][D];
    __shared__ float tops[WAVES][F::ROWS], weights[WAVES][F::ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int shift = a.pool.page_shift, runs = shift - 4;   // log2 of the runs of a page
    const int slot = i % F::SLOTS;
    const float digit = slot >= F::DIGITS ? 0.f : slot == F::DIGITS - 1 ? 1.f : slot == F::DIGITS - 2 ? 256.f : 65536.f;
    // v_perm selector of the slot's byte out of two words, zeros above; the slot without a digit takes zeros
    const uint32_t byte = F::DIGITS - 1 - slot, pick = slot < F::DIGITS ? 0x0C0C0000u | byte | (byte + 4) << 8 : 0x0C0C0C0Cu;
    // The workgroup's place: (part, row tile, head, sequence), the part fastest; or (head, piece), a piece being of one or
    // several sequences.
    int kv, seq, seq_end, tile0 = 0, part = 0;
    int first_step = 0, at_step = 0, end_step = 0, length = 1;   // the first step of `seq`, the piece's steps, and how many a piece has
    if (a.chunks) {
        kv = blockIdx.x % a.pool.heads;
        part = blockIdx.x / a.pool.heads;
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
        kv = at % a.pool.heads;
        seq = at / a.pool.heads;
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

        // The first step's keys and values are on their way while the rows' digits are made.
        // A step's page of the lane's run: of run i / 4 as the keys' operand has it, of run g for everything else
        const int32_t* entries = a.table + seq * a.table_stride;
        auto page_of = [&](int t, int run) {
            const int p0 = span.lo + t * KV_TILE + 16 * run;
            const int page = t < t_end && p0 < span.hi ? entries[p0 >> shift] : -1;
            return (unsigned)page < (unsigned)a.pool.pages ? page : -1;
        };
        uint4 k[4 * F::KK], v[F::NB];
        float ks = 0.f, vs = 0.f;
        auto load_keys = [&](int t, int kp) {
            const int64_t page = (int64_t)max(kp, 0) * a.pool.heads + kv;
            const int run = ((span.lo >> 4) + 4 * t + (i >> 2)) & ((1 << runs) - 1);
            const int8_t* from = a.pool.k + ((page << shift) + 16 * run + (i & 3)) * D + 16 * g;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int kk = 0; kk < F::KK; ++kk) k[b * F::KK + kk] = *(const uint4*)(from + 4 * b * D + 64 * kk);
        };
        auto load_values = [&](int t, int vp) {
            const int64_t page = (int64_t)max(vp, 0) * a.pool.heads + kv;
            const int run = ((span.lo >> 4) + 4 * t + g) & ((1 << runs) - 1);
            const int8_t* from = a.pool.v + (page << shift) * D + (run * D + i) * 16;
#pragma unroll
            for (int b = 0; b < F::NB; ++b) v[b] = *(const uint4*)(from + 256 * b);
        };
        auto load_scales = [&](int vp) {
            const int64_t page = (int64_t)max(vp, 0) * a.pool.heads + kv;
            ks = a.pool.k_scales[page];
            vs = vp >= 0 ? a.pool.v_scales[page] : 0.f;
        };
        int t = t_begin + wave;
        int kp = page_of(t, i >> 2), vp = page_of(t, g);
        if (t < t_end) {
            load_keys(t, kp);
            load_scales(vp);
            load_values(t, vp);
        }
        int kp_next = page_of(t + WAVES, i >> 2), vp_next = page_of(t + WAVES, g);
        // the rows' digits, and what a unit of the scores is in powers of two
        uint4 q[NT][F::KK];
        float unit[NT];
        int pos[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = r0 + n * F::RPT + i / F::SLOTS;
            const int of_seq = a.token_of(min(r, r1)), tok = s.first + of_seq, head = kv * a.group + min(r, r1) - of_seq * a.group;
            pos[n] = r <= r1 ? (int)max(s.pos_of_0 + tok, (int64_t)-1) : -1;
            const T* row = (const T*)a.q + tok * a.q_stride + (int64_t)head * D + 16 * g;
            float x[F::KK][16];
#pragma unroll
            for (int kk = 0; kk < F::KK; ++kk) {
                if (a.q_aligned) {
                    T raw[16];
#pragma unroll
                    for (int e = 0; e < (int)sizeof(T); ++e) ((uint4*)raw)[e] = ((const uint4*)(row + 64 * kk))[e];
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[kk][e] = to_f32(raw[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[kk][e] = to_f32(row[64 * kk + e]);
                }
            }
            uint32_t most = 0;   // as bits, where what is not a number is the largest
#pragma unroll
            for (int kk = 0; kk < F::KK; ++kk)
#pragma unroll
                for (int e = 0; e < 16; ++e) most = max(most, __float_as_uint(x[kk][e]) & 0x7FFFFFFFu);
            most = max(most, (uint32_t)__shfl_xor((int)most, 16));
            most = max(most, (uint32_t)__shfl_xor((int)most, 32));
            const bool finite = most < 0x7F800000u;
            int e2 = 0;
            const float mant = frexpf(finite && most ? __uint_as_float(most) : 1.f, &e2);   // in [1/2, 1)
            const float f = F::Q_MAX / mant;
            // (the row's power of two last: what it makes up for may be far from one)
            unit[n] = finite ? ldexpf(mant * (a.scale * (1.4426950408889634f * F::Q_ROUND / F::Q_MAX)), e2 - F::Q_BITS) : NAN;
#pragma unroll
            for (int kk = 0; kk < F::KK; ++kk) {
                uint32_t w[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    int t[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        t[j] = ((finite ? (int)rintf(ldexpf(x[kk][4 * b + j], -e2) * f) : 0) + F::BALANCE) ^ F::BALANCE;
                    w[b] = four_digits(t[0], t[1], t[2], t[3], pick);
                }
                q[n][kk] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        int pos_least = 0x7FFFFFFF, pos_most = -1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = r0 + n * F::RPT + i / F::SLOTS;
            if (r <= r1) { pos_least = min(pos_least, pos[n]); pos_most = max(pos_most, pos[n]); }
        }
        for (int o = 1; o < 16; o <<= 1) {
            pos_least = min(pos_least, __shfl_xor(pos_least, o));
            pos_most = max(pos_most, __shfl_xor(pos_most, o));
        }

        float m[NT], l[NT], acc[NT][F::PER][F::NB];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int p = 0; p < F::PER; ++p)
#pragma unroll
                for (int b = 0; b < F::NB; ++b) acc[n][p][b] = 0.f;
        }

        for (; t < t_end; t += WAVES) {
            const int p0 = span.lo + t * KV_TILE + 16 * g;   // the lane's first position
            // whether every row sees every position of the step
            const bool whole = span.lo + t * KV_TILE + KV_TILE - 1 <= pos_least && (a.window == 0 || span.lo + t * KV_TILE > pos_most - a.window) &&
                               __ballot(vp < 0) == 0;
            const float ks_now = ks, vs_now = vs;
            v4i sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    sc[n][b] = (v4i){0, 0, 0, 0};
#pragma unroll
                    for (int kk = 0; kk < F::KK; ++kk) sc[n][b] = mfma(k[b * F::KK + kk], q[n][kk], sc[n][b]);
                }
            const int vp_now = vp;
            kp = kp_next;
            vp = vp_next;
            if (t + WAVES < t_end) {
                load_keys(t + WAVES, kp);
                load_scales(vp);
            }
            kp_next = page_of(t + 2 * WAVES, i >> 2);
            vp_next = page_of(t + 2 * WAVES, g);

            // a row's weights go by the largest value scale of the pages that it sees
            auto share_of = [&](float mine, float most) { return most > 0.f ? mine / most * F::P_MAX : 0.f; };
            const float vs_all = max_over_groups(vs_now), cut_all = share_of(vs_now, vs_all);
            uint4 p_op[NT];
            float keep[NT], gain[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float by = unit[n] * ks_now;
                float x[16];
                float top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float f = (float)sc[n][e >> 2][e & 3] * digit;
                    f += dpp_f32<0xB1>(f);
                    if (F::SLOTS == 4) f += dpp_f32<0x4E>(f);
                    x[e] = f * by;
                }
                float vs_most = vs_all, cut = cut_all;
                if (!whole) {
                    const int last = vp_now < 0 ? -1 : pos[n] - p0, first = a.window > 0 ? pos[n] - a.window - p0 : -1;
                    const float vs_seen = last >= 0 && first < 15 ? vs_now : 0.f;
                    vs_most = max_over_groups(vs_seen);
                    cut = share_of(vs_seen, vs_most);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (e > last || e <= first) x[e] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, x[e]);
                top = max_over_groups(top);
                const float base = top == -INFINITY ? 0.f : top;   // (a row that is not finite has no top and stays that way)
                float sum = 0.f;
                int tt[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p = __builtin_amdgcn_exp2f(x[e] - base);
                    sum += p;
                    // the nearest whole number in the low 23 bits of a sum with 1.5 * 2^23, then its digits
                    tt[e] = (__float_as_int(fmaf(p, cut, 12582912.f)) + (F::BALANCE - (F::DIGITS == 3 ? 0x400000 : 0))) ^ F::BALANCE;
                }
                uint32_t w[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) w[b] = four_digits(tt[4 * b], tt[4 * b + 1], tt[4 * b + 2], tt[4 * b + 3], pick);
                p_op[n] = make_uint4(w[0], w[1], w[2], w[3]);
                const float m_new = fmaxf(m[n], top), m_base = m_new == -INFINITY ? 0.f : m_new;
                keep[n] = __builtin_amdgcn_exp2f(m[n] - m_base);
                const float g0 = __builtin_amdgcn_exp2f(base - m_base);
                const float part_gain = top == -INFINITY ? 1.f : g0;
                l[n] = l[n] * keep[n] + sum * part_gain;
                gain[n] = top == -INFINITY ? 0.f : g0 * (vs_most * F::P_LEFT);
                m[n] = m_new;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // of the rows whose sums the lane holds: (digits 3) row g, (2) rows 2 g and 2 g + 1
                float kr[F::PER], gr[F::PER];
#pragma unroll
                for (int p = 0; p < F::PER; ++p) {
                    const int from = 4 * g + 2 * p;
                    kr[p] = __shfl(keep[n], from);
                    gr[p] = __shfl(gain[n], from);
                }
#pragma unroll
                for (int b = 0; b < F::NB; ++b) {
                    const v4i c = mfma(p_op[n], v[b], (v4i){0, 0, 0, 0});
                    if (F::DIGITS == 3) {
                        const float x = fmaf((float)c[0], 65536.f * F::P_UNIT, fmaf((float)c[1], 256.f * F::P_UNIT, (float)c[2] * F::P_UNIT));
                        acc[n][0][b] = fmaf(x, gr[0], acc[n][0][b] * kr[0]);
                    } else {
#pragma unroll
                        for (int p = 0; p < F::PER; ++p) {
                            const float x = (float)(c[2 * p] * 256 + c[2 * p + 1]) * F::P_UNIT;
                            acc[n][p][b] = fmaf(x, gr[p], acc[n][p][b] * kr[p]);
                        }
                    }
                }
            }
            if (t + WAVES < t_end) load_values(t + WAVES, vp);
        }

        // the four waves' sums relative to their common maximum
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float lw = sum_over_groups(l[n]);
            const int r = n * F::RPT + i / F::SLOTS;
            if (g == 0 && slot == 0) { tops[wave][r] = m[n]; weights[wave][r] = lw; }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int p = 0; p < F::PER; ++p) {
                const int r = n * F::RPT + F::PER * g + p;
                const float mine = tops[wave][r];
                const float top = fmaxf(fmaxf(tops[0][r], tops[1][r]), fmaxf(tops[2][r], tops[3][r]));
                const float f = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - top);
#pragma unroll
                for (int b = 0; b < F::NB; ++b) sums[wave][r][16 * b + i] = acc[n][p][b] * f;
            }
        __syncthreads();
        for (int at = threadIdx.x; at < (r1 - r0 + 1) * D; at += 64 * WAVES) {
            const int r = at / D, d = at % D;
            const float top = fmaxf(fmaxf(tops[0][r], tops[1][r]), fmaxf(tops[2][r], tops[3][r]));
            float total = 0.f, lw = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                total += sums[w][r][d];
                // (a part whose scores are no numbers has no maximum and a sum that is none)
                lw += tops[w][r] == -INFINITY ? weights[w][r] : weights[w][r] * __builtin_amdgcn_exp2f(tops[w][r] - top);
            }
            const int of_seq = a.token_of(r0 + r), head = kv * a.group + r0 + r - of_seq * a.group;
            const int64_t row = s.first + of_seq;
            if (to < 0) {
                ((T*)a.out)[row * a.out_stride + (int64_t)head * D + d] = from_f32<T>(lw == 0.f ? 0.f : total / lw);
            } else {
                const int64_t place = a.chunks ? to + r : (a.part_row(seq, s, (int)row) * a.heads + head) * a.splits + part;
                a.part_o[place * D + d] = total;
                if (d == 0) a.part_ml[place] = make_float2(top, lw);
            }
        }
        __syncthreads();
      }
    }
}

template <typename T, int D>
static int launch(const Attend& a, int max_rows, hipStream_t s) {
    const int per = kv_few_rows(sizeof(T) == 4, D, max_rows), row_tiles = max_rows < 1 ? 1 : (max_rows - 1) / per + 1;
    const bool two = per > Few<T, D, 1>::RPT;
    const int64_t blocks = a.chunks ? (int64_t)a.chunks * a.pool.heads : (int64_t)a.seqs * a.pool.heads * row_tiles * a.splits;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    if (two) hipLaunchKernelGGL((kv_attention_few_kernel<T, D, (D < 256 ? 2 : 1)>), dim3((unsigned)blocks), dim3(64 * WAVES), 0, s, a, row_tiles);
    else hipLaunchKernelGGL((kv_attention_few_kernel<T, D, 1>), dim3((unsigned)blocks), dim3(64 * WAVES), 0, s, a, row_tiles);
    return lk_launch_status();
}

template <typename T>
static int by_dim(const Attend& a, int head_dim, int max_rows, hipStream_t s) {
    return head_dim == 64 ? launch<T, 64>(a, max_rows, s) : head_dim == 128 ? launch<T, 128>(a, max_rows, s) : launch<T, 256>(a, max_rows, s);
}

}  // namespace

int kv_attention_few(const Attend& a, int type, int head_dim, int max_rows, hipStream_t s) {
    if (type == LK_TYPE_F32) return by_dim<float>(a, head_dim, max_rows, s);
    if (type == LK_TYPE_F16) return by_dim<__half>(a, head_dim, max_rows, s);
    return by_dim<__hip_bfloat16>(a, head_dim, max_rows, s);
}
