// Attention over the 4-bit cache for many rows of a sequence: prompts and prefill chunks.
//
// As for a few rows (the operands and what a lane holds are the same), but a row's pieces are instructions of their own, and a workgroup's two waves
// have 16 NT rows (token, head of the group, so that the group's heads share what is read) and take steps of 32 positions in turn; they meet in
// LDS at the end. Nothing is shared before: no barrier, and each wave converts the codes for itself.
//
// The rows' pieces stay in LDS and the next step's keys are loaded when this one's scores are there, its values behind this one's products: bf16 heads of 128 then
// take 168 registers, three waves a SIMD. (In registers with two buffers two waves, weights of one piece: 2048 rows 57 us for 53, 700 rows behind 1000 52 for 35, calls.)
//
// A row's weights are taken relative to a maximum that is put up only where a score lies 2^SLACK above it: bf16 has f32's range, so that costs no
// bits, and a step without such a score needs no exchange between lanes and no correction. The sum of weights is a product with ones, of
// the weights as they went into the sums of values: their roundings cancel.
//
// Bound by the issue of vector and matrix instructions, which take turns on a SIMD: of a step of 32 rows x 32 positions, heads of 128, 52 matrix
// instructions of 16 cycles and 230 vector ones, 64 of them from codes to bf16. 2048 rows behind 14336 positions, 32 heads of 128, bf16: 770 us (calls), 669 TFLOP/s of the
// 1222 that a plain product reaches; 2048 rows alone 74.7 us (kernel trace). Not kept, with weights of one piece: 64 rows a wave (one wave a SIMD, 662 us for 642), 128
// rows that share the values' operands through LDS (598 for 616, and slower at every shorter size).

#include "kv_attention_mxfp4.h"

namespace {

constexpr int WAVES = 2, STEP = 32, TILES = STEP / 16;
constexpr float SLACK = 8.f;   // a power of two

template <typename T, int D>
struct Many {
    static constexpr bool FINE = sizeof(T) == 4;
    static constexpr int QP = FINE ? 3 : std::is_same<T, __half>::value ? 2 : 1;   // pieces of a query value
    // Pieces of a weight: 16 bits, 24 beside f32. (One, 8 bits, in bf16: 2048 rows alone 61 us for 74, behind 14336 625 for 770, calls, and outputs
    // off by 0.0020 of their size, root mean square, where 16 bits leave the output's own rounding, 0.0016.)
    static constexpr int SP = FINE ? 3 : 2;
    static constexpr int ROWS = mx_many_rows(FINE, D), NT = ROWS / 16, PITCH = D + 4, KS = D / 32, NB = D / 16, W = D / 32, PART = D / 32;
    static constexpr int QUERIES = NT * KS * QP * 64 * 16, HANDED = NT * 16 * PITCH * 4, LDS = QUERIES > HANDED ? QUERIES : HANDED;
};

// CAP: whether and how scores are capped (as a branch at run time the compiler takes the tanh always, and the result where it is asked for)
template <typename T, int D, int CAP>
__global__ __launch_bounds__(64 * WAVES, (mx_many_on_simd(sizeof(T) == 4, sizeof(T) == 2 && std::is_same<T, __half>::value, D))) void mx_many_kernel(AttendMx a) {
    using M = Many<T, D>;
    __shared__ uint4 lds[M::LDS / 16];   // the rows' operands, in the end half of the sums on their way to the other wave
    __shared__ float units[M::ROWS];
    __shared__ float tops[WAVES][M::ROWS], weights[WAVES][M::ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4, shift = a.mx.page_shift;
    unsigned block = blockIdx.x;
    const int kv = block % a.mx.heads;
    block /= a.mx.heads;
    const int part = block % a.splits;
    int seq = 0, tile = 0;
    if (!mx_tile_at(a, M::ROWS, block / a.splits, seq, tile)) return;
    seq = __builtin_amdgcn_readfirstlane(seq);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const KvSeq s(a, seq);
    const unsigned all_rows = (unsigned)s.tokens() * (unsigned)a.group, r0 = (unsigned)tile * M::ROWS, r1 = min(r0 + M::ROWS, all_rows) - 1;
    const KvSpan span(a, s, s.first + a.token_of(r0), s.first + a.token_of(r1));
    if (part >= span.parts) return;
    const int lo = __builtin_amdgcn_readfirstlane(span.lo), hi = __builtin_amdgcn_readfirstlane(span.hi);
    const int t_end = __builtin_amdgcn_readfirstlane(min(span.tiles, (part + 1) * span.per_part)) * (KV_TILE / STEP);
    int t = __builtin_amdgcn_readfirstlane(part * span.per_part) * (KV_TILE / STEP) + wave;
    // positions that some row of the tile sees: [seen_from, hi)
    const int seen_from = a.window > 0 ? (int)max((int64_t)0, s.pos_of_0 + s.first + a.token_of(r0) - a.window + 1) : 0;

    // (as memory that nobody writes, which scalar loads read: what a wave's vector loads wait for stays theirs)
    const auto* entries = (const __attribute__((address_space(4))) int32_t*)(uint64_t)(a.table + seq * a.table_stride);
    // A step's tile, from its first position; past the end the last one again, which is in the cache (a load that is left out at times
    // would be waited for at the next use of any).
    const int last_tile = (min(hi, lo + t_end * STEP) - 1) & ~15;
    auto at_tile = [&](int t, int b) { return min(lo + t * STEP + 16 * b, last_tile); };
    auto page_of = [&](int t, int b) { return entries[at_tile(t, b) >> shift]; };
    // (a page's address is the wave's own, a lane's place in a tile always the same)
    const uint32_t key_at = i * (D / 2) + g * (D / 8), key_power_at = i * M::PART + (D == 256 ? 2 * g : D == 64 ? g >> 1 : g);
    const uint32_t value_at = (g * 16 + i) * (D / 8), value_power_at = ((i * M::PART / 16) << shift) + 4 * g;
    MxWords<M::W> k[TILES], v[TILES];
    uint32_t kp[TILES], vp[TILES];   // powers: of the lane's block or two of a key; of four tokens' values
    const uint8_t *keys = a.mx.k + key_at, *key_powers = a.mx.k_powers + key_power_at, *values = a.mx.v + value_at, *value_powers = a.mx.v_powers + value_power_at;
    // a page's tokens among all: rows of either side are as long
    auto tokens_before = [&](int page) { return ((int64_t)((unsigned)page < (unsigned)a.mx.pages ? page : 0) * a.mx.heads + kv) << shift; };
    auto load_keys = [&](int t, const int (&pages)[TILES]) {
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
            const int64_t tok = tokens_before(pages[b]) + (at_tile(t, b) & ((1 << shift) - 1));
            k[b] = *(const MxWords<M::W>*)(keys + tok * (D / 2));
            if (D == 256) kp[b] = *(const uint16_t*)(key_powers + tok * M::PART);
            else kp[b] = key_powers[tok * M::PART];
        }
    };
    auto load_values = [&](int t, const int (&pages)[TILES]) {
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
            const int64_t page = tokens_before(pages[b]), tok = page + (at_tile(t, b) & ((1 << shift) - 1));
            v[b] = *(const MxWords<M::W>*)(values + tok * (D / 2));
            vp[b] = *(const uint32_t*)(value_powers + page * (M::PART - 1) + tok);
        }
    };
    int pages[TILES] = {}, next[TILES] = {};   // of this step and of the wave's next one
    if (t < t_end) {
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
            pages[b] = page_of(t, b);
            next[b] = page_of(t + WAVES, b);
        }
        load_keys(t, pages);
        load_values(t, pages);
    }

    const float under = mx_under<CAP>(a.scale, a.cap);
    // The rows' pieces as operands, in LDS, each wave half of them; and what a product, or its tanh, is in powers of two.
    uint4* const queries = lds;
    float unit[M::NT];
    int pos[M::NT];
#pragma unroll
    for (int n = 0; n < M::NT; ++n) {
        const unsigned r = r0 + 16 * n + i;
        const int of_seq = a.token_of(min(r, r1)), tok = s.first + of_seq, head = kv * a.group + (int)(min(r, r1) - (unsigned)of_seq * a.group);
        pos[n] = r <= r1 ? (int)max(s.pos_of_0 + tok, (int64_t)-1) : -1;
        if ((n & 1) != wave) continue;
        const T* row = (const T*)a.q + tok * a.q_stride + (int64_t)head * D + g * (D / 4);
        bool finite = true;
#pragma unroll
        for (int ks = 0; ks < M::KS; ++ks) {
            const MxEight<T> raw = *(const MxEight<T>*)(row + 8 * ks);
            uint32_t w[M::QP][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = to_f32(raw.v[2 * e]), y = to_f32(raw.v[2 * e + 1]);
                finite = finite && fabsf(x) < INFINITY && fabsf(y) < INFINITY;
                uint32_t both[M::QP];
                mx_cut<M::QP>(x, y, both);
#pragma unroll
                for (int p = 0; p < M::QP; ++p) w[p][e] = both[p];
            }
#pragma unroll
            for (int p = 0; p < M::QP; ++p) queries[((n * M::KS + ks) * M::QP + p) * 64 + lane] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
        }
        const uint64_t odd = __ballot(!finite);
        if (g == 0) units[16 * n + i] = (odd >> i & 0x0001000100010001ull) == 0 ? mx_unit<CAP>(a.scale, a.cap) : NAN;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < M::NT; ++n) unit[n] = units[16 * n + i];
    // positions that all rows see (of a window: behind the last one's first)
    const int pos_least = (int)max(s.pos_of_0 + s.first + a.token_of(r0), (int64_t)-1), pos_most = (int)max(s.pos_of_0 + s.first + a.token_of(r1), (int64_t)-1);

    float top[M::NT], base[M::NT];   // the product or tanh that weights are put to a new maximum above, and that maximum as a score
    v4f l[M::NT], acc[M::NT][M::NB];
#pragma unroll
    for (int n = 0; n < M::NT; ++n) {
        top[n] = -INFINITY;
        base[n] = 0.f;
        l[n] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < M::NB; ++b) acc[n][b] = (v4f){0.f, 0.f, 0.f, 0.f};
    }
    const mx_b8 ones = __builtin_bit_cast(mx_b8, make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u));

    for (; t < t_end; t += WAVES) {
        const int p0 = lo + t * STEP;
        int behind[TILES], absent = 0;
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
            behind[b] = page_of(t + 2 * WAVES, b);
            absent |= (unsigned)pages[b] < (unsigned)a.mx.pages && p0 + 16 * b < hi ? 0 : 1 << b;   // (behind the table's end: the last tile again)
        }
        // whether every row sees every position of the step
        const bool whole = p0 + STEP - 1 <= pos_least && (a.window == 0 || p0 > pos_most - a.window) && absent == 0;
        v4f sc[M::NT][TILES];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
#pragma unroll
            for (int n = 0; n < M::NT; ++n) sc[n][b] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < M::KS; ++ks) {
                const float power = D == 256 && ks >= M::KS / 2 ? mx_power_of<1>(kp[b]) : mx_power_of<0>(kp[b]);
                const mx_b8 op = mx_eight(k[b].w[ks], power);
#pragma unroll
                for (int n = 0; n < M::NT; ++n)
#pragma unroll
                    for (int p = 0; p < M::QP; ++p)
                        sc[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op, __builtin_bit_cast(mx_b8, queries[((n * M::KS + ks) * M::QP + p) * 64 + lane]), sc[n][b], 0, 0, 0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        load_keys(t + WAVES, next);
        mx_b8 share[M::NT][M::SP];
#pragma unroll
        for (int n = 0; n < M::NT; ++n) {
            float x[4 * TILES], most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4 * TILES; ++e) x[e] = sc[n][e >> 2][e & 3];
            if (CAP) {
#pragma unroll
                for (int e = 0; e < 4 * TILES; ++e) x[e] = mx_tanh<CAP>(x[e], under);
            }
            if (!whole) {
                asm volatile("");   // (stays a branch: the looks at eight positions would else be made in every step)
                const int last = pos[n] - p0 - 4 * g, first = a.window > 0 ? last - a.window : -0x40000000;
#pragma unroll
                for (int e = 0; e < 4 * TILES; ++e) {
                    const int at = 16 * (e >> 2) + (e & 3);
                    if (at > last || at <= first || (absent >> (e >> 2) & 1)) x[e] = -INFINITY;
                }
            }
#pragma unroll
            for (int e = 0; e < 4 * TILES; ++e) most = fmaxf(most, x[e]);
            if (__ballot(most > top[n])) {
                most = mx_max_over_groups(most);
                const bool first = top[n] == -INFINITY, up = most > top[n];
                const float to = up ? most * unit[n] : base[n], keep = first ? 1.f : __builtin_amdgcn_exp2f(base[n] - to);
                l[n] *= keep;
#pragma unroll
                for (int b = 0; b < M::NB; ++b) acc[n][b] *= keep;
                base[n] = to;
                top[n] = up ? most + SLACK / unit[n] : top[n];
            }
            uint32_t w[M::SP][2 * TILES];
#pragma unroll
            for (int e = 0; e < 2 * TILES; ++e) {
                uint32_t both[M::SP];
                mx_pieces<M::SP>(__builtin_amdgcn_exp2f(fmaf(x[2 * e], unit[n], -base[n])), __builtin_amdgcn_exp2f(fmaf(x[2 * e + 1], unit[n], -base[n])), both);
#pragma unroll
                for (int j = 0; j < M::SP; ++j) w[j][e] = both[j];
            }
#pragma unroll
            for (int j = 0; j < M::SP; ++j) share[n][j] = __builtin_bit_cast(mx_b8, make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]));
        }
        if (!whole) {
            // what no row sees may hold anything: its values count as zeros
#pragma unroll
            for (int b = 0; b < TILES; ++b) {
                uint32_t seen = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = p0 + 16 * b + 4 * g + j;
                    if (at >= seen_from && at < hi && !(absent >> b & 1)) seen |= 0xFFu << (8 * j);
                }
                vp[b] &= seen;
            }
        }
        float power[4 * TILES];
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
            power[4 * b] = mx_power_of<0>(vp[b]);
            power[4 * b + 1] = mx_power_of<1>(vp[b]);
            power[4 * b + 2] = mx_power_of<2>(vp[b]);
            power[4 * b + 3] = mx_power_of<3>(vp[b]);
        }
#pragma unroll
        for (int n = 0; n < M::NT; ++n)
#pragma unroll
            for (int j = 0; j < M::SP; ++j) l[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, share[n][j], l[n], 0, 0, 0);
#pragma unroll
        for (int byte = 0; byte < M::PART; ++byte) {   // columns 2 byte and 2 byte + 1 of the lane's sixteenth
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = (j & 3) * M::PART + byte;
                const uint32_t word = v[j >> 2].w[at >> 2];
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
            for (int n = 0; n < M::NT; ++n)
#pragma unroll
                for (int j = 0; j < M::SP; ++j) {
                    acc[n][2 * byte] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op0, share[n][j], acc[n][2 * byte], 0, 0, 0);
                    acc[n][2 * byte + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op1, share[n][j], acc[n][2 * byte + 1], 0, 0, 0);
                }
        }
        load_values(t + WAVES, next);
#pragma unroll
        for (int b = 0; b < TILES; ++b) {
            pages[b] = next[b];
            next[b] = behind[b];
        }
    }

    // The two waves' sums relative to their common maximum: each wave hands the other the half of the rows that it does not finish.
#pragma unroll
    for (int n = 0; n < M::NT; ++n)
        if (g == 0) {
            tops[wave][16 * n + i] = top[n] == -INFINITY ? -INFINITY : base[n];
            weights[wave][16 * n + i] = l[n][0];
        }
    __syncthreads();   // the last queries have been read
    float* const handed = (float*)lds;
#pragma unroll
    for (int n = 0; n < M::NT; ++n)
        if (n != wave) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int b = 0; b < M::NB; b += 4)
                    *(float4*)&handed[(n * 16 + i) * M::PITCH + (4 * g + e) * (D / 16) + b] = make_float4(acc[n][b][e], acc[n][b + 1][e], acc[n][b + 2][e], acc[n][b + 3][e]);
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < M::NT; ++n) {
        const unsigned r = r0 + 16 * n + i;
        if (n != wave || r > r1) continue;
        const float m0 = tops[0][16 * n + i], m1 = tops[1][16 * n + i], m = fmaxf(m0, m1);
        // (a part whose scores are no numbers has a sum that is none, and may have no maximum)
        const float f0 = m0 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m0 - m), f1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
        const float w0 = weights[0][16 * n + i], w1 = weights[1][16 * n + i], lw = (m0 == -INFINITY ? w0 : w0 * f0) + (m1 == -INFINITY ? w1 : w1 * f1);
        const float mine = n == 0 ? f0 : f1, others = n == 0 ? f1 : f0;
        const int of_seq = a.token_of(r), head = kv * a.group + (int)(r - (unsigned)of_seq * a.group);
        const int64_t row = s.first + of_seq, place = (a.part_row(seq, s, (int)row) * a.heads + head) * a.splits + part;
        const float by = span.parts > 1 ? 1.f : lw == 0.f ? 0.f : 1.f / lw;
        // the lane's rows 4 g + e of the operand are sixteenths of the head
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d0 = (4 * g + e) * (D / 16);
            float x[M::NB];
#pragma unroll
            for (int b = 0; b < M::NB; ++b) x[b] = fmaf(handed[(n * 16 + i) * M::PITCH + d0 + b], others, acc[n][b][e] * mine) * by;
            if (span.parts > 1) {
#pragma unroll
                for (int b = 0; b < M::NB; ++b) a.part_o[place * D + d0 + b] = x[b];
            } else {
                struct __attribute__((aligned(sizeof(T)))) Run { T v[M::NB]; } run;   // rows of out start on any value
#pragma unroll
                for (int b = 0; b < M::NB; ++b) run.v[b] = from_f32<T>(x[b]);
                *(Run*)((T*)a.out + row * a.out_stride + (int64_t)head * D + d0) = run;
            }
        }
        if (span.parts > 1 && g == 0) a.part_ml[place] = make_float2(m, lw);
    }
}

template <typename T, int D>
static int launch(const AttendMx& a, hipStream_t s) {
    const int64_t tiles = ((int64_t)a.rows * a.group + Many<T, D>::ROWS - 1) / Many<T, D>::ROWS + a.seqs, blocks = tiles * a.mx.heads * a.splits;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    const dim3 grid((unsigned)blocks), threads(64 * WAVES);
    const int cap = mx_cap_of(a.cap, sizeof(T) == 4);
    if constexpr (sizeof(T) == 2)
        if (cap == MX_NEAR) {
            hipLaunchKernelGGL((mx_many_kernel<T, D, MX_NEAR>), grid, threads, 0, s, a);
            return lk_launch_status();
        }
    if (cap == MX_FAR) hipLaunchKernelGGL((mx_many_kernel<T, D, MX_FAR>), grid, threads, 0, s, a);
    else hipLaunchKernelGGL((mx_many_kernel<T, D, MX_NONE>), grid, threads, 0, s, a);
    return lk_launch_status();
}

template <typename T>
static int by_dim(const AttendMx& a, int head_dim, hipStream_t s) {
    return head_dim == 64 ? launch<T, 64>(a, s) : head_dim == 128 ? launch<T, 128>(a, s) : launch<T, 256>(a, s);
}

}  // namespace

int kv_attention_mxfp4_many(const AttendMx& a, int type, int head_dim, hipStream_t s) {
    if (type == LK_TYPE_F32) return by_dim<float>(a, head_dim, s);
    if (type == LK_TYPE_F16) return by_dim<__half>(a, head_dim, s);
    return by_dim<__hip_bfloat16>(a, head_dim, s);
}
