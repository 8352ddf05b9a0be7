// Attention over the 8-bit cache for many rows of a sequence: prompts and prefill chunks.
//
// Rows are (token, head of the group) of one key / value head, so that the group's heads share the keys and values that are
// read. A team of four waves has 128 rows; a step is 64 positions, whose codes are turned into f16 (exactly) once for all
// rows on their way into LDS, values with the positions of a column together as they lie in the cache. Products are
// v_mfma_f32_32x32x16_f16, both turned round so that a lane keeps one row throughout:
//     scores   (32 positions) x (32 rows): lane l holds row l % 32, and the positions of its half of the lanes stand in the order in
//              which the next product wants them (the rows of the first operand are read from LDS in that order)
//     sums     (32 columns) x (32 rows): the weights go from the scores' registers straight into the operand
// so the running maximum, its corrections and the sum of weights are the lane's own, with one exchange between the two halves.
//
// Queries come in f16 scaled by a power of two of their row (bf16 fits with its 8 bits, f16 as it is); f32 ones as a high and a
// low half, two products each, as are its weights: 22 bits. A page's key scale goes onto the scores. Its value scale goes onto the
// weights, as a share of `ref`, a power of two above the largest value scale so far: as its logarithm, in the exponent that
// the weight is made from (off by 5e-7 of the weight at most, a last place of the logarithm), and back out of the sum of
// weights run by run.
//
// A row's sums go by 2^m, m a whole number about the largest of score + logarithm of the share among the positions that the row sees: so
// neither small scales nor large ones of pages that it does not see cost its weights bits in f16. They are put to a new m only where
// that lies 2^8 above: weights times shares up to 2^8 then, which stand LIFT = 2^7 above one and stay within 2^15, which f16 holds; one of
// 2^-21 still has all its bits, one of 2^-31 some. Where `ref` grows, m falls by as much and the sums of values stay as they are.
//
// A wave's step is 32 products of 32 cycles (twice as many in f32) and some 400 other instructions, 32 of them exponentials, which
// take four times as long. It is these that bound it, and what of them does not run beside products: so a product comes with
// six of them in turn, its operands read from LDS a group ahead, and nothing that is loaded is looked at before the step after.
// 2048 tokens of one prompt, 32 heads over 8 of 128 bf16 values: 70 us, 490 TFLOP/s of the causal half's products (two starts of 5 us a
// CU in it); the same behind 16384 tokens 700 us, 830 TFLOP/s, in f32 1110; 700 f32 rows over 2200 positions beside eleven single rows: 108 us.

#include "kv_attention.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4, THREADS = 64 * WAVES, RUNS = KV_TILE / 16;   // of a team
constexpr float LIFT = 7.f, SLACK = 8.f;   // powers of two
// Pages whose value scale is a share of 2^-FAR or less are as those without values: in the sum of weights, at a share of 2^-FAR. (A share
// goes down to 2^-247, and what it is taken back out with would leave f32.)
constexpr float FAR = 90.f, LEAST_SHARE = 0x1p-90f;

// Sixteen codes as f16, as they lie: 0x6400 + (code + 128) is the f16 number 1152 + code.
static __device__ __forceinline__ void to_halves(uint4 w, uint4* out) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = in[i] ^ 0x80808080u;
        const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
        const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
        const h2 a = __builtin_bit_cast(h2, lo) - bias, b = __builtin_bit_cast(h2, hi) - bias;
        r[2 * i] = __builtin_bit_cast(uint32_t, a);
        r[2 * i + 1] = __builtin_bit_cast(uint32_t, b);
    }
    out[0] = make_uint4(r[0], r[1], r[2], r[3]);
    out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// (the compiler takes a look at each operand for signalling NaN first)
static __device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// What the four lanes of the runs have together.
template <typename F>
static __device__ __forceinline__ float across_runs(float x, F both) {
    static_assert(RUNS == 4);
    x = both(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, true)));          // lanes 1, 0, 3, 2
    return both(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, true)));       // lanes 2, 3, 0, 1
}

// Teams of a workgroup, which take its steps in turn. Two, where the registers hold them, so that both waves of a SIMD have the same
// rows' work to do to the end: a prompt of 2048 tokens, 32 heads over 8 of 128 bf16 values, took 80 us with one team and two
// workgroups to a CU, of which the one with the longer rows ran on alone. f32 has no registers for the meeting of the teams
// (700 rows over 2200 positions: 178 us against 140), 256 columns none for a second wave on a SIMD.
constexpr int many_teams(bool fine, int head_dim) { return head_dim == 256 || fine ? 1 : 2; }
constexpr int many_waves(int head_dim) { return head_dim == 256 ? 1 : 2; }   // on a SIMD

template <typename T, int D>
struct Many {
    static constexpr bool FINE = sizeof(T) == 4;
    static constexpr int PARTS = FINE ? 2 : 1;
    static constexpr int KS = D / 16, NB = D / 32;
    static constexpr int K_PITCH = 2 * D + 16, V_PITCH = 2 * KV_TILE + 16;   // bytes; sixteen more: no bank conflicts
    static constexpr int K_BYTES = KV_TILE * K_PITCH, V_BYTES = D * V_PITCH;
    static constexpr int CHUNKS = KV_TILE * D / 16 / THREADS;   // of sixteen codes, a thread and side
    static constexpr int TEAMS = many_teams(FINE, D), TEAM_BYTES = 2 * (K_BYTES + V_BYTES);
    static constexpr int LDS = TEAMS * TEAM_BYTES;
    static_assert(TEAM_BYTES >= THREADS * D);   // half of the sums of a team, on their way to the other
};

// What a step's pages have for everybody.
struct __attribute__((aligned(16))) Step {
    float ks[RUNS];     // key scales; -1: the page is absent
    float share[RUNS];  // log2 of the value scale over `ref`; -FAR where the values do not show
    float bias[RUNS];   // that, and LIFT; -infinity where the values do not show
    float back[RUNS];   // 2^-bias, 0 where the values do not show
    uint32_t dead;      // a bit for each page whose values do not show: all zero, or LEAST_SHARE of `ref` at most
    float ref;          // a power of two, at least the largest value scale so far
    float drop, grow;   // log2 of how much `ref` has grown with this step, up to 100, and 2^drop
    float shrink;       // 2^-that of the rest
    int absent;         // whether a page is
};

// The row tile of that number among those of all sequences, from the last one on; false: there are fewer. Found by each wave.
static __device__ __forceinline__ bool tile_at(const Attend& a, int number, int& seq, int& tile) {
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](int i) {
        if (i >= a.seqs) return 0;
        const unsigned rows = (unsigned)KvSeq(a, i).tokens() * (unsigned)a.group;
        return (int)rows <= a.few_rows ? 0 : (int)((rows + KV_MANY_ROWS - 1) / KV_MANY_ROWS);
    };
    for (int base = (a.seqs - 1) & ~63; base >= 0; base -= 64) {
        const int mine = tiles_of(base + lane);
        int behind = mine;   // of this sequence and those behind it
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_down(behind, o);
            if (lane + o < 64) behind += v;
        }
        const uint64_t over = __ballot(behind > number);
        if (over) {
            const int l = 63 - __clzll((long long)over);
            seq = base + l;
            tile = __builtin_amdgcn_readlane(behind, l) - 1 - number;
            return true;
        }
        number -= __builtin_amdgcn_readfirstlane(behind);
    }
    return false;
}

template <typename T, int D>
__global__ __launch_bounds__(many_teams(sizeof(T) == 4, D) * THREADS, many_waves(D)) void kv_attention_many_kernel(Attend a, int row_tiles, int listed, int cus) {
    using M = Many<T, D>;
    extern __shared__ __align__(16) uint8_t lds_of_all[];
    __shared__ Step steps_of_all[M::TEAMS][2];
    __shared__ int pages_of_all[M::TEAMS][4][RUNS];
    __shared__ int64_t starts_of_all[M::TEAMS][4][RUNS];   // of a run's codes in the pool, on either side
    __shared__ float refs[M::TEAMS];
    __shared__ float2 meet[M::TEAMS][32 * WAVES];
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    const int tid = threadIdx.x % THREADS, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t* lds = lds_of_all + team * M::TEAM_BYTES;
    Step* steps = steps_of_all[team];
    auto pages = pages_of_all[team];
    auto starts = starts_of_all[team];
    const int col = lane & 31, half = lane >> 5;
    // Row tiles that see the most come first, so that what comes last is short. Where a CU has two workgroups at once they come in
    // rounds of one to a CU, every other one backwards: a CU with much of one has little of the other.
    unsigned at = blockIdx.x;
    if (M::TEAMS == 1 && D < 256) {
        const unsigned round = at / cus, first = round * cus, size = min((unsigned)cus, gridDim.x - first);
        if (round & 1) at = first + (size - 1 - (at - first));
    }
    const int part = at % a.splits;
    at /= a.splits;
    const int kv = at % a.pool.heads;
    at /= a.pool.heads;
    int seq = at % a.seqs, tile0 = row_tiles - 1 - (int)(at / a.seqs);
    if (listed && !tile_at(a, (int)at, seq, tile0)) return;
    const KvSeq s(a, seq);
    const unsigned all_rows = (unsigned)s.tokens() * (unsigned)a.group;   // below 2^31
    if ((int)all_rows <= a.few_rows) return;
    const int shift = a.pool.page_shift;
    const int32_t* entries = a.table + seq * a.table_stride;
    auto k_lds = [&](int buffer) { return lds + buffer * (M::K_BYTES + M::V_BYTES); };
    auto v_lds = [&](int buffer) { return lds + buffer * (M::K_BYTES + M::V_BYTES) + M::K_BYTES; };

    for (uint64_t tile = tile0; tile * KV_MANY_ROWS < all_rows; tile += row_tiles) {
        const unsigned r_tile = (unsigned)tile * KV_MANY_ROWS;
        const unsigned r_end = min(r_tile + KV_MANY_ROWS, all_rows);
        const KvSpan span(a, s, s.first + a.token_of(r_tile), s.first + a.token_of(r_end - 1));
        const int per_part = span.per_part, parts = span.parts;
        if (part >= parts) continue;
        // a team has every other step; steps are counted from its first
        const int t_begin = part * per_part, t_all = min(span.tiles, t_begin + per_part) - t_begin;
        const int turns = (t_all + M::TEAMS - 1) / M::TEAMS, t_end = (t_all - team + M::TEAMS - 1) / M::TEAMS;
        const int from_pos = span.lo + (t_begin + team) * KV_TILE;
        auto base_of = [&](int t) { return from_pos + t * M::TEAMS * KV_TILE; };   // below 2^31: contexts end 1024 positions before
        // the lane's row, and what its wave sees
        const unsigned r = r_tile + 32 * wave + col;
        const bool row_is = r < r_end;
        const unsigned r_in = min(r, r_end - 1);
        const int of_seq = a.token_of(r_in), tok = s.first + of_seq, head = kv * a.group + (int)r_in - of_seq * a.group;
        const int pos = (int)max(s.pos_of_0 + tok, (int64_t)-1);
        const unsigned w0 = min(r_tile + 32 * wave, r_end - 1), w1 = min(r_tile + 32 * wave + 31, r_end - 1);
        const int pos_least = (int)max(s.pos_of_0 + s.first + a.token_of(w0), (int64_t)-1), pos_most = (int)max(s.pos_of_0 + s.first + a.token_of(w1), (int64_t)-1);

        struct __attribute__((packed, aligned(sizeof(T)))) Eight { T of[8]; };   // (a row's alignment is its type's)
        const Eight* row = (const Eight*)((const T*)a.q + tok * a.q_stride + (int64_t)head * D + 8 * half);
        Eight in[M::KS];
#pragma unroll
        for (int k = 0; k < M::KS; ++k) in[k] = row[2 * k];
        h8 q[M::PARTS][M::KS];
        float unit = 0.f;
        v16f o[M::NB];
#pragma unroll
        for (int b = 0; b < M::NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][e] = 0.f;
        float m = -INFINITY, l = 0.f;

        // A step's codes: thread tid has chunk tid, tid + 256, .. of sixteen. Its pages have been in LDS since the step before.
        uint4 kc[M::CHUNKS], vc[M::CHUNKS];
        // Loads have no conditions and nothing of them is looked at before a step later: a wait for one would be a wait for all.
        const int run = tid & (RUNS - 1);
        auto entry = [&](int t) { return entries[min(base_of(t) + 16 * run, span.hi - 1) >> shift]; };   // (there is a step)
        auto list = [&](int t, int entry) {   // by the first lanes
            const int p0 = base_of(t) + 16 * run, off = p0 & ((1 << shift) - 1);
            const int page = p0 < span.hi && (unsigned)entry < (unsigned)a.pool.pages ? entry : -1;
            pages[t & 3][run] = page;
            starts[t & 3][run] = ((((int64_t)max(page, 0) * a.pool.heads + kv) << shift) + off) * D;
        };
        float ks = -1.f, vs = 0.f, ref = 0.f;
        int page_of_run = -1;
        auto fetch = [&](int t) {
            const int64_t* start = starts[t & 3];
            page_of_run = pages[t & 3][run];
            const int64_t at_scale = (int64_t)max(page_of_run, 0) * a.pool.heads + kv;
#pragma unroll
            for (int c = 0; c < M::CHUNKS; ++c) {   // (a run of either side is D chunks)
                const int n = tid + c * THREADS;
                kc[c] = *(const uint4*)(a.pool.k + start[n / D] + n % D * 16);
                vc[c] = *(const uint4*)(a.pool.v + start[n / D] + n % D * 16);
            }
            ks = a.pool.k_scales[at_scale];
            vs = a.pool.v_scales[at_scale];
        };
        auto store_chunk = [&](int t, int i) {   // keys and values in turn
            const int n = tid + i / 2 * THREADS;
            uint4 w[2];
            to_halves(i & 1 ? vc[i / 2] : kc[i / 2], w);
            uint4* to = (uint4*)(i & 1 ? v_lds(t & 1) + (n % D) * M::V_PITCH + (n / D) * 32 : k_lds(t & 1) + (n / (D / 16)) * M::K_PITCH + (n % (D / 16)) * 32);
            to[0] = w[0];
            to[1] = w[1];
        };
        auto store = [&](int t) {
#pragma unroll
            for (int i = 0; i < 2 * M::CHUNKS; ++i) store_chunk(t, i);
        };
        auto note = [&](int t) {
            if (wave == 1 && lane < RUNS) {
                Step& st = steps[t & 1];
                const float k1 = page_of_run < 0 ? -1.f : ks, v1 = page_of_run < 0 ? 0.f : vs;
                const float most = across_runs(v1, [](float x, float y) { return fmaxf(x, y); });
                const float least = across_runs(k1, [](float x, float y) { return fminf(x, y); });
                // the power of two above `most`, from its exponent
                const float now = most > 0.f ? fmaxf(ref, __uint_as_float(min((__float_as_uint(most) & 0x7F800000u) + 0x00800000u, 0x7F000000u))) : ref;
                const bool shows = v1 > now * LEAST_SHARE;
                const float share = shows ? __builtin_amdgcn_logf(v1 / now) : -FAR, bias = shows ? share + LIFT : -INFINITY;
                st.ks[lane] = k1;
                st.share[lane] = share;
                st.bias[lane] = bias;
                st.back[lane] = shows ? __builtin_amdgcn_exp2f(-bias) : 0.f;
                const uint32_t dead = (uint32_t)__ballot(!shows);
                if (lane == 0) {
                    // (up to the first scale the sums are zeros)
                    const int grown = ref > 0.f ? (int)((__float_as_uint(now) - __float_as_uint(ref)) >> 23) : 0, drop = min(grown, 100);
                    st.drop = (float)drop;
                    st.grow = __uint_as_float((uint32_t)(127 + drop) << 23);
                    st.shrink = grown - drop > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (grown - drop)) << 23);
                    st.ref = now;
                    st.absent = least < 0.f;
                    st.dead = dead;
                }
                ref = now;
            }
        };

        __syncthreads();   // the last row tile's reads of LDS
        int next = -1;
        if (t_all > 0) {   // (a team without a step: of no positions, and of page 0)
            const int e0 = entry(0), e1 = entry(1), e2 = entry(2);
            next = entry(3);
            if (wave == 2 && lane < RUNS) {
                list(0, e0);
                list(1, e1);
                list(2, e2);
            }
            __syncthreads();
            fetch(0);
            {
                uint32_t most = 0;
#pragma unroll
                for (int k = 0; k < M::KS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(to_f32(in[k].of[e])) & 0x7FFFFFFFu);
                most = max(most, (uint32_t)__shfl_xor((int)most, 32));
                const bool finite = most < 0x7F800000u;
                int e2 = 0;
                (void)frexpf(finite && most ? __uint_as_float(most) : 1.f, &e2);   // the row's largest is in [2^(e2 - 1), 2^e2)
#pragma unroll
                for (int k = 0; k < M::KS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = ldexpf(to_f32(in[k].of[e]), 14 - e2);   // below 2^14
                        const _Float16 hi = (_Float16)x;
                        q[0][k][e] = hi;
                        if (M::FINE) q[M::PARTS - 1][k][e] = (_Float16)(x - (float)hi);
                    }
                // the scale first: powers that it makes up for may be far from one
                unit = finite ? ldexpf(ldexpf(a.scale * 1.4426950408889634f, e2 / 2), e2 - e2 / 2 - 14) : NAN;
            }
            store(0);
            note(0);
            if (!M::FINE) fetch(1);
            __syncthreads();
        }
        float ref_of_sums = 0.f;
        for (int t = 0; t < turns; ++t) {
            const bool is = t < t_end;   // the other team may have one step more
            const int base = base_of(t);
            const Step& st = steps[t & 1];
            int after = -1;
            if (M::FINE) {
                after = entry(t + 4);
                fetch(t + 1);
            }
            float grow = 1.f;
            if (is) {
                ref_of_sums = st.ref;
                grow = st.grow;
            }
            // a wave whose rows see nothing of the step leaves it
            const bool sees = is && base <= pos_most && (a.window == 0 || base + KV_TILE - 1 > pos_least - a.window);
            v16f x[2];
            // First the scores, and the next step's codes into LDS meanwhile; then those of the step after it on their way. (f32 has no
            // registers for that: its next step's codes are loaded here and put into LDS at the end. 142 us against 164.)
            if (sees) {
                // row i = 8 b + 4 h + j of the operand is position 16 (b / 2) + 8 h + 4 (b % 2) + j
                const int from = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
                const uint8_t* kr = k_lds(t & 1) + from * M::K_PITCH + 16 * half;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[u][e] = 0.f;
                if constexpr (M::FINE) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int k = 0; k < M::KS; ++k) {
                            const h8 kk = *(const h8*)(kr + 32 * u * M::K_PITCH + 32 * k);
#pragma unroll
                            for (int p = 0; p < M::PARTS; ++p) x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk, q[p][k], x[u], 0, 0, 0);
                        }
                } else {   // four products at a time, the next ones' operands on their way from LDS
                    constexpr int FOURS = M::KS / 2;
                    static_assert(FOURS == 2 * M::CHUNKS);
                    h8 kk[2][4];
                    auto operands = [&](int i) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) kk[i & 1][j] = *(const h8*)(kr + 32 * (j & 1) * M::K_PITCH + 32 * (2 * i + j / 2));
                    };
                    operands(0);
#pragma unroll
                    for (int i = 0; i < FOURS; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (i + 1 < FOURS) operands(i + 1);
                        store_chunk(t + 1, i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[j & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk[i & 1][j], q[0][2 * i + j / 2], x[j & 1], 0, 0, 0);
                        if (i + 1 < FOURS) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                        }
                        __builtin_amdgcn_sched_group_barrier(0x200, 2, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else if (!M::FINE) store(t + 1);
            if (!M::FINE) {
                note(t + 1);
                if (wave == 2 && lane < RUNS) list(t + 3, next);
                next = entry(t + 4);
                fetch(t + 2);
            }
            if (grow > 1.f) {
                m -= st.drop;
                l = fminf(l * grow, 0x1p126f);
                const float shrink = st.shrink;
                if (shrink < 1.f) {
#pragma unroll
                    for (int b = 0; b < M::NB; ++b) o[b] *= shrink;
                }
            }
            if (sees) {
                // scores in powers of two; element e of x[u]: position base + 32 u + 16 (e / 8) + 8 half + e % 8
                const bool whole = base + KV_TILE - 1 <= pos_least && (a.window == 0 || base > pos_most - a.window) && !st.absent;
                float by[RUNS], share[RUNS], top = -INFINITY;
#pragma unroll
                for (int n = 0; n < RUNS; ++n) {
                    by[n] = st.ks[n] * unit;
                    share[n] = st.share[n];
                }
                if (!whole) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int p = base + 32 * u + 16 * (e / 8) + 8 * half + e % 8, n = 2 * u + e / 8;
                            const bool seen = p <= pos && (a.window == 0 || p > pos - a.window) && st.ks[n] >= 0.f;
                            x[u][e] = seen ? x[u][e] * by[n] : -INFINITY;
                        }
#pragma unroll
                    for (int n = 0; n < RUNS; ++n) by[n] = 1.f;
                }
#pragma unroll
                for (int n = 0; n < RUNS; ++n) {
                    const v16f& y = x[n / 2];
                    const int e = 8 * (n % 2);
                    const float part_top = max3(max3(max3(y[e], y[e + 1], y[e + 2]), y[e + 3], y[e + 4]), y[e + 5], max3(y[e + 6], y[e + 7], y[e + 7]));
                    top = fmaxf(top, fmaf(part_top, by[n], share[n]));
                }
                {
                    const auto r2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(r2[0]), __uint_as_float(r2[1]));
                }
                if (__ballot(top > m + SLACK || (m == -INFINITY && top > m)) != 0) {
                    const float m_new = fmaxf(m, ceilf(top));
                    const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                    l *= keep;
#pragma unroll
                    for (int b = 0; b < M::NB; ++b) o[b] *= keep;
                    m = m_new;
                }
                const float m_base = m == -INFINITY ? 0.f : m;
                if (st.dead) {   // positions of pages whose values do not show: in the sum of weights only
#pragma unroll
                    for (int n = 0; n < RUNS; ++n)
                        if (st.dead >> n & 1)
#pragma unroll
                            for (int e = 0; e < 8; ++e) l += __builtin_amdgcn_exp2f(fmaf(x[n / 2][8 * (n % 2) + e], by[n], -m_base));
                }
                // then the weights and sums
                const uint8_t* vl = v_lds(t & 1);
                h8 w[2][M::PARTS], vv[2][M::NB];
                auto operands = [&](int n) {
#pragma unroll
                    for (int b = 0; b < M::NB; ++b) vv[n & 1][b] = *(const h8*)(vl + (32 * b + col) * M::V_PITCH + 32 * n + 16 * half);
                };
                auto weights = [&](int n) {
                    const float add = st.bias[n] - m_base;
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const f2 y = {__builtin_amdgcn_exp2f(fmaf(x[n / 2][8 * (n % 2) + e], by[n], add)),
                                      __builtin_amdgcn_exp2f(fmaf(x[n / 2][8 * (n % 2) + e + 1], by[n], add))};
                        sum += y[0];
                        sum += y[1];
                        const h2 hi = __builtin_convertvector(y, h2);
                        w[n & 1][0][e] = hi[0];
                        w[n & 1][0][e + 1] = hi[1];
                        if (M::FINE) {
                            const f2 left = {y[0] - (float)hi[0], y[1] - (float)hi[1]};
                            const h2 lo = __builtin_convertvector(left, h2);
                            w[n & 1][M::PARTS - 1][e] = lo[0];
                            w[n & 1][M::PARTS - 1][e + 1] = lo[1];
                        }
                    }
                    l = fmaf(sum, st.back[n], l);
                };
                if constexpr (!M::FINE) {
                    operands(0);
                    weights(0);
                }
                // the next run's operands and weights while this one's products are on the matrix unit
#pragma unroll
                for (int n = 0; n < RUNS; ++n) {
                    if (!M::FINE) __builtin_amdgcn_sched_barrier(0);
                    if (M::FINE) {
                        operands(n);
                        weights(n);
                    } else if (n + 1 < RUNS) {
                        operands(n + 1);
                        weights(n + 1);
                    }
#pragma unroll
                    for (int b = 0; b < M::NB; ++b)
#pragma unroll
                        for (int p = 0; p < M::PARTS; ++p) o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[n & 1][b], w[n & 1][p], o[b], 0, 0, 0);
                    if constexpr (!M::FINE)
                        if (n + 1 < RUNS) {
                            __builtin_amdgcn_sched_group_barrier(0x100, M::NB, 0);
#pragma unroll
                            for (int b = 0; b < M::NB; ++b) {
                                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                                __builtin_amdgcn_sched_group_barrier(0x402, 36 / M::NB, 0);
                            }
                        }
                }
                if (!M::FINE) __builtin_amdgcn_sched_barrier(0);
            }
            if (M::FINE) {
                store(t + 1);
                note(t + 1);
                if (wave == 2 && lane < RUNS) list(t + 3, next);
                next = after;
            }
            __syncthreads();
        }
        l += __shfl_xor(l, 32);
        // element e of o[b]: column 32 b + 8 (e / 4) + 4 half + e % 4
        constexpr int MINE = M::NB / M::TEAMS;
        float back = ref_of_sums * 0.0078125f;   // 2^-LIFT
        if (M::TEAMS == 2) {
            // The teams' sums meet: each gives the other half of its columns. (The last step's end was a barrier.)
            if (team == 1)
#pragma unroll
                for (int b = 0; b < MINE; ++b) {
                    const v16f x = o[b];
                    o[b] = o[MINE + b];
                    o[MINE + b] = x;
                }
            auto slot = [&](int of, int n) { return (f4*)(lds_of_all + of * M::TEAM_BYTES) + n * THREADS + tid; };
#pragma unroll
            for (int b = 0; b < MINE; ++b)
#pragma unroll
                for (int e = 0; e < 16; e += 4) *slot(team, 4 * b + e / 4) = f4{o[MINE + b][e], o[MINE + b][e + 1], o[MINE + b][e + 2], o[MINE + b][e + 3]};
            if (half == 0) meet[team][32 * wave + col] = make_float2(m, l);
            if (tid == 0) refs[team] = back;
            __syncthreads();
            const float2 ml = meet[1 - team][32 * wave + col];
            const float m_both = fmaxf(m, ml.x);
            const float mine = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_both), other = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m_both);
            l = l * mine + ml.y * other;   // (what has no maximum has sums of zero, or none that is a number)
            m = m_both;
            const float mine_o = mine * back, other_o = other * refs[1 - team];
            back = 1.f;
#pragma unroll
            for (int b = 0; b < MINE; ++b)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f4 x = *slot(1 - team, 4 * b + e / 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[b][e + j] = o[b][e + j] * mine_o + x[j] * other_o;
                }
        }
        if (!row_is) continue;
        const int column = team * 32 * MINE + 4 * half;
        if (parts == 1) {
            const float f = l == 0.f ? 0.f : back / l;
            T* out = (T*)a.out + tok * a.out_stride + (int64_t)head * D + column;
#pragma unroll
            for (int b = 0; b < MINE; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) out[32 * b + 8 * (e / 4) + e % 4] = from_f32<T>(o[b][e] * f);
        } else {
            const int64_t to = (a.part_row(seq, s, tok) * a.heads + head) * a.splits + part;
            float* out = a.part_o + to * D + column;
#pragma unroll
            for (int b = 0; b < MINE; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) out[32 * b + 8 * (e / 4) + e % 4] = o[b][e] * back;
            if (half == 0 && team == 0) a.part_ml[to] = make_float2(m, l);
        }
    }
}

template <typename T, int D>
static int launch(const Attend& a, int max_rows, hipStream_t s) {
    // Workgroups to row tiles: as many to every sequence as the longest is said to have, or, where that is more, the tiles of all as a list
    // (at most one each that is not full). One prompt of 700 beside eleven single rows in f32: 816 workgroups and 109 us, 6336 otherwise, of
    // which each that finds nothing to do still holds a CU's LDS a while, and 137 us.
    const int row_tiles = max_rows < 1 ? 1 : (max_rows - 1) / KV_MANY_ROWS + 1;
    const int64_t spread = (int64_t)a.seqs * row_tiles, all = ((int64_t)a.rows * a.group - 1) / KV_MANY_ROWS + 1 + a.seqs;
    const bool listed = all < spread;
    const int64_t blocks = (listed ? all : spread) * a.pool.heads * a.splits;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    constexpr int bytes = Many<T, D>::LDS;
    // a kernel gets 64 KB of LDS unless the runtime is told otherwise
    if (bytes > 60 * 1024 &&
        hipFuncSetAttribute((const void*)kv_attention_many_kernel<T, D>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
        (void)hipGetLastError();
        return LK_ERR_LAUNCH;
    }
    hipLaunchKernelGGL((kv_attention_many_kernel<T, D>), dim3((unsigned)blocks), dim3(Many<T, D>::TEAMS * THREADS), bytes, s, a, listed ? 1 << 25 : row_tiles, listed, lk_device().cus);
    return lk_launch_status();
}

template <typename T>
static int by_dim(const Attend& a, int head_dim, int max_rows, hipStream_t s) {
    return head_dim == 64 ? launch<T, 64>(a, max_rows, s) : head_dim == 128 ? launch<T, 128>(a, max_rows, s) : launch<T, 256>(a, max_rows, s);
}

}  // namespace

int kv_attention_many(const Attend& a, int type, int head_dim, int max_rows, hipStream_t s) {
    if (type == LK_TYPE_F32) return by_dim<float>(a, head_dim, max_rows, s);
    if (type == LK_TYPE_F16) return by_dim<__half>(a, head_dim, max_rows, s);
    return by_dim<__hip_bfloat16>(a, head_dim, max_rows, s);
}
