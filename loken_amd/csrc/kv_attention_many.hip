// Attention over the 8-bit cache for many rows of a sequence: prompts and prefill chunks.
//
// Rows are (token, head of the group) of one key / value head, so that the group's heads share the keys and values that are
// read. A workgroup of four waves has 128 rows; a step is 64 positions, whose codes are turned into f16 (exactly) once for all
// rows on their way into LDS, values with the positions of a column together as they lie in the cache. Products are
// v_mfma_f32_32x32x16_f16, both turned round so that a lane keeps one row throughout:
//     scores   (32 positions) x (32 rows): lane l holds row l % 32, and the positions of its half of the lanes stand in the order in
//              which the next product wants them (the rows of the first operand are read from LDS in that order)
//     sums     (32 columns) x (32 rows): the weights go from the scores' registers straight into the operand
// so the running maximum, its corrections and the sum of weights are the lane's own, with one exchange between the two halves.
//
// Queries come in f16 scaled by a power of two of their row (bf16 fits with its 8 bits, f16 as it is); f32 ones as a high and a
// low half, two products each, as are its weights: 22 bits. A page's key scale goes onto the scores. Its value scale goes onto the
// weights, relative to the largest value scale so far, so that no scale is too small for f16: as its logarithm, in the exponent that
// the weight is made from (off by 5e-7 of the weight at most, a last place of the logarithm), and back out of the sum of
// weights run by run.
//
// The sums are put to a new maximum only where that lies 2^8 above the one they go by: weights up to 2^8 then, which stand
// LIFT = 2^7 above one and stay below 2^15, f16's largest; a weight of 2^-21 still has all its bits, one of 2^-31 some.

#include "kv_attention.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr int WAVES = 4, THREADS = 64 * WAVES, RUNS = KV_TILE / 16;
constexpr float LIFT = 7.f, SLACK = 8.f;   // powers of two

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

template <typename T, int D>
struct Many {
    static constexpr bool FINE = sizeof(T) == 4;
    static constexpr int PARTS = FINE ? 2 : 1;
    static constexpr int KS = D / 16, NB = D / 32;
    static constexpr int K_PITCH = 2 * D + 16, V_PITCH = 2 * KV_TILE + 16;   // bytes; sixteen more: no bank conflicts
    static constexpr int K_BYTES = KV_TILE * K_PITCH, V_BYTES = D * V_PITCH;
    static constexpr int BUFFERS = D < 256 ? 2 : 1;
    static constexpr int CHUNKS = KV_TILE * D / 16 / THREADS;   // of sixteen codes, a thread and side
    static constexpr int LDS = BUFFERS * (K_BYTES + V_BYTES);
};

// What a step's pages have for everybody.
struct Step {
    float ks[RUNS];     // key scales; -1: the page is absent
    float bias[RUNS];   // log2 of the value scale over `ref`, and LIFT; of a page whose values are all zero LIFT alone
    float back[RUNS];   // 2^-bias
    uint32_t live[RUNS];   // all bits, or none where the values are zero
    float shrink;       // what `ref` before this step is of it now
    float ref;          // the largest value scale so far
    int absent;         // whether a page is
    int pad;
};

template <typename T, int D>
__global__ __launch_bounds__(THREADS, D < 256 ? 2 : 1) void kv_attention_many_kernel(Attend a, int row_tiles, int cus) {
    using M = Many<T, D>;
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ Step steps[2];
    __shared__ int pages[2][RUNS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    // Workgroups in rounds of one to a CU, every other round backwards: row tiles that see the most come first, and where two rounds are
    // all there is a CU with much of one has little of the other.
    unsigned at = blockIdx.x;
    {
        const unsigned round = at / cus, first = round * cus, size = min((unsigned)cus, gridDim.x - first);
        if (round & 1) at = first + (size - 1 - (at - first));
    }
    const int part = at % a.splits;
    at /= a.splits;
    const int kv = at % a.pool.heads;
    at /= a.pool.heads;
    const int seq = at % a.seqs, tile0 = row_tiles - 1 - (int)(at / a.seqs);
    const KvSeq s(a, seq);
    const int64_t all_rows = (int64_t)s.tokens() * a.group;
    if (all_rows <= a.few_rows) return;
    const int shift = a.pool.page_shift;
    const int32_t* entries = a.table + seq * a.table_stride;
    auto k_lds = [&](int buffer) { return lds + buffer * (M::K_BYTES + M::V_BYTES); };
    auto v_lds = [&](int buffer) { return lds + buffer * (M::K_BYTES + M::V_BYTES) + M::K_BYTES; };

    for (int64_t r_tile = (int64_t)tile0 * KV_MANY_ROWS; r_tile < all_rows; r_tile += (int64_t)row_tiles * KV_MANY_ROWS) {
        const int64_t r_end = min(r_tile + KV_MANY_ROWS, all_rows);
        const KvSpan span(a, s, s.first + (int)(r_tile / a.group), s.first + (int)((r_end - 1) / a.group));
        const int per_part = span.per_part, parts = span.parts;
        if (part >= parts) continue;
        const int t_begin = part * per_part, t_end = min(span.tiles, t_begin + per_part);
        // the lane's row, and what its wave sees
        const int64_t r = r_tile + 32 * wave + col;
        const bool row_is = r < r_end;
        const int64_t r_in = min(r, r_end - 1);
        const int tok = s.first + (int)(r_in / a.group), head = kv * a.group + (int)(r_in % a.group);
        const int pos = (int)max(s.pos_of_0 + tok, (int64_t)-1);
        const int64_t w0 = min(r_tile + 32 * wave, r_end - 1), w1 = min(r_tile + 32 * wave + 31, r_end - 1);
        const int pos_least = (int)max(s.pos_of_0 + s.first + w0 / a.group, (int64_t)-1), pos_most = (int)max(s.pos_of_0 + s.first + w1 / a.group, (int64_t)-1);

        h8 q[M::PARTS][M::KS];
        float unit;
        {
            const T* row = (const T*)a.q + tok * a.q_stride + (int64_t)head * D + 8 * half;
            uint32_t most = 0;
#pragma unroll
            for (int k = 0; k < M::KS; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(to_f32(row[16 * k + e])) & 0x7FFFFFFFu);
            most = max(most, (uint32_t)__shfl_xor((int)most, 32));
            const bool finite = most < 0x7F800000u;
            int e2 = 0;
            (void)frexpf(finite && most ? __uint_as_float(most) : 1.f, &e2);   // the row's largest is in [2^(e2 - 1), 2^e2)
#pragma unroll
            for (int k = 0; k < M::KS; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = finite ? ldexpf(to_f32(row[16 * k + e]), 14 - e2) : 0.f;   // below 2^14
                    const _Float16 hi = (_Float16)x;
                    q[0][k][e] = hi;
                    if (M::FINE) q[M::PARTS - 1][k][e] = (_Float16)(x - (float)hi);
                }
            // the scale first: powers that it makes up for may be far from one
            unit = finite ? ldexpf(ldexpf(a.scale * 1.4426950408889634f, e2 / 2), e2 - e2 / 2 - 14) : NAN;
        }
        v16f o[M::NB];
#pragma unroll
        for (int b = 0; b < M::NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][e] = 0.f;
        float m = -INFINITY, l = 0.f;

        // A step's codes: thread tid has chunk tid, tid + 256, .. of sixteen. Its pages have been in LDS since the step before.
        uint4 kc[M::CHUNKS], vc[M::CHUNKS];
        auto entry = [&](int t) {   // of run tid, in the first lanes
            const int p0 = span.lo + t * KV_TILE + 16 * (tid & (RUNS - 1));
            const int page = t < t_end && p0 < span.hi ? entries[p0 >> shift] : -1;
            return (unsigned)page < (unsigned)a.pool.pages ? page : -1;
        };
        float ks = -1.f, vs = 0.f, ref = 0.f;
        auto fetch = [&](int t) {
            const int* page = pages[t & 1];
#pragma unroll
            for (int c = 0; c < M::CHUNKS; ++c) {
                const int n = tid + c * THREADS;
                const int token = n / (D / 16), run_v = n / D;
                const int off_k = (span.lo + t * KV_TILE + token) & ((1 << shift) - 1);
                kc[c] = *(const uint4*)(a.pool.k + ((((int64_t)max(page[token >> 4], 0) * a.pool.heads + kv) << shift) + off_k) * D + (n % (D / 16)) * 16);
                const int off_v = (span.lo + t * KV_TILE + 16 * run_v) & ((1 << shift) - 1);
                vc[c] = *(const uint4*)(a.pool.v + ((((int64_t)max(page[run_v], 0) * a.pool.heads + kv) << shift) + off_v) * D + (n % D) * 16);
            }
            if (tid < RUNS) {
                const int p = page[tid];
                const int64_t at_scale = (int64_t)max(p, 0) * a.pool.heads + kv;
                ks = a.pool.k_scales[at_scale];
                vs = a.pool.v_scales[at_scale];
                if (p < 0) { ks = -1.f; vs = 0.f; }
            }
        };
        auto store = [&](int t) {
            const int buffer = M::BUFFERS == 2 ? t & 1 : 0;
#pragma unroll
            for (int c = 0; c < M::CHUNKS; ++c) {
                const int n = tid + c * THREADS;
                uint4 w[2];
                to_halves(kc[c], w);
                uint4* to = (uint4*)(k_lds(buffer) + (n / (D / 16)) * M::K_PITCH + (n % (D / 16)) * 32);
                to[0] = w[0];
                to[1] = w[1];
                to_halves(vc[c], w);
                to = (uint4*)(v_lds(buffer) + (n % D) * M::V_PITCH + (n / D) * 32);
                to[0] = w[0];
                to[1] = w[1];
            }
            if (tid < RUNS) {
                Step& st = steps[t & 1];
                float most = vs, least = ks;
                for (int o = 1; o < RUNS; o <<= 1) { most = fmaxf(most, __shfl_xor(most, o)); least = fminf(least, __shfl_xor(least, o)); }
                const float now = fmaxf(ref, most);
                st.ks[tid] = ks;
                const float bias = vs > 0.f ? __builtin_amdgcn_logf(vs / now) + LIFT : LIFT;
                st.bias[tid] = bias;
                st.back[tid] = __builtin_amdgcn_exp2f(-bias);
                st.live[tid] = vs > 0.f ? 0xFFFFFFFFu : 0u;
                if (tid == 0) {
                    st.shrink = ref > 0.f ? ref / now : 1.f;   // (up to then the sums are zeros)
                    st.ref = now;
                    st.absent = least < 0.f;
                }
                ref = now;
            }
        };

        __syncthreads();   // the last row tile's reads of LDS
        int next = -1;
        if (tid < RUNS) {
            pages[t_begin & 1][tid] = entry(t_begin);
            next = entry(t_begin + 1);
        }
        __syncthreads();
        if (t_begin < t_end) {
            fetch(t_begin);
            store(t_begin);
        }
        if (tid < RUNS) pages[(t_begin + 1) & 1][tid] = next;
        __syncthreads();
        float ref_of_sums = 0.f;
        for (int t = t_begin; t < t_end; ++t) {
            const int buffer = M::BUFFERS == 2 ? t & 1 : 0;
            if (t + 1 < t_end) fetch(t + 1);
            if (tid < RUNS) next = entry(t + 2);
            const int base = span.lo + t * KV_TILE;
            const Step& st = steps[t & 1];
            ref_of_sums = st.ref;
            if (st.shrink < 1.f) {
                const float f = st.shrink;
#pragma unroll
                for (int b = 0; b < M::NB; ++b) o[b] *= f;
            }
            // a wave whose rows see nothing of the step leaves it
            if (base <= pos_most && (a.window == 0 || base + KV_TILE - 1 > pos_least - a.window)) {
                const uint8_t *kl = k_lds(buffer), *vl = v_lds(buffer);
                v16f x[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    // row i = 8 b + 4 h + j of the operand is position 16 (b / 2) + 8 h + 4 (b % 2) + j
                    const int from = 32 * u + 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
                    const uint8_t* kr = kl + from * M::K_PITCH + 16 * half;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[u][e] = 0.f;
#pragma unroll
                    for (int k = 0; k < M::KS; ++k) {
                        const h8 kk = *(const h8*)(kr + 32 * k);
#pragma unroll
                        for (int p = 0; p < M::PARTS; ++p) x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk, q[p][k], x[u], 0, 0, 0);
                    }
                }
                // scores in powers of two; element e of x[u]: position base + 32 u + 16 (e / 8) + 8 half + e % 8
                const bool whole = base + KV_TILE - 1 <= pos_least && (a.window == 0 || base > pos_most - a.window) && !st.absent;
                float by[RUNS], top = -INFINITY;
#pragma unroll
                for (int n = 0; n < RUNS; ++n) by[n] = st.ks[n] * unit;
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
                    float part_top = x[n / 2][8 * (n % 2)];
#pragma unroll
                    for (int e = 1; e < 8; ++e) part_top = fmaxf(part_top, x[n / 2][8 * (n % 2) + e]);
                    top = fmaxf(top, part_top * by[n]);
                }
                {
                    const auto r2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(r2[0]), __uint_as_float(r2[1]));
                }
                if (__ballot(top > m + SLACK || (m == -INFINITY && top > m)) != 0) {
                    const float m_new = fmaxf(m, top);
                    const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                    l *= keep;
#pragma unroll
                    for (int b = 0; b < M::NB; ++b) o[b] *= keep;
                    m = m_new;
                }
                const float m_base = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int n = 0; n < RUNS; ++n) {
                    h8 w[M::PARTS];
                    const float add = st.bias[n] - m_base;
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const f2 y = {__builtin_amdgcn_exp2f(fmaf(x[n / 2][8 * (n % 2) + e], by[n], add)),
                                      __builtin_amdgcn_exp2f(fmaf(x[n / 2][8 * (n % 2) + e + 1], by[n], add))};
                        sum += y[0];
                        sum += y[1];
                        const h2 hi = __builtin_convertvector(y, h2);
                        w[0][e] = hi[0];
                        w[0][e + 1] = hi[1];
                        if (M::FINE) {
                            const f2 left = {y[0] - (float)hi[0], y[1] - (float)hi[1]};
                            const h2 lo = __builtin_convertvector(left, h2);
                            w[M::PARTS - 1][e] = lo[0];
                            w[M::PARTS - 1][e + 1] = lo[1];
                        }
                    }
                    l = fmaf(sum, st.back[n], l);
#pragma unroll
                    for (int p = 0; p < M::PARTS; ++p) {   // values of a page whose scale is zero: zeros, whatever its codes are
                        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
                        w[p] = __builtin_bit_cast(h8, __builtin_bit_cast(u4, w[p]) & st.live[n]);
                    }
#pragma unroll
                    for (int b = 0; b < M::NB; ++b) {
                        const h8 vv = *(const h8*)(vl + (32 * b + col) * M::V_PITCH + 32 * n + 16 * half);
#pragma unroll
                        for (int p = 0; p < M::PARTS; ++p) o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv, w[p], o[b], 0, 0, 0);
                    }
                }
            }
            if (M::BUFFERS == 1) __syncthreads();
            if (t + 1 < t_end) store(t + 1);
            if (tid < RUNS) pages[t & 1][tid] = next;   // of step t + 2; those of t have been read
            __syncthreads();
        }
        l += __shfl_xor(l, 32);
        const float back = ref_of_sums * 0.0078125f;   // 2^-LIFT
        if (!row_is) continue;
        // element e of o[b]: column 32 b + 8 (e / 4) + 4 half + e % 4
        if (parts == 1) {
            const float f = l == 0.f ? 0.f : back / l;
            T* out = (T*)a.out + tok * a.out_stride + (int64_t)head * D + 4 * half;
#pragma unroll
            for (int b = 0; b < M::NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) out[32 * b + 8 * (e / 4) + e % 4] = from_f32<T>(o[b][e] * f);
        } else {
            const int64_t to = (a.part_row(seq, s, tok) * a.heads + head) * a.splits + part;
            float* out = a.part_o + to * D + 4 * half;
#pragma unroll
            for (int b = 0; b < M::NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) out[32 * b + 8 * (e / 4) + e % 4] = o[b][e] * back;
            if (half == 0) a.part_ml[to] = make_float2(m, l);
        }
    }
}

template <typename T, int D>
static int launch(const Attend& a, int max_rows, hipStream_t s) {
    const int row_tiles = max_rows < 1 ? 1 : (max_rows - 1) / KV_MANY_ROWS + 1;
    const int64_t blocks = (int64_t)a.seqs * a.pool.heads * row_tiles * a.splits;
    if (blocks > 0x7FFFFFFF) return LK_ERR_SIZE;
    constexpr int bytes = Many<T, D>::LDS;
    // a kernel gets 64 KB of LDS unless the runtime is told otherwise
    if (bytes > 60 * 1024 &&
        hipFuncSetAttribute((const void*)kv_attention_many_kernel<T, D>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
        (void)hipGetLastError();
        return LK_ERR_LAUNCH;
    }
    hipLaunchKernelGGL((kv_attention_many_kernel<T, D>), dim3((unsigned)blocks), dim3(THREADS), bytes, s, a, row_tiles, lk_device().cus);
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
