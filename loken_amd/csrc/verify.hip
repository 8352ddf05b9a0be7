// Drafted tokens against the target's distribution (lk_verify), and the token that follows those that are accepted.
//
// A row's distribution p is what sampling would draw from: weights of the words that top-k, top-p and min-p keep, as numbers of 2^-42, over their
// sum. Four launches:
//   pieces  each piece's largest word, and, of rows that no rule cuts, its sum of weights relative to that: one pass over these rows' words.
//   steps   sampling's histogram, of the other rows alone
//   kept    where the rules' last word is, as sampling finds it; of rows that nothing cuts the pieces' sums, put to the row's largest word. Then the
//           row's draft is looked at: accepted if u q < p.
//   judge   pieces of the row at which a sequence ends, which every workgroup finds itself. It sums what is left, max(p - q, 0) or p, round by round of
//           neighbouring words; the sequence's last workgroup finds the round in which the draw lies and goes through that again.
// Differences p - q are made in 64 bits and summed as integers of 2^-51, whose sums do not depend on an order.
//
// Bound by the passes over the logits, one of rows that nothing cuts, up to three of others, and by the issue of 30 instructions a weight. 158 rows of 151936
// bf16 words that nothing cuts: pieces 29 us (1.6 TB/s; the vector unit's), kept 8, judge 18; 320 rows of 128256 f32 words with every rule: 35 (4.7 TB/s, the copy
// rate), steps 39, kept 37, judge 27; five rows of 151936 with top-k: 32 in all, the chains of four launches. (Kernel trace.)

#include "sampling_core.h"

namespace {

struct Verify {
    Sampling s;
    Kept* kept;              // [rows]
    double* verdict;         // [rows]: p of the word that was drafted where it is accepted; -1: it is not
    const int32_t *drafted, *starts;
    int seqs, rows;
    const void* draft;
    int64_t draft_stride;
    const float *uniform, *draw;
    int32_t *tokens, *accepted;
    float* probs;
    double* sums;            // [rows][s.pieces]: weights of the pieces of rows that nothing cuts, relative to a piece's largest word
    uint32_t* tops;          // [rows][s.pieces][waves]: keys of the largest words, of rows of which a few are asked for
    int rounds, per_piece;   // rounds of a row as `judge` goes through it, and those of one of its workgroups
    uint64_t* left;          // [rows][rounds]: sums of the rounds, of a sequence's at its first row
    uint32_t* met;           // [rows]: pieces that have been summed
};

// Sum and maximum over the wave without the LDS crossbar, whose six exchanges in a row take longer than a round's weights.
template <int ctrl>
static __device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    return (uint64_t)(uint32_t)dpp_i32<ctrl>((int)(v >> 32)) << 32 | (uint32_t)dpp_i32<ctrl>((int)v);
}
static __device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
    v += dpp_u64<0xB1>(v);
    v += dpp_u64<0x4E>(v);
    v += dpp_u64<0x141>(v);
    v += dpp_u64<0x140>(v);
    uint64_t sum = 0;
#pragma unroll
    for (int l = 0; l < 64; l += 16)
        sum += (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, l);
    return sum;
}
static __device__ __forceinline__ double wave_sum_f64(double v) {
    auto step = [&](auto ctrl) { return __longlong_as_double((long long)dpp_u64<decltype(ctrl)::value>((uint64_t)__double_as_longlong(v))); };
    v += step(std::integral_constant<int, 0xB1>{});
    v += step(std::integral_constant<int, 0x4E>{});
    v += step(std::integral_constant<int, 0x141>{});
    v += step(std::integral_constant<int, 0x140>{});
    double sum = 0.0;
#pragma unroll
    for (int l = 0; l < 64; l += 16) {
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        sum += __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)b, l)));
    }
    return sum;
}
static __device__ __forceinline__ float wave_max(float v) {   // (of no numbers: -infinity)
    v = group_max32(v);
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 2^x for any x <= 0 (and 0 for what is no number), to 2e-13 of it; nothing is left of it below 2^-900.
static __device__ __forceinline__ double power_of_any(double below, double rate) {
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double x = fmax(below * rate, -900.0), y = x + magic;
    return power_at(x - (y - magic), (int)(uint32_t)__double_as_longlong(y));
}

// Whether a row is sampled from all of its words.
static __device__ __forceinline__ bool uncut(const Sampling& a, int row) {
    const int k = a.top_k ? a.top_k[row] : 0;
    return a.temperature[row] > 0.0f && !(k > 0 && k < a.vocab) && !(a.top_p && a.top_p[row] < 1.0f) && !(a.min_p && a.min_p[row] > 0.0f);
}

// Whether a row's top-k words are few beside the waves of the pieces: then those are found by the waves' largest words, without a histogram.
static __device__ __forceinline__ bool bounded(const Sampling& a, int row) {
    const int k = a.top_k ? a.top_k[row] : 0, tops = a.pieces * SAMPLE_WAVES;
    return a.temperature[row] > 0.0f && k > 0 && k < a.vocab && k <= tops / 2 && tops <= MOST_TOPS;
}

// WORDS a thread.
template <int WORDS, typename T>
__global__ __launch_bounds__(SAMPLE_WG) void verify_pieces_kernel(Verify v) {
    constexpr int VEC = 16 / sizeof(T), RUNS = WORDS / VEC;
    struct __attribute__((aligned(sizeof(T)))) Run { T v[VEC]; };
    __shared__ float most[SAMPLE_WAVES], least[SAMPLE_WAVES];
    __shared__ double sums[SAMPLE_WAVES];
    __shared__ int first;
    const Sampling& a = v.s;
    const int row = blockIdx.y, c = blockIdx.x, t = threadIdx.x, wave = t >> 6;
    const T* words = (const T*)a.logits + row * a.stride;
    const int begin = c * SAMPLE_WG * WORDS + t * VEC, end = min((c + 1) * SAMPLE_WG * WORDS, a.vocab);
    float x[WORDS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        const int i = begin + j * SAMPLE_WG * VEC;
        if (i + VEC <= end) {
            const Run r = *(const Run*)(words + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[j * VEC + e] = to_f32(r.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[j * VEC + e] = i + e < end ? to_f32(words[i + e]) : -INFINITY;
        }
    }
    if (t == 0 && c == 0) {
        a.floor_mass[row] = 0;
        a.arrived[row] = 0;
        v.met[row] = 0;
        v.tokens[row] = -1;
        if (v.probs) v.probs[row] = 0.0f;
    }
    const bool weigh = uncut(a, row), few = bounded(a, row);
    if (!weigh && !few)
        for (int i = c * SAMPLE_WG + t; i < BINS; i += a.pieces * SAMPLE_WG) {
            a.mass[(int64_t)row * BINS + i] = 0;
            a.count[(int64_t)row * BINS + i] = 0;
        }
    float top = -INFINITY, bottom = -INFINITY;   // (bottom: of what is turned round)
#pragma unroll
    for (int j = 0; j < WORDS; ++j) top = fmaxf(top, x[j]);   // (fmaxf passes over what is not a number)
    if (!weigh) {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) bottom = fmaxf(bottom, x[j] > -INFINITY ? -x[j] : -INFINITY);
        bottom = wave_max(bottom);
    }
    top = wave_max(top);
    if ((t & 63) == 0) {
        most[wave] = top;
        least[wave] = bottom;
        if (few) v.tops[((int64_t)row * a.pieces + c) * SAMPLE_WAVES + wave] = top > -INFINITY ? key_of(top) : 0;
    }
    if (t == 0) first = 0x7FFFFFFF;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SAMPLE_WAVES; ++w) {
        top = fmaxf(top, most[w]);
        bottom = fmaxf(bottom, least[w]);
    }
    if (most[wave] == top && top > -INFINITY) {   // the first of the largest words
        int at = WORDS;
#pragma unroll
        for (int j = WORDS - 1; j >= 0; --j) at = x[j] == top ? j : at;
        if (at < WORDS) atomicMin(&first, begin + at / VEC * (SAMPLE_WG * VEC) + at % VEC);
    }
    // Weights relative to the piece's largest word, summed in an order that is always the same.
    double sum = 0.0;
    Scale sc;
    if (weigh && sc.init(Peak{(uint64_t)key_of(top) << 32 | 1, key_of(0.0f), 0}, top > -INFINITY ? a.temperature[row] : 0.0f, 0.0f)) {
#pragma unroll 8
        for (int j = 0; j < WORDS; ++j) sum += sc.infinite ? (x[j] == INFINITY ? 1.0 : 0.0) : power_of_any((double)x[j] - (double)top, sc.rate);
        sum = wave_sum_f64(sum);
    }
    if ((t & 63) == 0) sums[wave] = sum;
    __syncthreads();
    if (t == 0) {
        sum = 0.0;
        for (int w = 0; w < SAMPLE_WAVES; ++w) sum += sums[w];
        if (weigh) v.sums[(int64_t)row * a.pieces + c] = sum;
        a.peaks[(int64_t)row * a.pieces + c] = Peak{top > -INFINITY ? (uint64_t)key_of(top) << 32 | (uint32_t)~first : 0, key_of(-bottom), 0};
    }
}

template <typename T>
__global__ __launch_bounds__(SAMPLE_WG, 4) void verify_steps_kernel(Sampling a) {
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    if (!uncut(a, blockIdx.y) && !bounded(a, blockIdx.y)) steps_of_row<T>(a, mass, count);
}

// A row's distribution.
struct Target {
    Scale sc;
    Kept kept;
    double by;      // 2^42 / kept weight
    bool floored;   // whether min-p is asked for
    bool plain;     // whether every word is in it, and the largest is a number
    __device__ __forceinline__ void init(const Sampling& a, const Kept& k, int row) {
        kept = k;
        const Peak peak{k.best, key_of(0.0f), 0};
        const float least = a.min_p ? a.min_p[row] : 0.0f;
        sc.init(peak, kept.kept ? a.temperature[row] : 1.0f, least);
        by = kept.kept ? 4398046511104.0 / (double)kept.kept : 1.0;
        floored = least > 0.0f;
        plain = kept.kept != 0 && kept.last == 0 && !floored && !sc.infinite;
    }
    __device__ __forceinline__ bool in(float v, int i) const {
        const uint64_t at = (uint64_t)key_of(v) << 32 | (uint32_t)~i;
        if (at == kept.best && kept.best != 0) return true;   // (also where min-p, of more than 1, keeps nothing)
        return kept.kept != 0 && sc.live(sc.below(v)) && at >= kept.last && !(floored && !sc.kept(sc.power(v)));
    }
    // p of a word that is in it. (Its weight as a number of 2^-42: 1024 more and less.)
    __device__ __forceinline__ double share(float v) const { return kept.kept == 0 ? 1.0 : ((power_of(sc.from_top(v), sc.rate) + 1024.0) - 1024.0) * by; }
};

// A row's distribution, and the word that was drafted behind it: how far it is accepted.
template <typename T, typename Q>
__global__ __launch_bounds__(SAMPLE_WG, 4) void verify_kept_kernel(Verify v) {
    __shared__ Shared sh;
    const int row = blockIdx.y;
    const Sampling& a = v.s;
    const bool whole = uncut(a, row);
    if (whole && (blockIdx.x || threadIdx.x >= 64)) return;
    const int word = v.drafted[row];
    const bool is_word = word >= 0 && word < a.vocab;
    const float x = is_word ? to_f32(((const T*)a.logits)[row * a.stride + word]) : -INFINITY;
    const double reach = v.draft ? (is_word ? (double)v.uniform[row] * (double)to_f32(((const Q*)v.draft)[row * v.draft_stride + word]) : 0.0) : (double)v.uniform[row];
    auto done = [&](const Kept& k) {
        v.kept[row] = k;
        Target target;
        target.init(a, k, row);
        const double p = is_word && target.in(x, word) ? target.share(x) : 0.0;
        v.verdict[row] = reach < p ? p : -1.0;
    };
    if (!whole) {
        const int tops = a.pieces * SAMPLE_WAVES;
        choose<true, T>(a, sh, done, bounded(a, row) ? v.tops + (int64_t)row * tops : nullptr, tops);
        return;
    }
    const Peak peak = peak_of_row(a, row);
    Scale sc;
    double sum = 0.0;
    if (sc.init(peak, a.temperature[row], 0.0f)) {
        for (int i = threadIdx.x; i < a.pieces; i += 64) {   // each lane's in the same order always
            const uint64_t of_piece = a.peaks[(int64_t)row * a.pieces + i].best;
            const float top = value_of((uint32_t)(of_piece >> 32));
            if (of_piece && sc.live(sc.below(top))) sum += v.sums[(int64_t)row * a.pieces + i] * power_of(sc.from_top(top), sc.rate);
        }
    }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x == 0) done(Kept{peak.best, 0, (uint64_t)(sum * 4398046511104.0 + 0.5)});
}

// What is left of a row's words: p, less the draft's share or without the word that was drafted for certain.
template <typename T, typename Q>
struct Left {
    static constexpr int VEC = 16 / sizeof(T), ROUND = SAMPLE_WG * VEC;
    struct __attribute__((aligned(sizeof(T)))) Words { T v[VEC]; };
    struct __attribute__((aligned(sizeof(Q)))) Shares { Q v[VEC]; };
    const T* row;
    const Q* draft;    // null: nothing is taken off
    int certain;       // -1: no word
    int vocab;
    struct Read { float x[VEC], q[VEC]; };
    // The thread's words of a round.
    __device__ __forceinline__ Read read(int round) const {
        const int i = round * ROUND + (int)threadIdx.x * VEC;
        Read r;
        float (&x)[VEC] = r.x, (&q)[VEC] = r.q;
        if (i + VEC <= vocab) {
            const Words w = *(const Words*)(row + i);
            Shares s;
            if (draft) s = *(const Shares*)(draft + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[e] = to_f32(w.v[e]);
                q[e] = draft ? to_f32(s.v[e]) : 0.0f;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[e] = i + e < vocab ? to_f32(row[i + e]) : -INFINITY;
                q[e] = draft && i + e < vocab ? to_f32(draft[i + e]) : 0.0f;
            }
        }
        return r;
    }
    // What is left of them, as integers of 2^-51.
    __device__ __forceinline__ void of_round(const Target& target, int round, const Read& r, uint64_t (&left)[VEC]) const {
        const int i = round * ROUND + (int)threadIdx.x * VEC;
        const float (&x)[VEC] = r.x, (&q)[VEC] = r.q;
        // (from 2^52 on a number's last place is one)
        auto whole = [](double p) { return (uint64_t)__double_as_longlong(fma(fmax(p, 0.0), 2251799813685248.0, 4503599627370496.0)) - 0x4330000000000000ull; };
        if (target.plain) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float v = target.sc.live(target.sc.top - x[e]) ? x[e] : -INFINITY;   // (else its weight is none)
                left[e] = whole(fma(power_of_any((double)v - (double)target.sc.top, target.sc.rate), target.by, -(double)q[e]));
            }
        } else {
            bool in[VEC], any = false;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                left[e] = 0;
                in[e] = target.in(x[e], i + e);
                any = any || in[e];
            }
            if (!__ballot(any)) return;
#pragma unroll
            for (int e = 0; e < VEC; ++e) left[e] = in[e] ? whole(target.share(x[e]) - (double)q[e]) : 0;
        }
        if (certain >= i && certain < i + VEC)
#pragma unroll
            for (int e = 0; e < VEC; ++e) left[e] = i + e == certain ? 0 : left[e];
    }
};

template <typename T, typename Q>
__global__ __launch_bounds__(SAMPLE_WG) void verify_judge_kernel(Verify v) {
    using L = Left<T, Q>;
    __shared__ uint64_t meet[SAMPLE_WAVES][2];
    __shared__ uint64_t sums[SAMPLE_WG], wanted;
    __shared__ int found, round_found;
    const Sampling& a = v.s;
    const int seq = blockIdx.y, c = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int first = min(max(v.starts[seq], 0), v.rows), end = min(max(v.starts[seq + 1], 0), v.rows), drafts = end - first - 1;
    if (drafts < 0) {
        if (c == 0 && t == 0) v.accepted[seq] = 0;
        return;
    }
    // The drafts that are accepted: a lane each, each wave for itself.
    int accepted = drafts;
    for (int j0 = 0; j0 < drafts && accepted == drafts; j0 += 64) {
        const uint64_t refused = __ballot(j0 + lane < drafts && v.verdict[first + min(j0 + lane, drafts)] < 0.0);
        if (refused) accepted = j0 + __ffsll((unsigned long long)refused) - 1;
    }
    const int row = first + accepted;
    const bool some = accepted < drafts;
    Target target;
    target.init(a, v.kept[row], row);
    L words{(const T*)a.logits + row * a.stride, some && v.draft ? (const Q*)v.draft + row * v.draft_stride : nullptr, some && !v.draft ? v.drafted[row] : -1, a.vocab};
    // The sums of rounds r0 .. r1 - 1, at `to`; the workgroup's rounds go through LDS.
    auto sum_rounds = [&](int r0, int r1, uint64_t* to) {
        sums[t] = 0;
        __syncthreads();
        auto next = words.read(r0);
        for (int r = r0; r < r1; ++r) {
            const auto now = next;
            next = words.read(r + 1 < r1 ? r + 1 : r0);   // (always: what is loaded at times is waited for each time)
            uint64_t left[L::VEC], mine = 0;
            words.of_round(target, r, now, left);
            for (uint64_t l : left) mine += l;
            mine = wave_sum_u64(mine);
            if (lane == 0 && mine) atomicAdd((unsigned long long*)&sums[r - r0], (unsigned long long)mine);
        }
        __syncthreads();
        for (int r = r0 + t; r < r1; r += SAMPLE_WG) __hip_atomic_store(&to[r], sums[r - r0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    uint64_t* left = v.left + (int64_t)first * v.rounds;
    sum_rounds(c * v.per_piece, min((c + 1) * v.per_piece, v.rounds), left);
    // as in sampling: once each wave's stores have gone where every XCD reads, the workgroup is counted, and the last one goes on
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) found = atomicAdd(&v.met[first], 1u) == gridDim.x - 1;
    __syncthreads();
    if (!found) return;

    // The round in which the draw lies: a round a thread.
    auto find_round = [&]() {
        const uint64_t mine = t < v.rounds ? __hip_atomic_load(&left[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        const uint64_t before = sum_before(mine, meet, 0);
        uint64_t total = 0;
        for (int w = 0; w < SAMPLE_WAVES; ++w) total += meet[w][0];
        const uint64_t target_sum = drawn_sum(v.draw[seq], total);
        if (total && before < target_sum && before + mine >= target_sum) {   // one thread's
            round_found = t;
            wanted = target_sum - before;
        }
        return total;
    };
    if (t == 0) {
        found = -1;
        round_found = 0;   // (shares of a draft that are far below 0 leave sums that wrap, and may leave no round)
    }
    uint64_t total = find_round();
    if (total == 0 && target.kept.best != 0) {   // nothing is left: p as it is, all of it by this workgroup
        words.draft = nullptr;
        words.certain = -1;
        __syncthreads();
        sum_rounds(0, v.rounds, left);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        total = find_round();
    }
    __syncthreads();
    if (total) {
        uint64_t of_words[L::VEC], held = 0;
        words.of_round(target, round_found, words.read(round_found), of_words);
        for (uint64_t l : of_words) held += l;
        uint64_t at = sum_before(held, meet, 1);
        if (at < wanted && at + held >= wanted) {   // one thread's
            int e = 0;
            for (uint64_t l : of_words) {
                at += l;
                if (at >= wanted) break;
                ++e;
            }
            found = round_found * L::ROUND + t * L::VEC + e;
        }
    }
    __syncthreads();
    const int token = found;
    for (int j = t; j <= accepted; j += SAMPLE_WG) {
        const bool last = j == accepted;
        if (last && token < 0) break;   // a row without words
        v.tokens[first + j] = last ? token : v.drafted[first + j];
        if (v.probs) v.probs[first + j] = (float)(last ? target.share(to_f32(words.row[token])) : v.verdict[first + j]);
    }
    if (t == 0) v.accepted[seq] = accepted;
}

template <typename T, typename Q>
static void launch(const Verify& v, bool wide, hipStream_t s) {
    const dim3 of_pieces(v.s.pieces, v.rows), of_rows(v.s.chunks, v.rows), of_seqs((v.rounds + v.per_piece - 1) / v.per_piece, v.seqs), threads(SAMPLE_WG);
    if (wide) hipLaunchKernelGGL((verify_pieces_kernel<16, T>), of_pieces, threads, 0, s, v);
    else hipLaunchKernelGGL((verify_pieces_kernel<8, T>), of_pieces, threads, 0, s, v);
    if (v.s.top_k || v.s.top_p || v.s.min_p) hipLaunchKernelGGL((verify_steps_kernel<T>), of_rows, threads, 0, s, v.s);
    hipLaunchKernelGGL((verify_kept_kernel<T, Q>), of_rows, threads, 0, s, v);
    hipLaunchKernelGGL((verify_judge_kernel<T, Q>), of_seqs, threads, 0, s, v);
}
template <typename T>
static void launch_draft(const Verify& v, bool wide, int draft_type, hipStream_t s) {
    if (draft_type == LK_TYPE_F16) launch<T, __half>(v, wide, s);
    else if (draft_type == LK_TYPE_BF16) launch<T, __hip_bfloat16>(v, wide, s);
    else launch<T, float>(v, wide, s);
}

}  // namespace

extern "C" int lk_verify(const void* logits, int type, int64_t stride, int rows, int vocab, const int32_t* drafted, const int32_t* starts, int seqs,
                         const void* draft, int draft_type, int64_t draft_stride, const float* uniform, const float* draw,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
                         int32_t* accepted, float* probs, void* stream) {
    const auto size_of = [](int t) { return t == LK_TYPE_F32 ? 4 : t == LK_TYPE_F16 || t == LK_TYPE_BF16 ? 2 : 0; };
    const int size = size_of(type), draft_size = draft ? size_of(draft_type) : 4;
    if (!size || !draft_size) return LK_ERR_TYPE;
    if (rows < 0 || rows > 65535 || seqs < 0 || seqs > 65535 || vocab <= 0 || stride < vocab || (draft && draft_stride < vocab)) return LK_ERR_ARG;
    if (vocab > LK_SAMPLE_VOCAB) return LK_ERR_SIZE;
    if (rows == 0 || seqs == 0) return LK_OK;
    if (!logits || !drafted || !starts || !uniform || !draw || !temperature || !tokens || !accepted || ((uintptr_t)logits & (size - 1)) ||
        ((uintptr_t)draft & (draft_size - 1)))
        return LK_ERR_ARG;
    Verify v{};
    v.s = Sampling{logits, stride, vocab, 0, 0, 0, nullptr, temperature, top_p, min_p, top_k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
    cut_rows(v.s, rows, size);
    // pieces of the first pass: 16 words a thread (half as many sums and largest words to bring together), 8 where that leaves CUs without two workgroups:
    // 320 bf16 rows of 151936 words 82 us (93 with 8), 40 rows 27.6 (29.1), 5 rows 24.1 (22.9), calls
    const int cus = lk_device().cus, most = SAMPLE_WG * 16;
    const bool wide = (int64_t)rows * ((vocab + most - 1) / most) >= 2 * cus;
    const int words = wide ? most : most / 2;
    v.s.pieces = (vocab + words - 1) / words;
    // rounds of the last one, as many to a workgroup as leave four workgroups to a CU
    const int round = SAMPLE_WG * 16 / size, of_seq = (4 * cus + seqs - 1) / seqs;
    v.rounds = (vocab + round - 1) / round;
    v.per_piece = (v.rounds + of_seq - 1) / of_seq;
    const size_t judged = sizeof(Kept) + 8 + (size_t)(v.s.pieces * (1 + SAMPLE_WAVES / 2) + v.rounds) * 8;
    LkScratch scratch((hipStream_t)stream);
    uint8_t* mem = (uint8_t*)scratch.get(LK_SCRATCH_SAMPLE, (size_t)rows * (judged + bytes_of_row(v.s) + 4));
    if (!mem) return LK_ERR_NOMEM;
    v.kept = (Kept*)mem;
    v.verdict = (double*)(v.kept + rows);
    v.sums = v.verdict + rows;
    v.left = (uint64_t*)(v.sums + (size_t)rows * v.s.pieces);
    v.tops = (uint32_t*)(v.left + (size_t)rows * v.rounds);
    place_rows(v.s, rows, mem + (size_t)rows * judged);
    v.met = v.s.arrived + rows;
    v.drafted = drafted;
    v.starts = starts;
    v.seqs = seqs;
    v.rows = rows;
    v.draft = draft;
    v.draft_stride = draft_stride;
    v.uniform = uniform;
    v.draw = draw;
    v.tokens = tokens;
    v.accepted = accepted;
    v.probs = probs;
    if (type == LK_TYPE_F32) launch_draft<float>(v, wide, draft_type, (hipStream_t)stream);
    else if (type == LK_TYPE_F16) launch_draft<__half>(v, wide, draft_type, (hipStream_t)stream);
    else launch_draft<__hip_bfloat16>(v, wide, draft_type, (hipStream_t)stream);
    return lk_launch_status();
}
