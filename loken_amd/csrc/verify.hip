// Drafted tokens against the target's distribution (lk_verify), and the token that follows those that are accepted.
//
// A row's distribution p is what sampling would draw from: weights as integers of 2^-42 of the words that top-k, top-p and min-p keep, over their
// sum. So the launches are sampling's (peak, steps, and its choice cut short where the kept words' last is known), and one more:
//   judge   pieces of the row at which a sequence ends. Every workgroup finds that row itself: drafts a lane each, accepted while u q < p. The pieces' sums
//           of what is left, max(p - q, 0) or p, meet; the sequence's last workgroup finds the piece in which the draw lies and goes through it again.
// Differences p - q are made in 64 bits and summed as integers of 2^-62, whose sums do not depend on an order.
//
// Bound by the passes over the logits: three of all rows (two where nothing cuts), one and a piece of one row of each sequence, and as much of the draft's row.

#include "sampling_core.h"

namespace {

constexpr double LEFT_ONE = 4611686018427387904.0;   // 2^62

struct Verify {
    Sampling s;
    const Kept* kept;        // [rows]
    const int32_t *drafted, *starts;
    int seqs, rows;
    const void* draft;
    int64_t draft_stride;
    const float *uniform, *draw;
    int32_t *tokens, *accepted;
    float* probs;
    uint64_t* left;          // [rows][chunks]: sums of the pieces, of a sequence's at its first row
    uint32_t* met;           // [rows]: pieces that have been summed
};

// A row's distribution.
struct Target {
    Scale sc;
    Kept kept;
    double by;   // 1 / kept weight
    __device__ __forceinline__ void init(const Sampling& a, const Kept& k, int row) {
        kept = k;
        const Peak peak{k.best, key_of(0.0f), 0};
        sc.init(peak, kept.kept ? a.temperature[row] : 1.0f, a.min_p ? a.min_p[row] : 0.0f);
        by = 1.0 / (double)kept.kept;
    }
    __device__ __forceinline__ double share(float v, int i) const {
        const uint64_t at = (uint64_t)key_of(v) << 32 | (uint32_t)~i;
        if (kept.kept == 0) return kept.best != 0 && at == kept.best ? 1.0 : 0.0;
        const bool in = sc.live(sc.below(v)) && at >= kept.last && sc.kept(sc.power(v));
        return in ? (double)sc.weight(v) * by : 0.0;
    }
};

// Where a row is asked for its distribution alone.
template <typename T>
__global__ __launch_bounds__(SAMPLE_WG, 4) void verify_kept_kernel(Verify v, Kept* kept) {
    __shared__ Shared sh;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const int row = blockIdx.y;
        v.met[row] = 0;
        v.tokens[row] = -1;
        if (v.probs) v.probs[row] = 0.0f;
    }
    choose<true, T>(v.s, sh, kept);
}

// What is left of a row's words: p, less the draft's share or without the word that was drafted for certain.
template <typename T, typename Q>
struct Left {
    const T* row;
    const Q* draft;    // null: nothing is taken off
    int certain;       // -1: no word
    // Rounds over neighbouring words begin .. end - 1, VEC of them a thread, that all threads come to; f(first word, what is left of the thread's
    // words) is false: the last round.
    template <class F>
    __device__ __forceinline__ void each_round(const Target& target, int begin, int end, F f) const {
        constexpr int VEC = 16 / sizeof(T);
        struct __attribute__((aligned(sizeof(T)))) Words { T v[VEC]; };
        struct __attribute__((aligned(sizeof(Q)))) Shares { Q v[VEC]; };
        for (int i0 = begin; i0 < end; i0 += SAMPLE_WG * VEC) {
            const int i = i0 + (int)threadIdx.x * VEC;
            float x[VEC], q[VEC];
            if (i + VEC <= end) {
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
                    x[e] = i + e < end ? to_f32(row[i + e]) : -INFINITY;
                    q[e] = draft && i + e < end ? to_f32(draft[i + e]) : 0.0f;
                }
            }
            uint64_t left[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const double p = target.share(x[e], i + e) - (double)q[e];
                left[e] = p > 0.0 && i + e != certain ? (uint64_t)fma(p, LEFT_ONE, 0.5) : 0;
            }
            if (!f(i, left)) return;
        }
    }
};

// Sum over the workgroup; meet[..][which] is free again past the barrier after next.
static __device__ __forceinline__ uint64_t sum_of_all(uint64_t mine, uint64_t (*meet)[2], int which) {
    for (int o = 32; o; o >>= 1) mine += __shfl_xor((unsigned long long)mine, o);
    if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6][which] = mine;
    __syncthreads();
    uint64_t all = 0;
    for (int w = 0; w < SAMPLE_WAVES; ++w) all += meet[w][which];
    return all;
}

template <typename T, typename Q>
__global__ __launch_bounds__(SAMPLE_WG) void verify_judge_kernel(Verify v) {
    __shared__ uint64_t meet[SAMPLE_WAVES][2];
    __shared__ int found;
    const Sampling& a = v.s;
    const int seq = blockIdx.y, c = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int first = min(max(v.starts[seq], 0), v.rows), end = min(max(v.starts[seq + 1], 0), v.rows), drafts = end - first - 1;
    if (drafts < 0) {
        if (c == 0 && t == 0) v.accepted[seq] = 0;
        return;
    }
    // p of the word that was drafted behind a row (0: no such word)
    auto share_of_draft = [&](int row) {
        const int word = v.drafted[row];
        if (word < 0 || word >= a.vocab) return 0.0;
        Target target;
        target.init(a, v.kept[row], row);
        return target.share(to_f32(((const T*)a.logits)[row * a.stride + word]), word);
    };
    // The drafts that are accepted: a lane each, each wave for itself.
    int accepted = drafts;
    for (int j0 = 0; j0 < drafts && accepted == drafts; j0 += 64) {
        bool refused = false;
        if (j0 + lane < drafts) {
            const int row = first + j0 + lane;
            const double p = share_of_draft(row);
            const double q = p > 0.0 && v.draft ? (double)to_f32(((const Q*)v.draft)[row * v.draft_stride + v.drafted[row]]) : 1.0;
            refused = !((double)v.uniform[row] * q < p);
        }
        const uint64_t all = __ballot(refused);
        if (all) accepted = j0 + __ffsll((unsigned long long)all) - 1;
    }
    const int row = first + accepted;
    const bool some = accepted < drafts;
    Target target;
    target.init(a, v.kept[row], row);
    Left<T, Q> words{(const T*)a.logits + row * a.stride, some && v.draft ? (const Q*)v.draft + row * v.draft_stride : nullptr, some && !v.draft ? v.drafted[row] : -1};
    uint64_t mine = 0;
    auto add = [&](int, const auto& left) {
        for (uint64_t l : left) mine += l;
        return true;
    };
    int begin = c * a.chunk, stop = min((c + 1) * a.chunk, a.vocab);
    words.each_round(target, begin, stop, add);
    const uint64_t here = sum_of_all(mine, meet, 0);
    uint64_t* sums = v.left + (int64_t)first * a.chunks;
    if (t == 0) __hip_atomic_store(&sums[c], here, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // as in sampling: once the store has gone where every XCD reads, the workgroup is counted, and the last one goes on
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) found = atomicAdd(&v.met[first], 1u) == (uint32_t)a.chunks - 1;
    __syncthreads();
    if (!found) return;

    uint64_t total = 0;
    for (int p = 0; p < a.chunks; ++p) total += __hip_atomic_load(&sums[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    uint64_t before = 0, wanted;   // what lies in front of `begin`, and the sum that is looked for
    if (total == 0) {   // nothing is left: p as it is, all of it by this workgroup
        words.draft = nullptr;
        words.certain = -1;
        mine = 0;
        words.each_round(target, 0, a.vocab, add);
        total = sum_of_all(mine, meet, 1);
        wanted = drawn_sum(v.draw[seq], total);
        begin = 0;
        stop = a.vocab;
    } else {
        wanted = drawn_sum(v.draw[seq], total);
        int p = 0;
        for (;; ++p) {
            const uint64_t of_piece = __hip_atomic_load(&sums[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (before + of_piece >= wanted || p == a.chunks - 1) break;
            before += of_piece;
        }
        begin = p * a.chunk;
        stop = min((p + 1) * a.chunk, a.vocab);
    }
    __syncthreads();
    if (t == 0) found = -1;
    if (total) {
        int which = 0;
        words.each_round(target, begin, stop, [&](int i, const auto& left) {
            uint64_t held = 0;
            for (uint64_t l : left) held += l;
            uint64_t at = before + sum_before(held, meet, which);
            if (at < wanted && at + held >= wanted) {   // one thread's
                int e = 0;
                for (uint64_t l : left) {
                    at += l;
                    if (at >= wanted) break;
                    ++e;
                }
                found = i + e;
            }
            for (int w = 0; w < SAMPLE_WAVES; ++w) before += meet[w][which];
            which ^= 1;
            return before < wanted;
        });
    }
    __syncthreads();
    const int token = found;
    for (int j = t; j <= accepted; j += SAMPLE_WG) {
        const bool last = j == accepted;
        if (last && token < 0) break;   // a row without words
        v.tokens[first + j] = last ? token : v.drafted[first + j];
        if (v.probs) v.probs[first + j] = (float)(last ? target.share(to_f32(words.row[token]), token) : share_of_draft(first + j));
    }
    if (t == 0) v.accepted[seq] = accepted;
}

template <typename T>
static void launch(const Verify& v, Kept* kept, int draft_type, hipStream_t s) {
    const dim3 of_rows(v.s.chunks, v.rows), of_seqs(v.s.chunks, v.seqs), threads(SAMPLE_WG);
    hipLaunchKernelGGL((sample_peak_kernel<T>), of_rows, threads, 0, s, v.s);
    hipLaunchKernelGGL((sample_steps_kernel<T>), of_rows, threads, 0, s, v.s);
    hipLaunchKernelGGL((verify_kept_kernel<T>), of_rows, threads, 0, s, v, kept);
    if (draft_type == LK_TYPE_F16) hipLaunchKernelGGL((verify_judge_kernel<T, __half>), of_seqs, threads, 0, s, v);
    else if (draft_type == LK_TYPE_BF16) hipLaunchKernelGGL((verify_judge_kernel<T, __hip_bfloat16>), of_seqs, threads, 0, s, v);
    else hipLaunchKernelGGL((verify_judge_kernel<T, float>), of_seqs, threads, 0, s, v);
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
    v.s = Sampling{logits, stride, vocab, 0, 0, nullptr, temperature, top_p, min_p, top_k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
    cut_rows(v.s, rows, size);
    const size_t judged = sizeof(Kept) + (size_t)v.s.chunks * 8;
    LkScratch scratch((hipStream_t)stream);
    uint8_t* mem = (uint8_t*)scratch.get(LK_SCRATCH_SAMPLE, (size_t)rows * (judged + bytes_of_row(v.s) + 4));
    if (!mem) return LK_ERR_NOMEM;
    Kept* kept = (Kept*)mem;
    v.kept = kept;
    v.left = (uint64_t*)(kept + rows);
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
    if (type == LK_TYPE_F32) launch<float>(v, kept, draft_type, (hipStream_t)stream);
    else if (type == LK_TYPE_F16) launch<__half>(v, kept, draft_type, (hipStream_t)stream);
    else launch<__hip_bfloat16>(v, kept, draft_type, (hipStream_t)stream);
    return lk_launch_status();
}
