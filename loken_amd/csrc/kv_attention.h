// What the attention kernels over the paged caches share: the call, which rows and positions a workgroup has, and partial results.
#pragma once
#include <math.h>

#include "kv_cache.h"

constexpr int KV_TILE = 64;   // positions of a step

struct Attend {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    KvPool pool;
    const int32_t *table, *lens, *starts;
    int64_t table_stride;
    int table_cols, seqs, rows, heads, group, window;
    float scale;
    bool q_aligned;   // rows of q start on 16 bytes
    // A context is cut into at most `splits` parts of at least `least_tiles` steps. With more than one the parts meet through
    // part_o [rows][heads][splits][head_dim] (sums relative to the part's maximum) and part_ml [rows][heads][splits] (that
    // maximum in powers of two, and the sum of weights); rows are those of the batch, or part_seq for each sequence (one
    // that has more is not cut).
    int splits, least_tiles, part_seq;
    float* part_o;
    float2* part_ml;
    // Or (few rows, `chunks` above 0): the steps of all sequences one after the other are cut into up to `chunks` pieces of equal
    // length, at least `least_tiles`, per key / value head, whatever sequences they belong to, and the parts are
    // [kv heads][chunks][2][rows of a workgroup]: what a piece has of the sequence that it starts inside of, and of the one that it ends in.
    int chunks;
    // The few-rows kernel takes the sequences of up to so many rows (token, head of the group), the other kernel the rest.
    int few_rows;
    // Row / group for rows below 2^31: ceil(2^shift / group), shift = 31 + ceil(log2 group).
    uint32_t group_inverse;
    int group_shift;
    __device__ __forceinline__ int token_of(unsigned row) const { return (int)(((uint64_t)row * group_inverse) >> group_shift); }
    __device__ __forceinline__ int64_t part_row(int seq, const struct KvSeq& s, int row) const;
};

// The rows of a sequence, as far as the batch holds them.
struct KvSeq {
    int first, end;        // rows [first, end)
    int64_t pos_of_0;      // position of row r is pos_of_0 + r
    int64_t limit;         // positions that the table has columns for
    __device__ __forceinline__ KvSeq(const Attend& a, int seq) {
        const int s = a.starts[seq], e = a.starts[seq + 1];
        // both within the batch, whatever stands there: a difference of what does not would pass 32 bits
        first = min(max(s, 0), a.rows);
        end = min(max(e, 0), a.rows);
        pos_of_0 = (int64_t)a.lens[seq] - e;
        limit = (int64_t)a.table_cols << a.pool.page_shift;
    }
    __device__ __forceinline__ int tokens() const { return max(end - first, 0); }
};

__device__ __forceinline__ int64_t Attend::part_row(int seq, const KvSeq& s, int row) const {
    return part_seq ? (int64_t)seq * part_seq + (row - s.first) : row;
}

// Steps [0, tiles) from position `lo` on cover what rows ra .. rb see.
struct KvSpan {
    int lo, hi, tiles;     // positions lo (a multiple of the step) .. hi - 1
    int per_part, parts;   // steps of a part, and how many parts
    __device__ __forceinline__ KvSpan(const Attend& a, const KvSeq& s, int ra, int rb) {
        const int64_t pa = s.pos_of_0 + ra, pb = s.pos_of_0 + rb;
        hi = (int)max((int64_t)0, min(pb + 1, s.limit));
        lo = a.window > 0 ? (int)max((int64_t)0, pa - a.window + 1) & ~(KV_TILE - 1) : 0;
        tiles = hi > lo ? (hi - lo + KV_TILE - 1) / KV_TILE : 0;
        per_part = max(tiles, 1);
        parts = 1;
        if (a.splits > 1 && !(a.part_seq && s.tokens() > a.part_seq)) {
            per_part = max(a.least_tiles, (tiles + a.splits - 1) / a.splits);
            parts = max(1, (tiles + per_part - 1) / per_part);
        }
    }
};

// The steps of a sequence as the pieces count them: none where it is not the few-rows kernel's, one where it is not cut (more rows
// than a workgroup has, or nothing to see).
static __device__ __forceinline__ int kv_steps_of(const Attend& a, int seq, int rows) {
    const KvSeq s(a, seq);
    const int64_t all = (int64_t)s.tokens() * a.group;
    if (all == 0 || all > a.few_rows) return 0;
    if (all > rows) return 1;
    return max(1, KvSpan(a, s, s.first, s.end - 1).tiles);
}

// Where sequences stand among the steps of all, found by a wave.
struct KvPieces {
    int total, length;   // steps, and those of a piece
    __device__ __forceinline__ KvPieces(const Attend& a, int rows) {
        total = 0;
        for (int base = 0; base < a.seqs; base += LK_WAVE) {
            const int seq = base + (threadIdx.x & 63);
            total += wave_sum_i32(seq < a.seqs ? kv_steps_of(a, seq, rows) : 0);
        }
        length = max(a.least_tiles, (total + a.chunks - 1) / a.chunks);
    }
    // The sequence that step `at` < total belongs to, and that sequence's first step.
    static __device__ __forceinline__ int sequence_at(const Attend& a, int rows, int at, int& first) {
        first = 0;
        for (int base = 0; base < a.seqs; base += LK_WAVE) {
            const int lane = threadIdx.x & 63, seq = base + lane;
            const int mine = seq < a.seqs ? kv_steps_of(a, seq, rows) : 0;
            int up_to = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(up_to, o);
                if (lane >= o) up_to += v;
            }
            const uint64_t over = __ballot(first + up_to > at);
            if (over) {
                const int l = __ffsll((unsigned long long)over) - 1;
                first += __shfl(up_to - mine, l);
                return base + l;
            }
            first += __shfl(up_to, 63);
        }
        return a.seqs;
    }
    // The first step of `seq`.
    static __device__ __forceinline__ int first_of(const Attend& a, int rows, int seq) {
        int before = 0;
        for (int base = 0; base < seq; base += LK_WAVE) {
            const int other = base + (threadIdx.x & 63);
            before += wave_sum_i32(other < seq ? kv_steps_of(a, other, rows) : 0);
        }
        return before;
    }
};

// Rows of a workgroup of the two kernels. The few-rows one takes two operands' rows in one pass over the keys where there are
// that many and the registers hold them (256 columns: not).
constexpr int KV_MANY_ROWS = 128;
constexpr int kv_few_rows(bool f32, int head_dim, int max_rows) {
    const int one = f32 ? 4 : 8;
    return head_dim < 256 && max_rows > one ? 2 * one : one;
}

int kv_attention_few(const Attend& a, int type, int head_dim, int max_rows, hipStream_t stream);
int kv_attention_many(const Attend& a, int type, int head_dim, int max_rows, hipStream_t stream);
// Joins the parts of a launch before it: of the few-rows kernel's sequences (`few`), `tokens` of whose rows a launch counts on, or of the others;
// `per` rows of a workgroup had the same parts.
int kv_attention_join(const Attend& a, int type, int head_dim, int per, bool few, int tokens, hipStream_t stream);
