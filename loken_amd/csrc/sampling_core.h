// What sampling and the check of drafted tokens share: words by their logits, weights as integers, a row's largest words, its histogram, and the
// search for the places where the rules cut. `choose` ends either in a row's token or in what it would be drawn from.
#pragma once
#include <math.h>

#include <type_traits>

#include "lk_common.h"
#include "stream_scratch.h"

#pragma clang fp contract(off)

namespace {

constexpr int BINS = 2048;        // steps of the histogram
constexpr int LIST = 2048;        // words that are sorted in LDS
constexpr int COUNTED = 256;      // words up to which each is counted to its place
constexpr int CROWD = 64;         // words of a step up to which they are
constexpr int SAMPLE_WG = 512, SAMPLE_WAVES = SAMPLE_WG / 64;
constexpr int ONE_BITS = 42;      // a weight of 1 is 2^42
constexpr float LIVE = 42.5f;     // words below 2^-42.5 weigh nothing

// 32 bits that order as the values do; equal values (both zeros) have equal bits.
static __device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
    return b ^ ((int)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
static __device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ ((int)key < 0 ? 0x80000000u : 0xFFFFFFFFu));
}

// Calls f(values, index of the first) for the words begin .. end - 1 of a row, sixteen bytes at a time (and single words behind the
// last such piece), the loads of AHEAD pieces out before the first is used.
template <int AHEAD, typename T, class F>
static __device__ __forceinline__ void each_piece(const T* __restrict__ row, int begin, int end, F f) {
    constexpr int VEC = 16 / sizeof(T);
    struct __attribute__((aligned(sizeof(T)))) Load { T v[VEC]; };   // rows start on any word
    const int step = SAMPLE_WG * VEC;
    auto hand = [&](const Load& raw, int i) {
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = to_f32(raw.v[e]);
        f(v, i);
    };
    int i = begin + (int)threadIdx.x * VEC;
    for (; i + (AHEAD - 1) * step + VEC <= end; i += AHEAD * step) {
        Load raw[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) raw[j] = *(const Load*)(row + i + j * step);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) hand(raw[j], i + j * step);
    }
    for (; i + VEC <= end; i += step) hand(*(const Load*)(row + i), i);
    const int rest = end - (end - begin) % VEC + (int)threadIdx.x;
    if (rest < end) {
        const float v[1] = {to_f32(row[rest])};
        f(v, rest);
    }
}
// The same word by word.
template <int AHEAD, typename T, class F>
static __device__ __forceinline__ void each_word(const T* __restrict__ row, int begin, int end, F f) {
    each_piece<AHEAD>(row, begin, end, [&](const auto& v, int i) {
        constexpr int N = sizeof(v) / sizeof(float);
#pragma unroll
        for (int e = 0; e < N; ++e) f(v[e], i + e);
    });
}

struct Peak {
    uint64_t best;     // key and the number turned round, of the largest word (the lowest number of equal ones); 0: none
    uint32_t lowest;   // key of the smallest word
    uint32_t pad;
};

static __device__ __forceinline__ void wave_peak(Peak& p) {
    for (int o = 32; o; o >>= 1) {
        const uint64_t b = __shfl_xor((unsigned long long)p.best, o);
        const uint32_t l = __shfl_xor(p.lowest, o);
        p.best = b > p.best ? b : p.best;
        p.lowest = l < p.lowest ? l : p.lowest;
    }
}

struct Sampling {
    const void* logits;
    int64_t stride;
    int vocab, chunk, chunks, pieces;   // words of a piece, pieces of a row, and pieces whose peaks are taken by themselves
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t* tokens;
    float* probs;
    Peak* peaks;          // [rows][pieces]
    uint64_t* mass;       // [rows][BINS]
    uint32_t* count;      // [rows][BINS]
    uint64_t* floor_mass; // [rows]: what min-p keeps
    uint64_t* list;       // [rows][chunks][LIST]: gathered words, where a row has several pieces
    uint32_t* listed;     // [rows][chunks]: how many each piece has
    uint32_t* arrived;    // [rows]: pieces that have been gathered
};

// What a row is sampled from, where it is asked for in place of a token: the words whose key and number (as Peak has them) are `last` or more
// and which min-p keeps, `kept` their weight; `kept` 0: the word `best` alone (0: none).
struct Kept {
    uint64_t best, last, kept;
};

// a b + c, c the same for all lanes: from scalar registers, where the compiler would copy it to the sum's register first: five of forty
// instructions a word, 256 rows of 151936 in bf16 47 us instead of 40.
static __device__ __forceinline__ double fma_by(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// 2^x, x = below * rate, -43 <= x <= 0. x = n + r, |r| <= 1/2; 2^r = 1 + r f(r), f the polynomial of degree 8
// through (2^r - 1) / r at the nine Chebyshev points of [-1/2, 1/2]: off by 2.8e-14. Its terms from r^5 on, which are below 2.4e-6 of
// the result, are made in 32 bits: off by 2e-13.
static __device__ __forceinline__ double power_at(double r, int n) {
    const float s = (float)r;
    const float high = fmaf(s, fmaf(s, fmaf(s, 1.0203121e-07f, 1.3255225e-06f), 1.5252687e-05f), 0.00015403455f);
    double p = fma_by(r, (double)high, 0.0013333558179043112);
    p = fma_by(r, p, 0.009618129159402558);
    p = fma_by(r, p, 0.055504108664760424);
    p = fma_by(r, p, 0.2402265069581299);
    p = fma_by(r, p, 0.6931471805599453);
    p = fma(r, p, 1.0);
    // times 2^n in the exponent
    return __longlong_as_double((long long)((uint64_t)__double_as_longlong(p) + ((uint64_t)(uint32_t)(n << 20) << 32)));
}
static __device__ __forceinline__ double power_of(double below, double rate) {
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double y = fma(below, rate, magic);
    return power_at(fma(below, rate, magic - y), (int)(uint32_t)__double_as_longlong(y));
}
// The same as an integer of 2^-42: 1024 more, and the last place is 2^-42: what the sum rounds to is the integer.
static __device__ __forceinline__ uint64_t weight_of(double below, double rate) {
    return (uint64_t)__double_as_longlong(power_of(below, rate) + 1024.0) - 0x4090000000000000ull;
}

// What a row's weights and steps go by.
struct Scale {
    float top;        // M; where it is infinite the words that are too count as 0, all others as none
    double rate;      // log2(e) / T
    float reach;      // words further below the top weigh nothing
    float steps;      // steps of the histogram per unit of the logit
    double least;     // log2(min_p)
    bool infinite;

    // From the row's peaks; false where there is nothing to weigh (no words, or the first of them is the choice).
    __device__ __forceinline__ bool init(const Peak& peak, float temperature, float min_p) {
        if (peak.best == 0 || !(temperature > 0.0f)) return false;
        top = value_of((uint32_t)(peak.best >> 32));
        infinite = top == INFINITY;
        float lowest = value_of(peak.lowest);
        if (infinite) top = lowest = 0.0f;
        rate = 1.4426950408889634 / (double)temperature;
        reach = fminf((float)(LIVE / rate), 3.402823466e38f);
        const float range = fminf(reach, top - lowest);
        steps = range > 0.0f ? (float)(BINS - 1) / range : 0.0f;
        if (!(steps <= 3.402823466e38f)) steps = 3.402823466e38f;
        least = min_p > 0.0f ? log2((double)min_p) : -1e300;
        return true;
    }
    // How far a word is below the top (not at all a number: for one that is none). The launches over pieces leave rows with an
    // infinite word to the workgroup that chooses alone, and ask less.
    __device__ __forceinline__ float below(float v) const { return infinite ? (v == INFINITY ? 0.0f : NAN) : top - v; }
    __device__ __forceinline__ bool live(float d) const { return d <= reach; }
    // The step of a live word, as a number that has not been cut to an integer.
    __device__ __forceinline__ float step(float d) const { return fminf(d * steps, (float)(BINS - 1)); }
    // v - M, to 64 bits, and its product with log2(e) / T: the difference first. Of v log2(e) / T - M log2(e) / T the rounding of the
    // second product stays, 2^-53 |M| / T, which is any size where |M| / T is: at M = 12.5 and T = 1e-17 the first word's power was -96.
    __device__ __forceinline__ double from_top(float v) const { return infinite ? 0.0 : (double)v - (double)top; }
    __device__ __forceinline__ double power(float v) const { return from_top(v) * rate; }
    __device__ __forceinline__ uint64_t weight(float v) const { return weight_of(from_top(v), rate); }
    // Whether min-p keeps a word.
    __device__ __forceinline__ bool kept(double power) const { return power >= least; }
};

static __device__ __forceinline__ Peak peak_of_row(const Sampling& a, int row) {
    Peak peak{0, 0xFFFFFFFFu, 0};
    for (int i = threadIdx.x & 63; i < a.pieces; i += 64) {
        const Peak p = a.peaks[(int64_t)row * a.pieces + i];
        peak.best = p.best > peak.best ? p.best : peak.best;
        peak.lowest = p.lowest < peak.lowest ? p.lowest : peak.lowest;
    }
    wave_peak(peak);
    return peak;
}

// Whether a row's histogram counts words, and whether it weighs them. The top-k words, where they are few, are all
// gathered: then their weights are taken from the list.
struct Wants {
    bool count, mass, above;
    __device__ __forceinline__ Wants(const Sampling& a, int row) {
        const int k = a.top_k ? a.top_k[row] : 0;
        count = k > 0 && k < a.vocab;
        mass = !(count && k <= LIST / 2);
        above = mass && a.min_p && a.min_p[row] > 0.0f;
    }
};

static_assert(BINS <= LIST, "the finer histogram stands where the list does");
struct Shared {
    uint64_t mass[BINS];      // running sums once scanned
    uint32_t count[BINS];
    uint64_t list[LIST], sums[LIST];   // both also a finer histogram, while there is no list
    uint64_t meet[SAMPLE_WAVES][2];
    uint64_t found;
    uint32_t low, high;
    int n, at;
};

// Running sums over the workgroup of what each thread brings; returns the sum before it. Ends past a barrier.
static __device__ __forceinline__ uint64_t sum_before(uint64_t mine, uint64_t (*meet)[2], int which) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t up_to = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t u = __shfl_up((unsigned long long)up_to, o);
        if (lane >= o) up_to += u;
    }
    if (lane == 63) meet[wave][which] = up_to;
    __syncthreads();
    uint64_t before = up_to - mine;
    for (int w = 0; w < SAMPLE_WAVES - 1; ++w) before += w < wave ? meet[w][which] : 0;
    return before;
}

// Running sums over the steps, of what the thread has of them (PER from PER t on), into `mass` and `count`.
constexpr int PER = BINS / SAMPLE_WG;
static __device__ __forceinline__ void scan_held(uint64_t (&m)[PER], uint32_t (&c)[PER], uint64_t* mass, uint32_t* count, uint64_t (*meet)[2]) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 1; i < PER; ++i) { m[i] += m[i - 1]; c[i] += c[i - 1]; }
    const uint64_t mb = sum_before(m[PER - 1], meet, 0);
    const uint32_t cb = (uint32_t)sum_before(c[PER - 1], meet, 1);
#pragma unroll
    for (int i = 0; i < PER; ++i) { mass[t * PER + i] = mb + m[i]; count[t * PER + i] = cb + c[i]; }
    __syncthreads();
}
// The same of a histogram in LDS, in place.
static __device__ __forceinline__ void scan_bins(uint64_t* mass, uint32_t* count, uint64_t (*meet)[2]) {
    uint64_t m[PER];
    uint32_t c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) { m[i] = mass[threadIdx.x * PER + i]; c[i] = count[threadIdx.x * PER + i]; }
    scan_held(m, c, mass, count, meet);
}

// The first of 0 .. n - 1 for which `is` holds, as it does for all behind it; n if for none. Each wave looks for itself, all its lanes
// at once: two looks into LDS, one after the other, where halves would take eleven.
static_assert(BINS <= 64 * 64 && LIST <= 64 * 64);
template <class F>
static __device__ __forceinline__ int first_where(int n, F is) {
    const int lane = threadIdx.x & 63, run = (n + 63) >> 6;
    uint64_t all = __ballot(lane * run < n && is(min(lane * run + run, n) - 1));
    if (!all) return n;
    const int from = (__ffsll((unsigned long long)all) - 1) * run;
    all = __ballot(lane < run && from + lane < n && is(min(from + lane, n - 1)));
    return from + __ffsll((unsigned long long)all) - 1;
}
// The first of n >= 1 running sums that reaches `target`, n - 1 if none does.
template <typename V>
static __device__ __forceinline__ int first_reaching(const V* sums, int n, uint64_t target) {
    return min(first_where(n, [&](int i) { return sums[i] >= target; }), n - 1);
}

// Sorts the n <= LIST words of the list, the largest first, and gives their running sums of weights. A word's number is part of
// what is compared, so the order the words came in does not show.
static __device__ __forceinline__ void sort_list(Shared& sh, int n, const Scale& sc) {
    const int t = threadIdx.x;
    if (n <= COUNTED) {
        // a word a thread: its place is the number of words in front of it
        constexpr int AT_ONCE = 8;
        if (t < AT_ONCE) sh.list[n + t] = 0;   // (the list has room for them)
        __syncthreads();
        const uint64_t mine = t < n ? sh.list[t] : ~0ull;
        const uint64_t weight = sc.weight(t < n ? value_of((uint32_t)(mine >> 32)) : sc.top);
        int place = 0;
        for (int i = 0; i < n; i += AT_ONCE) {
            uint64_t x[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) x[j] = sh.list[i + j];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) place += x[j] > mine;
        }
        __syncthreads();
        if (t < n) {
            sh.list[place] = mine;
            sh.sums[place] = weight;
        }
        __syncthreads();
        const uint64_t here = t < n ? sh.sums[t] : 0, before = sum_before(here, sh.meet, 0);
        if (t < n) sh.sums[t] = before + here;
        __syncthreads();
        return;
    }
    // More words: to their steps first, and then, among the words of a step, as above. 1000 words take 3 us; exchanges with a
    // barrier each, as for words of which many share a step, 16.
    static_assert(PER * SAMPLE_WG == LIST && PER % 2 == 0);
    uint32_t* start = (uint32_t*)sh.sums;   // of a step's words, while there are no sums
    uint64_t word[PER];
    int step[PER], slot[PER];
    for (int i = t; i < BINS; i += SAMPLE_WG) start[i] = 0;
    __syncthreads();
    bool crowd = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = i * SAMPLE_WG + t;
        word[i] = at < n ? sh.list[at] : 0;
        step[i] = at < n ? (int)sc.step(sc.below(value_of((uint32_t)(word[i] >> 32)))) : 0;
        slot[i] = at < n ? (int)atomicAdd(&start[step[i]], 1u) : 0;
        crowd = crowd || slot[i] >= CROWD;
    }
    const uint64_t crowds = __ballot(crowd);
    if ((t & 63) == 0) sh.meet[t >> 6][1] = crowds;
    __syncthreads();
    uint64_t any = 0;
    for (int w = 0; w < SAMPLE_WAVES; ++w) any |= sh.meet[w][1];
    if (any) {
        int size = 2 * COUNTED;
        while (size < n) size <<= 1;
        for (int i = n + t; i < size; i += SAMPLE_WG) sh.list[i] = 0;
        __syncthreads();
        for (int run = 2; run <= size; run <<= 1)
            for (int gap = run >> 1; gap > 0; gap >>= 1) {
                for (int j = t; j < size / 2; j += SAMPLE_WG) {
                    const int lo = 2 * j - (j & (gap - 1)), hi = lo + gap;
                    const uint64_t x = sh.list[lo], y = sh.list[hi];
                    if ((x < y) == ((lo & run) == 0)) { sh.list[lo] = y; sh.list[hi] = x; }
                }
                __syncthreads();
            }
    } else {
        uint32_t held[PER], all = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { held[i] = start[t * PER + i]; all += held[i]; }
        uint32_t before = (uint32_t)sum_before(all, sh.meet, 0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            start[t * PER + i] = before;
            before += held[i];
        }
        __syncthreads();
        int from[PER], to[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            from[i] = (int)start[step[i]];
            to[i] = step[i] + 1 < BINS ? (int)start[min(step[i] + 1, BINS - 1)] : n;
            if (i * SAMPLE_WG + t < n) sh.list[from[i] + slot[i]] = word[i];
        }
        __syncthreads();
        int place[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            place[i] = from[i];
            if (i * SAMPLE_WG + t < n)
                for (int j = from[i]; j < to[i]; ++j) place[i] += sh.list[j] > word[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * SAMPLE_WG + t < n) sh.list[place[i]] = word[i];
        __syncthreads();
    }
    uint64_t m[PER], ms = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = t * PER + i;
        if (at < n) ms += sc.weight(value_of((uint32_t)(sh.list[at] >> 32)));
        m[i] = ms;
    }
    const uint64_t before = sum_before(ms, sh.meet, 0);
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (t * PER + i < n) sh.sums[t * PER + i] = before + m[i];
    __syncthreads();
}

// floor(share * whole) + 1, at most `whole`, and ceil(share * whole), at least 1: the sums that the draw and top-p look for.
static __device__ __forceinline__ uint64_t drawn_sum(float u, uint64_t whole) {
    return min((uint64_t)floor((double)(u > 0.0f ? fminf(u, 1.0f) : 0.0f) * (double)whole) + 1, whole);
}
static __device__ __forceinline__ uint64_t nucleus_sum(float top_p, uint64_t whole) {
    const double wanted = ceil((double)fmaxf(top_p, 0.0f) * (double)whole);
    return wanted > 1.0 ? min((uint64_t)wanted, whole) : 1;
}

// A place in the row's order: the word, its weight, and the sum up to and with it.
struct Place {
    int token;
    uint64_t weight, sum;
};

// Searches of one row. All of it is inlined into the kernel, once, so that LDS is addressed as LDS: through generic
// addresses the compiler may step an address of the array at LDS offset 0 back and add the step in the load, and the
// hardware takes the address in front of LDS for one of memory.
template <typename T>
struct Searcher {
    const T* row;
    int vocab;
    Scale sc;
    // what the list holds: the words of steps b0 .. b1 (-1: none such), behind words that weigh base_mass, base_count of them
    int b0 = -1, b1 = -1, n = 0;
    uint64_t base_mass = 0;
    uint32_t base_count = 0;

    // The words of steps `from` .. `to` with keys low .. high (at most LIST), sorted, with their running sums.
    __device__ __forceinline__ void gather(Shared& sh, int from, int to, uint32_t low, uint32_t high) {
        const int t = threadIdx.x;
        __syncthreads();
        if (t == 0) sh.n = 0;
        __syncthreads();
        each_word<2>(row, 0, vocab, [&](float v, int i) {
            const float d = sc.below(v);
            const int b = (int)sc.step(d);
            const uint32_t key = key_of(v);
            if (sc.live(d) && b >= from && b <= to && key >= low && key <= high) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < LIST) sh.list[at] = (uint64_t)key << 32 | (uint32_t)~i;
            }
        });
        __syncthreads();
        n = min(sh.n, LIST);
        sort_list(sh, n, sc);
    }

    // The word at which the running number (by_mass: the running weight) reaches `target` >= 1, which some word does.
    __device__ __forceinline__ Place search(Shared& sh, bool by_mass, uint64_t target) {
        const int t = threadIdx.x;
        const int b = by_mass ? first_reaching(sh.mass, BINS, target) : first_reaching(sh.count, BINS, target);
        if (b < b0 || b > b1) {
            const uint32_t before = b > 0 ? sh.count[max(b - 1, 0)] : 0;
            const uint64_t mass_before = b > 0 ? sh.mass[max(b - 1, 0)] : 0;
            uint32_t low = 0, high = 0xFFFFFFFFu;
            b0 = b1 = b;
            base_mass = mass_before;
            base_count = before;
            if (sh.count[b] <= LIST) {   // all from the top on: what is looked for next is among them
                b0 = 0;
                base_mass = base_count = 0;
            } else if (sh.count[b] - before > LIST) {
                // A step that holds more words than the list: steps of their keys, finer each time, until the list takes
                // the words or all of them are equal.
                uint64_t* sub_mass = sh.list;
                uint32_t* sub_count = (uint32_t*)sh.sums;
                for (;;) {
                    __syncthreads();
                    if (t == 0) { sh.low = 0xFFFFFFFFu; sh.high = 0; }
                    for (int i = t; i < BINS; i += SAMPLE_WG) { sub_mass[i] = 0; sub_count[i] = 0; }
                    __syncthreads();
                    uint32_t lo = 0xFFFFFFFFu, hi = 0;
                    each_word<2>(row, 0, vocab, [&](float v, int) {
                        const uint32_t key = key_of(v);
                        const float d = sc.below(v);
                        const bool in = sc.live(d) && (int)sc.step(d) == b && key >= low && key <= high;
                        lo = in ? min(lo, key) : lo;
                        hi = in ? max(hi, key) : hi;
                    });
                    atomicMin(&sh.low, lo);
                    atomicMax(&sh.high, hi);
                    __syncthreads();
                    low = sh.low;
                    high = sh.high;
                    if (low >= high) return equal(sh, high, by_mass, target);
                    int shift = 0;
                    while (((high - low) >> shift) >= BINS) ++shift;
                    each_word<2>(row, 0, vocab, [&](float v, int) {
                        const uint32_t key = key_of(v);
                        const float d = sc.below(v);
                        if (sc.live(d) && (int)sc.step(d) == b && key >= low && key <= high) {
                            const uint32_t at = (high - key) >> shift;   // below BINS
                            atomicAdd((unsigned long long*)&sub_mass[at], (unsigned long long)sc.weight(v));
                            atomicAdd(&sub_count[at], 1u);
                        }
                    });
                    __syncthreads();
                    scan_bins(sub_mass, sub_count, sh.meet);
                    const int s = by_mass ? first_reaching(sub_mass, BINS, target - base_mass) : first_reaching(sub_count, BINS, target - base_count);
                    const uint32_t passed = s > 0 ? sub_count[max(s - 1, 0)] : 0, members = sub_count[s] - passed;
                    base_mass += s > 0 ? sub_mass[max(s - 1, 0)] : 0;
                    base_count += passed;
                    const uint32_t room = (1u << shift) - 1;
                    high -= (uint32_t)s << shift;
                    low = high - low > room ? high - room : low;
                    if (members <= LIST) break;
                }
            }
            gather(sh, b0, b1, low, high);
            if (low != 0 || high != 0xFFFFFFFFu) b0 = b1 = -1;   // a part of a step: no other search finds its words there
        }
        const int i = by_mass ? first_reaching(sh.sums, n, target - base_mass) : min(n, (int)(target - base_count)) - 1;
        const uint64_t sum = sh.sums[i], before = i > 0 ? sh.sums[max(i - 1, 0)] : 0;
        return {(int)~(uint32_t)sh.list[i], sum - before, base_mass + sum};
    }

    // More equal words than the list takes: the one whose turn it is, counted in the order of their numbers.
    __device__ __forceinline__ Place equal(Shared& sh, uint32_t key, bool by_mass, uint64_t target) {
        const int t = threadIdx.x;
        const uint64_t w = sc.weight(value_of(key));
        const uint32_t turn = (uint32_t)(by_mass ? (target - base_mass + w - 1) / w : target - base_count);
        uint32_t passed = 0;
        b0 = b1 = -1;
        for (int i0 = 0; i0 < vocab; i0 += SAMPLE_WG) {
            const int i = i0 + t;
            const float v = i < vocab ? to_f32(row[i]) : -INFINITY;
            const bool is = v > -INFINITY && key_of(v) == key;
            const uint64_t all = __ballot(is);
            if ((t & 63) == 0) sh.meet[t >> 6][0] = __popcll(all);
            __syncthreads();
            uint32_t here = 0, mine = 0;
            for (int wv = 0; wv < SAMPLE_WAVES; ++wv) {
                const uint32_t in_wave = (uint32_t)sh.meet[wv][0];
                mine += wv < (t >> 6) ? in_wave : 0;
                here += in_wave;
            }
            const uint32_t place = passed + mine + __popcll(all & ((1ull << (t & 63)) - 1)) + 1;
            if (is && place == turn) sh.n = i;
            passed += here;
            __syncthreads();
            if (passed >= turn) break;
        }
        return {sh.n, w, base_mass + turn * w};
    }
};

// The histogram of a piece of a row, into LDS arrays that are clear; the weight of what min-p keeps, of the thread's words.
template <bool COUNT, bool MASS, bool ABOVE, bool ALONE, typename T>
static __device__ __forceinline__ uint64_t weigh_as(const T* x, int begin, int end, const Scale& sc, uint64_t* mass, uint32_t* count) {
    uint64_t above = 0;
    each_piece<2>(x, begin, end, [&](const auto& v, int) {
        constexpr int N = sizeof(v) / sizeof(float);
        // first all weights (of words that weigh nothing something that is not used), side by side
        float d[N];
        uint64_t w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            d[e] = ALONE ? sc.below(v[e]) : sc.top - v[e];
            const double from_top = !MASS ? 0.0 : ALONE ? sc.from_top(v[e]) : (double)v[e] - (double)sc.top;
            w[e] = MASS ? weight_of(from_top, sc.rate) : 0;
            if (ABOVE) above += sc.live(d[e]) && sc.kept(from_top * sc.rate) ? w[e] : 0;
        }
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (sc.live(d[e])) {
                const int b = (int)(d[e] * sc.steps);   // (of a live word: below BINS)
                if (COUNT) atomicAdd(&count[b], 1u);
                if (MASS) atomicAdd((unsigned long long*)&mass[b], (unsigned long long)w[e]);
            }
    });
    return above;
}
template <typename T>
static __device__ __forceinline__ void steps_of_row(const Sampling& a, uint64_t (&mass)[BINS], uint32_t (&count)[BINS]) {
    const int row = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    Scale sc;
    if (!sc.init(peak_of_row(a, row), a.temperature[row], a.min_p ? a.min_p[row] : 0.0f) || sc.infinite) return;
    const Wants wants(a, row);
    for (int i = t; i < BINS; i += SAMPLE_WG) { mass[i] = 0; count[i] = 0; }
    __syncthreads();
    const T* x = (const T*)a.logits + row * a.stride;
    const int begin = c * a.chunk, end = min((c + 1) * a.chunk, a.vocab);
    uint64_t above = 0;
    if (!wants.mass) weigh_as<true, false, false, false>(x, begin, end, sc, mass, count);
    else if (!wants.count && !wants.above) weigh_as<false, true, false, false>(x, begin, end, sc, mass, count);
    else above = weigh_as<true, true, true, false>(x, begin, end, sc, mass, count);   // (what is not asked for is not read)
    if (wants.above) {
        for (int o = 32; o; o >>= 1) above += __shfl_xor((unsigned long long)above, o);
        if ((t & 63) == 0 && above) atomicAdd((unsigned long long*)&a.floor_mass[row], (unsigned long long)above);
    }
    __syncthreads();
    for (int i = t; i < BINS; i += SAMPLE_WG) {
        if (mass[i]) atomicAdd((unsigned long long*)&a.mass[(int64_t)row * BINS + i], (unsigned long long)mass[i]);
        if (count[i]) atomicAdd(&a.count[(int64_t)row * BINS + i], count[i]);
    }
}

// The choice by one workgroup alone, from the row itself: where the steps in question hold more words than are sorted at once.
template <bool KEPT, typename T, class F>
static __device__ __forceinline__ void choose_alone(const Sampling& a, int row, const Scale& sc, Shared& sh, uint64_t best, F done) {
    const int t = threadIdx.x;
    const T* x = (const T*)a.logits + row * a.stride;
    __syncthreads();
    for (int i = t; i < BINS; i += SAMPLE_WG) { sh.mass[i] = 0; sh.count[i] = 0; }
    if (t == 0) sh.found = 0;
    __syncthreads();
    uint64_t above = weigh_as<true, true, true, true>(x, 0, a.vocab, sc, sh.mass, sh.count);
    for (int o = 32; o; o >>= 1) above += __shfl_xor((unsigned long long)above, o);
    if ((t & 63) == 0) atomicAdd((unsigned long long*)&sh.found, (unsigned long long)above);
    __syncthreads();
    const uint64_t one = 1ull << ONE_BITS, kept_m = sh.found > one ? sh.found : one;
    scan_bins(sh.mass, sh.count, sh.meet);
    Searcher<T> at{x, a.vocab, sc};
    const uint64_t words = sh.count[BINS - 1], k = a.top_k && a.top_k[row] > 0 ? (uint64_t)a.top_k[row] : words;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f;
    uint64_t kept = sh.mass[BINS - 1], last = 0;
#pragma unroll 1
    for (int step = 0; step < (KEPT ? 2 : 3); ++step) {   // top-k, top-p, the draw
        uint64_t target = k;
        if (step == 0 && k >= words) continue;
        if (step == 1) {
            if (!(top_p < 1.0f)) continue;
            target = nucleus_sum(top_p, kept);
        }
        if (step == 2) {
            kept = min(kept, kept_m);
            target = drawn_sum(a.uniform[row], kept);
        }
        const Place p = at.search(sh, step > 0, target);
        if (step < 2) {
            kept = p.sum;
            if (KEPT) last = (uint64_t)key_of(to_f32(x[p.token])) << 32 | (uint32_t)~p.token;
        } else if (t == 0) {
            a.tokens[row] = p.token;
            if (a.probs) a.probs[row] = (float)((double)p.weight / (double)kept);
        }
    }
    if (KEPT && t == 0) done(Kept{best, last, min(kept, kept_m)});
}

// The top 16 bits of the k-th largest of n keys, the rest zeros: found by each wave, bit by bit.
constexpr int MOST_TOPS = 1024;
static __device__ __forceinline__ uint32_t bound_of(const uint32_t* keys, int n, int k) {
    constexpr int PER = MOST_TOPS / 64;
    const int lane = threadIdx.x & 63;
    uint32_t mine[PER], bound = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine[i] = i * 64 + lane < n ? keys[i * 64 + lane] : 0;
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t more = bound | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * 64 < n) reach += __popcll(__ballot(mine[i] >= more));
        bound = reach >= k ? more : bound;
    }
    return bound;
}

// The row's choice; with KEPT what it would be made from, which one thread hands to `done`. `tops`: keys of the largest words of so many parts of the row
// (null: none are known): top_k words are then at or above the k-th largest of them, and no histogram is needed to find them.
template <bool KEPT, typename T, class F>
static __device__ __forceinline__ void choose(const Sampling& a, Shared& sh, F done, const uint32_t* tops = nullptr, int n_tops = 0) {
    const int row = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    const T* x = (const T*)a.logits + row * a.stride;
    // everything that is read of the row's other launches, at once
    uint64_t mass[PER];
    uint32_t count[PER];
    if (!KEPT || !tops)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            mass[i] = a.mass[(int64_t)row * BINS + t * PER + i];
            count[i] = a.count[(int64_t)row * BINS + t * PER + i];
        }
    const uint64_t floor_mass = a.floor_mass[row];
    const Peak peak = peak_of_row(a, row);
    Scale sc;
    if (!sc.init(peak, a.temperature[row], a.min_p ? a.min_p[row] : 0.0f)) {   // no words, or the first of them
        if (c == 0 && t == 0) {
            if (KEPT) {
                done(Kept{peak.best, 0, 0});
            } else {
                a.tokens[row] = peak.best ? (int)~(uint32_t)peak.best : -1;
                if (a.probs) a.probs[row] = peak.best ? 1.0f : 0.0f;
            }
        }
        return;
    }
    if (sc.infinite) {   // words beside infinite ones are none: as rare as it is, not worth asking for in the pieces
        if (c == 0) choose_alone<KEPT, T>(a, row, sc, sh, peak.best, done);
        return;
    }
    const Wants wants(a, row);
    if (!KEPT || !tops) scan_held(mass, count, sh.mass, sh.count, sh.meet);   // (what is not counted or weighed is zeros)
    const uint64_t one = 1ull << ONE_BITS, kept_m = wants.above ? max(floor_mass, one) : ~0ull;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, u = KEPT ? 0.0f : a.uniform[row];
    const int k = wants.count ? a.top_k[row] : 0;
    const bool cut_k = KEPT && tops ? true : wants.count && (uint32_t)k < sh.count[BINS - 1];
    if (KEPT && wants.mass && !cut_k && !(top_p < 1.0f)) {   // no last word to look for
        if (c == 0 && t == 0) done(Kept{peak.best, 0, min(sh.mass[BINS - 1], kept_m)});
        return;
    }
    // The steps that are gathered: up to three ranges, [a0, a1] around the end of the top-k words, [b0, b1] around that of top-p's, which
    // is nearer to the top or touches it, [c0, c1] around the draw, nearer still. A range that touches the next one, where there is one
    // (its end is not below 0), is part of it.
    int a0 = BINS, a1 = -1, b0 = BINS, b1 = -1, c0 = BINS, c1 = -1;
    if (KEPT && tops) {   // the top-k words and what the bound lets in beside them
        a0 = 0;
        a1 = BINS - 1;
    } else if (!wants.mass) {   // the top-k words and the rest of their last step
        a0 = 0;
        a1 = first_reaching(sh.count, BINS, k);
    } else {
        auto before = [&](int b) { return b > 0 ? sh.mass[max(b - 1, 0)] : 0; };
        uint64_t least = sh.mass[BINS - 1], most = least;   // bounds of what is kept so far
        if (cut_k) {
            a0 = a1 = first_reaching(sh.count, BINS, k);
            least = before(a0) + 1;
            most = sh.mass[a0];
        }
        if (top_p < 1.0f) {
            b0 = first_reaching(sh.mass, BINS, nucleus_sum(top_p, least));
            b1 = first_reaching(sh.mass, BINS, nucleus_sum(top_p, most));
            least = before(b0) + 1;
            most = sh.mass[b1];
            if (a1 >= 0 && b1 >= a0 - 1) { a0 = min(a0, b0); b0 = BINS; b1 = -1; }
        }
        least = min(least, kept_m);
        most = min(most, kept_m);
        if (!KEPT) {
            c0 = first_reaching(sh.mass, BINS, drawn_sum(u, least));
            c1 = first_reaching(sh.mass, BINS, drawn_sum(u, most));
            if (b1 >= 0 && c1 >= b0 - 1) { b0 = min(b0, c0); c0 = BINS; c1 = -1; }
            else if (b1 < 0 && a1 >= 0 && c1 >= a0 - 1) { a0 = min(a0, c0); c0 = BINS; c1 = -1; }
        }
    }
    // A word's step s is in a range where s - (its first step), a difference without rounding, is at least 0 and below its length:
    // as bits, below that.
    if (a1 < 0) {   // what there is of ranges comes first
        a0 = b0; a1 = b1; b0 = BINS; b1 = -1;
        if (a1 < 0) { a0 = c0; a1 = c1; c0 = BINS; c1 = -1; }
    }
    const float fa = (float)a0, fb = (float)b0, fc = (float)c0;
    const uint32_t na = __float_as_uint((float)max(a1 + 1 - a0, 0)), nb = __float_as_uint((float)max(b1 + 1 - b0, 0)),
                   nc = __float_as_uint((float)max(c1 + 1 - c0, 0));
    if (t == 0) sh.n = 0;
    __syncthreads();
    auto take_words = [&](auto ranges) {
        constexpr int R = decltype(ranges)::value;
        each_piece<4>(x, c * a.chunk, min((c + 1) * a.chunk, a.vocab), [&](const auto& v, int i) {
            constexpr int N = sizeof(v) / sizeof(float);
            uint32_t hit = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float s = fminf((sc.top - v[e]) * sc.steps, (float)BINS);   // (past the last step, or no number: no range's)
                bool in = __float_as_uint(s - fa) < na;
                if (R > 1) in = in || __float_as_uint(s - fb) < nb || __float_as_uint(s - fc) < nc;
                hit |= (uint32_t)in << e;
            }
            while (hit) {
                const int e = __ffs((int)hit) - 1;
                hit &= hit - 1;
                float word = v[0];
#pragma unroll
                for (int j = 1; j < N; ++j) word = e == j ? v[j] : word;
                if (!sc.live(sc.top - word)) continue;   // (of the last step's words some weigh nothing)
                const int at = atomicAdd(&sh.n, 1);
                if (at < LIST) sh.list[at] = (uint64_t)key_of(word) << 32 | (uint32_t)~(i + e);
            }
        });
    };
    if (KEPT && tops) {
        const uint32_t bound = bound_of(tops, n_tops, k);
        each_word<4>(x, c * a.chunk, min((c + 1) * a.chunk, a.vocab), [&](float v, int i) {
            if (key_of(v) < bound || !sc.live(sc.top - v)) return;
            const int at = atomicAdd(&sh.n, 1);
            if (at < LIST) sh.list[at] = (uint64_t)key_of(v) << 32 | (uint32_t)~i;
        });
    } else if (nb == 0 && nc == 0) take_words(std::integral_constant<int, 1>{});
    else take_words(std::integral_constant<int, 3>{});
    __syncthreads();
    int n = sh.n;
    if (a.chunks > 1) {
        uint64_t* list = a.list + ((int64_t)row * a.chunks + c) * LIST;
        uint32_t* listed = a.listed + (int64_t)row * a.chunks;
        for (int i = t; i < min(n, LIST); i += SAMPLE_WG) __hip_atomic_store(&list[i], sh.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (t == 0) __hip_atomic_store(&listed[c], (uint32_t)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // Stores of agent scope go through the XCD's cache to where every XCD reads: once each wave has waited for its own, the
        // workgroup is counted, and the last one to be counted goes on with the row. (A fence writes the whole cache back, once a
        // wave: 64 rows took 150 us with two of them.)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t == 0) sh.at = atomicAdd(&a.arrived[row], 1u) == (uint32_t)a.chunks - 1;
        __syncthreads();
        if (!sh.at) return;
        list = a.list + (int64_t)row * a.chunks * LIST;
        // each wave takes pieces in turn; where a piece's words go is what the pieces before it hold
        const int lane = t & 63, wave = t >> 6;
        uint32_t all = 0;
        if (KEPT && tops && a.chunks <= 64) {   // a few words of each piece: eight threads to one, all pieces at once
            const uint32_t mine = lane < a.chunks ? __hip_atomic_load(&listed[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
            uint32_t up_to = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t v = __shfl_up(up_to, o);
                if (lane >= o) up_to += v;
            }
            const int piece = t >> 3;
            const uint32_t count = __shfl(mine, piece), to = __shfl(up_to, piece) - count;
            for (uint32_t i = t & 7; i < min(count, (uint32_t)LIST); i += 8)
                if (to + i < LIST) sh.list[to + i] = __hip_atomic_load(&list[(int64_t)piece * LIST + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            all = __shfl(up_to, 63);
        } else for (int p0 = 0; p0 < a.chunks; p0 += 64) {
            const uint32_t mine = p0 + lane < a.chunks ? __hip_atomic_load(&listed[p0 + lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
            uint32_t up_to = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t v = __shfl_up(up_to, o);
                if (lane >= o) up_to += v;
            }
            for (int j = wave; j < min(64, a.chunks - p0); j += SAMPLE_WAVES) {
                const uint32_t count = __shfl(mine, j), to = all + __shfl(up_to, j) - count;
                for (uint32_t i = lane; i < min(count, (uint32_t)LIST); i += 64)
                    if (to + i < LIST) sh.list[to + i] = __hip_atomic_load(&list[(int64_t)(p0 + j) * LIST + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            all += __shfl(up_to, 63);   // at most 2^20 words
        }
        n = (int)all;
    }
    if (n > LIST || n == 0) {
        choose_alone<KEPT, T>(a, row, sc, sh, peak.best, done);
        return;
    }
    __syncthreads();
    sort_list(sh, n, sc);
    // The list's running sums as the row's: each range starts at the weight of what lies in front of it.
    auto first_at = [&](int step) {   // the first word of the list whose step is not in front of `step`
        return first_where(n, [&](int i) { return sc.step(sc.top - value_of((uint32_t)(sh.list[i] >> 32))) >= (float)step; });
    };
    auto shift_of = [&](int step, int first) {
        return (wants.mass && step > 0 && step < BINS ? sh.mass[min(max(step - 1, 0), BINS - 1)] : 0) - (first > 0 ? sh.sums[max(first - 1, 0)] : 0);
    };
    const int in_a = a1 >= 0 ? first_at(a0) : n, in_b = b1 >= 0 ? first_at(b0) : in_a;
    const uint64_t shift_a = shift_of(a0, in_a), shift_b = shift_of(b0, in_b), shift_c = shift_of(c0, 0);
    __syncthreads();
    for (int i = t; i < n; i += SAMPLE_WG) sh.sums[i] += i >= in_a ? shift_a : i >= in_b ? shift_b : shift_c;
    __syncthreads();
    uint64_t kept = wants.mass ? sh.mass[BINS - 1] : sh.sums[n - 1];
    uint64_t last = 0;
    if (cut_k) {
        const int at = min(in_a + k - 1 - (int)(a0 > 0 ? sh.count[max(a0 - 1, 0)] : 0), n - 1);
        kept = sh.sums[at];
        last = sh.list[at];
    }
    if (top_p < 1.0f) {
        const int at = first_reaching(sh.sums, n, nucleus_sum(top_p, kept));
        kept = sh.sums[at];
        last = sh.list[at];
    }
    uint64_t above = kept_m;
    if (!wants.mass && a.min_p && a.min_p[row] > 0.0f) {   // what min-p keeps of the list, which is a prefix
        const int past = first_where(n, [&](int i) {
            const float v = value_of((uint32_t)(sh.list[i] >> 32));
            return !sc.kept(sc.power(v));
        });
        above = sh.sums[max(past, 1) - 1];
    }
    kept = min(kept, above);
    if (KEPT) {
        if (t == 0) done(Kept{peak.best, last, kept});
        return;
    }
    const int at = first_reaching(sh.sums, n, drawn_sum(u, kept));
    if (t == 0) {
        a.tokens[row] = (int)~(uint32_t)sh.list[at];
        if (a.probs) a.probs[row] = (float)((double)sc.weight(value_of((uint32_t)(sh.list[at] >> 32))) / (double)kept);
    }
}

// Pieces of a row: enough workgroups for two to a CU, of at least 4096 words.
static void cut_rows(Sampling& a, int rows, int size) {
    const int vec = SAMPLE_WG * 16 / size;
    int chunks = (2 * lk_device().cus + rows - 1) / rows;
    if (chunks > (a.vocab + 4095) / 4096) chunks = (a.vocab + 4095) / 4096;
    a.chunk = ((a.vocab + chunks - 1) / chunks + vec - 1) / vec * vec;
    a.pieces = a.chunks = (a.vocab + a.chunk - 1) / a.chunk;
}
// Bytes that a row needs between the launches, and where they are.
static size_t bytes_of_row(const Sampling& a) {
    return (size_t)BINS * 12 + 12 + a.pieces * sizeof(Peak) + a.chunks * (4 + (a.chunks > 1 ? (size_t)LIST * 8 : 0));
}
static void place_rows(Sampling& a, int rows, uint8_t* mem) {
    a.peaks = (Peak*)mem;
    a.mass = (uint64_t*)(a.peaks + (size_t)rows * a.pieces);
    a.list = a.mass + (size_t)rows * BINS;
    a.floor_mass = a.list + (a.chunks > 1 ? (size_t)rows * a.chunks * LIST : 0);
    a.count = (uint32_t*)(a.floor_mass + rows);
    a.listed = a.count + (size_t)rows * BINS;
    a.arrived = a.listed + (size_t)rows * a.chunks;
}

}  // namespace
