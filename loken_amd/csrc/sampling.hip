// The next token of each row of logits (lk_sample): temperature, top-k, top-p, min-p and a given uniform number.
//
// All three rules keep a prefix of the words in falling order of their logits, so a row needs no sorted vocabulary:
// the kept words' weight is S = min(S_k, S_p, S_m) of the three rules' prefixes, and the token is the first word
// whose running sum reaches floor(u S) + 1. Each of S_k, S_p and the token is one search in the running sums, by number or by
// weight: first in a histogram of the row over 2048 steps of the logit, then among the words of one step, which are gathered and
// sorted in LDS.
//
// Weights 2^x, x = (logit - M) log2(e) / T, decide between neighbours whose shares differ by one part in a million and
// less, so they are made to 1e-10 and summed exactly, as integers of 2^-42 (2^20 words of weight 1 fit 64 bits). Sums of
// integers do not depend on the order in which the LDS and global adds land.

#include <math.h>

#include "lk_common.h"
#include "stream_scratch.h"

#pragma clang fp contract(off)

namespace {

constexpr int BINS = 2048;        // steps of the histogram
constexpr int LIST = 2048;        // words that are sorted in LDS
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

// Calls f(value, index) for the words begin + thread, begin + thread + threads, .. below `end` of a row.
template <typename T, class F>
static __device__ __forceinline__ void each_word(const T* __restrict__ row, int begin, int end, F f) {
    constexpr int AHEAD = 8;
    const int step = blockDim.x;
    int i = begin + threadIdx.x;
    for (; i + (AHEAD - 1) * step < end; i += AHEAD * step) {
        T raw[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) raw[j] = row[i + j * step];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) f(to_f32(raw[j]), i + j * step);
    }
    for (; i < end; i += step) f(to_f32(row[i]), i);
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
    int vocab, chunk, chunks;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t* tokens;
    float* probs;
    Peak* peaks;          // [rows][chunks]
    uint64_t* mass;       // [rows][BINS], where a row has several chunks
    uint32_t* count;      // [rows][BINS]
    uint64_t* floor_mass; // [rows]: what min-p keeps
    uint32_t* arrived;    // [rows]
};

// The largest and the smallest word of a piece of a row; clears the row's histogram on the way.
template <typename T>
__global__ __launch_bounds__(SAMPLE_WG) void sample_peak_kernel(Sampling a) {
    __shared__ Peak meet[SAMPLE_WAVES];
    const int row = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    Peak p{0, 0xFFFFFFFFu, 0};
    each_word((const T*)a.logits + row * a.stride, c * a.chunk, min((c + 1) * a.chunk, a.vocab), [&](float v, int i) {
        if (v > -INFINITY) {
            const uint32_t key = key_of(v);
            const uint64_t word = (uint64_t)key << 32 | (uint32_t)~i;
            p.best = word > p.best ? word : p.best;
            p.lowest = key < p.lowest ? key : p.lowest;
        }
    });
    if (a.chunks > 1) {
        for (int i = c * SAMPLE_WG + t; i < BINS; i += a.chunks * SAMPLE_WG) {
            a.mass[(int64_t)row * BINS + i] = 0;
            a.count[(int64_t)row * BINS + i] = 0;
        }
        if (c == 0 && t == 0) { a.floor_mass[row] = 0; a.arrived[row] = 0; }
    }
    wave_peak(p);
    if ((t & 63) == 0) meet[t >> 6] = p;
    __syncthreads();
    if (t >= 64) return;
    p = t < SAMPLE_WAVES ? meet[t] : Peak{0, 0xFFFFFFFFu, 0};
    wave_peak(p);
    if (t == 0) a.peaks[(int64_t)row * a.chunks + c] = p;
}

// What a row's weights and steps go by.
struct Scale {
    float top;        // M
    double rate;      // log2(e) / T
    float reach;      // words further below the top weigh nothing
    float steps;      // steps of the histogram per unit of the logit
    double least;     // log2(min_p)
    __device__ __forceinline__ bool live(float v) const { return v > -INFINITY && (v == top || top - v <= reach); }
    __device__ __forceinline__ int bin(float v) const {
        const float at = (top - v) * steps;
        return v == top ? 0 : at < (float)(BINS - 1) ? (int)at : BINS - 1;
    }
    __device__ __forceinline__ double power(float v) const { return v == top ? 0.0 : ((double)v - (double)top) * rate; }
};

// 2^x, -43 <= x <= 0, as an integer of 2^-42: x = n + i / 256 + r, 2^(i / 256) from a table in LDS, 2^r by three terms
// (the fourth is below 2e-13) in 32 bits, whose error is 1e-10 of the result.
static __device__ __forceinline__ uint64_t weight_of(double x, const double* table) {
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double y = x * 256.0 + magic;
    const int k = (int)(uint32_t)__double_as_longlong(y);
    const float r = (float)fma(y - magic, -1.0 / 256.0, x);
    const float p = r * fmaf(r, fmaf(r, 0.05550411f, 0.2402265f), 0.6931472f);
    const double base = table[k & 255];
    const uint64_t bits = (uint64_t)__double_as_longlong(fma(base, (double)p, base));   // just below 1 where r is below 0 at i = 0
    const uint64_t m = (bits & 0xFFFFFFFFFFFFFull) | 0x10000000000000ull;
    const int shift = 52 - ONE_BITS - (k >> 8) + 1023 - (int)(bits >> 52);
    return (m + (1ull << (shift - 1))) >> shift;
}

static_assert(BINS <= LIST, "the finer histogram stands where the list does");
struct Shared {
    uint64_t mass[BINS];      // running sums once scanned
    uint32_t count[BINS];
    uint64_t list[LIST], sums[LIST];   // also a finer histogram, while there is no list
    double table[256];
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

// The histogram's running sums, in place.
static __device__ __forceinline__ void scan_bins(uint64_t* mass, uint32_t* count, uint64_t (*meet)[2]) {
    constexpr int PER = BINS / SAMPLE_WG;
    const int t = threadIdx.x;
    uint64_t m[PER], ms = 0;
    uint32_t c[PER], cs = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        m[i] = (ms += mass[t * PER + i]);
        c[i] = (cs += count[t * PER + i]);
    }
    const uint64_t mb = sum_before(ms, meet, 0);
    const uint32_t cb = (uint32_t)sum_before(cs, meet, 1);
#pragma unroll
    for (int i = 0; i < PER; ++i) { mass[t * PER + i] = mb + m[i]; count[t * PER + i] = cb + c[i]; }
    __syncthreads();
}

// The first of n >= 1 running sums that reaches `target`, n - 1 if none does. Every thread looks for itself.
template <typename V>
static __device__ __forceinline__ int first_reaching(const V* sums, int n, uint64_t target) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] >= target) hi = mid;
        else lo = mid + 1;
    }
    return lo;
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
        each_word(row, 0, vocab, [&](float v, int i) {
            const int b = sc.bin(v);
            const uint32_t key = key_of(v);
            if (sc.live(v) && b >= from && b <= to && key >= low && key <= high) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < LIST) sh.list[at] = (uint64_t)key << 32 | (uint32_t)~i;
            }
        });
        __syncthreads();
        n = min(sh.n, LIST);
        int size = 2;
        while (size < n) size <<= 1;
        for (int i = n + t; i < size; i += SAMPLE_WG) sh.list[i] = 0;
        __syncthreads();
        // sorted downwards; a word's number is part of what is compared, so the order the words came in does not show
        for (int run = 2; run <= size; run <<= 1)
            for (int gap = run >> 1; gap > 0; gap >>= 1) {
                for (int j = t; j < size / 2; j += SAMPLE_WG) {
                    const int lo = 2 * j - (j & (gap - 1)), hi = lo + gap;
                    const uint64_t x = sh.list[lo], y = sh.list[hi];
                    if ((x < y) == ((lo & run) == 0)) { sh.list[lo] = y; sh.list[hi] = x; }
                }
                __syncthreads();
            }
        constexpr int PER = LIST / SAMPLE_WG;
        uint64_t m[PER], ms = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = t * PER + i;
            if (at < n) ms += weight_of(sc.power(value_of((uint32_t)(sh.list[at] >> 32))), sh.table);
            m[i] = ms;
        }
        const uint64_t before = sum_before(ms, sh.meet, 0);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (t * PER + i < n) sh.sums[t * PER + i] = before + m[i];
        __syncthreads();
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
                    each_word(row, 0, vocab, [&](float v, int) {
                        const uint32_t key = key_of(v);
                        const bool in = sc.live(v) && sc.bin(v) == b && key >= low && key <= high;
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
                    each_word(row, 0, vocab, [&](float v, int) {
                        const uint32_t key = key_of(v);
                        if (sc.live(v) && sc.bin(v) == b && key >= low && key <= high) {
                            const uint32_t at = (high - key) >> shift;   // below BINS
                            atomicAdd((unsigned long long*)&sub_mass[at], (unsigned long long)weight_of(sc.power(v), sh.table));
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
        const uint64_t w = weight_of(sc.power(value_of(key)), sh.table);
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

template <typename T>
__global__ __launch_bounds__(SAMPLE_WG) void sample_kernel(Sampling a) {
    __shared__ Shared sh;
    __shared__ int is_last;
    const int row = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    const T* x = (const T*)a.logits + row * a.stride;
    Peak peak{0, 0xFFFFFFFFu, 0};
    for (int i = t & 63; i < a.chunks; i += 64) {
        const Peak p = a.peaks[(int64_t)row * a.chunks + i];
        peak.best = p.best > peak.best ? p.best : peak.best;
        peak.lowest = p.lowest < peak.lowest ? p.lowest : peak.lowest;
    }
    wave_peak(peak);
    const float temperature = a.temperature[row];
    if (peak.best == 0 || !(temperature > 0.0f)) {   // no words, or the first of them
        if (c == 0 && t == 0) {
            a.tokens[row] = peak.best ? (int)~(uint32_t)peak.best : -1;
            if (a.probs) a.probs[row] = peak.best ? 1.0f : 0.0f;
        }
        return;
    }
    Scale sc;
    sc.top = value_of((uint32_t)(peak.best >> 32));
    sc.rate = 1.4426950408889634 / (double)temperature;
    sc.reach = sc.top < INFINITY ? (float)(LIVE / sc.rate) : -1.0f;   // (beside an infinite word there is no other)
    const float range = fminf(sc.reach, sc.top - value_of(peak.lowest));
    sc.steps = range > 0.0f && range <= 3.402823466e38f ? (float)(BINS - 1) / range : 0.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    sc.least = min_p > 0.0f ? log2((double)min_p) : -1e300;
    if (t < 256) sh.table[t] = exp2((double)t / 256.0);
    for (int i = t; i < BINS; i += SAMPLE_WG) { sh.mass[i] = 0; sh.count[i] = 0; }
    if (t == 0) sh.found = 0;
    __syncthreads();
    uint64_t above = 0;   // what min-p keeps
    each_word(x, c * a.chunk, min((c + 1) * a.chunk, a.vocab), [&](float v, int) {
        if (!sc.live(v)) return;
        const double power = sc.power(v);
        const uint64_t w = weight_of(power, sh.table);
        const int b = sc.bin(v);
        atomicAdd((unsigned long long*)&sh.mass[b], (unsigned long long)w);
        atomicAdd(&sh.count[b], 1u);
        above += power >= sc.least ? w : 0;
    });
    for (int o = 32; o; o >>= 1) above += __shfl_xor((unsigned long long)above, o);
    if ((t & 63) == 0) atomicAdd((unsigned long long*)&sh.found, (unsigned long long)above);
    __syncthreads();
    if (a.chunks > 1) {
        uint64_t* mass = a.mass + (int64_t)row * BINS;
        uint32_t* count = a.count + (int64_t)row * BINS;
        for (int i = t; i < BINS; i += SAMPLE_WG)
            if (sh.count[i]) {
                atomicAdd((unsigned long long*)&mass[i], (unsigned long long)sh.mass[i]);
                atomicAdd(&count[i], sh.count[i]);
            }
        if (t == 0) atomicAdd((unsigned long long*)&a.floor_mass[row], (unsigned long long)sh.found);
        // this workgroup's adds are done before it is counted; the last one to be counted goes on with the row
        __threadfence();
        __syncthreads();
        if (t == 0) is_last = atomicAdd(&a.arrived[row], 1u) == (uint32_t)a.chunks - 1;
        __syncthreads();
        if (!is_last) return;
        __threadfence();
        for (int i = t; i < BINS; i += SAMPLE_WG) {
            sh.mass[i] = __hip_atomic_load(&mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sh.count[i] = __hip_atomic_load(&count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (t == 0) sh.found = __hip_atomic_load(&a.floor_mass[row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
    }
    const uint64_t one = 1ull << ONE_BITS, kept_m = sh.found > one ? sh.found : one;
    scan_bins(sh.mass, sh.count, sh.meet);
    Searcher<T> at{x, a.vocab, sc};
    const uint64_t words = sh.count[BINS - 1], k = a.top_k && a.top_k[row] > 0 ? (uint64_t)a.top_k[row] : words;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, u = a.uniform[row];
    uint64_t kept = sh.mass[BINS - 1];
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {   // top-k, top-p, the draw
        uint64_t target = k;
        if (step == 0 && k >= words) continue;
        if (step == 1) {
            if (!(top_p < 1.0f)) continue;
            const double wanted = ceil((double)fmaxf(top_p, 0.0f) * (double)kept);
            target = wanted > 1.0 ? min((uint64_t)wanted, kept) : 1;
        }
        if (step == 2) {
            kept = min(kept, kept_m);
            target = min((uint64_t)floor((double)(u > 0.0f ? fminf(u, 1.0f) : 0.0f) * (double)kept) + 1, kept);
        }
        const Place p = at.search(sh, step > 0, target);
        if (step < 2) {
            kept = p.sum;
        } else if (t == 0) {
            a.tokens[row] = p.token;
            if (a.probs) a.probs[row] = (float)((double)p.weight / (double)kept);
        }
    }
}

template <typename T>
static void launch(const Sampling& a, int rows, hipStream_t s) {
    const dim3 grid(a.chunks, rows);
    hipLaunchKernelGGL((sample_peak_kernel<T>), grid, dim3(SAMPLE_WG), 0, s, a);
    hipLaunchKernelGGL((sample_kernel<T>), grid, dim3(SAMPLE_WG), 0, s, a);
}

}  // namespace

extern "C" int lk_sample(const void* logits, int type, int64_t stride, int rows, int vocab, const float* uniform, const float* temperature,
                         const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* probs, void* stream) {
    const int size = type == LK_TYPE_F32 ? 4 : type == LK_TYPE_F16 || type == LK_TYPE_BF16 ? 2 : 0;
    if (!size) return LK_ERR_TYPE;
    if (rows < 0 || rows > 65535 || vocab <= 0 || stride < vocab) return LK_ERR_ARG;
    if (vocab > LK_SAMPLE_VOCAB) return LK_ERR_SIZE;
    if (rows == 0) return LK_OK;
    if (!logits || !uniform || !temperature || !tokens || ((uintptr_t)logits & (size - 1))) return LK_ERR_ARG;
    // pieces of a row: enough workgroups for two to a CU, at least 2048 words each
    int chunks = (2 * lk_device().cus + rows - 1) / rows;
    if (chunks > (vocab + 2047) / 2048) chunks = (vocab + 2047) / 2048;
    Sampling a{logits, stride, vocab, (vocab + chunks - 1) / chunks, 0, uniform, temperature, top_p, min_p, top_k, tokens, probs, nullptr, nullptr, nullptr, nullptr, nullptr};
    a.chunks = (vocab + a.chunk - 1) / a.chunk;
    const size_t of_row = (a.chunks > 1 ? (size_t)BINS * 12 + 16 : 0) + (size_t)a.chunks * sizeof(Peak);
    LkScratch scratch((hipStream_t)stream);
    uint8_t* mem = (uint8_t*)scratch.get(LK_SCRATCH_SAMPLE, (size_t)rows * of_row);
    if (!mem) return LK_ERR_NOMEM;
    a.peaks = (Peak*)mem;
    mem += (size_t)rows * a.chunks * sizeof(Peak);
    if (a.chunks > 1) {
        a.mass = (uint64_t*)mem;
        a.floor_mass = a.mass + (size_t)rows * BINS;
        a.count = (uint32_t*)(a.floor_mass + rows);
        a.arrived = a.count + (size_t)rows * BINS;
    }
    if (type == LK_TYPE_F32) launch<float>(a, rows, (hipStream_t)stream);
    else if (type == LK_TYPE_F16) launch<__half>(a, rows, (hipStream_t)stream);
    else launch<__hip_bfloat16>(a, rows, (hipStream_t)stream);
    return lk_launch_status();
}
