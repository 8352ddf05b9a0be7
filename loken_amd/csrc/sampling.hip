// The next token of each row of logits (lk_sample): temperature, top-k, top-p, min-p and a given uniform number.
//
// All three rules keep a prefix of the words in falling order of their logits, so a row needs no sorted vocabulary:
// the kept words' weight is S = min(S_k, S_p, S_m) of the three rules' prefixes, and the token is the first word
// whose running sum reaches floor(u S) + 1. Three launches, each over pieces of rows:
//   peak     the row's largest word, and its smallest
//   steps    a histogram of the row over 2048 steps of the logit: numbers of words, their weights, or both
//   choose   from the running sums over the steps: in which steps S_k, S_p and the token lie. Their words are gathered (a few
//            hundred of a vocabulary), and the last workgroup of the row sorts them and makes the choice.
// Where those steps hold more words than are sorted at once (thousands of equal logits), that workgroup searches the row
// itself, in steps of steps.
//
// Weights 2^x, x = (logit - M) log2(e) / T, decide between neighbours whose shares differ by one part in a million and
// less: were the sums off by 1e-10, one draw in 1e5 from a vocabulary of 1.5e5 words would give the next word. They are made to
// 2e-13 and summed exactly, as integers of 2^-42 (2^20 words of weight 1 fit 64 bits). Sums of integers do not depend on the order
// in which the LDS and global adds land.

#include "sampling_core.h"

namespace {

// The largest and the smallest word of a piece of a row; clears the row's histogram on the way.
template <typename T>
__global__ __launch_bounds__(SAMPLE_WG) void sample_peak_kernel(Sampling a) {
    __shared__ Peak meet[SAMPLE_WAVES];
    const int row = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    float best = -INFINITY, lowest = INFINITY;
    int at = 0x7FFFFFFF;
    each_word<4>((const T*)a.logits + row * a.stride, c * a.chunk, min((c + 1) * a.chunk, a.vocab), [&](float v, int i) {
        const bool more = v > best;   // a thread meets the words in rising order
        best = more ? v : best;
        at = more ? i : at;
        lowest = v > -INFINITY ? fminf(lowest, v) : lowest;   // (fminf passes over what is not a number)
    });
    for (int i = c * SAMPLE_WG + t; i < BINS; i += a.chunks * SAMPLE_WG) {
        a.mass[(int64_t)row * BINS + i] = 0;
        a.count[(int64_t)row * BINS + i] = 0;
    }
    if (c == 0 && t == 0) { a.floor_mass[row] = 0; a.arrived[row] = 0; }
    Peak p{best > -INFINITY ? (uint64_t)key_of(best) << 32 | (uint32_t)~at : 0, key_of(lowest), 0};
    wave_peak(p);
    if ((t & 63) == 0) meet[t >> 6] = p;
    __syncthreads();
    if (t >= 64) return;
    p = t < SAMPLE_WAVES ? meet[t] : Peak{0, 0xFFFFFFFFu, 0};
    wave_peak(p);
    if (t == 0) a.peaks[(int64_t)row * a.pieces + c] = p;
}

template <typename T>
__global__ __launch_bounds__(SAMPLE_WG, 4) void sample_steps_kernel(Sampling a) {
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    steps_of_row<T>(a, mass, count);
}

template <typename T>
__global__ __launch_bounds__(SAMPLE_WG, 4) void sample_choose_kernel(Sampling a) {
    __shared__ Shared sh;
    choose<false, T>(a, sh, [](const Kept&) {});
}

template <typename T>
static void launch(const Sampling& a, int rows, hipStream_t s) {
    const dim3 grid(a.chunks, rows);
    hipLaunchKernelGGL((sample_peak_kernel<T>), grid, dim3(SAMPLE_WG), 0, s, a);
    hipLaunchKernelGGL((sample_steps_kernel<T>), grid, dim3(SAMPLE_WG), 0, s, a);
    hipLaunchKernelGGL((sample_choose_kernel<T>), grid, dim3(SAMPLE_WG), 0, s, a);
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
    Sampling a{logits, stride, vocab, 0, 0, 0, uniform, temperature, top_p, min_p, top_k, tokens, probs, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
    cut_rows(a, rows, size);
    LkScratch scratch((hipStream_t)stream);
    uint8_t* mem = (uint8_t*)scratch.get(LK_SCRATCH_SAMPLE, (size_t)rows * bytes_of_row(a));
    if (!mem) return LK_ERR_NOMEM;
    place_rows(a, rows, mem);
    if (type == LK_TYPE_F32) launch<float>(a, rows, (hipStream_t)stream);
    else if (type == LK_TYPE_F16) launch<__half>(a, rows, (hipStream_t)stream);
    else launch<__hip_bfloat16>(a, rows, (hipStream_t)stream);
    return lk_launch_status();
}
