// What the kernels of lk_kv_attention_mxfp4 share: the call, and how 4-bit codes become operands of the matrix unit.
#pragma once
#include "kv_attention.h"
#include "kv_mxfp4.h"

// Parts, pieces and rows are those of the 8-bit cache's attention; `pool` of it holds sizes alone.
struct AttendMx : Attend {
    MxPool mx;
    float cap;   // above 0: scores are cap * tanh(score / cap)
};

typedef __bf16 mx_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_b8 __attribute__((ext_vector_type(8)));
typedef float mx_f2 __attribute__((ext_vector_type(2)));

// Byte `SEL` of `w`, two codes, times a power of two: as two bf16, exactly.
template <int SEL>
static __device__ __forceinline__ uint32_t mx_two(uint32_t w, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, SEL));
}
// A word, eight codes, as an operand of eight bf16.
static __device__ __forceinline__ mx_b8 mx_eight(uint32_t w, float power) {
    return __builtin_bit_cast(mx_b8, make_uint4(mx_two<0>(w, power), mx_two<1>(w, power), mx_two<2>(w, power), mx_two<3>(w, power)));
}
// Byte `I` of a word of powers where the conversion looks for it: it takes a number's exponent alone.
template <int I>
static __device__ __forceinline__ float mx_power_of(uint32_t w) {
    return __uint_as_float(I == 3 ? w >> 1 : w << (23 - 8 * I));
}

static __device__ __forceinline__ uint32_t mx_pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((mx_f2){a, b}, mx_b2));   // the nearest
}
// Two numbers as PIECES pairs of bf16 whose sums they are: to 8, 16 or 24 bits.
template <int PIECES>
static __device__ __forceinline__ void mx_pieces(float a, float b, uint32_t (&out)[PIECES]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        out[p] = mx_pack(a, b);
        if (p + 1 < PIECES) {
            a -= __uint_as_float(out[p] << 16);
            b -= __uint_as_float(out[p] & 0xFFFF0000u);
        }
    }
}

// Query values likewise, all of their bits: cut, not rounded, so that those beside f32's end have no infinity among their pieces.
template <int PIECES>
static __device__ __forceinline__ void mx_cut(float a, float b, uint32_t (&out)[PIECES]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        out[p] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
    }
}

// What a capped score is made of, from a product and what it is under the tanh, mx_under: tanh x = 1 - 2 / (e^2x + 1). A softmax does not see the 1: MX_NEAR leaves it
// off, -1 / (e^2x + 1), whose unit, mx_unit, is twice the cap. A score is then off by cap * 2^-23: for f16 and bf16 with caps up to 64, where that is below what their
// weights are held to. MX_FAR: the tanh, off by 1.2e-7; below a quarter by its series, to a few last places of x.
enum MxCap { MX_NONE, MX_NEAR, MX_FAR };
static inline int mx_cap_of(float cap, bool f32) { return !(cap > 0.f) ? MX_NONE : f32 || cap > 64.f ? MX_FAR : MX_NEAR; }
template <int CAP>
static __device__ __forceinline__ float mx_under(float scale, float cap) { return CAP == MX_NONE ? 0.f : scale / cap * (CAP == MX_NEAR ? 2.8853900817779268f : 1.f); }
template <int CAP>
static __device__ __forceinline__ float mx_unit(float scale, float cap) { return (CAP == MX_NONE ? scale : CAP == MX_NEAR ? 2.f * cap : cap) * 1.4426950408889634f; }
template <int CAP>
static __device__ __forceinline__ float mx_tanh(float product, float under) {
    const float x = product * under;
    if (CAP == MX_NEAR) return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x));
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * 2.8853900817779268f) + 1.f), s = x * x;
    const float near = fmaf(x * s, fmaf(s, fmaf(s, fmaf(s, 0.021869488f, -0.053968254f), 0.13333334f), -0.33333334f), x);
    return fabsf(x) < 0.25f ? near : far;
}

// The maximum over the four lanes l, l + 16, l + 32, l + 48.
static __device__ __forceinline__ float mx_max_over_groups(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int WORDS>
struct __attribute__((aligned(WORDS >= 4 ? 16 : 8))) MxWords { uint32_t w[WORDS]; };

// The row tile of that number among those of all sequences, from the last one on; false: there are fewer. Found by each wave.
static __device__ __forceinline__ bool mx_tile_at(const Attend& a, int rows_of_tile, int number, int& seq, int& tile) {
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](int i) {
        if (i >= a.seqs) return 0;
        const unsigned rows = (unsigned)KvSeq(a, i).tokens() * (unsigned)a.group;
        return (int)rows <= a.few_rows ? 0 : (int)((rows + rows_of_tile - 1) / rows_of_tile);
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

// Sequences of up to so many rows (token, head of a group) are the few-rows kernel's, and rows of its workgroups: those whose pieces fit one operand, else
// sixteen. (Sixteen columns, an operand a piece, for the one to four rows of 64 sequences of up to 8192 tokens in f32 83 us, in slots 73, kernel trace; for eight f32
// rows two operands of slots took 63 us, 64 x 2 behind up to 4096, where sixteen columns took 52, calls.)
constexpr int MX_FEW_ROWS = 16;
constexpr int mx_few_rows(bool f32, int max_rows) { return max_rows > (f32 ? 4 : 8) ? 16 : f32 ? 4 : 8; }
// Its waves on a SIMD, for that many rows: as many as the registers hold. Heads of 128 in three with one buffer of codes, for two with two: 64 sequences of up
// to 2000 tokens in pieces, bf16, 49 to 40 us (calls), 131072 tokens of one the same.
constexpr int mx_few_on_simd(bool f32, bool f16, int head_dim, int rows) { return head_dim == 256 && rows == 16 && (f32 || f16) ? 1 : head_dim == 128 && rows < 16 ? 3 : 2; }

// Rows of a workgroup of the many-rows kernel, and its waves on a SIMD, as the registers hold them. (Heads of 256 in two spill: 300 rows of two sequences
// behind 1000, weights of one piece, 42 us for 37, calls.)
constexpr int mx_many_rows(bool f32, int head_dim) { return head_dim == 256 && f32 ? 16 : 32; }
constexpr int mx_many_on_simd(bool f32, bool f16, int head_dim) {
    return head_dim == 64 ? (f32 || f16 ? 3 : 4) : head_dim == 128 ? (f32 || f16 ? 2 : 3) : 1;
}

int kv_attention_mxfp4_few(const AttendMx& a, int type, int head_dim, int max_rows, hipStream_t stream);
int kv_attention_mxfp4_many(const AttendMx& a, int type, int head_dim, hipStream_t stream);
