// The 8-bit key/value cache: its codes and scales (device), and the launchers behind
// shp_cache8_* (host).
//
// A code q of a block with scale s stands for the fp32 number fl(q * s).  A block's scale is
// max |x| over its tokens divided by the largest code (127, or 448 for e4m3), rounded once, and a
// code is the exact quotient x / s rounded once to the nearest code, ties to even: which way a
// quotient next to a tie falls does not depend on the order of the arithmetic.
#pragma once

#include "common.h"

namespace shp {

constexpr int kCacheTile = 64;  // tokens of a V tile, and of an attention step

// shp_cache8 with the counts the kernels derive from it.
struct Cache8 {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    int32_t* lengths;
    int n_seqs, kv, cap, block_log2;
};

struct Cache8Rows {
    const float *k, *v;
    int64_t k_seq, k_row, k_head, v_seq, v_row, v_head;
    const int32_t* counts;
    int n;
};

struct Cache8Query {
    const float* q;
    float* out;
    int64_t q_seq, q_row, q_head, o_seq, o_row, o_head;
    float* lse;  // attend: written where not null; weights: read
    const int32_t* counts;
    int n, heads, group;
    float scale;
    const float* acc_in;  // weights
    float* acc_out;
};

int cache8_append_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                         const Cache8Rows& r);
int cache8_read_launch(hipStream_t s, const Cache8& c, int head_dim, int format, int n, float* k,
                       float* v);
// How attention splits the tokens of a sequence, and the floats of scratch that takes (0: none).
struct Cache8Plan {
    int row_tiles;   // 16-row tiles a workgroup owns
    int row_blocks;  // workgroups over the rows of one KV head
    int splits;      // workgroups over the tokens of a sequence at most
    int least;       // tiles a workgroup takes at least
    size_t scratch;
};
Cache8Plan cache8_attend_plan(const Cache8& c, int head_dim, int64_t rows, int cu_count,
                              bool may_split);
int cache8_attend_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                         const Cache8Query& q, const Cache8Plan& p, float* scratch,
                         int* counters);
// How the accounts' rows and tokens are shared out, and the floats of scratch that takes (0: none).
struct Cache8WeightsPlan {
    int row_tiles;  // 16-row tiles a wavefront holds
    int groups;     // row groups of a KV head, each of `chunks` times that many rows
    int chunks;
    int row_waves;  // wavefronts of a workgroup side by side over groups; the rest share its tokens
    int workers;    // workgroups over the tokens
    size_t scratch;
};
Cache8WeightsPlan cache8_weights_plan(const Cache8& c, int head_dim, int64_t rows, bool may_group);
int cache8_weights_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                          const Cache8Query& q, const Cache8WeightsPlan& p, float* scratch);
int cache8_evict_launch(hipStream_t s, const Cache8& src, const Cache8& dst, int head_dim,
                        int format, const float* weights, int keep, int recent, int32_t* kept,
                        float* dst_weights);

struct LogprobArgs {
    const float* logits;
    int64_t row_stride;
    int rows, vocab, top;
    const int32_t* targets;
    float *logprob, *entropy;
    int32_t* top_ids;
    float* top_logprobs;
};
constexpr int kMaxTop = 64;  // alternatives a row can ask for
// Floats of scratch the rows' parts need (0: a workgroup takes a whole row).
size_t logprobs_scratch(int rows, int vocab);
int logprobs_launch(hipStream_t s, const LogprobArgs& a, float* scratch);

}  // namespace shp

#ifdef __HIPCC__
namespace shpd {

enum { kI8 = SHP_CACHE8_I8, kE4M3 = SHP_CACHE8_E4M3 };

constexpr float kScaleFloor = 0x1p-60f;  // keeps x / s and its remainder normal numbers

template <int FMT>
__device__ __forceinline__ float code_max() { return FMT == kI8 ? 127.0f : 448.0f; }

// The scale of a block whose largest |x| is `top` (NaN where some x is not finite).
template <int FMT>
__device__ __forceinline__ float block_scale(float top) {
    if (!(top <= 3.4028234663852886e+38f)) return __builtin_nanf("");
    return fmaxf(top / code_max<FMT>(), kScaleFloor);
}

// x / s rounded to odd: the quotient cut toward zero, its last bit set where something was cut
// off, so that a second rounding to fewer bits falls as that of the exact quotient would.  The
// remainder x - q s of a rounded quotient is exact in one fused step.
__device__ __forceinline__ float quotient_odd(float x, float s) {
    const float q = x / s;
    const float r = __builtin_fmaf(-q, s, x);
    int b = __float_as_int(q);
    // rounded away from zero (the remainder points back): one step toward zero, last bit set
    if (r != 0.0f) {
        if ((r < 0.0f) != (x < 0.0f)) b -= 1;
        b |= 1;
    }
    return __int_as_float(b);
}

// The codes (one word) of four numbers at scale s, inv = 1 / s rounded; of a block without a scale
// (NaN), 0.  x * inv is within 2^-23 of the quotient, which settles the code unless it lies next
// to the middle of two codes (about one number in 16,000): only then the quotient itself is formed
// (a division and its remainder, five times the work).
template <int FMT>
__device__ __forceinline__ unsigned encode4(const float* x, float s, float inv) {
    if (!(s > 0.0f)) return 0u;
    float y[4];
    if constexpr (FMT == kI8) {
        // adding 1.5 * 2^23 rounds to a whole number, whose low byte is the code
        constexpr float kWhole = 12582912.0f;
        float m[4], off = 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = x[i] * inv;
            m[i] = y[i] + kWhole;
            off = fminf(off, fabsf(fabsf(y[i] - (m[i] - kWhole)) - 0.5f));
        }
        if (off < 0x1p-15f) {  // 2^-23 of 127 is under 2^-16
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = quotient_odd(x[i], s) + kWhole;
        }
        const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(m[1]), __float_as_uint(m[0]), 0x0c0c0400u);
        const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(m[3]), __float_as_uint(m[2]), 0x04000c0cu);
        return lo | hi;
    } else {
        bool near = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = x[i] * inv;
            // the 20 bits behind a code's mantissa, 8 units around their middle; numbers that
            // become denormal codes have fewer bits
            const unsigned cut = (__float_as_uint(y[i]) & 0xfffffu) - 0x7fff8u;
            near |= cut <= 16u || (fabsf(y[i]) < 0x1p-6f && y[i] != 0.0f);
        }
        if (near) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = quotient_odd(x[i], s);
        }
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    }
}

// What byte `i` of a word of four codes stands for before the scale.
template <int FMT>
__device__ __forceinline__ float code_value(unsigned w, int i) {
    const unsigned b = (w >> (8 * i)) & 0xffu;
    if constexpr (FMT == kI8) return (float)(int)(int8_t)b;
    else return __builtin_amdgcn_cvt_f32_fp8((int)b, 0);
}

// Tokens sequence s holds, and how many of the n rows given for it are real, both within what can be.
__device__ __forceinline__ int seq_length(const shp::Cache8& c, int s) {
    return min(max(c.lengths[s], 0), c.cap);
}
__device__ __forceinline__ int seq_count(const int32_t* counts, int n, int s) {
    return counts ? min(max(counts[s], 0), n) : n;
}

}  // namespace shpd
#endif
