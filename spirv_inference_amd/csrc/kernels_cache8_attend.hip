// Attention over the 8-bit cache, and the accounts of the weight each cached token gets.
//
// A wavefront holds 16 * MT query rows (the rows of all query heads of a KV head, row r = new token
// r / group, head r % group) and walks the sequence's tokens 64 at a time, with the running maximum
// and sum of a softmax.  Codes are exact as fp16, q and the weights are cut into two fp16 pieces of
// 11 bits (both rounded to nearest, so an operand is off by 2^-23 of itself, or of 2^-15 of its row's
// largest where that is more), and the products run on
// v_mfma_f32_16x16x32_f16 with fp32 sums: twice the products of one fp16 pass at 8 times the rate of
// fp32's own matrix instructions.  Against 64 bits (norms) outputs are off by 1.6e-7 on 300 tokens, 4.3e-7
// for 512 rows on 8,190 and 4.9e-7 on 131,072; those of fp32 products by 2.6e-7, 1.6e-6 and 3.2e-6.
//
// Scores are computed transposed, S^T = K Q^T.  Row m of token tile j is given to token
// (m / 4) * 16 + 4 j + m % 4 of the 64: the lane (query l % 16, group g = l / 16) then holds the
// scores of tokens 16 g .. 16 g + 15, all of one block (one scale), and these are the k slots that
// the lane's 16 bytes of a dimension of V stand for in O^T = V^T P^T.  So K and V go from memory to
// the matrix cores without LDS, in 16-byte loads (but see stage_k), and P never leaves its registers.
//
// A row keeps the maximum m of its scores (in units of log2, rounded up to a whole number) and the sum
// of the weights e_t = 2^(score - m), in which V has no part.  What multiplies V's codes is w_t = e_t *
// (scale of V) * 2^(12 - k), k being the running maximum, rounded up, of log2(e_t * scale of V): the
// largest w_t of a row fill fp16's range whatever the scales are.  A token whose e_t * scale is 2^15
// times smaller than the row's largest has fewer bits of w_t, and one 2^37 times smaller none.
// (A single maximum, over log2(weight * scale), with the row's sum made of w_t / scale, is wrong where
// scales lie more than about 2^130 apart: the weight of the tokens with small values is lost.)  Scaling
// is by powers of two, which rounds nothing, and seldom: a maximum has to pass a whole number.
#include "cache8.h"
#include "coherent.h"
#include "gemm.h"

namespace {

using namespace shpd;
using shp::Cache8;
using shp::Cache8Query;
using shp::kCacheTile;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kLift = 12;  // w reaches 2^12: the low piece stays a normal fp16 number longer
constexpr int kRoom = 24;  // log2 of the room for sums of V over tokens
constexpr float kLargeScore = 262144.0f;  // |m| past which the rounding of a score shows in a weight
constexpr float kNoWeight = -126.0f;  // log2 of the smallest weight that counts: normal fp32 numbers
constexpr float kLeastLift = -114.0f;  // ... and that k follows, so that 2^(12 - k) * scale stays finite
constexpr float kNoValues = -1000.0f;  // k before the first token: below all that it can be
constexpr int kQBits = 14;      // a row of q is scaled to reach 2^13 .. 2^14

// Four codes as fp16 numbers.
template <int FMT>
__device__ __forceinline__ void codes4(unsigned w, h2& a, h2& b) {
    if constexpr (FMT == kI8) {
        // the bytes of c + 128 under an exponent of 1024, less 1152
        const unsigned u = w ^ 0x80808080u;
        const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(u, 0x64646464u, 0x01050104u)) + off;
        b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(u, 0x64646464u, 0x01070106u)) + off;
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
}
template <int FMT>
__device__ __forceinline__ h8 codes8(unsigned lo, unsigned hi) {
    h2 a, b, c, d;
    codes4<FMT>(lo, a, b);
    codes4<FMT>(hi, c, d);
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Two numbers as the sum of two fp16 each.
__device__ __forceinline__ void pieces(float x, float y, h2& hi, h2& lo) {
    hi = __builtin_convertvector(f2{x, y}, h2);
    lo = __builtin_convertvector(f2{x - (float)hi.x, y - (float)hi.y}, h2);
}

// f over the lane groups of 16, for every lane: two exchanges of rows of 16 and of 32 lanes.
template <class F>
__device__ __forceinline__ float over_groups(float x, F f) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float max_over_groups(float x) {
    return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_groups(float x) {
    return over_groups(x, [](float a, float b) { return a + b; });
}

// A KV head of a sequence and its query rows.
struct RowSpan {
    int s, h, len, count, rows;
};

// Row r (another one for each l % 16): the pieces of q * scale * log2 e in the B layout, scaled by a
// power of two, in `back` the inverse of that power, and in `limit` how many tokens the row sees.
// Rows behind the last repeat it.
template <int D>
__device__ __forceinline__ void load_q(const Cache8Query& q, const RowSpan& p, int r, h8* hi, h8* lo,
                                       float& back, int& limit) {
    const int g = (threadIdx.x & 63) >> 4;
    const bool real = r < p.rows;
    const int rr = real ? r : p.rows - 1, i = rr / q.group, head = p.h * q.group + rr - i * q.group;
    limit = max(p.len - p.count + i + 1, 0);
    const float* x = q.q + p.s * q.q_seq + i * q.q_row + head * q.q_head + 16 * g;
    f4 v[D / 16];
    float top = 0.0f;
#pragma unroll
    for (int a = 0; a < D / 64; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) v[4 * a + b] = *reinterpret_cast<const f4*>(x + 64 * a + 4 * b);
#pragma unroll
    for (int a = 0; a < D / 16; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            v[a][b] *= q.scale * kLog2e;
            top = fmaxf(top, fabsf(v[a][b]));
        }
    top = max_over_groups(top);
    const int e = kQBits - __builtin_amdgcn_frexp_expf(top);
    back = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
    for (int a = 0; a < D / 32; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const f4 t = v[2 * a + b / 2];
            h2 ph, pl;
            pieces(__builtin_amdgcn_ldexpf(t[2 * (b & 1)], e),
                   __builtin_amdgcn_ldexpf(t[2 * (b & 1) + 1], e), ph, pl);
            hi[a][2 * b] = ph.x;
            hi[a][2 * b + 1] = ph.y;
            lo[a][2 * b] = pl.x;
            lo[a][2 * b + 1] = pl.y;
        }
}

// K of a 64-token tile: raw[j][a] = 16 dimensions (64 a + 16 g) of token (m / 4) * 16 + 4 j + m % 4.
template <int D>
__device__ __forceinline__ void load_k(const uint8_t* tile, u4 raw[4][D / 64]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const uint8_t* p = tile + ((m >> 2) * 16 + (m & 3)) * D + 16 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int a = 0; a < D / 64; ++a)
            raw[j][a] = *reinterpret_cast<const u4*>(p + 4 * j * D + 64 * a);
}
// K's tiles of 128 dimensions go through LDS where 32 rows or more share one: lanes 0 to 15 of load_k
// read 16 bytes each of 16 rows, 16 cache lines, and tiles that many rows want come from L2, where that
// is what costs (512 rows on 8,190 tokens: attention 143 us so, 150 without, accounts 88 and 97 with 32
// rows a wavefront; rows of 64 dimensions are half as many lines and attention takes 94 and 91, and 16
// query rows, which memory bounds, 727 and 720).
template <int D, int MT>
constexpr bool kStaged = D == 128 && MT >= 2;
typedef const __attribute__((address_space(1))) void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// A wavefront's tile to LDS in whole rows, 1 KB a load, without passing its registers.  Piece p (16 bytes)
// of token t's row goes to place p ^ turn(t), turn(t) = t % 4 + 4 * (t / 16 % 2), so that the eight
// lanes that staged() serves at once take different banks.
__device__ __forceinline__ void stage_k(const uint8_t* tile, uint8_t* lds) {
    const int lane = threadIdx.x & 63, t = lane >> 3, at = t * 128 + 16 * ((lane & 7) ^ (t & 3));
#pragma unroll
    for (int i = 0; i < 8; ++i)
        __builtin_amdgcn_global_load_lds((GlobalPtr)(tile + i * 1024 + (at ^ (i & 2 ? 64 : 0))),
                                         (LdsPtr)(lds + i * 1024), 16, 0, 0);
}
// Until the wavefront's tile is there: the compiler does not promise to wait for these loads.
__device__ __forceinline__ void wait_staged() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// raw[j][a] of load_k.
__device__ __forceinline__ u4 staged(const uint8_t* lds, int j, int a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const int t = (m >> 2) * 16 + 4 * j + (m & 3);
    return *reinterpret_cast<const u4*>(lds + t * 128 + 16 * ((4 * a + g) ^ (m & 7)));
}
// V of a 64-token tile: raw[d] = tokens 16 g .. 16 g + 15 of dimension 16 d + m.
template <int D>
__device__ __forceinline__ void load_v(const uint8_t* tile, u4 raw[D / 16]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const uint8_t* p = tile + m * kCacheTile + 16 * g;
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
        raw[d] = *reinterpret_cast<const u4*>(p + d * 16 * kCacheTile);
}

// What a product of codes and pieces of q is multiplied by: finite where K's scale is, so that a product
// of zero is a score of zero however large q and K are.
__device__ __forceinline__ float score_factor(float kscale, float back) {
    return __builtin_elementwise_minimum(kscale * back, 3.4028234663852886e+38f);  // a NaN stays
}

// 2^(m - top), also where both are minus infinity or infinity.
__device__ __forceinline__ float factor_of(float m, float top) {
    return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

// What sums of weights times V are to be multiplied by, from the sum of the weights.
__device__ __forceinline__ float inverse(float l) {
    return l == 0.0f ? 0.0f : (float)(1 << kRoom) / l;
}

// The log of a row's sum from its maximum and sum of weights as the wavefronts keep them.
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// A workgroup's four wavefronts hold the same rows and take a tile each in turn; their parts meet in LDS
// at the end.  (Side by side over rows they would share tiles, but then few rows have to be cut into
// many shares of the tokens, whose parts go through memory: 512 rows x 4 heads on 8,190 tokens 171 us
// that way, 147 so, measured in one run.)  32 rows are what registers allow with two workgroups on a CU:
// 64 rows of 64 dimensions spilled and took 147 us where 32 take 88.  The tokens of a sequence are shared
// out over workgroups while that fills the GPU.
//
// With up to 16 rows reading the cache bounds it: 16 x 128,001-131,072 tokens x 8 heads x 128 (4.2 GB)
// 720 us, 5.9 TB/s, 24 sequences of 0-8,100 tokens 53 us, 3.8 TB/s (46 us where they are all as long as
// the average); a single sequence of 300 tokens takes 5.7 us, which is latency.  With more rows the vector
// unit, busy in 61 % of the cycles, and the matrix unit, busy in 37 %, do between them: 512 rows x 4 heads
// on 8,190 tokens x 8 heads x 128 (66.6 GFLOP, twice that as products of pieces) 143 us, 931 TFLOP/s of
// products.
// (Launch bounds: the wavefronts a SIMD that each variant reaches without spills.)
template <int D, int FMT, int MT>
__global__ __launch_bounds__(256, MT == 2 ? 2 : D == 64 ? 4 : 3) void cache8_attend_kernel(Cache8 c, Cache8Query q, int least,
                                                               float* part, int* counters) {
    constexpr int NO = D / 16;   // accumulators of 16 rows
    constexpr int PW = D + 4;    // floats of a row's part: sums, maximum, weight, two of padding
    // staged tiles of K, then parts of rows
    constexpr bool STAGED = kStaged<D, MT>;
    constexpr int EX = MT * (NO * 4 + 2) * 64, KB = STAGED ? 64 * D : 0;
    __shared__ __attribute__((aligned(16))) float ex[2][EX];
    static_assert(4 * KB <= 2 * EX * 4);
    __shared__ int arrived;
    constexpr int ROWS = 16 * MT, WAVES = 4;
    const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sh = blockIdx.x;
    RowSpan p;
    p.s = sh / c.kv;
    p.h = sh - p.s * c.kv;
    p.len = seq_length(c, p.s);
    p.count = seq_count(q.counts, q.n, p.s);
    p.rows = p.count * q.group;
    const int r0 = (int)(gridDim.y - 1 - blockIdx.y) * ROWS;  // those that see most begin first
    if (r0 >= p.rows) return;

    // tokens the workgroup's last row sees, in as many shares as there are workgroups for it, none of
    // fewer tiles than `least` but the last
    const int last = min(p.rows, r0 + ROWS) - 1;
    const int sees = max(p.len - p.count + last / q.group + 1, 0);
    const int tiles = (sees + kCacheTile - 1) / kCacheTile;
    const int share = max((tiles + (int)gridDim.z - 1) / (int)gridDim.z, least);
    const int splits = max((tiles + share - 1) / share, 1);
    if ((int)blockIdx.z >= splits) return;
    const int tile0 = (int)blockIdx.z * share, tile1 = min(tiles, tile0 + share);

    const uint8_t* kp = c.k + (int64_t)sh * c.cap * D;
    const uint8_t* vp = c.v + (int64_t)sh * c.cap * D;
    const int64_t sbase = (int64_t)sh * (c.cap >> c.block_log2);
    const int last_block = max(p.len - 1, 0) >> c.block_log2;
    uint8_t* const kl = reinterpret_cast<uint8_t*>(&ex[0][0]) + wave * KB;
    u4 kr[4][D / 64], vr[NO];
    float ks = 0.0f, vs = 0.0f;
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        if constexpr (STAGED) {
            stage_k(kp + (int64_t)tile * kCacheTile * D, kl);
        } else {
            load_k<D>(kp + (int64_t)tile * kCacheTile * D, kr);
        }
        load_v<D>(vp + (int64_t)tile * kCacheTile * D, vr);
        const int64_t b = sbase + min((tile * kCacheTile + 16 * g) >> c.block_log2, last_block);
        ks = c.k_scale[b];
        vs = c.v_scale[b];
    };

    float m[MT], l[MT], k[MT], back[MT];
    int limit[MT];
    f4 o[MT][NO];
    h8 qh[MT][D / 32], ql[MT][D / 32];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        load_q<D>(q, p, r0 + 16 * t + li, qh[t], ql[t], back[t], limit[t]);
        m[t] = -__builtin_inff();
        l[t] = 0.0f;
        k[t] = kNoValues;
#pragma unroll
        for (int d = 0; d < NO; ++d) o[t][d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    // tokens that every row sees
    const int open = max(p.len - p.count + r0 / q.group + 1, 0);

    for (int tile = tile0 + wave; tile < tile1; tile += WAVES) {
        const int t0 = tile * kCacheTile;
        // (the next tile's loads ahead of their use cost a wavefront of occupancy and 5 %)
        fetch(tile);
        if constexpr (STAGED) wait_staged();
        const bool edge = t0 + kCacheTile > open;
        f4 sc[MT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int t = 0; t < MT; ++t) sc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int a = 0; a < D / 32; ++a) {
                u4 w;
                if constexpr (STAGED) w = staged(kl, j, a >> 1);
                else w = kr[j][a >> 1];
                const h8 kf = a & 1 ? codes8<FMT>(w.z, w.w) : codes8<FMT>(w.x, w.y);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[t][a], sc[t][j], 0, 0, 0);
                    sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[t][a], sc[t][j], 0, 0, 0);
                }
            }
        }
        // sc[t][j][i]: token t0 + 16 g + 4 j + i, row r0 + 16 t + li
        const float ve = (float)__builtin_amdgcn_frexp_expf(vs);  // V's scale is under 2^ve
        h8 wh[MT][2], wl[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float f = score_factor(ks, back[t]);
            float mx = -__builtin_inff();
            if (edge) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (t0 + 16 * g + 4 * j + i >= limit[t]) sc[t][j][i] = -__builtin_inff();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[t][j][i]);
            // the best of the lane's 16 tokens (rounded: not to be fused with what it is compared with)
            const float best = __builtin_fmaf(mx, f, 0.0f);
            if (__any(best > m[t])) {
                const float top = fmaxf(m[t], __builtin_ceilf(max_over_groups(best)));
                const float step = m[t] == top ? 0.0f : m[t] - top;
                l[t] *= __builtin_amdgcn_exp2f(step);
                k[t] = fmaxf(k[t] + step, kNoValues);
                m[t] = top;
            }
            const float e = best - m[t];
            const bool on = e >= kNoWeight;  // not where the row sees none of the 16
            const float u = on ? fmaxf(e, kLeastLift) + ve : kNoValues;
            if (__any(u > k[t])) {
                const float top = fmaxf(k[t], __builtin_ceilf(max_over_groups(u)));
                const float down = __builtin_amdgcn_exp2f(k[t] - top);
#pragma unroll
                for (int d = 0; d < NO; ++d) o[t][d] *= down;
                k[t] = top;
            }
            const float lift = on ? __builtin_amdgcn_ldexpf(vs, kLift - (int)k[t]) : 0.0f;
            // score - m as one fused step; where scores are so large that their rounding would show
            // (a weight of 2^12, or none), rounded as the maximum was
            const bool large = fabsf(m[t]) > kLargeScore;
            float sum = 0.0f;
            if (edge || __any(large)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = sc[t][j][i];
                        const float y = large ? __builtin_fmaf(x, f, 0.0f) - m[t]
                                              : __builtin_fmaf(x, f, -m[t]);
                        sc[t][j][i] = t0 + 16 * g + 4 * j + i < limit[t]
                                          ? __builtin_amdgcn_exp2f(y) : 0.0f;
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[t][j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][j][i], f, -m[t]));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += sc[t][j][i];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    h2 ph, pl;
                    pieces(sc[t][j][2 * i] * lift, sc[t][j][2 * i + 1] * lift, ph, pl);
                    const int e = 4 * (j & 1) + 2 * i;
                    wh[t][j >> 1][e] = ph.x;
                    wh[t][j >> 1][e + 1] = ph.y;
                    wl[t][j >> 1][e] = pl.x;
                    wl[t][j >> 1][e + 1] = pl.y;
                }
            }
            l[t] += sum;
        }
        if (FMT == kE4M3 && t0 + kCacheTile > p.len) {
            // bytes behind the last token may be NaN codes, which a weight of zero does not cancel
#pragma unroll
            for (int d = 0; d < NO; ++d)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int left = p.len - t0 - 16 * g - 4 * w;
                    vr[d][w] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << 8 * left) - 1;
                }
        }
#pragma unroll
        for (int d = 0; d < NO; ++d) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const h8 vf = e ? codes8<FMT>(vr[d].z, vr[d].w) : codes8<FMT>(vr[d].x, vr[d].y);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wl[t][e], o[t][d], 0, 0, 0);
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wh[t][e], o[t][d], 0, 0, 0);
                }
            }
            // a dimension after the other: what else is begun early does not find registers
            if constexpr (STAGED) __builtin_amdgcn_sched_barrier(0);
        }
    }
    // the lane's numbers once more, which the loop's registers need not hold so
    const int ln = __lane_id(), row = ln & 15, quad = ln >> 4, tid = wave * 64 + ln;
    // the sums of the tokens' weights times V, 2^24 times smaller: with 4,194,304 tokens they are finite
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = sum_over_groups(l[t]);
#pragma unroll
        for (int d = 0; d < NO; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[t][d][i] = __builtin_amdgcn_ldexpf(o[t][d][i], (int)k[t] - kLift - kRoom);
    }

    // the wavefronts' parts, in pairs: the upper one's goes through LDS
    if constexpr (STAGED) __syncthreads();
#pragma unroll
    for (int step = WAVES / 2; step > 0; step >>= 1) {
        float* x = ex[wave & (step - 1)];
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int d = 0; d < NO; ++d)
                    *reinterpret_cast<f4*>(&x[((t * NO + d) * 64 + ln) * 4]) = o[t][d];
                x[(MT * NO * 4 + 2 * t) * 64 + ln] = m[t];
                x[(MT * NO * 4 + 2 * t + 1) * 64 + ln] = l[t];
            }
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float m1 = x[(MT * NO * 4 + 2 * t) * 64 + ln];
                const float l1 = x[(MT * NO * 4 + 2 * t + 1) * 64 + ln];
                const float top = fmaxf(m[t], m1);
                const float f0 = factor_of(m[t], top), f1 = factor_of(m1, top);
                l[t] = l[t] * f0 + l1 * f1;
                m[t] = top;
#pragma unroll
                for (int d = 0; d < NO; ++d)
                    o[t][d] = o[t][d] * f0 +
                              *reinterpret_cast<const f4*>(&x[((t * NO + d) * 64 + ln) * 4]) * f1;
            }
        __syncthreads();
    }

    // a row's place in out and lse
    auto place = [&](int r, int64_t& at, int64_t& at_lse) __attribute__((always_inline)) {
        const int i = r / q.group, head = p.h * q.group + r - i * q.group;
        at = p.s * q.o_seq + i * q.o_row + head * q.o_head;
        at_lse = ((int64_t)p.s * q.heads + head) * q.n + i;
    };
    if (splits == 1) {
        if (wave) return;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = r0 + 16 * t + row;
            if (r >= p.rows) continue;
            int64_t at, at_lse;
            place(r, at, at_lse);
            const float inv = inverse(l[t]);
#pragma unroll
            for (int d = 0; d < NO; ++d)
                *reinterpret_cast<f4*>(q.out + at + 16 * d + 4 * quad) = o[t][d] * inv;
            if (q.lse && quad == 0) q.lse[at_lse] = log_sum(m[t], l[t]);
        }
        return;
    }

    // Every share stores its rows' parts past the caches that other XCDs do not see; the last to
    // arrive joins them, and leaves the counter at zero for the next launch.
    const int unit = (int)blockIdx.y * (int)gridDim.x + sh, rows = min(p.rows - r0, ROWS);
    const __amdgpu_buffer_rsrc_t pr =
        buffer_rsrc(part + (int64_t)unit * gridDim.z * ROWS * PW, (int64_t)gridDim.z * ROWS * PW);
    if (wave == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = 16 * t + row;
            if (r >= rows) continue;
            const unsigned at = (unsigned)(((int)blockIdx.z * ROWS + r) * PW) * 4u;
#pragma unroll
            for (int d = 0; d < NO; ++d)
                st_coh16(pr, at + (16 * d + 4 * quad) * 4u,
                         make_float4(o[t][d].x, o[t][d].y, o[t][d].z, o[t][d].w));
            if (quad == 0) st_coh16(pr, at + D * 4u, make_float4(m[t], l[t], 0.f, 0.f));
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's parts are stored
    __syncthreads();
    if (tid == 0)
        arrived = __hip_atomic_fetch_add((SHP_GLOBAL int*)(counters + unit), 1, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != splits - 1) return;
    if (tid == 0)
        __hip_atomic_store((SHP_GLOBAL int*)(counters + unit), 0, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    // What the shares hold of the rows is on its way (B loads an output at a time) while their maxima and
    // sums, a share to one of 32 lanes, give the factors 2^(m_i - m) and the rows' m and l.  The join is
    // latency (64 rows x 4 heads of 8,190 tokens: 34.5 us in all with a row's shares one after the other and
    // 8 loads on their way, 32.6 so; 4 rows of 8 sequences 18.4, 17.2).
    constexpr int T = D / 4, NE = ROWS * T / 256, B = NE == 1 ? 16 : 8, NR = ROWS / 8;
    float* const factor = &ex[0][0];        // [ROWS][32]
    float* const total = factor + ROWS * 32;  // [ROWS][2]
    const int share_i = tid & 31;
    float4 ml[NR], x[NE][B];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        const int r = (tid >> 5) + 8 * k;
        ml[k] = make_float4(-__builtin_inff(), 0.f, 0.f, 0.f);
        if (share_i < splits && r < rows)
            ml[k] = ld_coh16(pr, (unsigned)((share_i * ROWS + r) * PW + D) * 4u, 0);
    }
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (i0 + i < splits)
#pragma unroll
                for (int n = 0; n < NE; ++n) {
                    const int e = tid + 256 * n, r = min(e / T, rows - 1);
                    x[n][i] = ld_coh16(pr, (unsigned)(((i0 + i) * ROWS + r) * PW + e % T * 4) * 4u, 0);
                }
    };
    load(0);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        float top = ml[k].x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float f = factor_of(ml[k].x, top);
        float sum = ml[k].y * f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        const int r = (tid >> 5) + 8 * k;
        factor[r * 32 + share_i] = f;
        if (share_i == 0) {
            total[2 * r] = top;
            total[2 * r + 1] = sum;
        }
    }
    __syncthreads();
    f4 sum[NE];
#pragma unroll
    for (int n = 0; n < NE; ++n) sum[n] = f4{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < splits; i0 += B) {
        if (i0) load(i0);
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (i0 + i < splits)
#pragma unroll
                for (int n = 0; n < NE; ++n)
                    sum[n] += f4{x[n][i].x, x[n][i].y, x[n][i].z, x[n][i].w} *
                              factor[(tid + 256 * n) / T * 32 + i0 + i];
    }
#pragma unroll
    for (int n = 0; n < NE; ++n) {
        const int e = tid + 256 * n, r = e / T, d = e % T * 4;
        if (r >= rows) continue;
        int64_t at, at_lse;
        place(r0 + r, at, at_lse);
        const float all = total[2 * r + 1];
        *reinterpret_cast<f4*>(q.out + at + d) = sum[n] * inverse(all);
        if (q.lse && d == 0) q.lse[at_lse] = log_sum(total[2 * r], all);
    }
}

// v[e] of lanes l and l ^ STEP added, for the half of the 2 * STEP indices whose STEP bit is the
// lane's own: after steps 8, 4, 2 and 1, v[0] is the sum of v[l % 16] over the 16 lanes.
template <int STEP>
__device__ __forceinline__ void halve(float* v) {
    const bool up = threadIdx.x & STEP;
#pragma unroll
    for (int e = 0; e < STEP; ++e) {
        const float mine = up ? v[e + STEP] : v[e], other = up ? v[e] : v[e + STEP];
        v[e] = mine + __shfl_xor(other, STEP);
    }
}

// Accounts.  A wavefront holds 16 * MT query rows, as for attention, and walks tiles of 64 tokens: the
// weights of a lane's 16 tokens are added over the row tiles, then over the 16 rows of its group, and
// lane l ends up with token l's.  Where a KV head has more rows than that, row groups leave their sums
// in `part` [group][head][capacity] and cache8_weights_join_kernel adds them in order; a group of
// several chunks of rows adds to what its own chunks before left there.  groups == 1 writes the
// accounts themselves.  A decode step is bound by reading K: 24 sequences of 500-8,100 tokens x 8 heads x
// 128 (113 MB) 30 us, 3.8 TB/s.  A prompt's chunk keeps the vector unit busy in 50 % of the cycles (exp2,
// the conversion of K, q's pieces) and the matrix unit in 25 %, and a quarter of the time no wavefront is
// there (the groups do not end together): 512 rows x 8 heads on 8,190 tokens x 4 heads x 64 (16.6
// GFLOP) 50.5 us, of which 5 are the join; 512 rows x 4 heads on 8 heads x 128 (33.3 GFLOP) 76 us.  The log
// sum enters in units of log2, rounded to fp32: against 64 bits the accounts of the chunk are off by
// 4.9e-8 (norms), fp32 torch's by 3.3e-8, those of the decode step by 2.5e-8 both.
template <int D, int FMT, int MT>
__global__ __launch_bounds__(256, 2) void cache8_weights_kernel(Cache8 c, Cache8Query q, int row_waves,
                                                             int groups, int chunks, float* part) {
    constexpr bool STAGED = kStaged<D, MT>;
    __shared__ __attribute__((aligned(16))) uint8_t tiles_k[STAGED ? 4 : 1][STAGED ? 64 * D : 16];
    const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sh = blockIdx.x, tok_waves = 4 / row_waves;
    const int group = (int)blockIdx.y * row_waves + wave % row_waves;
    const int worker = (int)blockIdx.z * tok_waves + wave / row_waves;
    const int workers = (int)gridDim.z * tok_waves;
    RowSpan p;
    p.s = sh / c.kv;
    p.h = sh - p.s * c.kv;
    p.len = seq_length(c, p.s);
    p.count = seq_count(q.counts, q.n, p.s);
    p.rows = p.count * q.group;
    const uint8_t* kp = c.k + (int64_t)sh * c.cap * D;
    const float* ksp = c.k_scale + (int64_t)sh * (c.cap >> c.block_log2);
    const int last_block = max(p.len - 1, 0) >> c.block_log2;
    const int64_t at0 = (int64_t)sh * c.cap;
    float* const out = groups == 1 ? q.acc_out + at0
                                   : part + ((int64_t)group * gridDim.x + sh) * c.cap;
    if (groups == 1 && p.rows == 0) {
        for (int t = worker * 64 + lane; t < p.len; t += workers * 64)
            out[t] = q.acc_in ? q.acc_in[at0 + t] : 0.0f;
        return;
    }

    int before = 0;  // tiles that the group's chunks so far have written
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int r0 = (group * chunks + chunk) * 16 * MT;
        if (r0 >= p.rows) return;
        const int last = min(p.rows, r0 + 16 * MT) - 1;
        const int tiles = (max(p.len - p.count + last / q.group + 1, 0) + kCacheTile - 1) / kCacheTile;
        const int open = max(p.len - p.count + r0 / q.group + 1, 0);  // seen by every row
        h8 qh[MT][D / 32], ql[MT][D / 32];
        float back[MT], at[MT];
        int limit[MT];
        bool whole = true;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = r0 + 16 * t + li;
            load_q<D>(q, p, r, qh[t], ql[t], back[t], limit[t]);
            const int i = min(r, p.rows - 1) / q.group, head = p.h * q.group + min(r, p.rows - 1) - i * q.group;
            const float lse = q.lse[((int64_t)p.s * q.heads + head) * q.n + i];
            // no such row, or one that saw nothing
            if (r >= p.rows || lse == -__builtin_inff()) limit[t] = 0;
            whole = whole && limit[t] > 0;
            at[t] = -lse * kLog2e;
        }
        const bool gaps = !__all(whole);
        int tile = worker;
        uint8_t* const kl = tiles_k[STAGED ? wave : 0];
        u4 kr[4][D / 64];
        float ks = 0.0f;
        auto fetch = [&](int t) __attribute__((always_inline)) {
            if constexpr (STAGED) stage_k(kp + (int64_t)t * kCacheTile * D, kl);
            else load_k<D>(kp + (int64_t)t * kCacheTile * D, kr);
            ks = ksp[min((t * kCacheTile + 16 * g) >> c.block_log2, last_block)];
        };
        if (tile < tiles) fetch(tile);
        if constexpr (STAGED) wait_staged();
        for (; tile < tiles; tile += workers) {
            const int t0 = tile * kCacheTile;
            float v[16], f[MT];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = 0.0f;
#pragma unroll
            for (int t = 0; t < MT; ++t) f[t] = score_factor(ks, back[t]);
            const bool edge = gaps || t0 + kCacheTile > open;
            f4 sc[MT][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int t = 0; t < MT; ++t) sc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int a = 0; a < D / 32; ++a) {
                    u4 w;
                    if constexpr (STAGED) w = staged(kl, j, a >> 1);
                    else w = kr[j][a >> 1];
                    const h8 kf = a & 1 ? codes8<FMT>(w.z, w.w) : codes8<FMT>(w.x, w.y);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[t][a], sc[t][j], 0, 0, 0);
                        sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[t][a], sc[t][j], 0, 0, 0);
                    }
                }
            }
            if (tile + workers < tiles) fetch(tile + workers);
            if (edge) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float w = __builtin_amdgcn_exp2f(
                            __builtin_fmaf(sc[t][e >> 2][e & 3], f[t], at[t]));
                        v[e] += t0 + 16 * g + e < limit[t] ? w : 0.0f;
                    }
            } else {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        v[e] += __builtin_amdgcn_exp2f(
                            __builtin_fmaf(sc[t][e >> 2][e & 3], f[t], at[t]));
            }
            // over the 16 rows of a lane group
            halve<8>(v);
            halve<4>(v);
            halve<2>(v);
            halve<1>(v);
            if constexpr (STAGED) wait_staged();  // before the store, which would be waited for too
            const int t = t0 + lane;
            if (t < p.len) {
                float sum = v[0];
                if (tile < before) sum = out[t] + sum;
                else if (groups == 1 && q.acc_in) sum = q.acc_in[at0 + t] + sum;
                out[t] = sum;
            }
        }
        before = tiles;
    }
}

// acc_out = acc_in + the row groups' sums: a lane a token, a wavefront every fourth group, in order.
__global__ __launch_bounds__(256) void cache8_weights_join_kernel(Cache8 c, Cache8Query q, int groups,
                                                                  int rows_of_group, const float* part) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sh = blockIdx.y, s = sh / c.kv, t = (int)blockIdx.x * 64 + lane;
    const int len = seq_length(c, s), count = seq_count(q.counts, q.n, s);
    if ((int)blockIdx.x * 64 >= len) return;
    const int64_t at = (int64_t)sh * c.cap + t, stride = (int64_t)gridDim.y * c.cap;
    // the groups with a row that sees token t
    const int first = max(t - (len - count), 0) * q.group / rows_of_group;
    const int end = t < len ? (count * q.group + rows_of_group - 1) / rows_of_group : 0;
    float sum = 0.0f;
#pragma unroll 8
    for (int i = first + wave; i < end; i += 4) sum += part[i * stride + at];
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave || t >= len) return;
    q.acc_out[at] = (q.acc_in ? q.acc_in[at] : 0.0f) +
                    ((sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]));
}

}  // namespace

namespace shp {

Cache8Plan cache8_attend_plan(const Cache8& c, int head_dim, int64_t rows, int cu_count,
                              bool may_split) {
    Cache8Plan p;
    // 32 rows a workgroup use each tile for twice the work, 16 leave room for more workgroups on a CU.
    // 32 pay where there is much of both, from 32 pairs of 32 rows and 64 tokens a CU with 128 dimensions
    // (64 rows x 4 heads on 8,190 tokens x 8 heads 33.0 us, 35.5 with 16 rows; 40: 36.6, 33.5; 16: 24.0,
    // 18.9) and 128 with 64, whose tiles cost half (512 rows x 8 heads on 8,190 tokens x 4 heads 88 us, 102;
    // 192: 52, 46; 128: 32, 34; 32 on 600 tokens 11.8, 8.5); and with 128 where blocks of 16 do not find
    // room at once, three on a CU (prompts of 500 x 4 x 8 heads 16.7 us, 21.2; of 350: 15.9, 12.5).
    const int64_t cu = std::max(cu_count, 1), heads = (int64_t)c.n_seqs * c.kv;
    const int64_t pairs = heads * ((rows + 31) / 32) * (c.cap / kCacheTile);
    const bool many = head_dim == 64 ? pairs >= 128 * cu
                                     : pairs >= 32 * cu || heads * ((rows + 15) / 16) > 3 * cu;
    p.row_tiles = rows > 16 && many ? 2 : 1;
    const int64_t per = 16 * p.row_tiles;
    p.row_blocks = (int)((rows + per - 1) / per);
    // Workgroups for 8 on every CU where a head has no more than 16 rows, which evens out sequences of
    // different length (64 x 3,000-6,000 tokens: 123 us, 134 with 4 and 127 with 16 a CU); for 3 with
    // more blocks of 16 (8 rows x 4 heads of 8 sequences on 4,000 tokens 25.6, 28.6 with 5), and for the
    // two that a CU holds at once with 32 (64 rows x 4 heads: 44 us with 4 a CU, 42 with one, where two
    // took 35).  A workgroup takes two tiles a wavefront or more (300 tokens 5.8 us, 7.1 from one tile; 4
    // rows of 8 sequences 17.2, 23.8; 1,000 tokens 8.3, 7.3), a sequence 32 shares at most, whose parts one
    // workgroup joins (32,000 tokens 24.6 us with 32, 29.9 with 16).
    const int64_t units = heads * p.row_blocks;
    const int64_t want = ((p.row_tiles == 2 ? 2 : p.row_blocks > 1 ? 3 : 8) * cu + units - 1) / units;
    p.least = 8;
    const int64_t most = (c.cap / kCacheTile + p.least - 1) / p.least;
    p.splits = (int)std::max<int64_t>(std::min<int64_t>(std::min(want, most), 32), 1);
    if (!may_split || units * (int64_t)sizeof(int) > (int64_t)kSplitCounterBytes) p.splits = 1;
    p.scratch = p.splits > 1 ? (size_t)units * per * p.splits * (head_dim + 4) : 0;
    return p;
}

int cache8_attend_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                         const Cache8Query& q, const Cache8Plan& p, float* scratch, int* counters) {
    const bool i8 = format == SHP_CACHE8_I8;
    auto kern = head_dim == 64
        ? (p.row_tiles == 1   ? (i8 ? cache8_attend_kernel<64, kI8, 1> : cache8_attend_kernel<64, kE4M3, 1>)
                              : (i8 ? cache8_attend_kernel<64, kI8, 2> : cache8_attend_kernel<64, kE4M3, 2>))
        : (p.row_tiles == 1   ? (i8 ? cache8_attend_kernel<128, kI8, 1> : cache8_attend_kernel<128, kE4M3, 1>)
                              : (i8 ? cache8_attend_kernel<128, kI8, 2> : cache8_attend_kernel<128, kE4M3, 2>));
    hipLaunchKernelGGL(kern, dim3(c.n_seqs * c.kv, p.row_blocks, p.splits), dim3(256), 0, s, c, q,
                       p.least, scratch, counters);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

// A row group a wavefront, as long as their sums fit 64 MiB.  With 16 rows about 8,192 wavefronts;
// with more, which take longer to load (their q is cut into pieces), no more than the 2,048 that are
// held at once (512 rows on 8,190 tokens 62 -> 51 us).  Each has four tiles or more.  64 rows a wavefront
// read K half as often as 32 and begin half as many times, which pays where there is work for all: from
// 8 pairs of 64 rows and 64 tokens for each wavefront that is held with 128 dimensions (8 heads of 1,024
// rows on 8,190 tokens 47.0 us, 51.3 with 32 rows; of 800: 57.4, 52.3) and from 4 with 64 (4 heads of
// 1,024 rows 20.4, 22.3; of 256: 13.7, 10.6; a last group of 32 rows costs more so: 16 heads of 800 rows
// on 4,000 tokens 37.7, 36.3).
Cache8WeightsPlan cache8_weights_plan(const Cache8& c, int head_dim, int64_t rows, bool may_group) {
    Cache8WeightsPlan p;
    const int64_t pairs = (int64_t)c.n_seqs * c.kv * ((rows + 63) / 64) * (c.cap / kCacheTile);
    p.row_tiles = rows <= 16 ? 1 : rows <= 32 || pairs < (head_dim == 128 ? 8 : 4) * 2048 ? 2 : 4;
    const int64_t per = 16 * p.row_tiles, all = std::max<int64_t>((rows + per - 1) / per, 1);
    const int64_t heads = (int64_t)c.n_seqs * c.kv, one = heads * c.cap;
    int64_t groups = may_group ? std::min(all, std::max<int64_t>((16ll << 20) / one, 1)) : 1;
    p.chunks = (int)((all + groups - 1) / groups);
    p.groups = (int)((all + p.chunks - 1) / p.chunks);
    p.row_waves = p.groups >= 4 ? 4 : p.groups >= 2 ? 2 : 1;
    const int64_t tok_waves = 4 / p.row_waves, tiles = c.cap / kCacheTile;
    const int64_t want = (p.row_tiles == 1 ? 8192 : 2048) / std::max<int64_t>(heads * p.groups, 1), most = (tiles + 3) / 4;
    p.workers = (int)((std::max<int64_t>(std::min(want, most), 1) + tok_waves - 1) / tok_waves);
    p.scratch = p.groups > 1 ? (size_t)(one * p.groups) : 0;
    return p;
}

int cache8_weights_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                          const Cache8Query& q, const Cache8WeightsPlan& p, float* scratch) {
    const bool i8 = format == SHP_CACHE8_I8;
    auto kern = head_dim == 64
        ? (p.row_tiles == 1   ? (i8 ? cache8_weights_kernel<64, kI8, 1> : cache8_weights_kernel<64, kE4M3, 1>)
           : p.row_tiles == 2 ? (i8 ? cache8_weights_kernel<64, kI8, 2> : cache8_weights_kernel<64, kE4M3, 2>)
                              : (i8 ? cache8_weights_kernel<64, kI8, 4> : cache8_weights_kernel<64, kE4M3, 4>))
        : (p.row_tiles == 1   ? (i8 ? cache8_weights_kernel<128, kI8, 1> : cache8_weights_kernel<128, kE4M3, 1>)
           : p.row_tiles == 2 ? (i8 ? cache8_weights_kernel<128, kI8, 2> : cache8_weights_kernel<128, kE4M3, 2>)
                              : (i8 ? cache8_weights_kernel<128, kI8, 4> : cache8_weights_kernel<128, kE4M3, 4>));
    hipLaunchKernelGGL(kern, dim3(c.n_seqs * c.kv, (p.groups + p.row_waves - 1) / p.row_waves, p.workers),
                       dim3(256), 0, s, c, q, p.row_waves, p.groups, p.chunks, scratch);
    SHP_HIP_CHECK(hipGetLastError());
    if (p.groups > 1) {
        hipLaunchKernelGGL(cache8_weights_join_kernel, dim3(c.cap / kCacheTile, c.n_seqs * c.kv),
                           dim3(256), 0, s, c, q, p.groups, 16 * p.row_tiles * p.chunks, scratch);
        SHP_HIP_CHECK(hipGetLastError());
    }
    return SHP_OK;
}

}  // namespace shp
