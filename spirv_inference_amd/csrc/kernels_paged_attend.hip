// Attention over the paged cache.
//
// A wavefront holds 16 * MT query rows (the rows of all query heads of a KV head, row r = new token
// r / group, head r % group) and walks the tokens that any of them sees, a tile at a time, with the
// running maximum and sum of a softmax.  fp16 and bf16 keys and values enter the matrix cores as they
// are; q and the weights are cut into two fp16 pieces of 11 bits (scaled by powers of two: an operand is
// off by 2^-23 of itself, or 2^-38 of the row's largest where that is more) or three bf16 pieces of 8
// bits (exact), so that fp32's accuracy costs two or three products at 16 times the rate of fp32's own,
// which fp32 caches use.
//
// Scores are computed transposed, S^T = K Q^T: the lane (query l % 16, group g = l / 16) then holds the
// scores of tokens 16 j + 4 g + i of a tile, and these are the k slots that it has to hold of P^T in
// O^T = V^T P^T.  Which dimension a row of V^T is does not matter to the product, so a lane takes dimensions
// that lie next to each other: V comes in loads of whole rows, 16-bit values are turned around within the
// lane (one byte permutation for two), and neither K, V nor P passes LDS.
//
// Weights are 2^(x - m), x being scores in units of log2 and m the running maximum, rounded up to a whole
// number and moved by a shift that is the same for all tokens: up for fp32 and bf16, so that sums of weights
// times V are no larger than V, down by 14 for fp16, so that the low piece stays a normal number
// longer.  Scaling is by powers of two, which rounds nothing, and seldom: a maximum has to pass a
// whole number.
#include "coherent.h"
#include "gemm.h"
#include "paged.h"

namespace {

using namespace shpd;
using shp::kTreeRows;
using shp::Paged;
using shp::PagedPlan;
using shp::PagedQuery;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef bf16 b8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLargeScore = 4194304.0f;  // |m| from which a shift would not be exact
constexpr int kQBits = 14;                 // fp16: a row of q is scaled to reach 2^13 .. 2^14
constexpr int kLift = 14;                  // fp16: weights reach 2^14

// How many pieces an fp32 operand is cut into beside values of this type.
template <class E> constexpr int kPieces = 1;
template <> constexpr int kPieces<_Float16> = 2;
template <> constexpr int kPieces<bf16> = 3;
template <class E> constexpr bool kF32 = sizeof(E) == 4;
// Tokens of a tile: 8 KB of K, 8 KB of V.
template <class E, int D> constexpr int kTile = 8192 / (D * (int)sizeof(E));

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
__device__ __forceinline__ int min_over_rows(int x) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int max_over_rows(int x) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}

// Two numbers as pieces, next to each other in a word of each.
template <class E>
__device__ __forceinline__ void cut(float x, float y, unsigned* piece) {
    if constexpr (sizeof(E) == 2 && kPieces<E> == 2) {
        const h2 hi = __builtin_convertvector(f2{x, y}, h2);
        const h2 lo = __builtin_convertvector(f2{x - (float)hi.x, y - (float)hi.y}, h2);
        piece[0] = __builtin_bit_cast(unsigned, hi);
        piece[1] = __builtin_bit_cast(unsigned, lo);
    } else {
        // the upper 16 bits, and what is left of the number, three times: nothing is rounded
        unsigned a = __float_as_uint(x), b = __float_as_uint(y);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            piece[p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            if (p == 2) break;
            a = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xffff0000u));
            b = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xffff0000u));
        }
    }
}

template <class E>
__device__ __forceinline__ f4 mfma32(u4 a, u4 b, f4 c) {
    if constexpr (kPieces<E> == 2)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// The bits of an infinity, and of 1 (16-bit types).
template <class E> constexpr unsigned kInf = kF32<E> ? 0x7f800000u : kPieces<E> == 2 ? 0x7c00u : 0x7f80u;
template <class E> constexpr unsigned kOne = kPieces<E> == 2 ? 0x3c00u : 0x3f80u;
// Whether the value with these bits is a NaN or the infinity of this sign.
template <class E>
__device__ __forceinline__ bool not_finite(unsigned x, int minus) {
    constexpr unsigned kSign = kF32<E> ? 0x80000000u : 0x8000u;
    const unsigned a = x & (kSign - 1);
    return a > kInf<E> || x == (minus ? kSign | kInf<E> : kInf<E>);
}
// Dimension d (of two in a word) of two tokens' words, side by side.
__device__ __forceinline__ unsigned dims_of(unsigned first, unsigned second, int d) {
    return __builtin_amdgcn_perm(second, first, d & 1 ? 0x07060302u : 0x05040100u);
}

// tanh: its series below 0.35 (the next term is 2^-26 of the value), 1 - 2 / (e^2|x| + 1) above.
__device__ __forceinline__ float tanh_of(float x) {
    const float a = fabsf(x), y = x * x;
    const float near = x + x * y * (-1.0f / 3 + y * (2.0f / 15 + y * (-17.0f / 315 + y * (62.0f / 2835 - y * (1382.0f / 155925)))));
    const float e = __builtin_amdgcn_exp2f(a * (2 * kLog2e));
    const float far = __builtin_copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f), x);
    return a < 0.35f ? near : far;
}

// Bits 0 .. n - 1.
__device__ __forceinline__ uint64_t below(int n) {
    return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// 2^(m - top), also where both are minus infinity or infinity.
__device__ __forceinline__ float factor_of(float m, float top) {
    return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}
// The log of a row's sum from its shifted maximum and sum of weights.
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// A drafted tree's rows: bit u of above[i] says that row u is row i or above it and within its window or
// the prefix, depth[i] how many rows are above row i.
struct Tree {
    uint64_t above[kTreeRows][kTreeRows / 64];
    uint16_t parent[kTreeRows], depth[kTreeRows];
};

// Which tokens a row sees: [first, len) of those in [lo, hi), before `prefix` or among its tree's.
struct Sight {
    int lo, hi, first, position, node;
};

template <class E, int D, int MT>
__global__ __launch_bounds__(256, 2) void paged_attend_kernel(Paged c, PagedQuery q, int least, float* part,
                                                              int* counters) {
    constexpr bool F32 = kF32<E>;
    constexpr int NP = kPieces<E>, NO = D / 16, TT = kTile<E, D>, NJ = TT / 16;
    constexpr int NQ = F32 ? D / 16 : D / 32;  // 16-byte pieces of a row of K that a lane takes
    constexpr int ROWS = 16 * MT, WAVES = 4, PW = D + 4;
    constexpr int EX = MT * (NO * 4 + 2) * 64;
    __shared__ __attribute__((aligned(16))) float ex[2][EX];
    static_assert(sizeof(Tree) <= sizeof(ex), "the tree lies where the wavefronts' parts go later");
    __shared__ int arrived;
    Tree& tree = *reinterpret_cast<Tree*>(&ex[0][0]);
    const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sh = blockIdx.x, s = sh / c.kv, h = sh - s * c.kv;
    const int len = paged_length(c, s), count = paged_count(q.counts, q.n, s), begin = len - count;
    const int nrows = count * q.group;
    const int r0 = (int)(gridDim.y - 1 - blockIdx.y) * ROWS;  // those that see most begin first
    if (r0 >= nrows) return;
    const bool drafted = q.parents != nullptr;
    const int window = q.window ? min(q.window, 1 << 30) : 1 << 30;
    const int prefix_all = q.prefix ? min(max(q.prefix[s], 0), len) : 0;
    const int prefix = drafted ? min(prefix_all, max(begin, 0)) : prefix_all;

    if (drafted) {
        const int i = threadIdx.x;
        if (i < count) {
            const int p = q.parents[(int64_t)s * q.n + i];
            tree.parent[i] = (uint16_t)(p >= 0 && p < i ? p : 0xffff);
        }
        __syncthreads();
        if (i < count) {
            uint64_t up[kTreeRows / 64] = {};
            int steps = 0;
            for (int u = i; u != 0xffff; u = tree.parent[u], ++steps)  // falls
                if (steps < window || begin + u < prefix_all) {
#pragma unroll
                    for (int w = 0; w < kTreeRows / 64; ++w)
                        up[w] |= u >> 6 == w ? 1ull << (u & 63) : 0ull;
                }
            tree.depth[i] = (uint16_t)(steps - 1);
#pragma unroll
            for (int w = 0; w < kTreeRows / 64; ++w) tree.above[i][w] = up[w];
        }
        __syncthreads();
    }

    // the lane's rows; those behind the last repeat it
    Sight see[MT];
    float slope[MT];
    const float* qrow[MT];
    int low = 0x7fffffff, high = 0, least_first = 0x7fffffff, open_lo = 0, open_hi = 0x7fffffff;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = min(r0 + 16 * t + li, nrows - 1), i = r / q.group, head = h * q.group + r - i * q.group;
        const int place = begin + i;
        Sight& v = see[t];
        v.node = i;
        v.position = drafted ? begin + tree.depth[i] : place;
        v.hi = drafted ? begin : place + 1;
        v.lo = max(v.position - window + 1, 0);
        v.first = q.first ? max(q.first[(int64_t)s * q.n + i], 0) : 0;
        if (place < 0) v.first = 0x7fffffff;  // sees nothing
        slope[t] = q.slopes ? q.slopes[head] * kLog2e : 0.0f;
        qrow[t] = q.q + s * q.q_seq + i * q.q_row + head * q.q_head;
        low = min(low, max(v.lo, v.first));
        high = max(high, place < 0 ? 0 : drafted ? place + 1 : v.hi);
        least_first = min(least_first, v.first);
        open_lo = max(open_lo, max(v.lo, v.first));
        open_hi = min(open_hi, v.hi);
    }
    low = min_over_rows(low);
    high = max_over_rows(high);
    least_first = min_over_rows(least_first);
    open_lo = max_over_rows(open_lo);
    open_hi = min_over_rows(open_hi);
    // a token of a tree may be nearer by position than by place
    if (drafted) low = min(low, max(begin, 0));

    // the tiles that any row sees a token of: of the prefix [a0, a0 + na), then [b0, b0 + nb)
    const int a0 = min(least_first, prefix) / TT, na = prefix > least_first ? (prefix + TT - 1) / TT - a0 : 0;
    const int b0 = na ? max(low / TT, a0 + na) : low / TT, nb = max((min(high, len) + TT - 1) / TT - b0, 0);
    const int tiles = na + nb;
    const int share = max((tiles + (int)gridDim.z - 1) / (int)gridDim.z, least);
    const int splits = max((tiles + share - 1) / share, 1);
    if ((int)blockIdx.z >= splits) return;
    const int tile0 = (int)blockIdx.z * share, tile1 = min(tiles, tile0 + share);

    // q's pieces in the B layout
    float m[MT], l[MT], back[MT];
    f4 o[MT][NO];
    u4 qp[MT][NQ][NP];
    const bool capped = q.cap > 0.0f;
    const float factor = capped ? q.scale / q.cap : q.scale * kLog2e;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t] = -__builtin_inff();
        l[t] = 0.0f;
        back[t] = 1.0f;
#pragma unroll
        for (int d = 0; d < NO; ++d) o[t][d] = f4{0.f, 0.f, 0.f, 0.f};
        if constexpr (F32) {
#pragma unroll
            for (int a = 0; a < NQ; ++a)
                qp[t][a][0] = __builtin_bit_cast(u4, *reinterpret_cast<const f4*>(qrow[t] + 16 * a + 4 * g) * factor);
        } else {
            f4 v[2 * NQ];
            float top = 0.0f;
#pragma unroll
            for (int a = 0; a < 2 * NQ; ++a) {
                v[a] = *reinterpret_cast<const f4*>(qrow[t] + 32 * (a >> 1) + 8 * g + 4 * (a & 1)) * factor;
#pragma unroll
                for (int b = 0; b < 4; ++b) top = fmaxf(top, fabsf(v[a][b]));
            }
            if constexpr (NP == 2) {
                top = max_over_groups(top);
                const int e = min(kQBits - __builtin_amdgcn_frexp_expf(top), 100);
                back[t] = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
                for (int a = 0; a < 2 * NQ; ++a)
#pragma unroll
                    for (int b = 0; b < 4; ++b) v[a][b] = __builtin_amdgcn_ldexpf(v[a][b], e);
            }
#pragma unroll
            for (int a = 0; a < NQ; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    unsigned piece[NP];
                    cut<E>(v[2 * a + (b >> 1)][2 * (b & 1)], v[2 * a + (b >> 1)][2 * (b & 1) + 1], piece);
#pragma unroll
                    for (int p = 0; p < NP; ++p) qp[t][a][p][b] = piece[p];
                }
        }
    }
    const float shift = NP == 2 ? (float)-kLift : (float)(32 - __builtin_clz(max(len, 1)));
    const E* const kb = (const E*)c.k;
    const E* const vb = (const E*)c.v;
    const int last = max(len - 1, 0);
    // what lies in a lane's registers of a tile: tokens 16 j + li of K, and of V those of its k slots
    constexpr int VW = F32 ? D / 64 : 1;         // loads of a row of V
    constexpr int VB = F32 ? 4 : D / 32;         // words of each
    typedef unsigned VWord __attribute__((ext_vector_type(VB)));

    for (int at = tile0 + wave; at < tile1; at += WAVES) {
        const int t0 = (at < na ? a0 + at : b0 + at - na) * TT;
        u4 kr[NJ][NQ];
        VWord vr[NJ][4][VW];
        uint64_t there = ~0ull;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int t = min(t0 + 16 * j, last & ~15);  // a page holds whole groups of 16
            int page = page_of(c, s, t);
            if (page < 0) {
                page = 0;
                there &= ~(0xffffull << (16 * j));
            }
            const int64_t row = row_of(c, page, h, t) * D;
#pragma unroll
            for (int a = 0; a < NQ; ++a)
                kr[j][a] = *reinterpret_cast<const u4*>(kb + row + li * D + (F32 ? 16 * a + 4 * g : 32 * a + 8 * g));
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < VW; ++w)
                    vr[j][i][w] = *reinterpret_cast<const VWord*>(vb + row + (4 * g + i) * D + (F32 ? 64 * w + 4 * li : NO * li));
        }
        // whether every row sees the whole tile
        const bool edge = (~there & below(TT)) || t0 < open_lo || t0 + TT > open_hi;
        f4 sc[MT][NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int t = 0; t < MT; ++t) sc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int a = 0; a < NQ; ++a)
#pragma unroll
                for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if constexpr (F32) {
#pragma unroll
                            for (int b = 0; b < 4; ++b)
                                sc[t][j] = mfma4(__uint_as_float(kr[j][a][b]), __uint_as_float(qp[t][a][0][b]), sc[t][j]);
                        } else {
                            sc[t][j] = mfma32<E>(kr[j][a], qp[t][a][p], sc[t][j]);
                        }
                    }
        }
        // sc[t][j][i]: token t0 + 16 j + 4 g + i, row r0 + 16 t + li
        uint64_t seen[MT];  // bit 16 j + i: the lane's tokens
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if constexpr (NP == 2) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) sc[t][j] *= back[t];
            }
            if (capped) {
                const float top = q.cap * kLog2e;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[t][j][i] = top * tanh_of(sc[t][j][i]);
            }
            if (q.slopes) {
                const bool mixed = drafted && t0 + TT > begin;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        int at_k = t0 + 16 * j + 4 * g + i;
                        if (mixed && at_k >= begin && at_k < len) at_k = begin + tree.depth[at_k - begin];
                        sc[t][j][i] -= slope[t] * fabsf((float)(see[t].position - at_k));
                    }
            }
            seen[t] = ~0ull;
            if (edge) {
                const Sight& v = see[t];
                uint64_t bits = (below(v.hi - t0) & ~below(v.lo - t0)) | below(prefix - t0);
                if (drafted && t0 + TT > begin) {
                    // the tree's bits from t0 on: those of rows t0 - begin ..
                    const uint64_t* up = tree.above[v.node];
                    const int u = t0 - begin;
                    if (u < 0) {
                        bits |= up[0] << -u;  // -u < TT
                    } else {
                        const int w = u >> 6, b = u & 63;
                        uint64_t x = w < kTreeRows / 64 ? up[w] >> b : 0ull;
                        if (b && w + 1 < kTreeRows / 64) x |= up[w + 1] << (64 - b);
                        bits |= x;
                    }
                }
                bits &= below(len - t0) & ~below(v.first == 0x7fffffff ? 64 : v.first - t0) & there;
                seen[t] = bits >> (4 * g);
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(seen[t] >> (16 * j + i) & 1)) sc[t][j][i] = -__builtin_inff();
            }
            float best = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) best = fmaxf(best, sc[t][j][i]);
            if (__any(best > m[t] - shift)) {
                float top = __builtin_ceilf(max_over_groups(best));
                if (fabsf(top) < kLargeScore) top += shift;
                top = fmaxf(m[t], top);
                const float down = factor_of(m[t], top);
                l[t] *= down;
#pragma unroll
                for (int d = 0; d < NO; ++d) o[t][d] *= down;
                m[t] = top;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = __builtin_amdgcn_exp2f(sc[t][j][i] - m[t]);
                    sc[t][j][i] = edge && !(seen[t] >> (16 * j + i) & 1) ? 0.0f : w;
                    sum += sc[t][j][i];
                }
            l[t] += sum;
        }

        // Where some row does not see some token, a value that is not finite would spoil that row too: such a
        // value is added to the rows that see it, as an infinity of its sign, a NaN as both, and taken out.
        if (edge) {
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int w = 0; w < VW; ++w)
#pragma unroll
                        for (int b = 0; b < VB; ++b) {
                            const unsigned x = vr[j][i][w][b] & 0x7fffffffu;
                            top = max(top, F32 ? x : max(x, (x & 0x7fffu) << 16));
                        }
            if (__any(top >= kInf<E> << (F32 ? 0 : 16))) {
#pragma unroll
                for (int d = 0; d < NO; ++d)
#pragma unroll
                    for (int minus = 0; minus < 2; ++minus)
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            f4 hits = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (F32) {
#pragma unroll
                                for (int j = 0; j < NJ; ++j)
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        hits = mfma4(not_finite<E>(vr[j][i][d >> 2][d & 3], minus) ? 1.0f : 0.0f,
                                                     seen[t] >> (16 * j + i) & 1 ? 1.0f : 0.0f, hits);
                            } else {
#pragma unroll
                                for (int e = 0; e < NJ / 2; ++e) {
                                    u4 x, y;
#pragma unroll
                                    for (int b = 0; b < 4; ++b) {
                                        const int j = 2 * e + (b >> 1), i = 2 * (b & 1);
                                        const unsigned v = dims_of(vr[j][i][0][d >> 1], vr[j][i + 1][0][d >> 1], d);
                                        x[b] = (not_finite<E>(v & 0xffffu, minus) ? kOne<E> : 0u) |
                                               (not_finite<E>(v >> 16, minus) ? kOne<E> << 16 : 0u);
                                        y[b] = (seen[t] >> (16 * j + i) & 1 ? kOne<E> : 0u) |
                                               (seen[t] >> (16 * j + i + 1) & 1 ? kOne<E> << 16 : 0u);
                                    }
                                    hits = mfma32<E>(x, y, hits);
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (hits[i] > 0.0f) o[t][d][i] += minus ? -__builtin_inff() : __builtin_inff();
                        }
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int w = 0; w < VW; ++w)
#pragma unroll
                            for (int b = 0; b < VB; ++b) {
                                unsigned& x = *(reinterpret_cast<unsigned*>(&vr[j][i][w]) + b);
                                if constexpr (F32) {
                                    if ((x & kInf<E>) == kInf<E>) x = 0u;
                                } else {
                                    if ((x & kInf<E>) == kInf<E>) x &= 0xffff0000u;
                                    if ((x >> 16 & kInf<E>) == kInf<E>) x &= 0xffffu;
                                }
                            }
            }
        }
        // O^T += V^T P^T
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < NO; ++d)
#pragma unroll
                        for (int t = 0; t < MT; ++t)
                            o[t][d] = mfma4(__uint_as_float(vr[j][i][d >> 2][d & 3]), sc[t][j][i], o[t][d]);
        } else {
#pragma unroll
            for (int e = 0; e < NJ / 2; ++e) {
                u4 wp[MT][NP];
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int j = 2 * e + (b >> 1), i = 2 * (b & 1);
                        unsigned piece[NP];
                        cut<E>(sc[t][j][i], sc[t][j][i + 1], piece);
#pragma unroll
                        for (int p = 0; p < NP; ++p) wp[t][p][b] = piece[p];
                    }
#pragma unroll
                for (int d = 0; d < NO; ++d) {
                    u4 vf;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int j = 2 * e + (b >> 1), i = 2 * (b & 1);
                        vf[b] = dims_of(vr[j][i][0][d >> 1], vr[j][i + 1][0][d >> 1], d);
                    }
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                        for (int t = 0; t < MT; ++t) o[t][d] = mfma32<E>(vf, wp[t][p], o[t][d]);
                }
            }
        }
    }

    // the lane's numbers once more, which the loop's registers need not hold so
    const int ln = __lane_id(), row = ln & 15, quad = ln >> 4, tid = wave * 64 + ln;
#pragma unroll
    for (int t = 0; t < MT; ++t) l[t] = sum_over_groups(l[t]);

    // the wavefronts' parts, in pairs: the upper one's goes through LDS (where the tree was)
    __syncthreads();
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

    // four dimensions next to each other of the lane's, and the first of them
    auto run = [&](int t, int n) __attribute__((always_inline)) {
        constexpr bool WIDE = !F32 && D == 128;  // a lane holds 8 dimensions in a row, not 4
        const int i = WIDE ? n >> 1 : n & 3, x = WIDE ? 4 * (n & 1) : 4 * (n >> 2);
        return f4{o[t][x][i], o[t][x + 1][i], o[t][x + 2][i], o[t][x + 3][i]};
    };
    auto dim = [&](int n) __attribute__((always_inline)) {
        return !F32 && D == 128 ? 32 * quad + 4 * n : 64 * (n >> 2) + 16 * quad + 4 * (n & 3);
    };
    // a row's place in out and lse
    auto place = [&](int r, int64_t& to, int64_t& to_lse) __attribute__((always_inline)) {
        const int i = r / q.group, head = h * q.group + r - i * q.group;
        to = s * q.o_seq + i * q.o_row + head * q.o_head;
        to_lse = ((int64_t)s * q.heads + head) * q.n + i;
    };
    if (splits == 1) {
        if (wave) return;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = r0 + 16 * t + row;
            if (r >= nrows) continue;
            int64_t to, to_lse;
            place(r, to, to_lse);
#pragma unroll
            for (int n = 0; n < NO; ++n)
                *reinterpret_cast<f4*>(q.out + to + dim(n)) = l[t] == 0.0f ? f4{0.f, 0.f, 0.f, 0.f} : run(t, n) / l[t];
            if (q.lse && quad == 0) q.lse[to_lse] = log_sum(m[t], l[t]);
        }
        return;
    }

    // Every share stores its rows' parts past the caches that other XCDs do not see; the last to
    // arrive joins them, and leaves the counter at zero for the next launch.
    const int unit = (int)blockIdx.y * (int)gridDim.x + sh, rows = min(nrows - r0, ROWS);
    const __amdgpu_buffer_rsrc_t pr =
        buffer_rsrc(part + (int64_t)unit * gridDim.z * ROWS * PW, (int64_t)gridDim.z * ROWS * PW);
    if (wave == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = 16 * t + row;
            if (r >= rows) continue;
            const unsigned to = (unsigned)(((int)blockIdx.z * ROWS + r) * PW) * 4u;
#pragma unroll
            for (int n = 0; n < NO; ++n) {
                const f4 x = run(t, n);
                st_coh16(pr, to + dim(n) * 4u, make_float4(x.x, x.y, x.z, x.w));
            }
            if (quad == 0) st_coh16(pr, to + D * 4u, make_float4(m[t], l[t], 0.f, 0.f));
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
    // sums, a share to one of 32 lanes, give the factors 2^(m_i - m) and the rows' m and l.
    constexpr int T = D / 4, NE = ROWS * T / 256, B = NE == 1 ? 16 : 8, NR = ROWS / 8;
    float* const factors = &ex[0][0];          // [ROWS][32]
    float* const total = factors + ROWS * 32;  // [ROWS][2]
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
        for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
        const float f = factor_of(ml[k].x, top);
        float sum = ml[k].y * f;
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
        const int r = (tid >> 5) + 8 * k;
        factors[r * 32 + share_i] = f;
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
                              factors[(tid + 256 * n) / T * 32 + i0 + i];
    }
#pragma unroll
    for (int n = 0; n < NE; ++n) {
        const int e = tid + 256 * n, r = e / T, d = e % T * 4;
        if (r >= rows) continue;
        int64_t to, to_lse;
        place(r0 + r, to, to_lse);
        const float all = total[2 * r + 1];
        *reinterpret_cast<f4*>(q.out + to + d) = all == 0.0f ? f4{0.f, 0.f, 0.f, 0.f} : sum[n] / all;
        if (q.lse && d == 0) q.lse[to_lse] = log_sum(total[2 * r], all);
    }
}

}  // namespace

namespace shp {

PagedPlan paged_attend_plan(const Paged& c, int head_dim, int64_t rows, int cu_count, bool may_split) {
    PagedPlan p;
    const int64_t cu = std::max(cu_count, 1), heads = (int64_t)c.n_seqs * c.kv;
    p.row_tiles = rows > 16 ? 2 : 1;
    const int64_t per = 16 * p.row_tiles;
    p.row_blocks = (int)((rows + per - 1) / per);
    const int64_t units = heads * p.row_blocks;
    const int64_t want = ((p.row_blocks > 1 ? 2 : 8) * cu + units - 1) / units;
    p.least = 8;
    const int64_t most = (c.cap / 16 + p.least - 1) / p.least;
    p.splits = (int)std::max<int64_t>(std::min<int64_t>(std::min(want, most), 32), 1);
    if (!may_split || units * (int64_t)sizeof(int) > (int64_t)kSplitCounterBytes) p.splits = 1;
    p.scratch = p.splits > 1 ? (size_t)units * per * p.splits * (head_dim + 4) : 0;
    return p;
}

int paged_attend_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedQuery& q,
                        const PagedPlan& p, float* scratch, int* counters) {
    with_format(format, [&](auto e) {
        using E = decltype(e);
        auto kern = head_dim == 64
                        ? (p.row_tiles == 1 ? paged_attend_kernel<E, 64, 1> : paged_attend_kernel<E, 64, 2>)
                        : (p.row_tiles == 1 ? paged_attend_kernel<E, 128, 1> : paged_attend_kernel<E, 128, 2>);
        hipLaunchKernelGGL(kern, dim3(c.n_seqs * c.kv, p.row_blocks, p.splits), dim3(256), 0, s, c, q, p.least,
                           scratch, counters);
    });
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

}  // namespace shp
