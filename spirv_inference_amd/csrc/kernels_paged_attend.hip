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
#include <cmath>
#include <type_traits>

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
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
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

// The bits of an infinity.
template <class E> constexpr unsigned kInf = kF32<E> ? 0x7f800000u : kPieces<E> == 2 ? 0x7c00u : 0x7f80u;
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

// All ones where bit n is set: selects by it need no scalar registers.
__device__ __forceinline__ unsigned mask_of(uint64_t bits, int n) {
    return (unsigned)__builtin_amdgcn_sbfe((int)(unsigned)(n < 32 ? bits : bits >> 32), n & 31, 1);
}

// 2^(m - top), also where both are minus infinity or infinity.
__device__ __forceinline__ float factor_of(float m, float top) {
    return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}
// What sums of weights times V are to be multiplied by, from the sum of the weights.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
// The log of a row's sum from its shifted maximum and sum of weights.
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// A drafted tree's rows: bit u of above[i] says that row u is row i of the workgroup's or above it and within its
// window or the prefix; depth[i] is how many rows are above row i of the tree.
struct Tree {
    uint64_t above[32][kTreeRows / 64];  // 32 query rows are of 32 tokens at most
    uint16_t parent[kTreeRows], depth[kTreeRows];
};

// A KV head of a sequence and its rows.
struct Unit {
    int s, h, len, count, begin, nrows;
    int window, prefix_all, prefix;  // prefix: of it what is no tree's
    bool drafted;
};

// What a workgroup does: a block of rows of a KV head, and of the tiles that they see the shares
// z * share .. of `shares`.  With target = 0 it is a place in the grid, and all tiles.  Else the blocks and the tiles
// of all sequences are counted and cut into shares of one size, `target` of them or less; a workgroup finds its own in
// their running sum, or that there is none for it.  A share is of one block, whose last may be shorter, so that blocks
// nearly as many as `target` are hardly cut: 24 sequences of 0-8,100 tokens x 8 heads have shares of 58 tiles where a
// workgroup's mean is 48 (82 us, 94 with a number of shares by sequence), trees of 60 rows of 16 sequences 123 and 73, and
// 64 such sequences have the longest whole, 254 and 127 (224 us, 190 of as many tokens in equal lengths).
struct Task {
    int s, h, len, count, block, z, share, shares, first;  // first: the place of its rows' first part and of their counter
    bool any;
};
// The running f over the lanes, in six steps that stay in registers; f(x, 0) = x.
template <class T, class F>
__device__ __forceinline__ T over_lanes(T x, F f) {
    auto step = [&](auto shift, auto rows) __attribute__((always_inline)) {
        const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), shift.value, rows.value, 0xf, false);
        x = f(x, __builtin_bit_cast(T, y));
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // from 1, 2, 4 and 8 lanes below in a row of 16
    step(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
    step(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
    step(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
    step(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // rows 1 and 3 from the last lane below
    step(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());  // rows 2 and 3 from lane 31
    return x;
}
template <class T>
__device__ __forceinline__ T last_lane(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
template <int T, int ROWS, int D>
__device__ __forceinline__ Task task_of(const Paged& c, const PagedQuery& q, int target, int least) {
    Task k;
    if (target == 0) {
        const int id = (int)blockIdx.x;
        k.s = (int)fdiv((unsigned)id, q.by_kv);
        k.h = id - k.s * c.kv;
        k.len = paged_length(c, k.s);
        k.count = paged_count(q.counts, q.n, k.s);
        k.block = (int)(gridDim.y - 1 - blockIdx.y);  // those that see most begin first
        k.z = 0;
        k.share = 1 << 30;
        k.shares = 1;
        k.first = 0;
        k.any = true;
        return k;
    }
    const int lane = threadIdx.x & 63;
    // a sequence's blocks, and the tiles that a block sees of it, no more than those that a window touches (with a
    // prefix all count: a row on 100,000 tokens x 8 heads x 128 in bf16 with a window of 4,096 14 us, and 37 with a
    // prefix of 4 as well)
    const int most = q.window && !q.prefix ? (min(q.window, 1 << 22) + q.n) / T + 2 : 1 << 22;
    int len, count, blocks, tiles;
    auto size = [&](int s0) __attribute__((always_inline)) {
        const bool real = s0 + lane < c.n_seqs;
        len = real ? paged_length(c, s0 + lane) : 0;
        count = real ? paged_count(q.counts, q.n, s0 + lane) : 0;
        blocks = (count * q.group + ROWS - 1) / ROWS;
        tiles = max(min((len + T - 1) / T, most), 1);
    };
    int top = 1, units = 0;
    float all = 0.0f;
    for (int s0 = 0; s0 < c.n_seqs; s0 += 64) {
        size(s0);
        all += (float)blocks * (float)tiles;
        top = max(top, tiles);
        units += blocks;
    }
    const auto add = [](auto a, auto b) { return a + b; };
    all = last_lane(over_lanes(all, add));
    units = last_lane(over_lanes(units, add)) * c.kv;
    top = last_lane(over_lanes(top, [](int a, int b) { return max(a, b); }));
    // running sums of the sequences' workgroups, 64 sequences at a time
    int mine, to;
    auto count_up = [&](int s0) __attribute__((always_inline)) {
        if (c.n_seqs > 64) size(s0);
        mine = c.kv * blocks * ((tiles + k.share - 1) / k.share);
        to = over_lanes(mine, add);
        return last_lane(to);
    };
    // `target` workgroups, or a whole number of times that
    const int room = max((units + target - 1) / target, 1) * target;
    // (32 shares of a block at most, 16 of 32 rows of 128 dimensions, whose parts one workgroup joins: at the
    // 30 GB/s that a CU reads it takes 9 us for 270 KB.  8 rows x 4 heads of 2 sequences on 100,000 tokens 132 us, 153
    // with twice as many; of 64 dimensions 57 with 32, 70 with 16)
    constexpr int kShares = ROWS * D <= 2048 ? 32 : 16;
    k.share = max(max((int)(all * (float)c.kv / (float)room), (top + kShares - 1) / kShares), least);
    int n;
    for (;; k.share += k.share / 16 + 1) {
        n = 0;
        for (int s0 = 0; s0 < c.n_seqs; s0 += 64) n += count_up(s0);
        if (n <= room) break;  // no more than `units` where a share has all tiles
    }
    // Workgroups with numbers 8 apart run on one XCD, one after the other: each XCD gets a run of the tasks, in which
    // blocks of rows that read the same tokens are neighbours.
    const int run = (n + 7) / 8, id = (int)(blockIdx.x & 7) * run + (int)(blockIdx.x >> 3);
    k.any = (int)(blockIdx.x >> 3) < run && id < n;
    for (int s0 = 0, sum = 0; k.any; s0 += 64) {
        const int all_here = c.n_seqs > 64 ? count_up(s0) : n;
        const uint64_t behind = __ballot(sum + to > id);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            k.s = s0 + at;
            k.len = __builtin_amdgcn_readlane(len, at);
            k.count = __builtin_amdgcn_readlane(count, at);
            const int nb = __builtin_amdgcn_readlane(blocks, at);
            const int start = sum + __builtin_amdgcn_readlane(to, at) - __builtin_amdgcn_readlane(mine, at);
            k.shares = (__builtin_amdgcn_readlane(tiles, at) + k.share - 1) / k.share;
            const int off = id - start, rest = off / nb;
            // those that see most first, every eighth one after the other: an XCD that gets a part of them gets a
            // part of each kind
            const int p = off - rest * nb, eighth = nb >> 3, more = nb & 7, head = more * (eighth + 1);
            const int x = p < head ? p / (eighth + 1) : more + (p - head) / max(eighth, 1);
            const int y = p < head ? p - x * (eighth + 1) : p - head - (x - more) * eighth;
            k.block = nb - 1 - (y * 8 + x);
            k.h = rest / k.shares;
            k.z = rest - k.h * k.shares;
            k.first = start + (k.h * nb + k.block) * k.shares;
            break;
        }
        sum += all_here;
    }
    return k;
}
__device__ __forceinline__ Unit unit_of(const PagedQuery& q, const Task& k) {
    Unit u;
    u.s = k.s;
    u.h = k.h;
    u.len = k.len;
    u.count = k.count;
    u.begin = u.len - u.count;
    u.nrows = u.count * q.group;
    u.drafted = q.parents != nullptr;
    u.window = q.window ? min(q.window, 1 << 30) : 1 << 30;
    u.prefix_all = q.prefix ? min(max(shared_int(q.prefix, k.s), 0), u.len) : 0;
    u.prefix = u.drafted ? min(u.prefix_all, max(u.begin, 0)) : u.prefix_all;
    return u;
}

// The workgroup's threads walk up the tree from a row each.  Its own rows are those from `own` on.
template <int THREADS>
__device__ __forceinline__ void climb(const PagedQuery& q, const Unit& u, int own, Tree& tree) {
    for (int i = threadIdx.x; i < u.count; i += THREADS) {
        const int p = q.parents[(int64_t)u.s * q.n + i];
        tree.parent[i] = (uint16_t)(p >= 0 && p < i ? p : 0xffff);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < u.count; i += THREADS) {
        uint64_t up[kTreeRows / 64] = {};
        int steps = 0;
        for (int v = i; v != 0xffff; v = tree.parent[v], ++steps)  // falls
            if (steps < u.window || u.begin + v < u.prefix_all) {
#pragma unroll
                for (int w = 0; w < kTreeRows / 64; ++w) up[w] |= v >> 6 == w ? 1ull << (v & 63) : 0ull;
            }
        tree.depth[i] = (uint16_t)(steps - 1);
        if (i >= own && i < own + 32) {
#pragma unroll
            for (int w = 0; w < kTreeRows / 64; ++w) tree.above[i - own][w] = up[w];
        }
    }
    __syncthreads();
}

// Bounds of what rows [ra, rb) see, the same for all lanes: nothing outside [low, high) and
// [least_first, prefix); each row all of [open_lo, open_hi), if that is not empty.
struct Span {
    int low, high, least_first, open_lo, open_hi;
};
__device__ __forceinline__ Span span_of(const PagedQuery& q, const Unit& u, int ra, int rb) {
    const int i0 = (int)fdiv((unsigned)ra, q.by_group), i1 = (int)fdiv((unsigned)(rb - 1), q.by_group);
    const int p0 = u.begin + i0, p1 = u.begin + i1;
    Span v;
    // a tree's rows are at positions from begin up to their place
    v.low = max((u.drafted ? u.begin : p0) - u.window + 1, 0);
    v.high = max(p1 + 1, 0);
    v.open_lo = p0 < 0 ? 0x7fffffff : max(p1 - u.window + 1, 0);
    v.open_hi = u.drafted ? u.begin : p0 + 1;
    v.least_first = 0;
    if (q.first) {
        int a = 0x7fffffff, b = 0;
        for (int i = i0 + (threadIdx.x & 63); i <= i1; i += 64) {
            const int f = max(q.first[(int64_t)u.s * q.n + i], 0);
            a = min(a, f);
            b = max(b, f);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            a = min(a, __shfl_xor(a, o));
            b = max(b, __shfl_xor(b, o));
        }
        v.least_first = __builtin_amdgcn_readfirstlane(a);
        v.low = max(v.low, v.least_first);
        v.open_lo = max(v.open_lo, __builtin_amdgcn_readfirstlane(b));
    }
    return v;
}

// The tiles of T tokens that any row of a span sees a token of: of the prefix [a0, a0 + na), then from b0 on.
template <int T>
struct Tiles {
    int a0, na, b0, all;
    __device__ __forceinline__ Tiles(const Unit& u, const Span& v) {
        a0 = v.least_first / T;
        na = u.prefix > v.least_first ? (u.prefix + T - 1) / T - a0 : 0;
        b0 = na ? max(v.low / T, a0 + na) : v.low / T;
        all = na + max((min(v.high, u.len) + T - 1) / T - b0, 0);
    }
    __device__ __forceinline__ int begin(int k) const { return (k < na ? a0 + k : b0 + k - na) * T; }
};

// Which tokens a row sees: [first, len) of those in [lo, hi), before the prefix or among its tree's.
struct Sight {
    int lo, hi, first, position, node;  // node: of the workgroup's
};

// 16 * MT rows of a wavefront, and what it has of their softmax.  LARGE: the cap is large.
template <class E, int D, int MT, bool LARGE>
struct Wave {
    static constexpr bool F32 = kF32<E>;
    static constexpr int NP = kPieces<E>, NO = D / 16, TT = kTile<E, D>, NJ = TT / 16;
    static constexpr int NQ = F32 ? D / 16 : D / 32;  // 16-byte pieces of a row of K that a lane takes
    static constexpr int VW = F32 ? D / 64 : 1;       // loads of a row of V
    static constexpr int VB = F32 ? 4 : D / 32;       // words of each
    static constexpr int PW = D + 4;                  // floats of a row's part: sums, maximum, weight, two of padding
    typedef unsigned VWord __attribute__((ext_vector_type(VB)));
    // The lowest of three pieces of 32 rows of 128 dimensions stays in LDS, which the registers do not hold with
    // the other two (a tree of 60 rows x 4 heads 16 times on 4,100 tokens: 610 us where they spill).
    static constexpr int NL = NP == 3 && MT == 2 && D == 128 ? 1 : 0, NR = NP - NL;

    f4 o[MT][NO];
    u4 qp[MT][NQ][NR];
    float m[MT], l[MT], slope[MT], back[MT];
    Sight see[MT];
    int lift[LARGE ? MT : 1];  // the power of two that a row's products lack

    // Rows from r0 on; those behind the last repeat it.  raw: the lane's part of them.
    __device__ __forceinline__ void begin(const PagedQuery& q, const Unit& u, const uint16_t* depth, int node0, int r0, f4 raw[MT][2 * D / 32]) {
        const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = min(r0 + 16 * t + li, u.nrows - 1), i = (int)fdiv((unsigned)r, q.by_group);
            const int head = u.h * q.group + r - i * q.group, place = u.begin + i;
            const float* x = q.q + u.s * q.q_seq + i * q.q_row + head * q.q_head;
#pragma unroll
            for (int a = 0; a < D / 16; ++a)
                raw[t][a] = *reinterpret_cast<const f4*>(x + (F32 ? 16 * a + 4 * g : 32 * (a >> 1) + 8 * g + 4 * (a & 1)));
            Sight& v = see[t];
            v.node = i - node0;
            v.position = u.drafted ? u.begin + depth[i] : place;
            v.hi = u.drafted ? u.begin : place + 1;
            v.lo = max(v.position - u.window + 1, 0);
            v.first = q.first ? max(q.first[(int64_t)u.s * q.n + i], 0) : 0;
            if (place < 0) v.first = 0x7fffffff;  // sees nothing
            slope[t] = q.slopes ? q.slopes[head] * kLog2e : 0.0f;
        }
    }
    // The rows' pieces in the B layout, times the scale; nothing seen yet.  low: those that LDS holds.
    __device__ __forceinline__ void pieces(const PagedQuery& q, f4 v[MT][2 * D / 32], u4* low, bool mine) {
        const float factor = LARGE ? q.factor : q.cap > 0.0f ? q.scale / q.cap : q.scale * kLog2e;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            back[t] = 1.0f;
            if constexpr (LARGE) {
                float top = 0.0f;
#pragma unroll
                for (int a = 0; a < D / 16; ++a)
#pragma unroll
                    for (int b = 0; b < 4; ++b) top = fmaxf(top, fabsf(v[t][a][b]));
                const int e = __builtin_amdgcn_frexp_expf(max_over_groups(top));
                lift[t] = e + q.lift;
#pragma unroll
                for (int a = 0; a < D / 16; ++a)
#pragma unroll
                    for (int b = 0; b < 4; ++b) v[t][a][b] = __builtin_amdgcn_ldexpf(v[t][a][b], -e);
            }
#pragma unroll
            for (int a = 0; a < D / 16; ++a) v[t][a] *= factor;
            if constexpr (F32) {
#pragma unroll
                for (int a = 0; a < NQ; ++a) qp[t][a][0] = __builtin_bit_cast(u4, v[t][a]);
            } else {
                if constexpr (NP == 2) {
                    float top = 0.0f;
#pragma unroll
                    for (int a = 0; a < 2 * NQ; ++a)
#pragma unroll
                        for (int b = 0; b < 4; ++b) top = fmaxf(top, fabsf(v[t][a][b]));
                    top = max_over_groups(top);
                    const int e = min(kQBits - __builtin_amdgcn_frexp_expf(top), 100);
                    back[t] = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
                    for (int a = 0; a < 2 * NQ; ++a)
#pragma unroll
                        for (int b = 0; b < 4; ++b) v[t][a][b] = __builtin_amdgcn_ldexpf(v[t][a][b], e);
                }
#pragma unroll
                for (int a = 0; a < NQ; ++a) {
                    u4 lowest;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        unsigned piece[NP];
                        cut<E>(v[t][2 * a + (b >> 1)][2 * (b & 1)], v[t][2 * a + (b >> 1)][2 * (b & 1) + 1], piece);
#pragma unroll
                        for (int p = 0; p < NR; ++p) qp[t][a][p][b] = piece[p];
                        lowest[b] = piece[NP - 1];
                    }
                    if (NL && mine) low[(t * NQ + a) * 64 + (threadIdx.x & 63)] = lowest;
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // the sums take the registers that the rows had
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            m[t] = -__builtin_inff();
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < NO; ++d) o[t][d] = f4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // A tile from token t0 on.  key(j, a) gives 16 bytes of token 16 j + l % 16, value(j, i, w) words of token
    // 16 j + 4 g + i; `there` says which of its tokens have a page.
    // number(token, dimension) is one of the tile's values.
    template <class K, class V, class N>
    __device__ __forceinline__ void step(const PagedQuery& q, const Unit& u, const uint64_t (*above)[kTreeRows / 64],
                                         const uint16_t* depth, const Span& span, float shift,
                                         int t0, uint64_t there, const u4* low, K key, V value, N number) {
        const int g = (threadIdx.x & 63) >> 4;
        // whether some row does not see some token
        // (a tile of the prefix in front of the window as well, though all rows see it whole)
        const bool edge = (~there & below(TT)) || t0 < span.open_lo || t0 + TT > span.open_hi;
        f4 sc[MT][NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) sc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int a = 0; a < NQ; ++a) {
            if constexpr (NL) {
                u4 lowest[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) lowest[t] = low[(t * NQ + a) * 64 + (threadIdx.x & 63)];
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int t = 0; t < MT; ++t) sc[t][j] = mfma32<E>(key(j, a), lowest[t], sc[t][j]);
            }
#pragma unroll
            for (int p = NR - 1; p >= 0; --p)
#pragma unroll
                for (int b = 0; b < (F32 ? 4 : 1); ++b)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            if constexpr (F32)
                                sc[t][j] = mfma4(__uint_as_float(key(j, a)[b]), __uint_as_float(qp[t][a][0][b]), sc[t][j]);
                            else
                                sc[t][j] = mfma32<E>(key(j, a), qp[t][a][p], sc[t][j]);
                        }
        }
        // sc[t][j][i]: token t0 + 16 j + 4 g + i, row r0 + 16 t + li
        uint64_t seen[MT];  // the row's tokens of the tile
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if constexpr (NP == 2) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) sc[t][j] *= back[t];
            }
            if constexpr (LARGE) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[t][j][i] = 2.0f * (q.half * tanh_of(__builtin_amdgcn_ldexpf(sc[t][j][i], lift[t])));
            } else if (q.cap > 0.0f) {
                const float top = q.cap * kLog2e;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[t][j][i] = top * tanh_of(sc[t][j][i]);
            }
            if (q.slopes) {
                if (u.drafted && t0 + TT > u.begin) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = t0 + 16 * j + 4 * g + i, up = min(max(at - u.begin, 0), max(u.count - 1, 0));
                            const int position = at < u.begin ? at : u.begin + depth[up];
                            sc[t][j][i] -= slope[t] * fabsf((float)(see[t].position - position));
                        }
                } else {
                    const float far = (float)(see[t].position - t0 - 4 * g);
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[t][j][i] -= slope[t] * fabsf(far - (float)(16 * j + i));
                }
            }
            seen[t] = ~0ull;
            if (edge) {
                const Sight& v = see[t];
                uint64_t bits = (below(v.hi - t0) & ~below(v.lo - t0)) | below(u.prefix - t0);
                if (u.drafted && t0 + TT > u.begin) {
                    // the tree's bits from t0 on: those of rows t0 - begin ..
                    const uint64_t* up = above[v.node];
                    const int from = t0 - u.begin;
                    if (from < 0) {
                        bits |= up[0] << -from;  // -from < TT
                    } else {
                        const int w = from >> 6, b = from & 63;
                        uint64_t x = w < kTreeRows / 64 ? up[w] >> b : 0ull;
                        if (b && w + 1 < kTreeRows / 64) x |= up[w + 1] << (64 - b);
                        bits |= x;
                    }
                }
                bits &= below(u.len - t0) & ~below(v.first == 0x7fffffff ? 64 : v.first - t0) & there;
                seen[t] = bits;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned w = mask_of(bits >> (4 * g), 16 * j + i);
                        sc[t][j][i] = __uint_as_float((__float_as_uint(sc[t][j][i]) & w) | (0xff800000u & ~w));
                    }
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
            if (edge) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = __builtin_amdgcn_exp2f(sc[t][j][i] - m[t]);
                        sc[t][j][i] = __uint_as_float(__float_as_uint(w) & mask_of(seen[t] >> (4 * g), 16 * j + i));
                        sum += sc[t][j][i];
                    }
            } else {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[t][j][i] = __builtin_amdgcn_exp2f(sc[t][j][i] - m[t]);
                        sum += sc[t][j][i];
                    }
            }
            l[t] += sum;
        }

        VWord vr[NJ][4][VW];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < VW; ++w) vr[j][i][w] = value(j, i, w);
        // Where some row does not see some token, a value that is not finite would spoil that row too: such a
        // value is added to the rows that see it and taken out.
        if (edge && not_finite(vr)) {
#pragma unroll 1
                for (int token = 0; token < TT; ++token)
#pragma unroll
                    for (int d = 0; d < NO; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = number(token, dim_of(g, d, i));
#pragma unroll
                            for (int t = 0; t < MT; ++t)
                                if (!(fabsf(x) <= 3.4028234663852886e+38f) && (seen[t] >> token & 1)) o[t][d][i] += x;
                        }
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int w = 0; w < VW; ++w)
#pragma unroll
                            for (int b = 0; b < VB; ++b) {
                                unsigned x = vr[j][i][w][b];
                                if constexpr (F32) {
                                    if ((x & kInf<E>) == kInf<E>) x = 0u;
                                } else {
                                    if ((x & kInf<E>) == kInf<E>) x &= 0xffff0000u;
                                    if ((x >> 16 & kInf<E>) == kInf<E>) x &= 0xffffu;
                                }
                                vr[j][i][w][b] = x;
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

    // The dimension that o[t][d][i] of lane group g is.
    static __device__ __forceinline__ int dim_of(int g, int d, int i) {
        return !F32 && D == 128 ? 32 * g + 8 * i + d : 64 * (d >> 2) + 16 * g + 4 * i + (d & 3);
    }
    // Whether some of a tile's values is an infinity or a NaN.
    static __device__ __forceinline__ bool not_finite(const VWord vr[NJ][4][VW]) {
        // the largest exponents, of 16-bit values in both halves of a word
        us2 top2 = {0, 0};
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < VW; ++w)
#pragma unroll
                    for (int b = 0; b < VB; ++b) {
                        const unsigned x = vr[j][i][w][b];
                        if constexpr (F32) top = max(top, x & 0x7fffffffu);
                        else top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(us2, x & 0x7fff7fffu));
                    }
        if constexpr (!F32) top = max((unsigned)top2.x, (unsigned)top2.y);
        return __any(top >= kInf<E>);
    }
    // Four dimensions next to each other of the lane's, and the first of them.
    __device__ __forceinline__ f4 run(int t, int n) const {
        constexpr bool WIDE = !F32 && D == 128;  // a lane holds 8 dimensions in a row, not 4
        const int i = WIDE ? n >> 1 : n & 3, x = WIDE ? 4 * (n & 1) : 4 * (n >> 2);
        return f4{o[t][x][i], o[t][x + 1][i], o[t][x + 2][i], o[t][x + 3][i]};
    }
    static __device__ __forceinline__ int dim(int quad, int n) {
        return !F32 && D == 128 ? 32 * quad + 4 * n : 64 * (n >> 2) + 16 * quad + 4 * (n & 3);
    }
    // The results of rows r0 .., which saw all of their tokens.
    __device__ __forceinline__ void store(const PagedQuery& q, const Unit& u, int r0) const;
    // The same as parts of the rows, `row` floats in front of the first.
    __device__ __forceinline__ void store_part(__amdgpu_buffer_rsrc_t to, int row, int rows) const {
        const int ln = __lane_id(), li = ln & 15, quad = ln >> 4;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = 16 * t + li;
            if (r >= rows) continue;
            const unsigned at = (unsigned)((row + r) * PW) * 4u;
#pragma unroll
            for (int n = 0; n < NO; ++n) {
                const f4 x = run(t, n);
                st_coh16(to, at + dim(quad, n) * 4u, make_float4(x.x, x.y, x.z, x.w));
            }
            if (quad == 0) st_coh16(to, at + D * 4u, make_float4(m[t], l[t], 0.f, 0.f));
        }
    }
};

// A row's place in out and lse.
__device__ __forceinline__ void place_of(const PagedQuery& q, const Unit& u, int r, int64_t& to, int64_t& to_lse) {
    const int i = (int)fdiv((unsigned)r, q.by_group), head = u.h * q.group + r - i * q.group;
    to = u.s * q.o_seq + i * q.o_row + head * q.o_head;
    to_lse = ((int64_t)u.s * q.heads + head) * q.n + i;
}

template <class E, int D, int MT, bool LARGE>
__device__ __forceinline__ void Wave<E, D, MT, LARGE>::store(const PagedQuery& q, const Unit& u, int r0) const {
    const int ln = __lane_id(), li = ln & 15, quad = ln >> 4;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = r0 + 16 * t + li;
        if (r >= u.nrows) continue;
        int64_t to, to_lse;
        place_of(q, u, r, to, to_lse);
        const float inv = inverse(l[t]);
#pragma unroll
        for (int n = 0; n < NO; ++n) *reinterpret_cast<f4*>(q.out + to + dim(quad, n)) = run(t, n) * inv;
        if (q.lse && quad == 0) q.lse[to_lse] = log_sum(m[t], l[t]);
    }
}

// The workgroup has stored its part of rows r0 .. r0 + rows - 1 past the caches that other XCDs do not
// see; the last of `splits` to arrive joins the parts, 32 rows at a time, and leaves the counter at zero
// for the next launch.  `room`: (32 + 2) * min(ROWS, 32) floats of LDS.
template <int D, int ROWS>
__device__ __forceinline__ void join(const PagedQuery& q, const Unit& u, __amdgpu_buffer_rsrc_t pr, int* counter, int splits,
                                     int r0, int rows, float* room, int* arrived) {
    constexpr int PW = D + 4, RB = ROWS < 32 ? ROWS : 32;
    const int tid = threadIdx.x;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's parts are stored
    __syncthreads();
    if (tid == 0)
        *arrived = __hip_atomic_fetch_add((SHP_GLOBAL int*)counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*arrived != splits - 1) return;
    if (tid == 0) __hip_atomic_store((SHP_GLOBAL int*)counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // What the shares hold of the rows is on its way (B loads an output at a time) while their maxima and
    // sums, a share to one of 32 lanes, give the factors 2^(m_i - m) and the rows' m and l.
    constexpr int T = D / 4, NE = RB * T / 256, B = NE == 1 ? 16 : 8, NR = RB / 8;
    float* const factors = room;            // [RB][32]
    float* const total = factors + RB * 32;  // [RB][2]
    const int share_i = tid & 31;
    for (int rb = 0; rb < rows; rb += RB) {
        const int left = min(rows - rb, RB);
        float4 ml[NR], x[NE][B];
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int r = (tid >> 5) + 8 * k;
            ml[k] = make_float4(-__builtin_inff(), 0.f, 0.f, 0.f);
            if (share_i < splits && r < left)
                ml[k] = ld_coh16(pr, (unsigned)((share_i * ROWS + rb + r) * PW + D) * 4u, 0);
        }
        auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < B; ++i)
                if (i0 + i < splits)
#pragma unroll
                    for (int n = 0; n < NE; ++n) {
                        const int e = tid + 256 * n, r = min(e / T, left - 1);
                        x[n][i] = ld_coh16(pr, (unsigned)(((i0 + i) * ROWS + rb + r) * PW + e % T * 4) * 4u, 0);
                    }
        };
        load(0);
        if (rb) __syncthreads();  // the factors of the rows before have been used
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
            if (r >= left) continue;
            int64_t to, to_lse;
            place_of(q, u, r0 + rb + r, to, to_lse);
            const float all = total[2 * r + 1];
            *reinterpret_cast<f4*>(q.out + to + d) = sum[n] * inverse(all);
            if (q.lse && d == 0) q.lse[to_lse] = log_sum(total[2 * r], all);
        }
    }
}

// Few rows, or a long way through the tokens: the four wavefronts of a workgroup hold the same rows and take a tile
// each in turn; their parts meet in LDS at the end.  Many rows that see little each (SIDE): a workgroup is one
// wavefront, which takes all tiles.  K and V go from memory to registers.
//
// With 16 rows reading the cache bounds it: 16 x 128,001-131,072 tokens x 8 heads x 128 in fp16 (8.5 GB) 1,410 us,
// 6.0 TB/s; 24 sequences of 0-8,100 tokens in bf16 with capped scores (399 MB) 82 us, 4.9 TB/s; 300 tokens 8.7 us, which
// is latency (a CU reads 30 GB/s, and shares cost 3 us for their parts' way through memory).  With more rows the vector
// and the matrix unit do: a SIMD runs instructions of the two side by side only in small part (48 products and 192
// additions, each 0.36 us by itself for a thousand rounds of one wavefront, take 0.61 interleaved as well as they can be), so
// that the kernel's time is nearly the sum of both: 60-row trees of 16 sequences in bf16 90 us, 38 % of it products and
// 37 % other instructions; documents in 4,090 tokens 151 us, 38 % and 46 %.  512 rows x 4 heads on 8,190 tokens x 8 heads x
// 128 in fp32 655 us, 102 TFLOP/s, its matrix unit busy for 68 % and its vector unit for 6 %: a tile has 16 tokens
// there, and a step of the softmax, lookups and the wait for K and V come after every 128 products.  (Loads of K and V
// that ran ahead into LDS gained nothing, nor did wavefronts of different priority.)
// (Launch bounds: the wavefronts a SIMD that each variant reaches with few spills, which are outside the loop.  With a
// large cap 16 rows of 128 dimensions in bf16 reach two: 24 sequences 83 us, 98 with three.)
template <class E, int D, int MT, bool SIDE, bool LARGE>
__global__ __launch_bounds__(SIDE ? 64 : 256, MT == 1 ? (D == 64 ? 4 : LARGE ? 2 : 3) : 2) void paged_attend_kernel(
    Paged c, PagedQuery q, int target, int least, float* part, int* counters) {
    typedef Wave<E, D, MT, LARGE> W;
    constexpr int NO = W::NO, TT = W::TT, NJ = W::NJ, NQ = W::NQ, WAVES = SIDE ? 1 : 4, PW = W::PW;
    constexpr int ROWS = 16 * MT, EX = MT * (NO * 4 + 2) * 64;  // floats of a wavefront's part
    constexpr bool F32 = W::F32;
    __shared__ __attribute__((aligned(16))) float ex[SIDE ? 1 : WAVES / 2][SIDE ? 4 : EX];
    __shared__ u4 lowest[W::NL ? MT * NQ * 64 : 1];
    __shared__ Tree tree;
    __shared__ int arrived;
    const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Task task = task_of<TT, ROWS, D>(c, q, target, least);
    if (!task.any) return;
    const Unit u = unit_of(q, task);
    const int r0 = task.block * ROWS;
    if (r0 >= u.nrows) return;
    const Span span = span_of(q, u, r0, min(r0 + ROWS, u.nrows));
    const Tiles<TT> tiles(u, span);
    const int splits = min(max((tiles.all + task.share - 1) / task.share, 1), task.shares);
    if (task.z >= splits) return;
    const int tile0 = task.z * task.share, tile1 = task.z == splits - 1 ? tiles.all : tile0 + task.share;
    const int node0 = (int)fdiv((unsigned)r0, q.by_group);  // the first row's token
    if (u.drafted) climb<64 * WAVES>(q, u, node0, tree);

    W x;
    {
        f4 raw[MT][D / 16];
        x.begin(q, u, tree.depth, node0, r0, raw);
        x.pieces(q, raw, lowest, wave == 0);
    }
    if (W::NL && !SIDE) __syncthreads();
    const float shift = W::NP == 2 ? (float)-kLift : (float)(32 - __builtin_clz(max(u.len, 1)));
    const E* const kb = (const E*)c.k;
    const E* const vb = (const E*)c.v;
    const int last = max(u.len - 1, 0) & ~15;
    for (int at = tile0 + wave; at < tile1; at += WAVES) {
        const int t0 = tiles.begin(at);
        uint64_t there = ~0ull;  // the tokens that have a page, of which each holds whole groups of 16
        int pages[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) pages[j] = shared_page_of(c, u.s, min(t0 + 16 * j, last));
        int64_t row[NJ];
        u4 kr[NJ][NQ];
        typename W::VWord vr[NJ][4][W::VW];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (pages[j] < 0) there &= ~(0xffffull << (16 * j));
            row[j] = row_of(c, max(pages[j], 0), u.h, min(t0 + 16 * j, last)) * D;
#pragma unroll
            for (int a = 0; a < NQ; ++a)
                kr[j][a] = *reinterpret_cast<const u4*>(kb + row[j] + li * D + (F32 ? 16 * a + 4 * g : 32 * a + 8 * g));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < W::VW; ++w)
                    vr[j][i][w] = *reinterpret_cast<const typename W::VWord*>(
                        vb + row[j] + (4 * g + i) * D + (F32 ? 64 * w + 4 * li : NO * li));
        // all of them on their way before the first is used: left to itself the compiler keeps few
        __builtin_amdgcn_sched_barrier(0);
        x.step(q, u, tree.above, tree.depth, span, shift, t0, there, lowest,
               [&](int j, int a) __attribute__((always_inline)) { return kr[j][a]; },
               [&](int j, int i, int w) __attribute__((always_inline)) { return vr[j][i][w]; },
               [&](int token, int d) __attribute__((always_inline)) {
                   const int t = min(t0 + token, u.len - 1);
                   return (float)vb[row_of(c, max(page_of(c, u.s, t), 0), u.h, t) * D + d];
               });
    }

#pragma unroll
    for (int t = 0; t < MT; ++t) x.l[t] = sum_over_groups(x.l[t]);
    if constexpr (SIDE) {
        x.store(q, u, r0);
    } else {
        const int ln = __lane_id();
        // the wavefronts' parts, in pairs: the upper one's goes through LDS
#pragma unroll
        for (int step = WAVES / 2; step > 0; step >>= 1) {
            float* e = ex[wave & (step - 1)];
            if (wave >= step && wave < 2 * step)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
#pragma unroll
                    for (int d = 0; d < NO; ++d)
                        *reinterpret_cast<f4*>(&e[((t * NO + d) * 64 + ln) * 4]) = x.o[t][d];
                    e[(MT * NO * 4 + 2 * t) * 64 + ln] = x.m[t];
                    e[(MT * NO * 4 + 2 * t + 1) * 64 + ln] = x.l[t];
                }
            __syncthreads();
            if (wave < step)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const float m1 = e[(MT * NO * 4 + 2 * t) * 64 + ln];
                    const float l1 = e[(MT * NO * 4 + 2 * t + 1) * 64 + ln];
                    const float top = fmaxf(x.m[t], m1);
                    const float f0 = factor_of(x.m[t], top), f1 = factor_of(m1, top);
                    x.l[t] = x.l[t] * f0 + l1 * f1;
                    x.m[t] = top;
#pragma unroll
                    for (int d = 0; d < NO; ++d)
                        x.o[t][d] = x.o[t][d] * f0 +
                                    *reinterpret_cast<const f4*>(&e[((t * NO + d) * 64 + ln) * 4]) * f1;
                }
            __syncthreads();
        }
        if (splits == 1) {
            if (wave == 0) x.store(q, u, r0);
            return;
        }
        const int rows = min(u.nrows - r0, ROWS);
        const __amdgpu_buffer_rsrc_t pr = buffer_rsrc(part + (int64_t)task.first * ROWS * PW, (int64_t)splits * ROWS * PW);
        if (wave == 0) x.store_part(pr, task.z * ROWS, rows);
        join<D, ROWS>(q, u, pr, counters + task.first, splits, r0, rows, &ex[0][0], &arrived);
    }
}

}  // namespace

namespace shp {

PagedPlan paged_attend_plan(const Paged& c, int head_dim, int format, int64_t rows, int cu_count, bool may_split) {
    PagedPlan p;
    const bool f32 = format == SHP_PAGED_F32;
    const int cu = std::max(cu_count, 1), tile = 8192 / (head_dim * (f32 ? 4 : 2));
    const int64_t heads = (int64_t)c.n_seqs * c.kv, tiles = (c.cap + tile - 1) / tile;
    // 32 rows a workgroup use each tile for twice the work (60 rows x 4 heads of 16 sequences on 4,100 tokens x 8
    // heads x 128 in bf16 180 us, with 16 rows 287; prompts of 1,000 tokens 80 and 104).  fp32's products take so
    // long that 16 rows, twice the workgroups, are better until there are 32 pairs of 32 rows and a tile a CU (24
    // rows x 8 heads on 700 tokens x 4 heads x 64 11 us and 15, prompts of 200 tokens 20 and 30).
    p.rows = rows > 16 && (!f32 || heads * ((rows + 31) / 32) * tiles >= 32 * cu) ? 32 : 16;
    // Where blocks of 32 rows are seven times as many as CUs, one wavefront takes all tiles of a block: it begins and
    // ends once, not four times (4,000 tokens with a window of 500 113 us, 155 the other way; prompts of 100 tokens of
    // 32 sequences 29 and 54; 2,000 tokens x 8 heads 127 and 130; trees of 60 rows of 16 sequences 252 and 188, for
    // whose 1,024 blocks it is not taken).  In fp32 the products outweigh that (prompts of 1,000 tokens 247 and 186).
    p.side = !f32 && rows > 64 && heads * ((rows + 31) / 32) >= 7 * cu;
    p.row_blocks = (int)((rows + p.rows - 1) / p.rows);
    const int64_t units = heads * p.row_blocks;
    // Two workgroups on every CU, or a whole number of times that (of 32 rows a CU holds no more, of 16 three or four:
    // trees of 60 rows in 16 sequences 91 us, 104 with one and a half times as many), none with fewer tiles than pay for the parts' way
    // through memory, about 3 us: more where there are many blocks anyway (one row of 64 sequences on 1,000 tokens
    // x 8 heads 32 us with 32 tiles, 46 with 4; of one sequence on 700 tokens 11.4 with 4, 14.8 with 16).
    p.target = 2 * cu;
    p.least = (int)std::min<int64_t>(std::max<int64_t>((units / 8 + 3) / 4 * 4, 4), 32);
    const int64_t shares = (tiles + p.least - 1) / p.least;  // of the longest sequence there can be
    const int64_t grid = std::min((units + p.target - 1) / p.target * p.target, units * shares) + 8;  // (8: XCDs' runs are rounded up)
    // Without shares a block has one workgroup, however long its sequence: 131,000 tokens x 128 in bf16 beside 127 or 159
    // sequences of 500 take 1.9 ms (160 of 500 67 us); beside a chunk of 512 rows 15 sequences of 8,000 tokens with one row
    // each 1,015 us (96 in a call of their own, and the chunk 188).
    if (p.side || !may_split || shares == 1 || units > 2 * p.target || c.n_seqs > 512 ||
        grid * (int64_t)sizeof(int) > (int64_t)kSplitCounterBytes) {
        p.target = 0;
        p.grid = (int)heads;
        p.scratch = 0;
    } else {
        p.grid = (int)grid;
        p.row_blocks = 1;
        p.scratch = (size_t)grid * p.rows * (head_dim + 4);
    }
    return p;
}

namespace {
template <class E, int D, bool LARGE>
auto kernel_of(int rows, bool side) {
    if constexpr (sizeof(E) == 2)
        if (side) return paged_attend_kernel<E, D, 2, true, LARGE>;
    return rows == 16 ? paged_attend_kernel<E, D, 1, false, LARGE> : paged_attend_kernel<E, D, 2, false, LARGE>;
}
template <class E, int D>
auto kernel_of(int rows, bool side, bool large) {
    return large ? kernel_of<E, D, true>(rows, side) : kernel_of<E, D, false>(rows, side);
}
}  // namespace

int paged_attend_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedQuery& query,
                        const PagedPlan& p, float* scratch, int* counters) {
    PagedQuery q = query;
    q.by_kv = shpd::fast_div((unsigned)c.kv);
    q.by_group = shpd::fast_div((unsigned)q.group);
    const bool large = q.cap >= kLargeCap;
    if (large) {
        // A row of q enters the products as numbers up to 1, scale and cap with their digits only, so that pieces of
        // 16 bits hold them; the powers of two come back behind the sums (a denormal score loses 2^-150 of the cap,
        // 2^-22 at most).  Half of the cap is finite in units of log2 as well.  Kernels of their own: instructions for
        // this in the others, behind a branch, cost 1 to 3 % of calls that never take it.
        const int down = std::ilogb(q.cap), up = q.scale == 0.0f ? 0 : std::ilogb(q.scale);
        q.lift = up - down;
        q.factor = std::ldexp(q.scale, -up) / std::ldexp(q.cap, -down);
        q.half = q.cap * 0.5f * kLog2e;
    }
    with_format(format, [&](auto e) {
        using E = decltype(e);
        auto kern = head_dim == 64 ? kernel_of<E, 64>(p.rows, p.side, large) : kernel_of<E, 128>(p.rows, p.side, large);
        hipLaunchKernelGGL(kern, dim3(p.grid, p.row_blocks), dim3(p.side ? 64 : 256), 0, s, c, q, p.target, p.least, scratch, counters);
    });
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

}  // namespace shp
