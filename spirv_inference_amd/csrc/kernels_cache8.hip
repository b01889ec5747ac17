// The 8-bit key/value cache: writing new rows, reading values back, and eviction.
//
// All of them move bytes and are bound by memory, or by latency where a call is small.  A workgroup
// owns the tokens of one V tile (64; 128 with blocks of 128) of K or of V of one head, so that a
// block's scale is settled inside one workgroup and V's 64-byte rows are written whole.
#include "cache8.h"

namespace {

using namespace shpd;
using shp::Cache8;
using shp::Cache8Rows;
using shp::kCacheTile;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

__device__ __forceinline__ float magnitude(float x) {
    // a NaN fails the comparison and counts as an infinity
    return fabsf(x) <= 3.4028234663852886e+38f ? fabsf(x) : __builtin_inff();
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// Positive floats in LDS that take maxima: their bits order as they do.
__device__ __forceinline__ void raise(unsigned* p, float x) { atomicMax(p, __float_as_uint(x)); }

// Where the code of dimension d of token t lies in a head's K or V.
template <int D, bool V>
__device__ __forceinline__ int64_t code_at(int t, int d) {
    if constexpr (V) return (int64_t)(t / kCacheTile) * (D * kCacheTile) + d * kCacheTile + t % kCacheTile;
    else return (int64_t)t * D + d;
}

// Where the scale of token t of a head lies.
__device__ __forceinline__ int64_t block_at(const Cache8& c, int sh, int t) {
    return ((int64_t)sh * c.cap + t) >> c.block_log2;
}

struct Scales {
    unsigned top[8];         // of each block of the span, as raise() keeps it
    float now[8], inv[8], was[8];
};

// ---- append ----------------------------------------------------------------------------------
// The new rows of one span, of K or V of one head.  Rows are read once, into registers; V's codes
// turn through LDS.  Prompts of 4 x up to 2,000 rows x 8 heads x 128 (2,316 rows, 24 MB): 11.4 us; a kernel
// that read rows twice, wrote single bytes and divided for every code took 18.8.
template <int D, int FMT, int SPAN, bool V>
__device__ __forceinline__ void append_span(const Cache8& c, const Cache8Rows& r, Scales& sc,
                                            uint8_t* lds) {
    constexpr int Q = D / 4, NP = SPAN * Q / kThreads, PITCH = SPAN + 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int sh = blockIdx.y, s = sh / c.kv, h = sh - s * c.kv, B = 1 << c.block_log2;
    const int len = seq_length(c, s), start = len - seq_count(r.counts, r.n, s);
    const int first = max(start, 0), t0 = (first / SPAN + (int)blockIdx.x) * SPAN;
    const int a = max(first, t0), t1 = min(len, t0 + SPAN);
    if (a >= t1) return;
    const float* x = V ? r.v + s * r.v_seq + h * r.v_head : r.k + s * r.k_seq + h * r.k_head;
    const int64_t row = V ? r.v_row : r.k_row;
    uint8_t* codes = (V ? c.v : c.k) + (int64_t)sh * c.cap * D;
    float* scale = (V ? c.v_scale : c.k_scale) + block_at(c, sh, t0);
    const int nb = SPAN >> c.block_log2;

    f4 v[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const int p = e * kThreads + tid, t = t0 + p / Q;
        v[e] = t >= a && t < t1 ? *reinterpret_cast<const f4*>(x + (t - start) * row + p % Q * 4)
                                : f4{0.f, 0.f, 0.f, 0.f};
    }
    if (tid < 8) sc.top[tid] = 0;
    __syncthreads();
    // a wavefront's rows of one step are of one block, and so are those of neighbouring steps
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, magnitude(v[e][i]));
        const int t = (e * kThreads + tid) / Q;
        const bool flush = e + 1 == NP || ((t ^ (t + kThreads / Q)) >> c.block_log2) != 0;
        if (__builtin_amdgcn_readfirstlane(flush)) {
            top = wave_max(top);
            if (lane == 0) raise(&sc.top[t >> c.block_log2], top);
            top = 0.0f;
        }
    }
    __syncthreads();
    if (tid < nb) {
        const int b0 = t0 + tid * B;
        if (b0 + B > a && b0 < t1) {
            float now = block_scale<FMT>(__uint_as_float(sc.top[tid])), was = now;
            if (b0 < a) {  // behind tokens of an earlier call
                was = scale[tid];
                if (!(now < was) && !(was >= 0.0f)) now = was;  // a NaN stays
                if (now < was) now = was;
            }
            scale[tid] = now;
            sc.now[tid] = now;
            sc.inv[tid] = 1.0f / now;
            sc.was[tid] = was;
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const int p = e * kThreads + tid, lt = p / Q, d = p % Q * 4, t = t0 + lt;
        if (t < a || t >= t1) continue;
        const int b = lt >> c.block_log2;
        const float y[4] = {v[e][0], v[e][1], v[e][2], v[e][3]};
        const unsigned w = encode4<FMT>(y, sc.now[b], sc.inv[b]);
        if constexpr (V) {
#pragma unroll
            for (int i = 0; i < 4; ++i) lds[(d + i) * PITCH + lt] = (uint8_t)(w >> (8 * i));
        } else {
            *reinterpret_cast<unsigned*>(codes + (int64_t)t * D + d) = w;
        }
    }
    // earlier tokens of the first block, where its scale grew
    const int b = (a - t0) >> c.block_log2, b0 = t0 + b * B;
    const float now = sc.now[b], inv = sc.inv[b], was = sc.was[b];
    const bool grown = now > was;
    auto again = [&](unsigned w) {
        const float y[4] = {code_value<FMT>(w, 0) * was, code_value<FMT>(w, 1) * was,
                            code_value<FMT>(w, 2) * was, code_value<FMT>(w, 3) * was};
        return encode4<FMT>(y, now, inv);
    };
    if constexpr (!V) {
        if (grown)
            for (int e = tid; e < (a - b0) * Q; e += kThreads) {
                unsigned* p = reinterpret_cast<unsigned*>(codes + (int64_t)b0 * D) + e;
                *p = again(*p);
            }
    } else {
        __syncthreads();
        // words of four tokens of a dimension, from the first that changes
        constexpr int W = SPAN / 4;
        const int w = tid % W, t = t0 + 4 * w, from = grown ? b0 : a;
        if (t + 4 <= from || t >= t1) return;
#pragma unroll 4
        for (int d = tid / W; d < D; d += kThreads / W) {
            unsigned* p = reinterpret_cast<unsigned*>(codes + code_at<D, true>(t, d));
            const unsigned fresh = *reinterpret_cast<const unsigned*>(&lds[d * PITCH + 4 * w]);
            if (t >= a && t + 4 <= t1) {
                *p = fresh;
                continue;
            }
            const unsigned old = grown && t < a ? again(*p) : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool isnew = t + i >= a && t + i < t1;
                if (isnew || (t + i >= from && t + i < a))
                    reinterpret_cast<uint8_t*>(p)[i] = (uint8_t)((isnew ? fresh : old) >> (8 * i));
            }
        }
    }
}

template <int D, int FMT, int SPAN>
__global__ __launch_bounds__(kThreads) void cache8_append_kernel(Cache8 c, Cache8Rows r) {
    __shared__ Scales sc;
    __shared__ __attribute__((aligned(16))) uint8_t lds[D * (SPAN + 4)];
    if (blockIdx.z) append_span<D, FMT, SPAN, true>(c, r, sc, lds);
    else append_span<D, FMT, SPAN, false>(c, r, sc, lds);
}

// Up to kFew rows a sequence, as decode steps append them: a wavefront for K or V and each of the two
// blocks they can touch, D / 64 dimensions a lane, without LDS or barriers.  64 sequences x 4 heads x
// 64: 3.3 us; a span of 64 tokens a workgroup took 6.6.
constexpr int kFew = 4;
template <int D, int FMT>
__global__ __launch_bounds__(kThreads) void cache8_append_few_kernel(Cache8 c, Cache8Rows r) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sh = blockIdx.x, s = sh / c.kv, h = sh - s * c.kv, B = 1 << c.block_log2;
    const bool isv = wave & 1;
    const int len = seq_length(c, s), start = len - seq_count(r.counts, r.n, s);
    const int t0 = ((max(start, 0) >> c.block_log2) + (wave >> 1)) << c.block_log2;
    const int a = max(start, t0), t1 = min(len, t0 + B);
    if (a >= t1) return;
    const float* x = (isv ? r.v + s * r.v_seq + h * r.v_head : r.k + s * r.k_seq + h * r.k_head) + lane;
    const int64_t row = isv ? r.v_row : r.k_row;
    uint8_t* codes = (isv ? c.v : c.k) + (int64_t)sh * c.cap * D;
    float* scale = (isv ? c.v_scale : c.k_scale) + block_at(c, sh, t0);
    auto at = [&](int t, int d) { return codes + (isv ? code_at<D, true>(t, d) : code_at<D, false>(t, d)); };
    float v[kFew][E], top = 0.0f, was = a > t0 ? *scale : 0.0f;
#pragma unroll
    for (int i = 0; i < kFew; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[i][e] = a + i < t1 ? x[(a + i - start) * row + 64 * e] : 0.0f;
            top = fmaxf(top, magnitude(v[i][e]));
        }
    float now = block_scale<FMT>(wave_max(top));
    if (a > t0) {
        if (!(now < was) && !(was >= 0.0f)) now = was;  // a NaN stays
        if (now < was) now = was;
    } else {
        was = now;
    }
    if (lane == 0) *scale = now;
    const float inv = 1.0f / now;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float y[4] = {v[0][e], v[1][e], v[2][e], v[3][e]};
        const unsigned w = encode4<FMT>(y, now, inv);
#pragma unroll
        for (int i = 0; i < kFew; ++i)
            if (a + i < t1) *at(a + i, lane + 64 * e) = (uint8_t)(w >> (8 * i));
    }
    if (now > was)  // earlier tokens of the block, four at a time
        for (int t = t0; t < a; t += 4)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    y[i] = t + i < a ? code_value<FMT>(*at(t + i, lane + 64 * e), 0) * was : 0.0f;
                const unsigned w = encode4<FMT>(y, now, inv);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i < a) *at(t + i, lane + 64 * e) = (uint8_t)(w >> (8 * i));
            }
}

// ---- read ------------------------------------------------------------------------------------
// The values of one tile of the newest n tokens; tiles before the first token are zeros.  V turns
// through LDS.  268 MB of values from 67 MB of codes: 52 us (112 reading V byte by byte).
template <int D, int FMT>
__global__ __launch_bounds__(kThreads) void cache8_read_kernel(Cache8 c, int n, float* k, float* v) {
    constexpr int Q = D / 4, NP = kCacheTile * Q / kThreads, PITCH = kCacheTile + 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[D * PITCH];
    const int tid = threadIdx.x, sh = blockIdx.y, s = sh / c.kv;
    const bool isv = blockIdx.z == 1;
    float* const out = (isv ? v : k);
    if (!out) return;
    const int start = seq_length(c, s) - n;  // the token of row 0
    const int t0 = ((start >> 6) + (int)blockIdx.x) * kCacheTile;
    if (t0 >= start + n) return;
    const bool held = t0 >= 0;
    const uint8_t* codes = (isv ? c.v : c.k) + ((int64_t)sh * c.cap + max(t0, 0)) * D;
    const float* scale = (isv ? c.v_scale : c.k_scale) + block_at(c, sh, max(t0, 0));
    float* const o = out + (int64_t)sh * n * D;
    if (isv && held) {
#pragma unroll
        for (int e = 0; e < D * kCacheTile / 16 / kThreads; ++e) {
            const int p = e * kThreads + tid;
            const u4 w = reinterpret_cast<const u4*>(codes)[p];
            unsigned* to = reinterpret_cast<unsigned*>(&lds[p / 4 * PITCH + p % 4 * 16]);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = w[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const int p = e * kThreads + tid, lt = p / Q, d = p % Q * 4, i = t0 + lt - start;
        if (i < 0 || i >= n) continue;
        f4 x = {0.f, 0.f, 0.f, 0.f};
        if (held) {
            unsigned w;
            if (isv) {
                w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) w |= (unsigned)lds[(d + j) * PITCH + lt] << (8 * j);
            } else {
                w = *reinterpret_cast<const unsigned*>(codes + lt * D + d);
            }
            const float sx = scale[lt >> c.block_log2];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = code_value<FMT>(w, j) * sx;
        }
        *reinterpret_cast<f4*>(o + (int64_t)i * D + d) = x;
    }
}

// ---- eviction --------------------------------------------------------------------------------

// A float as an unsigned number of the same order: NaN lowest, both zeros alike.
__device__ __forceinline__ unsigned order_of(float x) {
    if (!(x == x)) return 0u;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kSelect = 1024;

struct Select {
    unsigned part[2][16];
    unsigned hist[256];
    unsigned found[2];
};

// Sum over the workgroup of a count that each wavefront has, for everybody.  `turn` alternates.
__device__ __forceinline__ unsigned group_sum(unsigned wave_count, Select& m, int turn) {
    const int tid = threadIdx.x;
    if ((tid & 63) == 0) m.part[turn][tid >> 6] = wave_count;
    __syncthreads();
    unsigned all = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) all += m.part[turn][q];
    return all;
}

// Sum of the counts of all threads before this one.
__device__ __forceinline__ unsigned before_me(unsigned count, Select& m, int turn) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned upto = count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned u = __shfl_up(upto, o);
        if (lane >= o) upto += u;
    }
    if (lane == 63) m.part[turn][wave] = upto;
    __syncthreads();
    unsigned base = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) base += q < wave ? m.part[turn][q] : 0u;
    return base + upto - count;
}

// Counts a digit; a wavefront whose lanes all have the same adds once.
__device__ __forceinline__ void count_digit(bool have, unsigned digit, Select& m) {
    const unsigned long long who = __ballot(have);
    if (!who) return;
    const unsigned one = __shfl(digit, __ffsll(who) - 1);
    if (__ballot(have && digit == one) == who) {
        if ((threadIdx.x & 63) == 0) atomicAdd(&m.hist[one], (unsigned)__popcll(who));
    } else if (have) {
        atomicAdd(&m.hist[digit], 1u);
    }
}

// The largest digit that `need` keys reach, and how many have a larger one: one wavefront looks,
// four digits a lane from the largest on, and everybody gets them.
__device__ __forceinline__ void find_digit(unsigned need, Select& m) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < 64) {
        unsigned n[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += n[i] = m.hist[255 - 4 * tid - i];
        unsigned upto = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned u = __shfl_up(upto, o);
            if (tid >= o) upto += u;
        }
        unsigned above = upto - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (above < need && above + n[i] >= need) {
                m.found[0] = 255 - 4 * tid - i;
                m.found[1] = above;
            }
            above += n[i];
        }
    }
    __syncthreads();
}

// Which of `old` tokens are the `need` heaviest (0 < need < old), each thread holding E of them in
// order: the smallest key that stays is found by counting its digits, eight bits at a time, in LDS.
// Latency bounds it: 4 heads of 936 weights 6.3 us, 128 heads of up to 7,934 13.4 (a ballot a bit
// instead of the digits: 14 and 22).
template <int E>
__device__ __forceinline__ void select_held(const float* __restrict__ w, int old, unsigned need,
                                            int32_t* out, float* ow, Select& m) {
    typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
    const int tid = threadIdx.x, i0 = tid * E;
    float x[E];
    unsigned key[E];
    if constexpr (E == 1) x[0] = i0 < old ? w[i0] : 0.0f;
#pragma unroll
    for (int e = 0; e + 4 <= E; e += 4) {
        if (i0 + e + 4 <= old) {
            const f4u v = *reinterpret_cast<const f4u*>(w + i0 + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[e + j] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[e + j] = i0 + e + j < old ? w[i0 + e + j] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = order_of(x[e]);
    unsigned last = 0;     // the smallest key that stays, as far as it is known
    unsigned spare = need;  // how many of the keys equal to it so far stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) m.hist[tid] = 0;
        __syncthreads();
        const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
#pragma unroll
        for (int e = 0; e < E; ++e)
            count_digit(i0 + e < old && (key[e] & mask) == last, (key[e] >> shift) & 255, m);
        find_digit(spare, m);
        last |= m.found[0] << shift;
        spare -= m.found[1];
    }
    unsigned equal = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) equal += i0 + e < old && key[e] == last;
    equal = before_me(equal, m, 0);
    unsigned stay = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        bool s = i0 + e < old && key[e] >= last;
        if (s && key[e] == last) s = equal++ < spare;
        stay |= (unsigned)s << e;
    }
    unsigned at = before_me((unsigned)__popc(stay), m, 1);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (stay >> e & 1) {
            out[at] = i0 + e;
            if (ow) ow[at] = x[e];
            ++at;
        }
}

// The same for more tokens than the workgroup's registers hold; each digit reads the weights again.
__device__ __forceinline__ void select_long(const float* __restrict__ w, int old, unsigned need,
                                            int32_t* out, float* ow, Select& m) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned key = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) m.hist[tid] = 0;
        __syncthreads();
        const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i0 = 0; i0 < old; i0 += kSelect) {
            const unsigned o = order_of(i0 + tid < old ? w[i0 + tid] : 0.0f);
            count_digit(i0 + tid < old && (o & mask) == key, (o >> shift) & 255, m);
        }
        find_digit(need, m);
        key |= m.found[0] << shift;
        need -= m.found[1];
    }
    unsigned base = 0, equal = 0;
    for (int i0 = 0; i0 < old; i0 += kSelect) {
        const int i = i0 + tid;
        const float x = i < old ? w[i] : 0.0f;
        const unsigned o = order_of(x);
        const bool eq = i < old && o == key;
        const unsigned long long below = (1ull << lane) - 1, be = __ballot(eq);
        const unsigned all = group_sum((unsigned)__popcll(be), m, 0);
        unsigned before = equal + (unsigned)__popcll(be & below);
        for (int q = 0; q < wave; ++q) before += m.part[0][q];
        equal += all;
        const bool stay = i < old && (o > key || (eq && before < need));
        const unsigned long long bs = __ballot(stay);
        const unsigned out_all = group_sum((unsigned)__popcll(bs), m, 1);
        unsigned at = base + (unsigned)__popcll(bs & below);
        for (int q = 0; q < wave; ++q) at += m.part[1][q];
        base += out_all;
        if (stay) {
            out[at] = i;
            if (ow) ow[at] = x;
        }
        __syncthreads();
    }
}

// One sequence and head: which of its tokens stay, in their order.
__global__ __launch_bounds__(kSelect) void cache8_select_kernel(Cache8 src, Cache8 dst,
                                                                const float* __restrict__ weights,
                                                                int keep, int recent, int32_t* kept,
                                                                float* dst_weights) {
    __shared__ Select m;
    const int sh = blockIdx.x, s = sh / src.kv, tid = threadIdx.x;
    const int len = seq_length(src, s);
    const float* w = weights + (int64_t)sh * src.cap;
    int32_t* const out = kept + (int64_t)sh * keep;
    float* const ow = dst_weights ? dst_weights + (int64_t)sh * dst.cap : nullptr;
    const int n = min(len, keep);
    if (sh % src.kv == 0 && tid == 0) dst.lengths[s] = n;
    for (int i = n + tid; i < keep; i += kSelect) out[i] = -1;
    if (ow)
        for (int i = n + tid; i < dst.cap; i += kSelect) ow[i] = 0.0f;
    if (len <= keep) {
        for (int i = tid; i < len; i += kSelect) {
            out[i] = i;
            if (ow) ow[i] = w[i];
        }
        return;
    }
    const int old = len - recent;  // tokens that compete
    for (int i = tid; i < recent; i += kSelect) {
        out[keep - recent + i] = old + i;
        if (ow) ow[keep - recent + i] = w[old + i];
    }
    const unsigned need = keep - recent;
    if (need == 0) return;
    if (old <= kSelect) select_held<1>(w, old, need, out, ow, m);
    else if (old <= 8 * kSelect) select_held<8>(w, old, need, out, ow, m);
    else if (old <= 32 * kSelect) select_held<32>(w, old, need, out, ow, m);
    else select_long(w, old, need, out, ow, m);
}

// The scales of the blocks of a span of dst, from the maxima in sc.top, for everybody.
template <int FMT>
__device__ __forceinline__ void settle_scales(const Cache8& dst, float* scale, int t0, int t1,
                                              Scales& sc) {
    __syncthreads();
    const int b = threadIdx.x;
    if (b < 8 && t0 + (b << dst.block_log2) < t1) {
        const float now = block_scale<FMT>(__uint_as_float(sc.top[b]));
        scale[b] = now;
        sc.now[b] = now;
        sc.inv[b] = 1.0f / now;
    }
    __syncthreads();
}

// One span of K of dst, made from the kept tokens of src, whose rows are read 16 bytes a lane.
template <int D, int FMT, int SPAN>
__device__ __forceinline__ void gather_k(const Cache8& src, const Cache8& dst, const int32_t* id,
                                         int t0, int t1, Scales& sc) {
    constexpr int R = D / 16, NP = SPAN * R / kThreads;  // NP pieces of 16 dimensions of a token
    const int tid = threadIdx.x, lane = tid & 63, sh = blockIdx.y;
    const uint8_t* from = src.k + (int64_t)sh * src.cap * D;
    uint8_t* to = dst.k + (int64_t)sh * dst.cap * D;
    u4 raw[NP];
    float was[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const int p = e * kThreads + tid, t = t0 + p / R;
        raw[e] = u4{0u, 0u, 0u, 0u};
        was[e] = 0.0f;
        if (t < t1) {
            const int i = id[t];
            raw[e] = *reinterpret_cast<const u4*>(from + (int64_t)i * D + p % R * 16);
            was[e] = src.k_scale[block_at(src, sh, i)];
        }
    }
    __syncthreads();  // sc.top is clear
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(code_value<FMT>(raw[e][i >> 2], i & 3)));
        // the wavefront's tokens of this step are of one block
        top = wave_max(magnitude(top * was[e]));
        if (lane == 0) raise(&sc.top[(e * kThreads + tid) / R >> dst.block_log2], top);
    }
    settle_scales<FMT>(dst, dst.k_scale + block_at(dst, sh, t0), t0, t1, sc);
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const int p = e * kThreads + tid, lt = p / R;
        if (t0 + lt >= t1) continue;
        const float now = sc.now[lt >> dst.block_log2], inv = sc.inv[lt >> dst.block_log2];
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = code_value<FMT>(raw[e][i], j) * was[e];
            w[i] = encode4<FMT>(y, now, inv);
        }
        *reinterpret_cast<u4*>(to + (int64_t)(t0 + lt) * D + p % R * 16) = w;
    }
}

// One span of V: a lane makes words of four tokens of a dimension, whose bytes it reads one by one.
// The 64 tokens of a span come from few tiles (their places rise), so a wavefront's loads share
// lines, and lines are all that reading whole tiles would fetch too.  128 heads, 1,900-8,190 tokens of
// 128 to 2,048, K and V: 64 us for 216 MB, of which the kept tokens are 134; with a lane a token, which
// then writes single bytes, 79; with whole tiles read and their bytes sorted out in LDS 76.
template <int D, int FMT, int SPAN>
__device__ __forceinline__ void gather_v(const Cache8& src, const Cache8& dst, const int32_t* id,
                                         int t0, int t1, Scales& sc) {
    constexpr int W = SPAN / 4, STEP = kThreads / W, NW = D / STEP;
    const int tid = threadIdx.x, sh = blockIdx.y, n = t1 - t0, w = tid % W, d0 = tid / W;
    const uint8_t* from = src.v + (int64_t)sh * src.cap * D;
    uint8_t* to = dst.v + (int64_t)sh * dst.cap * D;
    float was[4];
    unsigned at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // behind the last token: the last one's bytes, which do not count
        const int t = id[t0 + min(4 * w + i, n - 1)];
        at[i] = (unsigned)code_at<D, true>(t, d0);
        was[i] = src.v_scale[block_at(src, sh, t)];
    }
    unsigned char b[NW][4];
#pragma unroll
    for (int e = 0; e < NW; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) b[e][i] = from[at[i] + e * STEP * kCacheTile];
    __syncthreads();  // sc.top is clear
    float most[4] = {0.f, 0.f, 0.f, 0.f}, top = 0.0f;
#pragma unroll
    for (int e = 0; e < NW; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = fmaxf(most[i], fabsf(code_value<FMT>(b[e][i], 0)));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (4 * w + i < n) top = fmaxf(top, magnitude(most[i] * was[i]));
    raise(&sc.top[4 * w >> dst.block_log2], top);
    settle_scales<FMT>(dst, dst.v_scale + block_at(dst, sh, t0), t0, t1, sc);
    if (4 * w >= n) return;
    const float now = sc.now[4 * w >> dst.block_log2], inv = sc.inv[4 * w >> dst.block_log2];
#pragma unroll
    for (int e = 0; e < NW; ++e) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            y[i] = 4 * w + i < n ? code_value<FMT>(b[e][i], 0) * was[i] : 0.0f;
        const unsigned c = encode4<FMT>(y, now, inv);
        uint8_t* p = to + code_at<D, true>(t0 + 4 * w, d0 + e * STEP);
        if (4 * w + 4 <= n) {
            *reinterpret_cast<unsigned*>(p) = c;
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (4 * w + i < n) p[i] = (uint8_t)(c >> (8 * i));
        }
    }
}

template <int D, int FMT, int SPAN>
__global__ __launch_bounds__(kThreads) void cache8_gather_kernel(Cache8 src, Cache8 dst,
                                                                 const int32_t* kept, int keep) {
    __shared__ Scales sc;
    const int sh = blockIdx.y, s = sh / src.kv, t0 = (int)blockIdx.x * SPAN;
    const int t1 = min(min(seq_length(src, s), keep), t0 + SPAN);
    if (t0 >= t1) return;
    if (threadIdx.x < 8) sc.top[threadIdx.x] = 0;
    const int32_t* id = kept + (int64_t)sh * keep;
    if (blockIdx.z) gather_v<D, FMT, SPAN>(src, dst, id, t0, t1, sc);
    else gather_k<D, FMT, SPAN>(src, dst, id, t0, t1, sc);
}

// KERN<head_dim, format, span> for a cache.
#define SHP_CACHE8_SPAN(KERN, SPAN, head_dim, format)                                             \
    ((head_dim) == 64 ? ((format) == SHP_CACHE8_I8 ? KERN<64, kI8, SPAN> : KERN<64, kE4M3, SPAN>) \
                      : ((format) == SHP_CACHE8_I8 ? KERN<128, kI8, SPAN> : KERN<128, kE4M3, SPAN>))

int span_of(const Cache8& c) { return c.block_log2 == 7 ? 128 : 64; }

}  // namespace

namespace shp {

int cache8_append_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                         const Cache8Rows& r) {
    if (r.n <= kFew) {
        auto kern = head_dim == 64
            ? (format == SHP_CACHE8_I8 ? cache8_append_few_kernel<64, kI8> : cache8_append_few_kernel<64, kE4M3>)
            : (format == SHP_CACHE8_I8 ? cache8_append_few_kernel<128, kI8> : cache8_append_few_kernel<128, kE4M3>);
        hipLaunchKernelGGL(kern, dim3(c.n_seqs * c.kv), dim3(kThreads), 0, s, c, r);
        SHP_HIP_CHECK(hipGetLastError());
        return SHP_OK;
    }
    // n rows end anywhere: they touch at most this many spans
    const int span = span_of(c), spans = (std::min(r.n, c.cap) + span - 2) / span + 1;
    hipLaunchKernelGGL(span == 128 ? SHP_CACHE8_SPAN(cache8_append_kernel, 128, head_dim, format)
                                   : SHP_CACHE8_SPAN(cache8_append_kernel, 64, head_dim, format),
                       dim3(spans, c.n_seqs * c.kv, 2), dim3(kThreads), 0, s, c, r);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

int cache8_read_launch(hipStream_t s, const Cache8& c, int head_dim, int format, int n, float* k,
                       float* v) {
    const int tiles = (n + kCacheTile - 2) / kCacheTile + 1;
    auto kern = head_dim == 64
        ? (format == SHP_CACHE8_I8 ? cache8_read_kernel<64, kI8> : cache8_read_kernel<64, kE4M3>)
        : (format == SHP_CACHE8_I8 ? cache8_read_kernel<128, kI8> : cache8_read_kernel<128, kE4M3>);
    hipLaunchKernelGGL(kern, dim3(tiles, c.n_seqs * c.kv, 2), dim3(kThreads), 0, s, c, n, k, v);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

int cache8_evict_launch(hipStream_t s, const Cache8& src, const Cache8& dst, int head_dim,
                        int format, const float* weights, int keep, int recent, int32_t* kept,
                        float* dst_weights) {
    hipLaunchKernelGGL(cache8_select_kernel, dim3(src.n_seqs * src.kv), dim3(kSelect), 0, s, src, dst,
                       weights, keep, recent, kept, dst_weights);
    SHP_HIP_CHECK(hipGetLastError());
    const int span = span_of(dst), spans = (std::min(keep, src.cap) + span - 1) / span;
    hipLaunchKernelGGL(span == 128 ? SHP_CACHE8_SPAN(cache8_gather_kernel, 128, head_dim, format)
                                   : SHP_CACHE8_SPAN(cache8_gather_kernel, 64, head_dim, format),
                       dim3(spans, src.n_seqs * src.kv, 2), dim3(kThreads), 0, s, src, dst, kept,
                       keep);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

}  // namespace shp
