// How likely tokens are: log probability of a given id, entropy and the likeliest ids of each row
// of logits, from one read of the row.
//
// A workgroup holds 32 logits a thread in registers: their maximum m, Z = sum exp(x - m) and X = sum
// exp(x - m) (x - m) give log p = x - m - log Z and the entropy log Z - X / Z, a sum of two numbers
// that are not negative.  exp(d) is exp2(d * log2 e) with a rounded product, off by 2^-24 of d log2 e; |d| e^d
// is under 0.37, so that costs a sum less than its own rounding.  Against 64 bits results are off by 6.7e-8
// (1 x 32,000) and 9.5e-8 (1,500 x 131,071), norms; those of fp32 torch by 4.5e-8 and 5.0e-8.
//
// From 256 rows on a workgroup takes a row, chunk after chunk, and reading bounds it: 1,500 x
// 131,071 with 20 alternatives (786 MB) 160 us, 4.9 TB/s, 146 without alternatives.  It has 256 threads,
// from 1,024 rows on 128 (4,000 x 40,000 133 us, 148 with 256; 600 x 32,000 40, 30).  Fewer rows are cut
// into parts of 32,768 logits for workgroups of 1,024, and joined: 1 x 32,000 8.1 us (17 the other
// way), 128 x 32,000 12.2 (26); 300 x 131,071 take 69 and 72, 600 x 32,000 28 and 35.
#include "cache8.h"

namespace {

using shp::kMaxTop;
using shp::LogprobArgs;
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kHeld = 32;
constexpr int kFewThreads = 1024, kFewSpan = kFewThreads * kHeld, kManyThreads = 256;
constexpr int kManyRows = 256, kMostRows = 1024, kMostThreads = 128;
constexpr int kCandidates = 448;  // logits of a chunk that are put in order by counting
constexpr float kLog2e = 1.4426950408889634f;

// A float as an unsigned number of the same order: NaN lowest, both zeros alike.
__device__ __forceinline__ unsigned order_of(float x) {
    if (!(x == x)) return 0u;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// A logit and its id as one number: larger is better, of equal logits the lower id.
__device__ __forceinline__ unsigned long long rank_of(float x, int id) {
    return ((unsigned long long)order_of(x) << 32) | (unsigned)(0x7fffffff - id);
}

// The id in a rank that was raised by one (0: nothing).
__device__ __forceinline__ int id_of(unsigned long long r) {
    return 0x7fffffff - (int)(unsigned)(r - 1);
}

struct Sums {
    float m, z, x;
};

// Adds a part to sums whose maximum is t.m already.  Of a part that holds nothing but the type's lowest
// numbers d * z would be minus infinity and f zero: d stays where their product is finite for every
// length of a row, which also leaves alone what holds nothing but minus infinity (z is 0, and d may be
// a NaN).  Logits that are plus infinity or NaN are in z and x.
__device__ __forceinline__ void add_part(Sums& t, float m, float z, float x) {
    const float d = fmaxf(m - t.m, -1e28f), f = __builtin_amdgcn_exp2f(d * kLog2e);
    t.z += z * f;
    t.x += (x + d * z) * f;
}

__device__ __forceinline__ float lp_of(float x, const Sums& t) {
    // no sum at all: nothing but minus infinity
    return t.z == 0.0f ? __builtin_nanf("") : (x - t.m) - logf(t.z);
}

// What a row's sums give, by one thread.
__device__ __forceinline__ void finish(const LogprobArgs& a, int row, const Sums& t) {
    if (a.logprob) {
        const int id = a.targets[row];
        const float x = id >= 0 && id < a.vocab ? a.logits[row * a.row_stride + id] : -__builtin_inff();
        a.logprob[row] = lp_of(x, t);
    }
    if (a.entropy) a.entropy[row] = t.z == 0.0f ? __builtin_nanf("") : logf(t.z) - t.x / t.z;
}

__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor(v, o);
        v = u > v ? u : v;
    }
    return v;
}

// Parts of a row: m, Z, X, and the ranks of its best `top` ids.
struct Part {
    float m, z, x, pad;
    unsigned long long rank[kMaxTop];
};

template <int T>
struct Shared {
    float m[2][T / 64], z[2][T / 64], x[2][T / 64];
    unsigned bests[T];                        // the threads' best logits, as order_of
    unsigned long long held[kCandidates + kMaxTop];  // ranks of candidates, raised by one
    unsigned long long tops[kMaxTop];                // the best in order
    int count[T / 64];
    float threshold;
    int found;
    int added[3];  // candidates of the chunk before, of this one, and zero for the next
};

// 32 logits a thread from i0 on, minus infinity from `end` on.
template <int T>
__device__ __forceinline__ void load_logits(const float* x, int i0, int end, float* v) {
#pragma unroll
    for (int p = 0; p < kHeld / 4; ++p) {
        const int i = i0 + (p * T + (int)threadIdx.x) * 4;
        if (i + 4 <= end) {
            const f4u t = *reinterpret_cast<const f4u*>(x + i);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * p + c] = t[c];
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * p + c] = i + c < end ? x[i + c] : -__builtin_inff();
        }
    }
}

template <int T>
__device__ __forceinline__ int id_at(int i0, int e) {
    return i0 + ((e >> 2) * T + (int)threadIdx.x) * 4 + (e & 3);
}

// A logit that `top` groups of threads reach with the best they hold, so that `top` logits or more do
// (if that many groups hold one): one wavefront halves the range of the groups' best until no more
// than twice as many pass.  Up to 24 alternatives take 64 groups, one a lane, at a ballot a turn (a row
// of 32,000, 5 alternatives: 9.5 us by threads, 8.2 by groups; 24: 11.3 and 10.5).  More would let
// through many logits too many, which all have to be put in order (32: 11.3 and 13.9; 64: 13.7 and
// 22.9), and take the threads one by one.  For everybody behind the next barrier.
template <int T>
__device__ __forceinline__ void find_threshold(int top, Shared<T>& sm) {
    const int tid = threadIdx.x;
    if (tid >= 64) return;
    unsigned b[T / 64], best = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) {
        b[i] = sm.bests[i * 64 + tid];
        best = max(best, b[i]);
    }
    const bool groups = top <= 24;
    unsigned lo = best, hi = best;
    if (!groups)
#pragma unroll
        for (int i = 0; i < T / 64; ++i) lo = min(lo, b[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, (unsigned)__shfl_xor((int)lo, o));
        hi = max(hi, (unsigned)__shfl_xor((int)hi, o));
    }
    while (hi - lo > 1) {
        const unsigned next = lo + (hi - lo) / 2;
        int n = 0;
        if (groups) {
            n = __popcll(__ballot(best >= next));
        } else {
#pragma unroll
            for (int i = 0; i < T / 64; ++i) n += __popcll(__ballot(b[i] >= next));
        }
        if (n < top) {
            hi = next;
        } else {
            lo = next;
            if (n <= 2 * top) break;
        }
    }
    // as a float of that order; 0: some groups hold nothing, and the others pass all they have
    if (tid == 0)
        sm.threshold = lo & 0x80000000u ? __uint_as_float(lo ^ 0x80000000u)
                       : lo             ? __uint_as_float(~lo) : -__builtin_inff();
}

// Adds the logits of a chunk that are no worse than `least` behind the `have` candidates, in any order.
// Behind a barrier *added is their number, also of those that did not fit.
template <int T>
__device__ __forceinline__ void collect(const float* v, int i0, int end, float mine, float least,
                                        int have, int* added, Shared<T>& sm) {
    if (!(mine >= least)) return;
#pragma unroll
    for (int e = 0; e < kHeld; ++e) {
        const int id = id_at<T>(i0, e);
        if (v[e] >= least && id < end) {
            const int c = have + atomicAdd(added, 1);
            if (c < kCandidates) sm.held[c] = rank_of(v[e], id) + 1;
        }
    }
}

// The same where too many logits are as large (plateaus, ties, a few threads that hold all the large
// ones) or too few are numbers: exactly the `top` best of the chunk, which is read again.  The key of
// the last of them is the threshold's, if that is what the plateau is at, or found by halving the
// range of keys; of the logits that have it the first are taken, T after T.
template <int T>
__device__ __forceinline__ void collect_exactly(const float* x, int i0, int end, int top, int have,
                                                Shared<T>& sm) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto total = [&](int mine) {  // over the workgroup
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o);
        __syncthreads();
        if (lane == 0) sm.count[wave] = mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) all += sm.count[w];
        return all;
    };
    auto reach = [&](unsigned key) {  // logits of this key or a larger one
        int n = 0;
#pragma unroll 8
        for (int i = i0 + tid; i < end; i += T) n += order_of(x[i]) >= key;
        return total(n);
    };
    const int want = min(top, end - i0);
    unsigned last = order_of(sm.threshold);
    if (reach(last) < want || (last < ~0u && reach(last + 1) >= want)) {
        last = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned next = last | 1u << bit;
            if (reach(next) >= want) last = next;
        }
    }
    __syncthreads();
    if (tid == 0) sm.found = have;
    __syncthreads();
    for (int i = i0 + tid; i < end; i += T)
        if (order_of(x[i]) > last) sm.held[atomicAdd(&sm.found, 1)] = rank_of(x[i], i) + 1;
    __syncthreads();
    int got = sm.found;  // under have + want: the last one's key is not among them
    for (int j = i0; j < end && got < have + want; j += T) {
        const int i = j + tid;
        const bool is = i < end && order_of(x[i]) == last;
        const unsigned long long who = __ballot(is);
        __syncthreads();
        if (lane == 0) sm.count[wave] = __popcll(who);
        __syncthreads();
        int at = got + __popcll(who & ((1ull << lane) - 1));
#pragma unroll
        for (int w = 0; w < T / 64; ++w) {
            at += w < wave ? sm.count[w] : 0;
            got += sm.count[w];
        }
        if (is && at < have + want) sm.held[at] = rank_of(x[i], i) + 1;
    }
    __syncthreads();
}

// Puts the candidates in order, by counting how many are better than each, and keeps `top`: in
// sm.tops, and as the candidates that later ones join where there are any.
template <int T, bool LOOP>
__device__ __forceinline__ int order_candidates(int n, int top, Shared<T>& sm) {
    for (int i = threadIdx.x; i < n; i += T) {
        const unsigned long long r = sm.held[i];
        int better = 0;
        for (int j = 0; j < n; ++j) better += sm.held[j] > r;
        if (better < top) sm.tops[better] = r;
    }
    n = min(n, top);
    __syncthreads();
    if (!LOOP) return n;
    if ((int)threadIdx.x < n) sm.held[threadIdx.x] = sm.tops[threadIdx.x];
    __syncthreads();
    return n;
}

// The logits [p * span, + span) of a row, in chunks of 32 a thread.  LOOP: several chunks, the next
// one on its way while one is worked on; once a row has a full list of candidates a chunk costs one
// barrier, behind which the chunk before is looked at again if it had too many.
template <int T, bool LOOP>
__global__ __launch_bounds__(T, 4) void logprobs_kernel(LogprobArgs a, int parts, int span,
                                                                   Part* out) {
    constexpr int CHUNK = T * kHeld;
    __shared__ Shared<T> sm;
    const int row = blockIdx.x / parts, p = blockIdx.x - row * parts;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = a.logits + row * a.row_stride;
    const int begin = p * span, end = min(a.vocab, begin + span);
    Sums t = {-__builtin_inff(), 0.0f, 0.0f};
    int have = 0;          // candidates
    float least = 0.0f;    // what a logit must reach once there is a full list of the best
    bool full = false;
    float next[LOOP ? kHeld : 1];
    if (LOOP) load_logits<T>(x, begin, end, next);
    if (tid < 3) sm.added[tid] = 0;
    auto order = [&]() __attribute__((always_inline)) {
        have = order_candidates<T, LOOP>(have, a.top, sm);
        full = have == a.top;
        if (LOOP && full) {
            const unsigned o = (unsigned)((sm.tops[a.top - 1] - 1) >> 32);
            least = o & 0x80000000u ? __uint_as_float(o ^ 0x80000000u)
                    : o             ? __uint_as_float(~o) : -__builtin_inff();
        }
    };
    // the candidates of the chunk from i0 on, whose number is at hand behind a barrier
    auto settle = [&](int i0, int added) __attribute__((always_inline)) {
        const int most = min(a.top, end - i0);
        if (have + added > kCandidates || (!full && added < most)) {
            collect_exactly<T>(x, i0, min(end, i0 + CHUNK), a.top, have, sm);
            added = min(most, CHUNK);
        }
        have += added;
    };
    int turn = 0, last = 0, now = 1, coming = 2;  // the turns of sm.added
    for (int i0 = begin; i0 < end; i0 += CHUNK, turn ^= 1) {
        float v[kHeld];
        if constexpr (LOOP) {
#pragma unroll
            for (int e = 0; e < kHeld; ++e) v[e] = next[e];
            if (i0 + CHUNK < end) load_logits<T>(x, i0 + CHUNK, end, next);
        } else {
            load_logits<T>(x, i0, end, v);
        }
        // each wavefront's own maximum and sums, then everybody joins them
        float mine = -__builtin_inff();  // the thread's best
#pragma unroll
        for (int e = 0; e < kHeld; ++e) mine = fmaxf(mine, v[e]);
        float m = mine;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float at = m == -__builtin_inff() ? 0.0f : m;
        float z = 0.0f, s = 0.0f;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const float d = v[e] - at, w = __builtin_amdgcn_exp2f(d * kLog2e);
            z += w;
            s += w * fmaxf(d, -3.4028234663852886e+38f);  // minus infinity adds nothing
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            z += __shfl_xor(z, o);
            s += __shfl_xor(s, o);
        }
        if (lane == 0) {
            sm.m[turn][wave] = m;
            sm.z[turn][wave] = z;
            sm.x[turn][wave] = s;
        }
        const bool any = i0 + tid * 4 < end;  // the thread holds a logit
        if (!any) mine = __builtin_nanf("");
        if (!full) sm.bests[tid] = any ? order_of(mine) : 0;
        __syncthreads();
        const Sums before = t;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) t.m = fmaxf(t.m, sm.m[turn][w]);
        t.z = t.x = 0.0f;
        add_part(t, before.m, before.z, before.x);
#pragma unroll
        for (int w = 0; w < T / 64; ++w) add_part(t, sm.m[turn][w], sm.z[turn][w], sm.x[turn][w]);
        if (!a.top) continue;
        if (LOOP && full) {
            settle(i0 - CHUNK, sm.added[last]);
            if (tid == 0) sm.added[coming] = 0;
            if (have > 2 * a.top + 32) order();  // and a closer bound from here on
            collect<T>(v, i0, end, mine, least, have, &sm.added[now], sm);
            const int free = last;
            last = now;
            now = coming;
            coming = free;
        } else {
            find_threshold<T>(a.top, sm);
            __syncthreads();
            collect<T>(v, i0, end, mine, sm.threshold, have, &sm.added[now], sm);
            __syncthreads();
            settle(i0, sm.added[now]);
            order();
            if (LOOP) {
                if (tid == 0) sm.added[now] = 0;
                __syncthreads();
            }
        }
    }
    if (LOOP && a.top && end - begin > CHUNK) {
        __syncthreads();
        settle((end - begin - 1) / CHUNK * CHUNK + begin, sm.added[last]);
        order();
    }
    if (parts > 1) {
        Part* part = out + blockIdx.x;
        if (tid == 0) {
            part->m = t.m;
            part->z = t.z;
            part->x = t.x;
        }
        if (tid < a.top) part->rank[tid] = tid < have ? sm.tops[tid] : 0;
        return;
    }
    if (tid == 0) finish(a, row, t);
    if (tid < a.top) {
        const int id = id_of(sm.tops[tid]);
        a.top_ids[(int64_t)row * a.top + tid] = id;
        a.top_logprobs[(int64_t)row * a.top + tid] = lp_of(x[id], t);
    }
}

// Joins a row's parts.  The best of each part come in order, so the merged ones are found by place:
// how many of all are better.  With more of them than fit LDS, one after the other.
constexpr int kJoin = 256, kJoinHeld = 2048;
__global__ __launch_bounds__(kJoin) void logprobs_join_kernel(LogprobArgs a, int chunks,
                                                              const Part* parts) {
    __shared__ unsigned long long held[kJoinHeld];
    __shared__ unsigned long long best[kJoin / 64];
    const int row = blockIdx.x, tid = threadIdx.x;
    const Part* part = parts + (int64_t)row * chunks;
    const int n = chunks * a.top;
    const bool fits = n <= kJoinHeld;
    if (fits)
        for (int i = tid; i < n; i += kJoin) held[i] = part[i / a.top].rank[i % a.top];
    Sums t = {-__builtin_inff(), 0.0f, 0.0f};
    for (int c = 0; c < chunks; ++c) t.m = fmaxf(t.m, part[c].m);
    for (int c = 0; c < chunks; ++c) add_part(t, part[c].m, part[c].z, part[c].x);
    if (tid == 0) finish(a, row, t);
    auto put = [&](int k, unsigned long long r) {
        const int id = id_of(r);
        a.top_ids[(int64_t)row * a.top + k] = id;
        a.top_logprobs[(int64_t)row * a.top + k] = lp_of(a.logits[row * a.row_stride + id], t);
    };
    if (fits) {
        __syncthreads();
        for (int i = tid; i < n; i += kJoin) {
            const unsigned long long r = held[i];
            if (!r) continue;
            int better = 0;
            for (int j = 0; j < n && better < a.top; ++j) better += held[j] > r;
            if (better < a.top) put(better, r);
        }
        return;
    }
    unsigned long long above = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        unsigned long long r = 0;
        for (int i = tid; i < n; i += kJoin) {
            const unsigned long long q = part[i / a.top].rank[i % a.top];
            if (q < above && q > r) r = q;
        }
        r = wave_max(r);
        if ((tid & 63) == 0) best[tid >> 6] = r;
        __syncthreads();
        above = best[0];
        for (int w = 1; w < kJoin / 64; ++w) above = best[w] > above ? best[w] : above;
        if (tid == 0) put(k, above);
        __syncthreads();
    }
}

int parts_of(int rows, int vocab) { return rows >= kManyRows ? 1 : (vocab + kFewSpan - 1) / kFewSpan; }

}  // namespace

namespace shp {

size_t logprobs_scratch(int rows, int vocab) {
    const int p = parts_of(rows, vocab);
    return p > 1 ? (size_t)rows * p * (sizeof(Part) / sizeof(float)) : 0;
}

int logprobs_launch(hipStream_t s, const LogprobArgs& a, float* scratch) {
    const int p = parts_of(a.rows, a.vocab);
    Part* out = reinterpret_cast<Part*>(scratch);
    if (a.rows >= kMostRows)
        hipLaunchKernelGGL((logprobs_kernel<kMostThreads, true>), dim3(a.rows), dim3(kMostThreads), 0, s, a, 1,
                           a.vocab, out);
    else if (a.rows >= kManyRows)
        hipLaunchKernelGGL((logprobs_kernel<kManyThreads, true>), dim3(a.rows), dim3(kManyThreads), 0, s, a, 1,
                           a.vocab, out);
    else
        hipLaunchKernelGGL((logprobs_kernel<kFewThreads, false>), dim3(a.rows * p), dim3(kFewThreads), 0, s, a, p,
                           kFewSpan, out);
    SHP_HIP_CHECK(hipGetLastError());
    if (p > 1) {
        hipLaunchKernelGGL(logprobs_join_kernel, dim3(a.rows), dim3(kJoin), 0, s, a, p, out);
        SHP_HIP_CHECK(hipGetLastError());
    }
    return SHP_OK;
}

}  // namespace shp
