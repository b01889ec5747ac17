// How likely tokens are: log probability of a given id, entropy and the likeliest ids of each row
// of logits, from one read of the row.
//
// A workgroup holds up to 32,768 logits of a row in registers, 32 a thread: their maximum m, Z =
// sum exp(x - m) and X = sum exp(x - m) (x - m) give log p = x - m - log Z and the entropy log Z -
// X / Z, a sum of two numbers that are not negative.  A longer row goes to several workgroups and
// its parts are joined.
#include "cache8.h"

namespace {

using shp::kMaxTop;
using shp::LogprobArgs;
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 1024, kHeld = 32, kChunk = kThreads * kHeld;
constexpr int kCandidates = 512;  // logits at a row's threshold that are put in order by counting
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

// Adds a part to sums whose maximum is t.m already.
__device__ __forceinline__ void add_part(Sums& t, float m, float z, float x) {
    if (z == 0.0f) return;  // nothing but minus infinity
    const float d = m - t.m, f = __builtin_amdgcn_exp2f(d * kLog2e);
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

__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobArgs a, int chunks, Part* parts) {
    __shared__ float red[3][16];
    __shared__ unsigned long long best[2][16];
    __shared__ unsigned bests[kThreads];
    __shared__ unsigned long long candidates[kCandidates];
    __shared__ float threshold;
    __shared__ int found;
    const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = a.logits + row * a.row_stride;
    const int i0 = chunk * kChunk, end = min(a.vocab, i0 + kChunk);
    float v[kHeld];
#pragma unroll
    for (int p = 0; p < kHeld / 4; ++p) {
        const int i = i0 + (p * kThreads + tid) * 4;
        if (i + 4 <= end) {
            const f4u t = *reinterpret_cast<const f4u*>(x + i);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * p + c] = t[c];
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * p + c] = i + c < end ? x[i + c] : -__builtin_inff();
        }
    }
    // each wavefront's own maximum and sums, then everybody joins the sixteen
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
        red[0][wave] = m;
        red[1][wave] = z;
        red[2][wave] = s;
    }
    const bool any = i0 + tid * 4 < end;  // the thread holds a logit
    bests[tid] = any ? order_of(mine) : 0;
    if (tid == 0) found = 0;
    __syncthreads();
    Sums t = {-__builtin_inff(), 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 16; ++w) t.m = fmaxf(t.m, red[0][w]);
#pragma unroll
    for (int w = 0; w < 16; ++w) add_part(t, red[0][w], red[1][w], red[2][w]);
    Part* part = parts + blockIdx.x;
    if (tid == 0) {
        if (chunks == 1) finish(a, row, t);
        else {
            part->m = t.m;
            part->z = t.z;
            part->x = t.x;
        }
    }
    if (!a.top) return;
    const bool one = chunks == 1;
    auto put = [&](int k, unsigned long long r) {
        if (!one) {
            part->rank[k] = r;
        } else if (r) {
            const int id = id_of(r);
            a.top_ids[(int64_t)row * a.top + k] = id;
            a.top_logprobs[(int64_t)row * a.top + k] = lp_of(x[id], t);
        }
    };

    // A threshold that `top` threads reach with the best they hold, so that `top` logits or more do:
    // one wavefront halves the range of the threads' best until no more than twice as many pass.
    if (tid < 64) {
        unsigned b[kThreads / 64], lo = ~0u, hi = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 64; ++i) {
            b[i] = bests[i * 64 + tid];
            lo = min(lo, b[i]);
            hi = max(hi, b[i]);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            lo = min(lo, (unsigned)__shfl_xor((int)lo, o));
            hi = max(hi, (unsigned)__shfl_xor((int)hi, o));
        }
        for (int turn = 0; turn < 24 && hi - lo > 1; ++turn) {
            const unsigned next = lo + (hi - lo) / 2;
            int n = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 64; ++i) n += __popcll(__ballot(b[i] >= next));
            if (n < a.top) {
                hi = next;
            } else {
                lo = next;
                if (n <= 2 * a.top) break;
            }
        }
        // as a float of that order; lo 0: some threads hold nothing, and the others all they have
        if (tid == 0) threshold = lo & 0x80000000u ? __uint_as_float(lo ^ 0x80000000u)
                                  : lo            ? __uint_as_float(~lo) : -__builtin_inff();
    }
    __syncthreads();
    const float least = threshold;
    if (any && mine >= least) {
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const int id = i0 + ((e >> 2) * kThreads + tid) * 4 + (e & 3);
            if (id < end && v[e] >= least) {
                const int c = atomicAdd(&found, 1);
                if (c < kCandidates) candidates[c] = rank_of(v[e], id) + 1;
            }
        }
    }
    __syncthreads();
    const int n = found;
    if (n <= kCandidates && n >= min(a.top, end - i0)) {
        // a candidate's place is how many are better; their order in LDS does not matter
        for (int i = tid; i < n; i += kThreads) {
            const unsigned long long r = candidates[i];
            int better = 0;
            for (int j = 0; j < n; ++j) better += candidates[j] > r;
            if (better < a.top) put(better, r);
        }
        for (int k = n + tid; k < a.top; k += kThreads) put(k, 0);  // a chunk of few logits
        return;
    }

    // Too many logits about as large as the best (ties, or a few threads that hold them all), or too
    // few that are numbers: the best of what each thread holds, and whoever gives the best of all looks for its next.
    unsigned taken = 0;
    auto next_best = [&]() {
        unsigned long long r = 0;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const int id = i0 + ((e >> 2) * kThreads + tid) * 4 + (e & 3);
            const unsigned long long q = id < end && !(taken >> e & 1) ? rank_of(v[e], id) + 1 : 0;
            r = q > r ? q : r;
        }
        return r;
    };
    unsigned long long own = next_best();
    for (int k = 0; k < a.top; ++k) {
        const unsigned long long w = wave_max(own);
        if (lane == 0) best[k & 1][wave] = w;
        __syncthreads();
        unsigned long long r = best[k & 1][0];
        for (int q = 1; q < 16; ++q) r = best[k & 1][q] > r ? best[k & 1][q] : r;
        if (r && own == r) {
            const int o = id_of(r) - i0;
            taken |= 1u << ((o >> 2) / kThreads * 4 + (o & 3));
            own = next_best();
        }
        if (tid == 0) put(k, r);
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

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

namespace shp {

size_t logprobs_scratch(int rows, int vocab, int top) {
    (void)top;
    const int c = chunks_of(vocab);
    return c > 1 ? (size_t)rows * c * (sizeof(Part) / sizeof(float)) : 0;
}

int logprobs_launch(hipStream_t s, const LogprobArgs& a, float* scratch) {
    const int c = chunks_of(a.vocab);
    Part* parts = reinterpret_cast<Part*>(scratch);
    hipLaunchKernelGGL(logprobs_kernel, dim3(a.rows * c), dim3(kThreads), 0, s, a, c, parts);
    SHP_HIP_CHECK(hipGetLastError());
    if (c > 1) {
        hipLaunchKernelGGL(logprobs_join_kernel, dim3(a.rows), dim3(kJoin), 0, s, a, c, parts);
        SHP_HIP_CHECK(hipGetLastError());
    }
    return SHP_OK;
}

}  // namespace shp
