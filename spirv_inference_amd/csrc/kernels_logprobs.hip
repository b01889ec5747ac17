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

struct Sums {
    float m, z, x;
};

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
    float m = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < kHeld; ++e) m = fmaxf(m, v[e]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = red[0][0];
    for (int w = 1; w < 16; ++w) m = fmaxf(m, red[0][w]);
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
        red[1][wave] = z;
        red[2][wave] = s;
    }
    __syncthreads();
    z = red[1][0];
    s = red[2][0];
    for (int w = 1; w < 16; ++w) {
        z += red[1][w];
        s += red[2][w];
    }
    const Sums t = {m, z, s};
    Part* part = parts + blockIdx.x;
    if (tid == 0) {
        if (chunks == 1) finish(a, row, t);
        else {
            part->m = m;
            part->z = z;
            part->x = s;
        }
    }
    if (!a.top) return;
    // the best of what each thread holds; whoever gives the best of all looks for its next
    unsigned taken = 0;
    auto mine = [&]() {
        unsigned long long r = 0;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const int id = i0 + ((e >> 2) * kThreads + tid) * 4 + (e & 3);
            const unsigned long long q = id < end && !(taken >> e & 1) ? rank_of(v[e], id) + 1 : 0;
            r = q > r ? q : r;
        }
        return r;
    };
    unsigned long long own = mine();
    for (int k = 0; k < a.top; ++k) {
        const unsigned long long w = wave_max(own);
        if (lane == 0) best[k & 1][wave] = w;
        __syncthreads();
        unsigned long long r = best[k & 1][0];
        for (int q = 1; q < 16; ++q) r = best[k & 1][q] > r ? best[k & 1][q] : r;
        const int id = 0x7fffffff - (int)(unsigned)(r - 1);
        if (r && own == r) {
            const int o = id - i0;
            taken |= 1u << ((o >> 2) / kThreads * 4 + (o & 3));
            own = mine();
        }
        if (tid == 0) {
            if (chunks > 1) part->rank[k] = r;
            else {
                a.top_ids[(int64_t)row * a.top + k] = id;
                a.top_logprobs[(int64_t)row * a.top + k] = lp_of(x[id], t);
            }
        }
    }
}

// Joins a row's parts: one wavefront.
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobArgs a, int chunks,
                                                           const Part* parts) {
    const int row = blockIdx.x, lane = threadIdx.x;
    const Part* part = parts + (int64_t)row * chunks;
    Sums t = {-__builtin_inff(), 0.0f, 0.0f};
    for (int c = 0; c < chunks; ++c) t.m = fmaxf(t.m, part[c].m);
    for (int c = 0; c < chunks; ++c) {
        const float z = part[c].z;
        if (z == 0.0f) continue;
        const float d = part[c].m - t.m, f = __builtin_amdgcn_exp2f(d * kLog2e);
        t.z += z * f;
        t.x += (part[c].x + d * z) * f;
    }
    if (lane == 0) finish(a, row, t);
    const int n = chunks * a.top;
    unsigned long long above = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        unsigned long long r = 0;
        for (int i = lane; i < n; i += 64) {
            const unsigned long long q = part[i / a.top].rank[i % a.top];
            if (q < above && q > r) r = q;
        }
        above = wave_max(r);
        if (lane == 0) {
            const int id = 0x7fffffff - (int)(unsigned)(above - 1);
            a.top_ids[(int64_t)row * a.top + k] = id;
            a.top_logprobs[(int64_t)row * a.top + k] = lp_of(a.logits[row * a.row_stride + id], t);
        }
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
        hipLaunchKernelGGL(logprobs_join_kernel, dim3(a.rows), dim3(64), 0, s, a, c, parts);
        SHP_HIP_CHECK(hipGetLastError());
    }
    return SHP_OK;
}

}  // namespace shp
