// The paged cache's appends, with the rotation by position on the way, and the acceptance of drafted
// trees.
#include "paged.h"

namespace {

using namespace shpd;
using shp::kTreeRows;
using shp::Paged;
using shp::PagedRows;
using shp::PagedTree;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

// cos and sin of position * freq.  The product is formed in 64 bits: exact for positions below 2^29 (freq has 24
// bits), beyond that and in quarter turns rounded to 2^-53 of itself.  What is left without the whole quarter turns
// is at most an eighth of a turn, where the Taylor series end within 2^-29 after x^11 and x^10.
__device__ __forceinline__ void turn(double position, float freq, float& c, float& s) {
    constexpr double kQuarters = 0.63661977236758134308, kQuarter = 1.57079632679489661923;
    const double t = position * (double)freq * kQuarters, n = __builtin_rint(t);
    const float x = (float)((t - n) * kQuarter), y = x * x;
    const int m = (int)(long long)n & 3;
    const float sine = x + x * y * (-1.0f / 6 + y * (1.0f / 120 + y * (-1.0f / 5040 + y * (1.0f / 362880 - y * (1.0f / 39916800)))));
    const float cosine = 1.0f + y * (-0.5f + y * (1.0f / 24 + y * (-1.0f / 720 + y * (1.0f / 40320 - y * (1.0f / 3628800)))));
    s = m & 1 ? cosine : sine;
    c = m & 1 ? sine : cosine;
    if (m & 2) s = -s;
    if (m == 1 || m == 2) c = -c;
}

// Four numbers next to each other.
template <class E>
__device__ __forceinline__ void store4(E* p, f4 v) {
    typedef E e4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<e4*>(p) = __builtin_convertvector(v, e4);
}

// A thread takes 8 dimensions of a head of a row: two runs of 4, which are those of a pair where
// dimensions j and j + rot / 2 are turned together.  blockIdx.x is a row of a sequence, and heads are
// q's, k's and v's one after the other.  Memory bounds prompts: 4 of up to 2,000 rows of 32 + 8 + 8 heads x 128
// into bf16 (104 MB) 19.5 us, 5.3 TB/s, with angles made once for four heads as well; a token of 64 sequences
// takes 3.8 us, which is latency.
template <class E, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(Paged c, PagedRows r) {
    constexpr int T = D / 8;
    const int s = blockIdx.x / r.n, i = blockIdx.x - s * r.n;
    const int count = paged_count(r.counts, r.n, s);
    if (i >= count) return;
    const int begin = paged_length(c, s) - count, place = begin + i;
    const int heads = r.heads + 2 * c.kv;
    const int page = place >= 0 ? page_of(c, s, place) : -1;
    for (int e = blockIdx.y * 256 + threadIdx.x; e < heads * T; e += gridDim.y * 256) {
        const int head = e / T, t = e - head * T;
        const bool is_q = head < r.heads, is_v = head >= r.heads + c.kv;
        const int h = is_q ? head : is_v ? head - r.heads - c.kv : head - r.heads;
        if (!is_q && page < 0) continue;
        const bool turned = !is_v && t < r.rot / 8;
        const int d0 = turned && !r.interleaved ? 4 * t : 8 * t;
        const int d1 = turned && !r.interleaved ? d0 + r.rot / 2 : d0 + 4;
        const float* x = is_q   ? r.q + s * r.q_seq + i * r.q_row + h * r.q_head
                         : is_v ? r.v + s * r.v_seq + i * r.v_row + h * r.v_head
                                : r.k + s * r.k_seq + i * r.k_row + h * r.k_head;
        f4 a = *reinterpret_cast<const f4*>(x + d0), b = *reinterpret_cast<const f4*>(x + d1);
        if (turned) {
            const double position = (double)begin + (r.offsets ? r.offsets[(int64_t)s * r.n + i] : i);  // of 33 bits
            f4 co, si;
#pragma unroll
            for (int j = 0; j < 4; ++j) turn(position, r.inv_freq[4 * t + j], ((float*)&co)[j], ((float*)&si)[j]);
            if (r.interleaved) {
                const f4 x0 = {a.x, a.z, b.x, b.z}, x1 = {a.y, a.w, b.y, b.w};
                const f4 y0 = x0 * co - x1 * si, y1 = x1 * co + x0 * si;
                a = f4{y0.x, y1.x, y0.y, y1.y};
                b = f4{y0.z, y1.z, y0.w, y1.w};
            } else {
                const f4 x0 = a, x1 = b;
                a = x0 * co - x1 * si;
                b = x1 * co + x0 * si;
            }
        }
        if (is_q) {
            float* y = r.q_out + s * r.o_seq + i * r.o_row + h * r.o_head;
            *reinterpret_cast<f4*>(y + d0) = a;
            *reinterpret_cast<f4*>(y + d1) = b;
        } else {
            E* y = (E*)(is_v ? c.v : c.k) + row_of(c, page, h, place) * D;
            store4(y + d0, a);
            store4(y + d1, b);
        }
    }
}

// A workgroup takes a sequence, whose length it reads before it writes it.  Which row follows which is
// settled for all rows at once: row j follows its parent if its id is the one chosen there, and of
// several the first does.  Then the path is a chain.  It rises, so that a row only moves to the front,
// past rows that are moved or dropped: eight rows at a time are read and then written, and a thread
// moves the same 16 bytes of each, so that nothing is overwritten that has still to be read.  Latency bounds
// it: 2.9 us for a tree of 24 rows in fp32, 5.2 us for 64 of 60 rows x 8 heads x 128 in bf16.
template <class E, int D>
__global__ __launch_bounds__(256) void paged_accept_kernel(Paged c, PagedTree t) {
    __shared__ int follow[kTreeRows], path[kTreeRows], from[kTreeRows], to[kTreeRows];
    const int s = blockIdx.x, tid = threadIdx.x;
    const int len = paged_length(c, s), count = paged_count(t.counts, t.n, s), begin = len - count;
    const int32_t *parents = t.parents + (int64_t)s * t.n, *tokens = t.tokens + (int64_t)s * t.n;
    const int32_t* choices = t.choices + (int64_t)s * t.n;
    const bool any = count > 0 && begin >= 0;
    follow[tid] = kTreeRows;
    __syncthreads();
    if (tid > 0 && tid < count) {
        const int p = parents[tid];
        if (p >= 0 && p < tid && tokens[tid] == choices[p]) atomicMin(&follow[p], tid);
    }
    __syncthreads();
    int kept = 0, last = 0;
    if (any)
        for (int node = 0; node < count; node = follow[node]) {  // rises
            if (tid == 0) path[kept] = node;
            last = node;
            ++kept;
        }
    __syncthreads();
    if (tid < kept) {
        const int a = begin + path[tid], b = begin + tid;
        const int pa = page_of(c, s, a), pb = page_of(c, s, b);
        from[tid] = pa;
        to[tid] = pa < 0 ? -1 : pb;
    }
    if (tid < t.n) t.path[(int64_t)s * t.n + tid] = tid < kept ? path[tid] : -1;
    if (tid == 0) {
        t.accepted[s] = kept;
        t.next[s] = kept ? choices[last] : -1;
        t.lengths_out[s] = any ? begin + kept : len;
    }
    __syncthreads();
    constexpr int W = D * sizeof(E) / 16, B = 8;
    for (int e = tid; e < 2 * c.kv * W; e += 256) {
        const int head = e / W, w = e - head * W, h = head % c.kv;
        u4* const x = (u4*)(head < c.kv ? c.k : c.v) + w;
        for (int j0 = 1; j0 < kept; j0 += B) {
            u4 v[B];
#pragma unroll
            for (int j = 0; j < B; ++j)
                if (j0 + j < kept && to[j0 + j] >= 0)
                    v[j] = x[row_of(c, from[j0 + j], h, begin + path[j0 + j]) * W];
#pragma unroll
            for (int j = 0; j < B; ++j)
                if (j0 + j < kept && to[j0 + j] >= 0)
                    x[row_of(c, to[j0 + j], h, begin + j0 + j) * W] = v[j];
        }
    }
}

}  // namespace

namespace shp {

int paged_append_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedRows& r) {
    const int64_t rows = (int64_t)c.n_seqs * r.n;  // 16,000,000 at most
    const int64_t units = (int64_t)(r.heads + 2 * c.kv) * (head_dim / 8);
    const dim3 grid((unsigned)rows, (unsigned)std::min<int64_t>((units + 255) / 256, 65535));
    with_format(format, [&](auto e) {
        using E = decltype(e);
        auto kern = head_dim == 64 ? paged_append_kernel<E, 64> : paged_append_kernel<E, 128>;
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, r);
    });
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

int paged_accept_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedTree& t) {
    with_format(format, [&](auto e) {
        using E = decltype(e);
        auto kern = head_dim == 64 ? paged_accept_kernel<E, 64> : paged_accept_kernel<E, 128>;
        hipLaunchKernelGGL(kern, dim3(c.n_seqs), dim3(256), 0, s, c, t);
    });
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

}  // namespace shp
