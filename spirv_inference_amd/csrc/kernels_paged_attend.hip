// Attention over the paged cache.
#include "paged.h"

namespace {

using namespace shpd;
using shp::kTreeRows;
using shp::Paged;
using shp::PagedQuery;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// A wavefront takes a row of a query head and walks its sequence's tokens 64 at a time: a lane has a
// token's score, then the weights go round and a lane has D / 64 dimensions of the output.
template <class E, int D>
__global__ __launch_bounds__(64) void paged_attend_kernel(Paged c, PagedQuery q) {
    __shared__ float qs[D];
    __shared__ int above[kTreeRows];  // rows from the row up to this one, -1: not above it
    const int lane = threadIdx.x, head = blockIdx.x, s = blockIdx.z;
    const int h = head / q.group;
    const int len = paged_length(c, s), count = paged_count(q.counts, q.n, s), begin = len - count;
    // weights are 2^room times smaller, so that sums of them times V are no larger than V
    const int room = 32 - __builtin_clz(max(len, 1));
    const float small = __builtin_ldexpf(1.0f, -room);
    for (int i = blockIdx.y; i < count; i += gridDim.y) {
        __syncthreads();
        const float* x = q.q + s * q.q_seq + i * q.q_row + head * q.q_head;
        for (int d = lane; d < D; d += 64) qs[d] = x[d] * q.scale;
        const int place = begin + i;
        int position = place;
        if (q.parents) {
            for (int u = lane; u < kTreeRows; u += 64) above[u] = -1;
            __syncthreads();
            int steps = 0;
            for (int u = i;;) {
                if (lane == 0) above[u] = steps;
                const int p = q.parents[(int64_t)s * q.n + u];
                if (p < 0 || p >= u) break;
                u = p;
                ++steps;
            }
            position = begin + steps;
        }
        __syncthreads();
        const int first = q.first ? q.first[(int64_t)s * q.n + i] : 0;
        const int prefix = q.prefix ? q.prefix[s] : 0;
        const float slope = q.slopes ? q.slopes[head] : 0.0f;
        float m = -__builtin_inff(), l = 0.0f, o[D / 64] = {};
        for (int t0 = 0; t0 < len && place >= 0; t0 += 64) {
            const int t = t0 + lane;
            int far = position - t;
            bool sees = t < len, kin = t <= place;
            const int page = t < len ? page_of(c, s, t) : -1;
            if (q.parents && t >= begin && t < len) {
                const int up = above[t - begin];
                kin = up >= 0;
                far = up;
                sees = sees && kin;
            }
            sees = sees && page >= 0 && t >= first &&
                   ((kin && (q.window == 0 || far < q.window)) || t < prefix);
            float y = -__builtin_inff();
            if (sees) {
                const E* k = (const E*)c.k + row_of(c, page, h, t) * D;
                y = 0.0f;
                for (int d = 0; d < D; ++d) y = __builtin_fmaf(qs[d], (float)k[d], y);
                if (q.cap > 0.0f) y = q.cap * tanhf(y / q.cap);
                y -= slope * fabsf((float)far);
            }
            const float top = fmaxf(m, wave_max(y));
            const float w = sees ? expf(y - top) * small : 0.0f;
            const float down = m == top ? 1.0f : expf(m - top);
            l = l * down + wave_sum(w);
#pragma unroll
            for (int d = 0; d < D / 64; ++d) o[d] *= down;
            m = top;
            for (int j = 0; j < 64; ++j) {
                if (!__shfl((int)sees, j)) continue;
                const float wj = __shfl(w, j);
                const int pj = __shfl(page, j);
                const E* v = (const E*)c.v + row_of(c, pj, h, t0 + j) * D;
#pragma unroll
                for (int d = 0; d < D / 64; ++d) o[d] = __builtin_fmaf(wj, (float)v[64 * d + lane], o[d]);
            }
        }
        float* out = q.out + s * q.o_seq + i * q.o_row + head * q.o_head;
#pragma unroll
        for (int d = 0; d < D / 64; ++d) out[64 * d + lane] = l == 0.0f ? 0.0f : o[d] / l;
        if (q.lse && lane == 0)
            q.lse[((int64_t)s * q.heads + head) * q.n + i] = l == 0.0f ? -__builtin_inff() : m + logf(l / small);
    }
}

}  // namespace

namespace shp {

int paged_attend_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedQuery& q) {
    const dim3 grid(q.heads, std::min(q.n, 65535), c.n_seqs);
    with_format(format, [&](auto e) {
        using E = decltype(e);
        auto kern = head_dim == 64 ? paged_attend_kernel<E, 64> : paged_attend_kernel<E, 128>;
        hipLaunchKernelGGL(kern, grid, dim3(64), 0, s, c, q);
    });
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

}  // namespace shp
