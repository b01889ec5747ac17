// The 8-bit key/value cache: writing new rows, reading values back, and eviction.
#include "cache8.h"

namespace {

using namespace shpd;
using shp::Cache8;
using shp::Cache8Rows;
using shp::kCacheTile;
typedef float f4 __attribute__((ext_vector_type(4)));

// Largest |x| of a workgroup's threads, infinite where one saw an infinity or a NaN.
__device__ __forceinline__ float group_max(float x, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
    for (int w = 1; w < (int)blockDim.x >> 6; ++w) x = fmaxf(x, red[w]);
    return x;
}

__device__ __forceinline__ float top_of(f4 x) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // a NaN fails the comparison and counts as an infinity
        t = fmaxf(t, fabsf(x[i]) <= 3.4028234663852886e+38f ? fabsf(x[i]) : __builtin_inff());
    return t;
}

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

// One block of K or V of one head that gets new rows; grid (blocks a call can touch, seqs * kv, 2).
template <int D, int FMT, bool V>
__device__ __forceinline__ void append_block(const Cache8& c, const Cache8Rows& r, float* red) {
    const int sh = blockIdx.y, s = sh / c.kv, h = sh - s * c.kv, B = 1 << c.block_log2;
    const int len = seq_length(c, s), start = len - seq_count(r.counts, r.n, s);
    const int t0 = (max(start, 0) >> c.block_log2 << c.block_log2) + (int)blockIdx.x * B;
    const int a = max(start, t0), t1 = min(len, t0 + B);
    if (a >= t1) return;
    const float* x = V ? r.v + s * r.v_seq + h * r.v_head : r.k + s * r.k_seq + h * r.k_head;
    const int64_t row = V ? r.v_row : r.k_row;
    uint8_t* codes = (V ? c.v : c.k) + (int64_t)sh * c.cap * D;
    float* scale = (V ? c.v_scale : c.k_scale) + block_at(c, sh, t0);

    constexpr int Q = D / 4;
    float top = 0.0f;
    for (int e = threadIdx.x; e < (t1 - a) * Q; e += 256)
        top = fmaxf(top, top_of(*reinterpret_cast<const f4*>(x + (a - start + e / Q) * row + e % Q * 4)));
    float now = block_scale<FMT>(group_max(top, red));
    const float was = a > t0 ? *scale : now;
    __syncthreads();  // everybody has read the old scale
    if (!(now < was) && a > t0 && !(was >= 0.0f)) now = was;  // a NaN stays
    if (now < was) now = was;
    if (threadIdx.x == 0) *scale = now;
    for (int e = threadIdx.x; e < (t1 - a) * Q; e += 256) {
        const int t = a + e / Q, d = e % Q * 4;
        const f4 v = *reinterpret_cast<const f4*>(x + (t - start) * row + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            codes[code_at<D, V>(t, d + i)] = (uint8_t)encode<FMT>(v[i], now);
    }
    if (now > was)
        for (int e = threadIdx.x; e < (a - t0) * D; e += 256) {
            uint8_t* p = codes + code_at<D, V>(t0 + e / D, e % D);
            *p = (uint8_t)encode<FMT>(code_value<FMT>(*p, 0) * was, now);
        }
}

template <int D, int FMT>
__global__ __launch_bounds__(256) void cache8_append_kernel(Cache8 c, Cache8Rows r) {
    __shared__ float red[4];
    if (blockIdx.z) append_block<D, FMT, true>(c, r, red);
    else append_block<D, FMT, false>(c, r, red);
}

// Thread = 4 dimensions of one of the newest n tokens of a head.
template <int D, int FMT>
__global__ __launch_bounds__(256) void cache8_read_kernel(Cache8 c, int n, float* k, float* v) {
    const int sh = blockIdx.y, s = sh / c.kv;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int i = (int)(e / (D / 4)), d = (int)(e % (D / 4)) * 4;
    if (i >= n) return;
    const int t = seq_length(c, s) - n + i;
    f4 kx = {0.f, 0.f, 0.f, 0.f}, vx = kx;
    if (t >= 0) {
        const int64_t base = (int64_t)sh * c.cap * D;
        const int64_t b = block_at(c, sh, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (k) kx[j] = code_value<FMT>(c.k[base + code_at<D, false>(t, d + j)], 0) * c.k_scale[b];
            if (v) vx[j] = code_value<FMT>(c.v[base + code_at<D, true>(t, d + j)], 0) * c.v_scale[b];
        }
    }
    const int64_t o = ((int64_t)sh * n + i) * D + d;
    if (k) *reinterpret_cast<f4*>(k + o) = kx;
    if (v) *reinterpret_cast<f4*>(v + o) = vx;
}

// A float as an unsigned number of the same order: NaN lowest, both zeros alike.
__device__ __forceinline__ unsigned order_of(float x) {
    if (!(x == x)) return 0u;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One sequence and head: which of its tokens stay.  The smallest key that stays is found eight
// bits at a time by counting; the tokens then go out in their order.
__global__ __launch_bounds__(1024) void cache8_select_kernel(Cache8 src, Cache8 dst,
                                                             const float* __restrict__ weights,
                                                             int keep, int recent, int32_t* kept,
                                                             float* dst_weights) {
    __shared__ unsigned hist[256];
    __shared__ unsigned part[16];
    __shared__ unsigned found[2];
    const int sh = blockIdx.x, s = sh / src.kv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = seq_length(src, s);
    const float* w = weights + (int64_t)sh * src.cap;
    int32_t* const out = kept + (int64_t)sh * keep;
    float* const ow = dst_weights ? dst_weights + (int64_t)sh * dst.cap : nullptr;
    const int m = min(len, keep);
    if (sh % src.kv == 0 && tid == 0) dst.lengths[s] = m;
    for (int i = m + tid; i < keep; i += 1024) out[i] = -1;
    if (ow)
        for (int i = m + tid; i < dst.cap; i += 1024) ow[i] = 0.0f;
    if (len <= keep) {
        for (int i = tid; i < len; i += 1024) {
            out[i] = i;
            if (ow) ow[i] = w[i];
        }
        return;
    }
    const int old = len - recent;    // tokens that compete
    unsigned need = keep - recent;   // how many of them stay
    unsigned key = 0;                // of the last one that stays
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int i = tid; i < old; i += 1024) {
                const unsigned o = order_of(w[i]);
                if ((o & mask) == key) atomicAdd(&hist[(o >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                unsigned above = 0;
                int b = 255;
                while (above + hist[b] < need) above += hist[b--];
                found[0] = (unsigned)b;
                found[1] = above;
            }
            __syncthreads();
            key |= found[0] << shift;
            need -= found[1];
            __syncthreads();
        }
    }
    // in order: larger keys, the first `need` equal ones, the newest
    const bool none = keep == recent;
    unsigned base = 0, equal = 0;
    for (int i0 = 0; i0 < old && !none; i0 += 1024) {
        const int i = i0 + tid;
        const float x = i < old ? w[i] : 0.0f;
        const unsigned o = order_of(x);
        const bool eq = i < old && o == key, gt = i < old && o > key;
        // places of the equal ones first, as they decide who stays
        const unsigned long long be = __ballot(eq);
        if (lane == 0) part[wave] = (unsigned)__popcll(be);
        __syncthreads();
        unsigned before = equal, all = equal;
        for (int q = 0; q < 16; ++q) {
            if (q < wave) before += part[q];
            all += part[q];
        }
        before += (unsigned)__popcll(be & ((1ull << lane) - 1));
        const bool stay = gt || (eq && before < need);
        equal = all;
        __syncthreads();
        const unsigned long long bs = __ballot(stay);
        if (lane == 0) part[wave] = (unsigned)__popcll(bs);
        __syncthreads();
        unsigned at = base;
        for (int q = 0; q < 16; ++q) {
            if (q < wave) at += part[q];
            base += part[q];
        }
        at += (unsigned)__popcll(bs & ((1ull << lane) - 1));
        if (stay) {
            out[at] = i;
            if (ow) ow[at] = x;
        }
        __syncthreads();
    }
    for (int i = tid; i < recent; i += 1024) {
        out[keep - recent + i] = old + i;
        if (ow) ow[keep - recent + i] = w[old + i];
    }
}

// One block of K or V of dst, made from the kept tokens of src.
template <int D, int FMT, bool V>
__device__ __forceinline__ void gather_block(const Cache8& src, const Cache8& dst,
                                             const int32_t* kept, int keep, float* red) {
    const int sh = blockIdx.y, s = sh / src.kv, B = 1 << dst.block_log2;
    const int t0 = (int)blockIdx.x * B, t1 = min(min(seq_length(src, s), keep), t0 + B);
    if (t0 >= t1) return;
    const int32_t* id = kept + (int64_t)sh * keep;
    const uint8_t* from = (V ? src.v : src.k) + (int64_t)sh * src.cap * D;
    const float* from_scale = V ? src.v_scale : src.k_scale;
    uint8_t* to = (V ? dst.v : dst.k) + (int64_t)sh * dst.cap * D;
    auto value = [&](int e) {
        const int t = id[t0 + e / D], d = e % D;
        return code_value<FMT>(from[code_at<D, V>(t, d)], 0) *
               from_scale[block_at(src, sh, t)];
    };
    float top = 0.0f;
    for (int e = threadIdx.x; e < (t1 - t0) * D; e += 256) {
        const float x = value(e);
        top = fmaxf(top, top_of(f4{x, 0.f, 0.f, 0.f}));
    }
    const float scale = block_scale<FMT>(group_max(top, red));
    if (threadIdx.x == 0)
        (V ? dst.v_scale : dst.k_scale)[block_at(dst, sh, t0)] = scale;
    for (int e = threadIdx.x; e < (t1 - t0) * D; e += 256)
        to[code_at<D, V>(t0 + e / D, e % D)] = (uint8_t)encode<FMT>(value(e), scale);
}

template <int D, int FMT>
__global__ __launch_bounds__(256) void cache8_gather_kernel(Cache8 src, Cache8 dst,
                                                            const int32_t* kept, int keep) {
    __shared__ float red[4];
    if (blockIdx.z) gather_block<D, FMT, true>(src, dst, kept, keep, red);
    else gather_block<D, FMT, false>(src, dst, kept, keep, red);
}

}  // namespace

namespace shp {

// KERN<head_dim, format> for a cache's head_dim and format.
#define SHP_CACHE8_KERNEL(KERN, head_dim, format)                                   \
    ((head_dim) == 64 ? ((format) == SHP_CACHE8_I8 ? KERN<64, shpd::kI8> : KERN<64, shpd::kE4M3>) \
                      : ((format) == SHP_CACHE8_I8 ? KERN<128, shpd::kI8> : KERN<128, shpd::kE4M3>))

int cache8_append_launch(hipStream_t s, const Cache8& c, int head_dim, int format,
                         const Cache8Rows& r) {
    const int B = 1 << c.block_log2;
    // n rows end anywhere: they touch at most this many blocks
    const int blocks = (std::min(r.n, c.cap) + B - 2) / B + 1;
    hipLaunchKernelGGL(SHP_CACHE8_KERNEL(cache8_append_kernel, head_dim, format),
                       dim3(blocks, c.n_seqs * c.kv, 2), dim3(256), 0, s, c, r);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

int cache8_read_launch(hipStream_t s, const Cache8& c, int head_dim, int format, int n, float* k,
                       float* v) {
    const unsigned gx = (unsigned)(((int64_t)n * (head_dim / 4) + 255) / 256);
    hipLaunchKernelGGL(SHP_CACHE8_KERNEL(cache8_read_kernel, head_dim, format),
                       dim3(gx, c.n_seqs * c.kv), dim3(256), 0, s, c, n, k, v);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

int cache8_evict_launch(hipStream_t s, const Cache8& src, const Cache8& dst, int head_dim,
                        int format, const float* weights, int keep, int recent, int32_t* kept,
                        float* dst_weights) {
    hipLaunchKernelGGL(cache8_select_kernel, dim3(src.n_seqs * src.kv), dim3(1024), 0, s, src, dst,
                       weights, keep, recent, kept, dst_weights);
    SHP_HIP_CHECK(hipGetLastError());
    const int B = 1 << dst.block_log2, blocks = (std::min(keep, src.cap) + B - 1) / B;
    hipLaunchKernelGGL(SHP_CACHE8_KERNEL(cache8_gather_kernel, head_dim, format),
                       dim3(blocks, src.n_seqs * src.kv, 2), dim3(256), 0, s, src, dst, kept, keep);
    SHP_HIP_CHECK(hipGetLastError());
    return SHP_OK;
}

}  // namespace shp
