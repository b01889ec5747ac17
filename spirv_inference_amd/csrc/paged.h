// The paged key/value cache: where a token of a sequence lies (device), and the launchers behind
// shp_paged_* (host).
#pragma once

#include "common.h"
#include "fastdiv.h"

namespace shp {

constexpr int kTreeRows = 256;  // rows of a drafted tree at most

// shp_paged with the counts the kernels derive from it.
struct Paged {
    void *k, *v;
    const int32_t* table;
    const int32_t* lengths;
    int n_seqs, kv, n_pages, page_log2, max_pages, cap;  // cap: tokens a table has room for
};

struct PagedRows {
    const float *k, *v, *q;
    float* q_out;
    int64_t k_seq, k_row, k_head, v_seq, v_row, v_head, q_seq, q_row, q_head, o_seq, o_row, o_head;
    const int32_t *counts, *offsets;
    const float* inv_freq;
    int n, heads, rot;  // heads: of q, 0 for none
    bool interleaved;
};
int paged_append_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedRows& r);

struct PagedQuery {
    const float* q;
    float* out;
    int64_t q_seq, q_row, q_head, o_seq, o_row, o_head;
    float* lse;
    const int32_t* counts;
    const float* slopes;
    const int32_t *prefix, *first, *parents;
    int n, heads, group, window;
    float scale, cap;
    shpd::FastDiv by_kv, by_group;  // set by the launch
    // and where the cap is large: scale / cap = factor * 2^lift, half the cap in units of log2
    float factor, half;
    int lift;
};
// Caps from here on are large: 16-bit pieces of scale / cap * q and the cap in units of log2 leave their range.
constexpr float kLargeCap = 0x1p64f;
// How attention shares out rows and tokens, and the floats of scratch that takes (0: none).
struct PagedPlan {
    int rows;              // a workgroup owns: 16 or 32
    bool side;             // a workgroup is one wavefront, else four, which share the tokens
    int target;            // workgroups that the tokens are shared out for; 0: a workgroup takes all of them
    int least;             // tiles a workgroup takes at least
    int grid, row_blocks;  // workgroups: over KV heads and blocks of rows, or (row_blocks 1) over shares
    size_t scratch;
};
PagedPlan paged_attend_plan(const Paged& c, int head_dim, int format, int64_t rows, int cu_count, bool may_split);
int paged_attend_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedQuery& q,
                        const PagedPlan& p, float* scratch, int* counters);

struct PagedTree {
    const int32_t *counts, *parents, *tokens, *choices;
    int32_t *path, *accepted, *next, *lengths_out;
    int n;
};
int paged_accept_launch(hipStream_t s, const Paged& c, int head_dim, int format, const PagedTree& t);

}  // namespace shp

#ifdef __HIPCC__
namespace shpd {

typedef __bf16 bf16;

// Tokens sequence s holds, and how many of the n rows given for it are real, both within what can be.
__device__ __forceinline__ int paged_length(const shp::Paged& c, int s) {
    return min(max(c.lengths[s], 0), c.cap);
}
__device__ __forceinline__ int paged_count(const int32_t* counts, int n, int s) {
    return counts ? min(max(counts[s], 0), n) : n;
}

// The page of a sequence that holds token t (0 <= t < cap), -1 where there is none.
__device__ __forceinline__ int page_of(const shp::Paged& c, int s, int t) {
    const int p = c.table[(int64_t)s * c.max_pages + (t >> c.page_log2)];
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}
// What the launch only reads, at an index that all lanes share: by the scalar unit.
__device__ __forceinline__ int shared_int(const int32_t* p, int64_t i) {
    typedef const __attribute__((address_space(4))) int32_t* Constant;
    return ((Constant)(uintptr_t)p)[i];
}
// page_of where all lanes ask for the same sequence and token.
__device__ __forceinline__ int shared_page_of(const shp::Paged& c, int s, int t) {
    const int p = shared_int(c.table, __builtin_amdgcn_readfirstlane(s) * (int64_t)c.max_pages +
                                          (__builtin_amdgcn_readfirstlane(t) >> c.page_log2));
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}
// Rows before the row of KV head h and token t, which lies in `page`.
__device__ __forceinline__ int64_t row_of(const shp::Paged& c, int page, int h, int t) {
    return (((int64_t)page * c.kv + h) << c.page_log2) + (t & ((1 << c.page_log2) - 1));
}

// Calls f with a value of the type that a cache of this format holds.
template <class F>
inline auto with_format(int format, F f) {
    switch (format) {
        case SHP_PAGED_F32: return f(float());
        case SHP_PAGED_F16: return f(_Float16());
        default: return f(bf16());
    }
}

}  // namespace shpd
#endif
