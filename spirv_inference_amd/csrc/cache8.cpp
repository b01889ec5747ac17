// The C ABI of the 8-bit cache and of token log probabilities: argument checks, scratch and
// timing around the launchers.  Arguments are checked before the context, so a refusal needs no
// device.
#include <array>
#include <cmath>
#include <vector>

#include "cache8.h"
#include "runtime.h"

namespace shp {
namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool aligned4(const void* p) { return ((uintptr_t)p & 3) == 0; }
template <class... P>
bool aligned4(const void* p, P... rest) { return aligned4(p) && aligned4(rest...); }

int bad(const char* where, const char* what, int code = SHP_ERR_INVALID) {
    return fail(code, std::string(where) + ": " + what);
}

int check_cache(const char* where, const shp_cache8* c, Cache8* out) {
    if (!c) return bad(where, "null cache");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->lengths)
        return bad(where, "null array in the cache");
    if (c->format != SHP_CACHE8_I8 && c->format != SHP_CACHE8_E4M3)
        return bad(where, "unknown format", SHP_ERR_UNSUPPORTED);
    if (c->head_dim != 64 && c->head_dim != 128)
        return bad(where, "head_dim must be 64 or 128", SHP_ERR_UNSUPPORTED);
    int lb = 0;
    while (lb < 7 && (16 << lb) != c->block) ++lb;
    if (lb > 3) return bad(where, "block must be 16, 32, 64 or 128", SHP_ERR_UNSUPPORTED);
    if (c->n_seqs < 1 || c->n_kv_heads < 1 || (int64_t)c->n_seqs * c->n_kv_heads > 65535)
        return bad(where, "n_seqs * n_kv_heads must be 1 to 65535", SHP_ERR_SHAPE);
    if (c->capacity < 1 || c->capacity > (1 << 22) || c->capacity % 64 || c->capacity % c->block)
        return bad(where, "capacity must be a multiple of 64 and of block, at most 4194304",
                   SHP_ERR_SHAPE);
    if (!aligned16(c->k) || !aligned16(c->v))
        return bad(where, "k and v must be 16-byte aligned");
    if (!aligned4(c->k_scale) || !aligned4(c->v_scale) || !aligned4(c->lengths))
        return bad(where, "scales and lengths must be 4-byte aligned");
    *out = Cache8{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, c->lengths,
                  c->n_seqs, c->n_kv_heads, c->capacity, lb + 4};
    return SHP_OK;
}

int check_rows(const char* where, const char* what, const float* p, int64_t seq, int64_t row,
               int64_t head) {
    if (!p) return bad(where, (std::string("null ") + what).c_str());
    if (!aligned16(p) || (seq | row | head) & 3)
        return bad(where, (std::string(what) + " rows must be 16-byte aligned").c_str());
    return SHP_OK;
}

struct Range {
    uintptr_t from, bytes;
    Range(const void* p, int64_t n) : from((uintptr_t)p), bytes(p ? (uintptr_t)n : 0) {}
    bool meets(const Range& o) const {
        return bytes && o.bytes && from < o.from + o.bytes && o.from < from + bytes;
    }
};
std::array<Range, 5> ranges(const Cache8& c, int head_dim) {
    const int64_t n = (int64_t)c.n_seqs * c.kv * c.cap, scales = (n >> c.block_log2) * 4;
    return {Range(c.k, n * head_dim), Range(c.v, n * head_dim), Range(c.k_scale, scales),
            Range(c.v_scale, scales), Range(c.lengths, c.n_seqs * 4ll)};
}
// Whether what an eviction writes overlaps what it reads, or something else that it writes.
bool evict_overlaps(const Cache8& s, const Cache8& d, int head_dim, const shp_cache8_evict_args& a) {
    const int64_t heads = (int64_t)s.n_seqs * s.kv;
    std::vector<Range> in(1, Range(a.weights, heads * s.cap * 4));
    std::vector<Range> out = {Range(a.kept, heads * a.keep * 4), Range(a.dst_weights, heads * d.cap * 4)};
    for (const Range& r : ranges(s, head_dim)) in.push_back(r);
    for (const Range& r : ranges(d, head_dim)) out.push_back(r);
    for (size_t i = 0; i < out.size(); ++i) {
        for (const Range& r : in)
            if (out[i].meets(r)) return true;
        for (size_t j = 0; j < i; ++j)
            if (out[i].meets(out[j])) return true;
    }
    return false;
}

// What attention and its accounts have in common.
int check_query(const char* where, const Cache8& c, const float* q, int64_t q_seq, int64_t q_row,
                int64_t q_head, int n, int heads, float scale) {
    if (n < 0) return bad(where, "n < 0");
    if (heads < 1 || heads % c.kv) return bad(where, "n_heads must be a multiple of n_kv_heads", SHP_ERR_SHAPE);
    if ((int64_t)n * (heads / c.kv) > 500000)
        return bad(where, "more than 500000 rows for a KV head", SHP_ERR_UNSUPPORTED);
    if (!std::isfinite(scale)) return bad(where, "scale is not finite");
    return check_rows(where, "q", q, q_seq, q_row, q_head);
}

}  // namespace
}  // namespace shp

using shp::bad;
using shp::Cache8;
using shp::Ctx;

extern "C" {

int shp_cache8_append(shp_ctx* ctx, const shp_cache8* cache, const shp_cache8_append_args* a) {
    const char* const me = "shp_cache8_append";
    Cache8 c;
    int rc = shp::check_cache(me, cache, &c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    if (a->n < 0) return bad(me, "n < 0");
    rc = shp::check_rows(me, "k", a->k, a->k_seq, a->k_row, a->k_head);
    if (!rc) rc = shp::check_rows(me, "v", a->v, a->v_seq, a->v_row, a->v_head);
    if (rc) return rc;
    if (!shp::aligned4(a->counts)) return bad(me, "counts must be 4-byte aligned");
    if (!ctx) return bad(me, "null ctx");
    if (a->n == 0) return SHP_OK;
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    const shp::Cache8Rows r = {a->k, a->v, a->k_seq, a->k_row, a->k_head, a->v_seq, a->v_row,
                               a->v_head, a->counts, a->n};
    return x->timed("cache8_append", [&] {
        return shp::cache8_append_launch(x->stream, c, cache->head_dim, cache->format, r);
    });
}

int shp_cache8_read(shp_ctx* ctx, const shp_cache8* cache, int32_t n, float* k, float* v) {
    const char* const me = "shp_cache8_read";
    Cache8 c;
    int rc = shp::check_cache(me, cache, &c);
    if (rc) return rc;
    if (n < 0 || n > c.cap) return bad(me, "n must be 0 to capacity", SHP_ERR_SHAPE);
    if (!shp::aligned16(k) || !shp::aligned16(v)) return bad(me, "outputs must be 16-byte aligned");
    if (!ctx) return bad(me, "null ctx");
    if (n == 0 || (!k && !v)) return SHP_OK;
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    return x->timed("cache8_read", [&] {
        return shp::cache8_read_launch(x->stream, c, cache->head_dim, cache->format, n, k, v);
    });
}

int shp_cache8_attend(shp_ctx* ctx, const shp_cache8* cache, const shp_cache8_attend_args* a) {
    const char* const me = "shp_cache8_attend";
    Cache8 c;
    int rc = shp::check_cache(me, cache, &c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    rc = shp::check_query(me, c, a->q, a->q_seq, a->q_row, a->q_head, a->n, a->n_heads, a->scale);
    if (!rc) rc = shp::check_rows(me, "out", a->out, a->o_seq, a->o_row, a->o_head);
    if (rc) return rc;
    if (!shp::aligned4(a->counts, a->lse)) return bad(me, "counts and lse must be 4-byte aligned");
    if (!ctx) return bad(me, "null ctx");
    if (a->n == 0) return SHP_OK;
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    const int group = a->n_heads / c.kv;
    shp::Cache8Plan plan = shp::cache8_attend_plan(c, cache->head_dim, (int64_t)a->n * group,
                                                   x->cu_count, true);
    float* scratch = nullptr;
    if (plan.scratch) {
        rc = x->scratch(plan.scratch, &scratch);
        if (rc) return rc;
        if (!scratch)
            plan = shp::cache8_attend_plan(c, cache->head_dim, (int64_t)a->n * group, x->cu_count,
                                           false);
    }
    shp::Cache8Query q{};
    q.q = a->q; q.q_seq = a->q_seq; q.q_row = a->q_row; q.q_head = a->q_head;
    q.out = a->out; q.o_seq = a->o_seq; q.o_row = a->o_row; q.o_head = a->o_head;
    q.lse = a->lse; q.counts = a->counts;
    q.n = a->n; q.heads = a->n_heads; q.group = group; q.scale = a->scale;
    return x->timed("cache8_attend", [&] {
        return shp::cache8_attend_launch(x->stream, c, cache->head_dim, cache->format, q, plan,
                                         scratch, (int*)x->workspace);
    });
}

int shp_cache8_weights(shp_ctx* ctx, const shp_cache8* cache, const shp_cache8_weights_args* a) {
    const char* const me = "shp_cache8_weights";
    Cache8 c;
    int rc = shp::check_cache(me, cache, &c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    rc = shp::check_query(me, c, a->q, a->q_seq, a->q_row, a->q_head, a->n, a->n_heads, a->scale);
    if (rc) return rc;
    if (!a->lse || !a->acc_out) return bad(me, "null lse or acc_out");
    if (!shp::aligned4(a->counts, a->lse, a->acc_in, a->acc_out))
        return bad(me, "counts, lse, acc_in and acc_out must be 4-byte aligned");
    if (!ctx) return bad(me, "null ctx");
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    shp::Cache8Query q{};
    q.q = a->q; q.q_seq = a->q_seq; q.q_row = a->q_row; q.q_head = a->q_head;
    q.lse = const_cast<float*>(a->lse); q.counts = a->counts;
    q.n = a->n; q.heads = a->n_heads; q.group = a->n_heads / c.kv; q.scale = a->scale;
    q.acc_in = a->acc_in; q.acc_out = a->acc_out;
    const int64_t rows = (int64_t)q.n * q.group;
    shp::Cache8WeightsPlan plan = shp::cache8_weights_plan(c, cache->head_dim, rows, true);
    float* scratch = nullptr;
    if (plan.scratch) {
        rc = x->scratch(plan.scratch, &scratch);
        if (rc) return rc;
        if (!scratch) plan = shp::cache8_weights_plan(c, cache->head_dim, rows, false);
    }
    return x->timed("cache8_weights", [&] {
        return shp::cache8_weights_launch(x->stream, c, cache->head_dim, cache->format, q, plan,
                                          scratch);
    });
}

int shp_cache8_evict(shp_ctx* ctx, const shp_cache8* src, const shp_cache8* dst,
                     const shp_cache8_evict_args* a) {
    const char* const me = "shp_cache8_evict";
    Cache8 s, d;
    int rc = shp::check_cache(me, src, &s);
    if (!rc) rc = shp::check_cache(me, dst, &d);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    if (src->n_seqs != dst->n_seqs || src->n_kv_heads != dst->n_kv_heads ||
        src->head_dim != dst->head_dim || src->block != dst->block || src->format != dst->format)
        return bad(me, "the caches differ in more than capacity", SHP_ERR_SHAPE);
    if (s.k == d.k || s.v == d.v || s.k_scale == d.k_scale || s.v_scale == d.v_scale ||
        s.lengths == d.lengths)
        return bad(me, "the caches share memory");
    if (a->keep < 1 || a->keep > d.cap || a->recent < 0 || a->recent > a->keep)
        return bad(me, "needs 1 <= keep <= dst capacity and 0 <= recent <= keep", SHP_ERR_SHAPE);
    if (!a->weights || !a->kept) return bad(me, "null weights or kept");
    if (!shp::aligned4(a->weights, a->kept, a->dst_weights))
        return bad(me, "weights, kept and dst_weights must be 4-byte aligned");
    if (a->dst_weights == a->weights) return bad(me, "dst_weights is weights");
    if (!ctx) return bad(me, "null ctx");
    if (shp::evict_overlaps(s, d, src->head_dim, *a))
        return bad(me, "what is written shares memory with what is read or written");
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    return x->timed("cache8_evict", [&] {
        return shp::cache8_evict_launch(x->stream, s, d, src->head_dim, src->format, a->weights,
                                        a->keep, a->recent, a->kept, a->dst_weights);
    });
}

int shp_token_logprobs(shp_ctx* ctx, const shp_logprobs_args* a) {
    const char* const me = "shp_token_logprobs";
    if (!a) return bad(me, "null arguments");
    if (a->rows < 0 || a->vocab < 1) return bad(me, "rows < 0 or vocab < 1", SHP_ERR_SHAPE);
    if (!a->logits || !shp::aligned4(a->logits)) return bad(me, "null or unaligned logits");
    if (a->rows > 1 && a->row_stride < a->vocab)
        return bad(me, "row_stride is less than vocab", SHP_ERR_SHAPE);
    if (a->n_top < 0 || a->n_top > shp::kMaxTop || a->n_top > a->vocab)
        return bad(me, "n_top must be 0 to 64 and at most vocab", SHP_ERR_SHAPE);
    if (!a->targets != !a->logprob) return bad(me, "targets and logprob go together");
    if (a->n_top && (!a->top_ids || !a->top_logprobs))
        return bad(me, "n_top without top_ids or top_logprobs");
    if (!shp::aligned4(a->targets, a->logprob, a->entropy, a->top_ids, a->top_logprobs))
        return bad(me, "targets and outputs must be 4-byte aligned");
    if (a->rows > 16000000 || a->vocab > (1 << 30))
        return bad(me, "more than 16000000 rows or 2^30 logits a row", SHP_ERR_UNSUPPORTED);
    if (!ctx) return bad(me, "null ctx");
    if (a->rows == 0) return SHP_OK;
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    const shp::LogprobArgs l = {a->logits, a->row_stride, a->rows, a->vocab, a->n_top, a->targets,
                                a->logprob, a->entropy, a->top_ids, a->top_logprobs};
    float* scratch = nullptr;
    const size_t need = shp::logprobs_scratch(a->rows, a->vocab);
    if (need) {
        int rc = x->scratch(need, &scratch);
        if (rc) return rc;
        if (!scratch)
            return bad(me, "the workspace is too small and cannot grow while the stream is being "
                           "captured: run the call once before", SHP_ERR_UNSUPPORTED);
    }
    return x->timed("token_logprobs",
                    [&] { return shp::logprobs_launch(x->stream, l, scratch); });
}

}  // extern "C"
