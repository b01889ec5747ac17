// The C ABI of the paged cache: argument checks and timing around the launchers.  Arguments are
// checked before the context, so a refusal needs no device.
#include <cmath>

#include "paged.h"
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

int check_paged(const char* where, const shp_paged* c, Paged* out) {
    if (!c) return bad(where, "null cache");
    if (!c->k || !c->v || !c->table || !c->lengths) return bad(where, "null array in the cache");
    if (c->format != SHP_PAGED_F32 && c->format != SHP_PAGED_F16 && c->format != SHP_PAGED_BF16)
        return bad(where, "unknown format", SHP_ERR_UNSUPPORTED);
    if (c->head_dim != 64 && c->head_dim != 128)
        return bad(where, "head_dim must be 64 or 128", SHP_ERR_UNSUPPORTED);
    int lb = 0;
    while (lb < 5 && (16 << lb) != c->page_size) ++lb;
    if (lb > 4) return bad(where, "page_size must be 16, 32, 64, 128 or 256", SHP_ERR_UNSUPPORTED);
    if (c->n_seqs < 1 || c->n_kv_heads < 1 || (int64_t)c->n_seqs * c->n_kv_heads > 65535)
        return bad(where, "n_seqs * n_kv_heads must be 1 to 65535", SHP_ERR_SHAPE);
    if (c->n_pages < 1) return bad(where, "n_pages must be positive", SHP_ERR_SHAPE);
    if (c->max_pages < 1 || (int64_t)c->max_pages * c->page_size > (1 << 22))
        return bad(where, "max_pages must be positive, max_pages * page_size at most 4194304", SHP_ERR_SHAPE);
    if (!aligned16(c->k) || !aligned16(c->v))
        return bad(where, "k and v must be 16-byte aligned");
    if (!aligned4(c->table, c->lengths))
        return bad(where, "table and lengths must be 4-byte aligned");
    *out = Paged{c->k, c->v, c->table, c->lengths, c->n_seqs, c->n_kv_heads, c->n_pages, lb + 4,
                 c->max_pages, c->max_pages * c->page_size};
    return SHP_OK;
}

int check_rows(const char* where, const char* what, const float* p, int64_t seq, int64_t row,
               int64_t head) {
    if (!p) return bad(where, (std::string("null ") + what).c_str());
    if (!aligned16(p) || (seq | row | head) & 3)
        return bad(where, (std::string(what) + " rows must be 16-byte aligned").c_str());
    return SHP_OK;
}

int check_heads(const char* where, const Paged& c, int n, int heads) {
    if (heads < 1 || heads % c.kv)
        return bad(where, "n_heads must be a multiple of n_kv_heads", SHP_ERR_SHAPE);
    if ((int64_t)n * (heads / c.kv) > 500000)
        return bad(where, "more than 500000 rows for a KV head", SHP_ERR_UNSUPPORTED);
    return SHP_OK;
}

struct Range {
    uintptr_t from, bytes;
    Range(const void* p, int64_t n) : from((uintptr_t)p), bytes(p ? (uintptr_t)n : 0) {}
    bool meets(const Range& o) const {
        return bytes && o.bytes && from < o.from + o.bytes && o.from < from + bytes;
    }
};

// Whether an array that acceptance writes overlaps another one of the call.  Only lengths_out may be
// an array that is read: a sequence's length is read before it is written.
bool accept_overlaps(const shp_paged& c, const shp_paged_accept_args& a) {
    const int64_t all = (int64_t)c.n_seqs * a.n * 4, one = c.n_seqs * 4ll;
    const int64_t pages = (int64_t)c.n_pages * c.n_kv_heads * c.page_size * c.head_dim *
                          (c.format == SHP_PAGED_F32 ? 4 : 2);
    const Range out[] = {Range(a.path, all), Range(a.accepted, one), Range(a.next, one),
                         Range(a.lengths_out, one), Range(c.k, pages), Range(c.v, pages)};
    const Range in[] = {Range(a.parents, all), Range(a.tokens, all), Range(a.choices, all),
                        Range(a.counts, one), Range(c.table, (int64_t)c.n_seqs * c.max_pages * 4),
                        Range(c.lengths, one)};
    for (int i = 0; i < 6; ++i) {
        for (int j = 0; j < 6; ++j)
            if (out[i].meets(in[j]) && !(i == 3 && j == 5 && a.lengths_out == c.lengths)) return true;
        for (int j = 0; j < i; ++j)
            if (out[i].meets(out[j])) return true;
    }
    return false;
}

}  // namespace
}  // namespace shp

using shp::bad;
using shp::Ctx;
using shp::Paged;

extern "C" {

int shp_paged_append(shp_ctx* ctx, const shp_paged* cache, const shp_paged_append_args* a) {
    const char* const me = "shp_paged_append";
    Paged c;
    int rc = shp::check_paged(me, cache, &c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    if (a->n < 0) return bad(me, "n < 0");
    rc = shp::check_rows(me, "k", a->k, a->k_seq, a->k_row, a->k_head);
    if (!rc) rc = shp::check_rows(me, "v", a->v, a->v_seq, a->v_row, a->v_head);
    if (rc) return rc;
    if (!a->q != !a->q_out) return bad(me, "q and q_out go together");
    if (a->q) {
        rc = shp::check_rows(me, "q", a->q, a->q_seq, a->q_row, a->q_head);
        if (!rc) rc = shp::check_rows(me, "q_out", a->q_out, a->o_seq, a->o_row, a->o_head);
        if (!rc) rc = shp::check_heads(me, c, a->n, a->n_heads);
        if (rc) return rc;
        if (a->q == a->q_out && (a->q_seq != a->o_seq || a->q_row != a->o_row || a->q_head != a->o_head))
            return bad(me, "q_out is q with other strides");
    } else {
        rc = shp::check_heads(me, c, a->n, c.kv);
        if (rc) return rc;
    }
    if ((int64_t)c.n_seqs * a->n > 16000000) return bad(me, "more than 16000000 rows", SHP_ERR_UNSUPPORTED);
    if (a->rot < 0 || a->rot > cache->head_dim || a->rot % 8)
        return bad(me, "rot must be a multiple of 8, 0 to head_dim", SHP_ERR_SHAPE);
    if (a->rot && !a->inv_freq) return bad(me, "rot without inv_freq");
    if (!shp::aligned4(a->counts, a->offsets, a->inv_freq))
        return bad(me, "counts, offsets and inv_freq must be 4-byte aligned");
    if (!ctx) return bad(me, "null ctx");
    if (a->n == 0) return SHP_OK;
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    shp::PagedRows r{};
    r.k = a->k; r.k_seq = a->k_seq; r.k_row = a->k_row; r.k_head = a->k_head;
    r.v = a->v; r.v_seq = a->v_seq; r.v_row = a->v_row; r.v_head = a->v_head;
    r.q = a->q; r.q_seq = a->q_seq; r.q_row = a->q_row; r.q_head = a->q_head;
    r.q_out = a->q_out; r.o_seq = a->o_seq; r.o_row = a->o_row; r.o_head = a->o_head;
    r.counts = a->counts; r.offsets = a->offsets; r.inv_freq = a->inv_freq;
    r.n = a->n; r.heads = a->q ? a->n_heads : 0; r.rot = a->rot; r.interleaved = a->interleaved != 0;
    return x->timed("paged_append", [&] {
        return shp::paged_append_launch(x->stream, c, cache->head_dim, cache->format, r);
    });
}

int shp_paged_attend(shp_ctx* ctx, const shp_paged* cache, const shp_paged_attend_args* a) {
    const char* const me = "shp_paged_attend";
    Paged c;
    int rc = shp::check_paged(me, cache, &c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    if (a->n < 0) return bad(me, "n < 0");
    rc = shp::check_heads(me, c, a->n, a->n_heads);
    if (!rc) rc = shp::check_rows(me, "q", a->q, a->q_seq, a->q_row, a->q_head);
    if (!rc) rc = shp::check_rows(me, "out", a->out, a->o_seq, a->o_row, a->o_head);
    if (rc) return rc;
    if (a->q == a->out && (a->q_seq != a->o_seq || a->q_row != a->o_row || a->q_head != a->o_head))
        return bad(me, "out is q with other strides");
    if (!std::isfinite(a->scale)) return bad(me, "scale is not finite");
    if (!std::isfinite(a->cap) || a->cap < 0 || (a->cap > 0 && !std::isfinite(a->scale / a->cap)))
        return bad(me, "cap must be finite, and 0 or large enough for scale / cap");
    if (a->cap == 0 && !std::isfinite(a->scale * 1.4426950408889634f))  // q is multiplied by it
        return bad(me, "scale times log2 e must be finite");
    if (a->window < 0) return bad(me, "window < 0");
    if (a->parents && a->n > shp::kTreeRows)
        return bad(me, "a tree of more than 256 rows", SHP_ERR_UNSUPPORTED);
    if (!shp::aligned4(a->counts, a->lse, a->slopes, a->prefix, a->first, a->parents))
        return bad(me, "counts, lse, slopes, prefix, first and parents must be 4-byte aligned");
    if (!ctx) return bad(me, "null ctx");
    if (a->n == 0) return SHP_OK;
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    shp::PagedQuery q{};
    q.q = a->q; q.q_seq = a->q_seq; q.q_row = a->q_row; q.q_head = a->q_head;
    q.out = a->out; q.o_seq = a->o_seq; q.o_row = a->o_row; q.o_head = a->o_head;
    q.lse = a->lse; q.counts = a->counts; q.slopes = a->slopes;
    q.prefix = a->prefix; q.first = a->first; q.parents = a->parents;
    q.n = a->n; q.heads = a->n_heads; q.group = a->n_heads / c.kv; q.window = a->window;
    q.scale = a->scale; q.cap = a->cap;
    const int64_t rows = (int64_t)q.n * q.group;
    shp::PagedPlan plan = shp::paged_attend_plan(c, cache->head_dim, cache->format, rows, x->cu_count, true);
    float* scratch = nullptr;
    if (plan.scratch) {
        rc = x->scratch(plan.scratch, &scratch);
        if (rc) return rc;
        if (!scratch) plan = shp::paged_attend_plan(c, cache->head_dim, cache->format, rows, x->cu_count, false);
    }
    return x->timed("paged_attend", [&] {
        return shp::paged_attend_launch(x->stream, c, cache->head_dim, cache->format, q, plan, scratch,
                                        (int*)x->workspace);
    });
}

// Internal hook for tests, not in spirv_hip.h: how attention shares out n rows of n_heads heads on the context's
// device (without a context: on 256 CUs).  out4: rows of a block, 1 where a wavefront takes a block by itself, 1
// where tokens are shared out, workgroups.
int shp_paged_attend_plan(shp_ctx* ctx, const shp_paged* cache, int32_t n, int32_t n_heads, int32_t* out4) {
    const char* const me = "shp_paged_attend_plan";
    Paged c;
    int rc = shp::check_paged(me, cache, &c);
    if (rc) return rc;
    if (n < 1 || !out4) return bad(me, "n < 1 or null out4");
    rc = shp::check_heads(me, c, n, n_heads);
    if (rc) return rc;
    const int cu = ctx ? reinterpret_cast<Ctx*>(ctx)->cu_count : 256;
    const shp::PagedPlan p = shp::paged_attend_plan(c, cache->head_dim, cache->format, (int64_t)n * (n_heads / c.kv), cu, true);
    out4[0] = p.rows;
    out4[1] = p.side;
    out4[2] = p.scratch != 0;
    out4[3] = p.grid * p.row_blocks;
    return SHP_OK;
}

int shp_paged_accept(shp_ctx* ctx, const shp_paged* cache, const shp_paged_accept_args* a) {
    const char* const me = "shp_paged_accept";
    Paged c;
    int rc = shp::check_paged(me, cache, &c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    if (a->n < 1) return bad(me, "n < 1");
    if (a->n > shp::kTreeRows) return bad(me, "a tree of more than 256 rows", SHP_ERR_UNSUPPORTED);
    if (!a->parents || !a->tokens || !a->choices) return bad(me, "null parents, tokens or choices");
    if (!a->path || !a->accepted || !a->next || !a->lengths_out)
        return bad(me, "null path, accepted, next or lengths_out");
    if (!shp::aligned4(a->counts, a->parents, a->tokens, a->choices, a->path, a->accepted, a->next,
                       a->lengths_out))
        return bad(me, "all arrays must be 4-byte aligned");
    if (shp::accept_overlaps(*cache, *a))
        return bad(me, "what is written shares memory with what is read or written");
    if (!ctx) return bad(me, "null ctx");
    Ctx* x = reinterpret_cast<Ctx*>(ctx);
    SHP_HIP_CHECK(hipSetDevice(x->device));
    const shp::PagedTree t = {a->counts, a->parents, a->tokens, a->choices, a->path, a->accepted,
                              a->next, a->lengths_out, a->n};
    return x->timed("paged_accept", [&] {
        return shp::paged_accept_launch(x->stream, c, cache->head_dim, cache->format, t);
    });
}

}  // extern "C"
