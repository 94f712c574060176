/*
 * sequence.cpp - host side of the sequence operators (kernels in
 * csrc/kernels/{rope,cache,paged_attn,seq_attn,cache4,paged_attn4,linear_attn}.hpp): argument checks
 * (seq_rules.h) and launches. They need no model and keep no state.
 */
#include <hip/hip_runtime.h>

#include <cstring>

#include "ctx.h"
#include "seq_rules.h"

using namespace prism;

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int log2_of(int32_t n) { return __builtin_ctz((unsigned)n); }
int hd_index(int32_t hd) { return log2_of(hd) - 4; }
/* what the kernels divide by d with */
uint32_t inverse(int32_t d) { return d > 1 ? (uint32_t)((uint64_t(1) << 32) / (uint32_t)d) : UINT32_MAX; }

/* The context's device while a call enqueues its work, the caller's after it. */
class OnDevice {
  public:
    explicit OnDevice(int device) {
        err_ = hipGetDevice(&before_);
        if (err_ == hipSuccess && before_ != device) {
            err_ = hipSetDevice(device);
            changed_ = err_ == hipSuccess;
        }
    }
    ~OnDevice() {
        if (changed_) (void)hipSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    hipError_t error() const { return err_; }

  private:
    int before_ = 0;
    bool changed_ = false;
    hipError_t err_ = hipSuccess;
};

/* grid workgroups of `threads` on the context's device */
int launch(prism_ctx* c, hipFunction_t f, const char* what, int64_t grid, unsigned threads, void* args, void* stream) {
    if (!seq_grid_ok(grid, threads))
        return fail(c, PRISM_ERR_UNSUPPORTED, "%s: %lld workgroups are more than one launch takes", what, (long long)grid);
    OnDevice on(c->device);
    if (on.error() != hipSuccess)
        return fail(c, PRISM_ERR_HIP, "hipSetDevice(%d): %s", c->device, hipGetErrorString(on.error()));
    void* params[] = {args};
    const hipError_t e =
        hipModuleLaunchKernel(f, (unsigned)grid, 1, 1, threads, 1, 1, 0, (hipStream_t)stream, params, nullptr);
    if (e != hipSuccess) return fail(c, PRISM_ERR_HIP, "hipModuleLaunchKernel(%s): %s", what, hipGetErrorString(e));
    return PRISM_OK;
}

template <class P, class F>
int checked(prism_ctx* c, const P* p, const char* what, F check) {
    if (!c) return fail(nullptr, PRISM_ERR_INVALID, "context is NULL");
    if (!p) return fail(c, PRISM_ERR_INVALID, "%s: push is NULL", what);
    const char* why = "";
    const int rc = check(*p, &why);
    return rc ? fail(c, rc, "%s: %s", what, why) : PRISM_OK;
}

}  // namespace

extern "C" int prism_rope(prism_ctx* c, const prism_rope_push* p, const void* in, const int32_t* pos, void* out,
                          void* stream) {
    if (const int rc = checked(c, p, "rope", check_rope)) return rc;
    if (p->n_tokens == 0) return PRISM_OK;
    if (!in || !pos || !out) return fail(c, PRISM_ERR_INVALID, "rope: NULL buffer");
    if (!aligned16(in) || !aligned16(out)) return fail(c, PRISM_ERR_INVALID, "rope: buffers must be 16-byte aligned");
    if (in == out && (p->in_token_stride != p->out_token_stride || p->in_head_stride != p->out_head_stride))
        return fail(c, PRISM_ERR_INVALID, "rope: in place needs equal strides");
    RopeArgs a;
    memset(&a, 0, sizeof a);
    a.in = static_cast<const uint16_t*>(in);
    a.out = static_cast<uint16_t*>(out);
    a.pos = pos;
    a.in_token_stride = p->in_token_stride;
    a.in_head_stride = p->in_head_stride;
    a.out_token_stride = p->out_token_stride;
    a.out_head_stride = p->out_head_stride;
    a.pos_stride = p->pos_stride;
    a.n_tokens = p->n_tokens;
    a.n_heads = p->n_heads;
    a.head_dim = p->head_dim;
    a.adjacent = p->layout == PRISM_ROPE_ADJACENT;
    a.n_pairs = rope_axes(*p, a.axis_end);
    a.one_ladder = p->ladder == PRISM_ROPE_ONE_LADDER;
    a.turn = (p->inverse ? -1.0 : 1.0) / 6.283185307179586476925286766559;
    a.log2_base = std::log2(p->base);
    a.copy = in != out;
    a.tile = rope_tile(p->n_tokens, a.n_pairs);
    const bool loose = !a.adjacent && a.n_pairs % 8 != 0;
    return launch(c, c->f_rope[p->dtype][loose], "rope", ((int64_t)p->n_tokens + a.tile - 1) / a.tile, 256, &a, stream);
}

extern "C" int prism_cache_append(prism_ctx* c, const prism_append_push* p, const void* k, const void* v,
                                  const int32_t* seq_of, const int32_t* pos_of, const int32_t* table, void* k_pages,
                                  void* v_pages, void* stream) {
    if (const int rc = checked(c, p, "cache append", check_append)) return rc;
    const prism_cache_desc& d = p->cache;
    if (p->n_new == 0 || d.n_seqs == 0 || d.n_pages == 0 || d.table_pages == 0) return PRISM_OK;
    if (!k || !v || !seq_of || !pos_of || !table || !k_pages || !v_pages)
        return fail(c, PRISM_ERR_INVALID, "cache append: NULL buffer");
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages))
        return fail(c, PRISM_ERR_INVALID, "cache append: buffers must be 16-byte aligned");
    AppendArgs a;
    memset(&a, 0, sizeof a);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.k_pages = static_cast<uint16_t*>(k_pages);
    a.v_pages = static_cast<uint16_t*>(v_pages);
    a.table = table;
    a.seq_of = seq_of;
    a.pos_of = pos_of;
    a.k_token_stride = p->k_token_stride;
    a.k_head_stride = p->k_head_stride;
    a.v_token_stride = p->v_token_stride;
    a.v_head_stride = p->v_head_stride;
    a.n_new = p->n_new;
    a.n_seqs = d.n_seqs;
    a.n_kv_heads = d.n_kv_heads;
    a.head_dim = d.head_dim;
    a.page_log2 = log2_of(d.page_size);
    a.n_pages = d.n_pages;
    a.table_pages = d.table_pages;
    const int64_t chunks = (int64_t)p->n_new * d.n_kv_heads * (d.head_dim / 8);
    return launch(c, c->f_append, "cache append", (chunks + 255) / 256, 256, &a, stream);
}

namespace {

int64_t paged_workspace_of(const prism_paged_attn_push* p, bool four) {
    if (!p) return fail(nullptr, PRISM_ERR_INVALID, "paged attention: push is NULL");
    const char* why = "";
    const int rc = check_paged(*p, &why);
    if (rc) return fail(nullptr, rc, "paged attention: %s", why);
    return paged_workspace(*p, four ? paged4_plan(*p) : paged_plan(*p));
}

/* k_scales, v_scales: of a 4-bit cache */
int paged(prism_ctx* c, const prism_paged_attn_push* p, bool four, const void* q, const void* k_pages, const void* v_pages,
          const void* k_scales, const void* v_scales, const int32_t* table, const int32_t* lengths, void* out,
          void* workspace, int64_t workspace_bytes, void* stream) {
    if (const int rc = checked(c, p, "paged attention", check_paged)) return rc;
    const prism_cache_desc& d = p->cache;
    if (d.n_seqs == 0) return PRISM_OK;
    if (!q || !lengths || !out) return fail(c, PRISM_ERR_INVALID, "paged attention: NULL buffer");
    if (d.n_pages > 0 && d.table_pages > 0 && (!k_pages || !v_pages || !table || (four && (!k_scales || !v_scales))))
        return fail(c, PRISM_ERR_INVALID, "paged attention: NULL cache");
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_scales) || !aligned16(v_scales) ||
        !aligned16(out))
        return fail(c, PRISM_ERR_INVALID, "paged attention: buffers must be 16-byte aligned");
    const PagedPlan plan = four ? paged4_plan(*p) : paged_plan(*p);
    const int64_t need = paged_workspace(*p, plan);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(c, PRISM_ERR_INVALID, "paged attention: workspace of %lld bytes, %lld needed, 16-byte aligned",
                    workspace ? (long long)workspace_bytes : 0LL, (long long)need);
    PagedAttnArgs a;
    memset(&a, 0, sizeof a);
    a.q = static_cast<const uint16_t*>(q);
    a.k_pages = static_cast<const uint16_t*>(k_pages);
    a.v_pages = static_cast<const uint16_t*>(v_pages);
    a.k_scales = static_cast<const uint8_t*>(k_scales);
    a.v_scales = static_cast<const uint8_t*>(v_scales);
    a.table = table;
    a.lengths = lengths;
    a.out = static_cast<uint16_t*>(out);
    a.q_seq_stride = p->q_seq_stride;
    a.q_head_stride = p->q_head_stride;
    a.out_seq_stride = p->out_seq_stride;
    a.out_head_stride = p->out_head_stride;
    a.n_seqs = d.n_seqs;
    a.n_heads = p->n_heads;
    a.n_kv_heads = d.n_kv_heads;
    a.page_log2 = log2_of(d.page_size);
    a.n_pages = d.n_pages;
    a.table_pages = d.n_pages > 0 ? d.table_pages : 0;
    a.left = p->left;
    a.sinks = p->sinks;
    a.scale_log2 = seq_scale_log2(p->scale);
    a.head_tiles = plan.head_tiles;
    a.waves = plan.waves;
    a.splits = plan.splits;
    a.ws = static_cast<float*>(workspace);
    if (four) {
        a.each = paged4_each(*p, plan);
        a.group = p->n_heads / d.n_kv_heads;
        a.by_splits = inverse(plan.splits);
        a.by_tiles = inverse(plan.head_tiles);
        a.by_kv = inverse(d.n_kv_heads);
    }
    const int i = hd_index(d.head_dim), kind = plan.many ? 2 : p->n_heads / d.n_kv_heads - 1;
    const hipFunction_t f = four ? c->f_paged4[d.dtype][i][kind] : c->f_paged[d.dtype][i][kind];
    const int rc = launch(c, f, "paged attention", plan.grid, 256, &a, stream);
    if (rc || plan.splits == 1) return rc;
    return launch(c, four ? c->f_paged4_join[d.dtype][i] : c->f_paged_join[d.dtype][i], "paged attention's join", (int64_t)d.n_seqs * p->n_heads, 256, &a, stream);
}

}  // namespace

extern "C" int64_t prism_paged_attn_workspace(const prism_paged_attn_push* p) { return paged_workspace_of(p, false); }

extern "C" int prism_paged_attn(prism_ctx* c, const prism_paged_attn_push* p, const void* q, const void* k_pages,
                                const void* v_pages, const int32_t* table, const int32_t* lengths, void* out,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    return paged(c, p, false, q, k_pages, v_pages, nullptr, nullptr, table, lengths, out, workspace, workspace_bytes, stream);
}

extern "C" int64_t prism_paged_attn4_workspace(const prism_paged_attn_push* p) { return paged_workspace_of(p, true); }

extern "C" int prism_paged_attn4(prism_ctx* c, const prism_paged_attn_push* p, const void* q, const prism_cache_pages* g,
                                 const int32_t* table, const int32_t* lengths, void* out, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
    if (c && p && !g) return fail(c, PRISM_ERR_INVALID, "paged attention: pages is NULL");
    return paged(c, p, true, q, g ? g->k : nullptr, g ? g->v : nullptr, g ? g->k_scales : nullptr, g ? g->v_scales : nullptr,
                 table, lengths, out, workspace, workspace_bytes, stream);
}

extern "C" int prism_seq_attn(prism_ctx* c, const prism_seq_attn_push* p, const void* q, const void* k, const void* v,
                              const int32_t* cu_q, const int32_t* cu_k, void* out, void* stream) {
    if (const int rc = checked(c, p, "sequence attention", check_seq)) return rc;
    if (p->n_seqs == 0 || p->n_q == 0) return PRISM_OK;
    if (!q || !out || (p->n_k > 0 && (!k || !v))) return fail(c, PRISM_ERR_INVALID, "sequence attention: NULL buffer");
    if ((!cu_q && p->n_q % p->n_seqs) || (!cu_k && p->n_k % p->n_seqs))
        return fail(c, PRISM_ERR_INVALID, "sequence attention: %d sequences of equal length do not fill the rows", p->n_seqs);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(c, PRISM_ERR_INVALID, "sequence attention: buffers must be 16-byte aligned");
    SeqAttnArgs a;
    memset(&a, 0, sizeof a);
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.out = static_cast<uint16_t*>(out);
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.q_token_stride = p->q_token_stride;
    a.q_head_stride = p->q_head_stride;
    a.k_token_stride = p->k_token_stride;
    a.k_head_stride = p->k_head_stride;
    a.v_token_stride = p->v_token_stride;
    a.v_head_stride = p->v_head_stride;
    a.out_token_stride = p->out_token_stride;
    a.out_head_stride = p->out_head_stride;
    a.n_seqs = p->n_seqs;
    a.n_q = p->n_q;
    a.n_k = p->n_k;
    a.n_heads = p->n_heads;
    a.n_kv_heads = p->n_kv_heads;
    a.left = p->left;
    a.right = p->right;
    a.sinks = p->sinks;
    a.scale_log2 = seq_scale_log2(p->scale);
    const SeqPlan plan = seq_plan(*p);
    a.tile_heads = plan.tile_heads;
    a.tile_q = plan.tile_q;
    return launch(c, c->f_seq[p->dtype][hd_index(p->head_dim)][plan.kind], "sequence attention", plan.grid,
                  plan.kind == SEQ_FOUR ? 256 : 512, &a, stream);
}

namespace {

/* the pools that a call needs, and their alignment */
int check_pages(prism_ctx* c, const char* what, const prism_cache_pages* g, int32_t format) {
    const bool four = format == PRISM_CACHE_4;
    if (!g) return fail(c, PRISM_ERR_INVALID, "%s: pages is NULL", what);
    if (!g->k || !g->v || (four && (!g->k_scales || !g->v_scales))) return fail(c, PRISM_ERR_INVALID, "%s: NULL cache", what);
    if (!aligned16(g->k) || !aligned16(g->v) || (four && (!aligned16(g->k_scales) || !aligned16(g->v_scales))))
        return fail(c, PRISM_ERR_INVALID, "%s: buffers must be 16-byte aligned", what);
    return PRISM_OK;
}

}  // namespace

extern "C" int prism_rope_append(prism_ctx* c, const prism_rope_append_push* p, const void* q, const void* k, const void* v,
                                 const int32_t* pos, void* q_out, const int32_t* seq_of, const int32_t* pos_of,
                                 const int32_t* table, const prism_cache_pages* g, void* stream) {
    const char* what = "rope append";
    if (const int rc = checked(c, p, what, check_rope_append)) return rc;
    if (p->n_new == 0) return PRISM_OK;
    const prism_cache_desc& d = p->cache;
    const bool kept = d.n_seqs > 0 && d.n_pages > 0 && d.table_pages > 0; /* some row may have a place */
    if (!kept && p->n_heads == 0) return PRISM_OK;
    if (!k || !v || (kept && (!seq_of || !pos_of || !table)) || (p->n_axes > 0 && !pos) || (p->n_heads > 0 && (!q || !q_out)))
        return fail(c, PRISM_ERR_INVALID, "%s: NULL buffer", what);
    if (kept)
        if (const int rc = check_pages(c, what, g, p->format)) return rc;
    if (!aligned16(k) || !aligned16(v) || (p->n_heads > 0 && (!aligned16(q) || !aligned16(q_out))))
        return fail(c, PRISM_ERR_INVALID, "%s: buffers must be 16-byte aligned", what);
    if (p->n_heads > 0 && q == q_out && (p->q_token_stride != p->out_token_stride || p->q_head_stride != p->out_head_stride))
        return fail(c, PRISM_ERR_INVALID, "%s: in place needs equal strides", what);
    RopeAppendArgs a;
    memset(&a, 0, sizeof a);
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.q_out = static_cast<uint16_t*>(q_out);
    if (kept) {
        a.k_pages = static_cast<uint8_t*>(g->k);
        a.v_pages = static_cast<uint8_t*>(g->v);
        a.k_scales = static_cast<uint8_t*>(g->k_scales);
        a.v_scales = static_cast<uint8_t*>(g->v_scales);
    }
    a.pos = pos;
    a.table = table;
    a.seq_of = seq_of;
    a.pos_of = pos_of;
    a.q_token_stride = p->q_token_stride;
    a.q_head_stride = p->q_head_stride;
    a.k_token_stride = p->k_token_stride;
    a.k_head_stride = p->k_head_stride;
    a.v_token_stride = p->v_token_stride;
    a.v_head_stride = p->v_head_stride;
    a.out_token_stride = p->out_token_stride;
    a.out_head_stride = p->out_head_stride;
    a.pos_stride = p->pos_stride;
    a.n_new = p->n_new;
    a.n_heads = p->n_heads;
    a.n_kv_heads = kept ? d.n_kv_heads : 0; /* no place: no work but the queries' */
    a.by_heads = inverse(a.n_heads);
    a.by_kv = inverse(a.n_kv_heads);
    if (p->n_axes > 0) {
        a.n_pairs = rope_axes(turn_of(*p, 1, 0, 0), a.axis_end);
        a.log2_base = std::log2(p->base);
    }
    a.adjacent = p->layout == PRISM_ROPE_ADJACENT;
    a.one_ladder = p->ladder == PRISM_ROPE_ONE_LADDER;
    a.turn = 1.0 / 6.283185307179586476925286766559;
    a.tile = append_tile(p->n_new, a.n_heads + 2 * a.n_kv_heads, d.head_dim);
    a.n_seqs = d.n_seqs;
    a.page_log2 = log2_of(d.page_size);
    a.n_pages = d.n_pages;
    a.table_pages = d.table_pages;
    return launch(c, c->f_rope_append[d.dtype][p->format == PRISM_CACHE_4][hd_index(d.head_dim)], what,
                  ((int64_t)p->n_new + a.tile - 1) / a.tile, 256, &a, stream);
}

extern "C" int prism_cache_read(prism_ctx* c, const prism_cache_read_push* p, const prism_cache_pages* g,
                                const int32_t* seq_of, const int32_t* pos_of, const int32_t* table, void* k, void* v,
                                void* stream) {
    const char* what = "cache read";
    if (const int rc = checked(c, p, what, check_cache_read)) return rc;
    if (p->n_rows == 0) return PRISM_OK;
    const prism_cache_desc& d = p->cache;
    const bool kept = d.n_seqs > 0 && d.n_pages > 0 && d.table_pages > 0;
    if (!k || !v || (kept && (!seq_of || !pos_of || !table))) return fail(c, PRISM_ERR_INVALID, "%s: NULL buffer", what);
    if (kept)
        if (const int rc = check_pages(c, what, g, p->format)) return rc;
    if (!aligned16(k) || !aligned16(v)) return fail(c, PRISM_ERR_INVALID, "%s: buffers must be 16-byte aligned", what);
    CacheReadArgs a;
    memset(&a, 0, sizeof a);
    if (kept) {
        a.k_pages = static_cast<const uint8_t*>(g->k);
        a.v_pages = static_cast<const uint8_t*>(g->v);
        a.k_scales = static_cast<const uint8_t*>(g->k_scales);
        a.v_scales = static_cast<const uint8_t*>(g->v_scales);
        a.n_seqs = d.n_seqs; /* else no row has a place */
    }
    a.table = table;
    a.seq_of = seq_of;
    a.pos_of = pos_of;
    a.k = static_cast<uint16_t*>(k);
    a.v = static_cast<uint16_t*>(v);
    a.k_token_stride = p->k_token_stride;
    a.k_head_stride = p->k_head_stride;
    a.v_token_stride = p->v_token_stride;
    a.v_head_stride = p->v_head_stride;
    a.n_rows = p->n_rows;
    a.n_kv_heads = d.n_kv_heads;
    a.by_kv = inverse(d.n_kv_heads);
    a.page_log2 = log2_of(d.page_size);
    a.n_pages = d.n_pages;
    a.table_pages = d.table_pages;
    const int64_t chunks = (int64_t)p->n_rows * d.n_kv_heads * (d.head_dim / 8);
    return launch(c, c->f_cache_read[d.dtype][p->format == PRISM_CACHE_4][hd_index(d.head_dim)], what, (chunks + 255) / 256, 256, &a, stream);
}

namespace {

LinearAttnArgs linear_args(const prism_linear_attn_push* p, const void* q, const void* k, const void* v, const float* rates,
                           const int32_t* cu, const int32_t* state_of, const float* state_in, void* out, float* state_out) {
    LinearAttnArgs a;
    memset(&a, 0, sizeof a);
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.rates = rates;
    a.cu = cu;
    a.state_of = state_of;
    a.state_in = state_in;
    a.out = static_cast<uint16_t*>(out);
    a.state_out = state_out;
    a.q_token_stride = p->q_token_stride;
    a.q_head_stride = p->q_head_stride;
    a.k_token_stride = p->k_token_stride;
    a.k_head_stride = p->k_head_stride;
    a.v_token_stride = p->v_token_stride;
    a.v_head_stride = p->v_head_stride;
    a.out_token_stride = p->out_token_stride;
    a.out_head_stride = p->out_head_stride;
    a.n_seqs = p->n_seqs;
    a.n_tokens = p->n_tokens;
    a.n_heads = p->n_heads;
    a.n_kv_heads = p->n_kv_heads;
    a.n_states = p->n_states;
    a.scale = p->scale;
    return a;
}

}  // namespace

extern "C" int64_t prism_linear_attn_workspace(const prism_linear_attn_push* p) {
    if (!p) return fail(nullptr, PRISM_ERR_INVALID, "linear attention: push is NULL");
    const char* why = "";
    const int rc = check_linear(*p, &why);
    if (rc) return fail(nullptr, rc, "linear attention: %s", why);
    return linear_workspace(*p, linear_plan(*p));
}

extern "C" int prism_linear_attn(prism_ctx* c, const prism_linear_attn_push* p, const void* q, const void* k, const void* v,
                                 const float* rates, const int32_t* cu, const int32_t* state_of, const float* state_in,
                                 void* out, float* state_out, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "linear attention";
    if (const int rc = checked(c, p, what, check_linear)) return rc;
    if (p->n_seqs == 0) return PRISM_OK;
    if (!rates || (p->n_tokens > 0 && (!q || !k || !v || !out))) return fail(c, PRISM_ERR_INVALID, "%s: NULL buffer", what);
    if (!cu && p->n_tokens % p->n_seqs)
        return fail(c, PRISM_ERR_INVALID, "%s: %d sequences of equal length do not fill the rows", what, p->n_seqs);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(state_in) || !aligned16(state_out))
        return fail(c, PRISM_ERR_INVALID, "%s: buffers must be 16-byte aligned", what);
    const LinearPlan plan = linear_plan(*p);
    const int64_t need = linear_workspace(*p, plan);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(c, PRISM_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed, 16-byte aligned", what,
                    workspace ? (long long)workspace_bytes : 0LL, (long long)need);
    LinearAttnArgs a = linear_args(p, q, k, v, rates, cu, state_of, state_in, out, state_out);
    a.segment = plan.segment;
    a.ws = static_cast<float*>(workspace);
    const int i = hd_index(p->head_dim);
    /* a wave for 16 channels of the values (of 128, for 32); below 64, four waves by query tiles for what has queries */
    const unsigned states = p->head_dim < 128 ? 4 * p->head_dim : 256, threads = std::max(states, 256u);
    const int64_t grid = plan.segments * p->n_heads;
    if (plan.split)
        if (const int rc = launch(c, c->f_linear_states[p->dtype][i], what, grid, states, &a, stream)) return rc;
    return launch(c, c->f_linear[p->dtype][i], what, grid, threads, &a, stream);
}

extern "C" int prism_linear_step(prism_ctx* c, const prism_linear_attn_push* p, const void* q, const void* k, const void* v,
                                 const float* rates, const int32_t* state_of, const float* state_in, void* out,
                                 float* state_out, void* stream) {
    const char* what = "linear step";
    if (const int rc = checked(c, p, what, check_linear_step)) return rc;
    if (p->n_seqs == 0) return PRISM_OK;
    if (!rates || !q || !k || !v || !out || (p->n_states > 0 && (!state_in || !state_out)))
        return fail(c, PRISM_ERR_INVALID, "%s: NULL buffer", what);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(state_in) || !aligned16(state_out))
        return fail(c, PRISM_ERR_INVALID, "%s: buffers must be 16-byte aligned", what);
    LinearAttnArgs a = linear_args(p, q, k, v, rates, nullptr, state_of, state_in, out, state_out);
    const int64_t items = (int64_t)p->n_seqs * p->n_heads; /* a wave each; of 128 channels, four */
    return launch(c, c->f_linear_step[p->dtype][hd_index(p->head_dim)], what, p->head_dim == 128 ? items : (items + 3) / 4, 256, &a, stream);
}
