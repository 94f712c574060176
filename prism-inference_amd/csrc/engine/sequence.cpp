/*
 * sequence.cpp - host side of the sequence operators (kernels in
 * csrc/kernels/{rope,cache,paged_attn,seq_attn}.hpp): argument checks
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

extern "C" int64_t prism_paged_attn_workspace(const prism_paged_attn_push* p) {
    if (!p) return fail(nullptr, PRISM_ERR_INVALID, "paged attention: push is NULL");
    const char* why = "";
    const int rc = check_paged(*p, &why);
    if (rc) return fail(nullptr, rc, "paged attention: %s", why);
    return paged_workspace(*p, paged_plan(*p));
}

extern "C" int prism_paged_attn(prism_ctx* c, const prism_paged_attn_push* p, const void* q, const void* k_pages,
                                const void* v_pages, const int32_t* table, const int32_t* lengths, void* out,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    if (const int rc = checked(c, p, "paged attention", check_paged)) return rc;
    const prism_cache_desc& d = p->cache;
    if (d.n_seqs == 0) return PRISM_OK;
    if (!q || !lengths || !out) return fail(c, PRISM_ERR_INVALID, "paged attention: NULL buffer");
    if (d.n_pages > 0 && d.table_pages > 0 && (!k_pages || !v_pages || !table))
        return fail(c, PRISM_ERR_INVALID, "paged attention: NULL cache");
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out))
        return fail(c, PRISM_ERR_INVALID, "paged attention: buffers must be 16-byte aligned");
    const PagedPlan plan = paged_plan(*p);
    const int64_t need = paged_workspace(*p, plan);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(c, PRISM_ERR_INVALID, "paged attention: workspace of %lld bytes, %lld needed, 16-byte aligned",
                    workspace ? (long long)workspace_bytes : 0LL, (long long)need);
    PagedAttnArgs a;
    memset(&a, 0, sizeof a);
    a.q = static_cast<const uint16_t*>(q);
    a.k_pages = static_cast<const uint16_t*>(k_pages);
    a.v_pages = static_cast<const uint16_t*>(v_pages);
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
    const int i = hd_index(d.head_dim), kind = plan.many ? 2 : p->n_heads / d.n_kv_heads - 1;
    const int rc = launch(c, c->f_paged[d.dtype][i][kind], "paged attention", plan.grid, 256, &a, stream);
    if (rc || plan.splits == 1) return rc;
    return launch(c, c->f_paged_join[d.dtype][i], "paged attention's join", (int64_t)d.n_seqs * p->n_heads, 256, &a, stream);
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
