/* The sequence operators' checks, splits and index arithmetic
 * (csrc/engine/seq_rules.h, csrc/seq_index.h) for ctypes. */
#include "../prism-inference_amd/csrc/engine/seq_rules.h"
#include "../prism-inference_amd/csrc/seq_index.h"

using namespace prism;

extern "C" {
int rope_check(const prism_rope_push* p) { const char* w; return check_rope(*p, &w); }
int append_check(const prism_append_push* p) { const char* w; return check_append(*p, &w); }
int paged_check(const prism_paged_attn_push* p) { const char* w; return check_paged(*p, &w); }
int seq_check(const prism_seq_attn_push* p) { const char* w; return check_seq(*p, &w); }
int axes(const prism_rope_push* p, int32_t* axis_end) { return rope_axes(*p, axis_end); }
int tile(long long n_tokens, int n_pairs) { return rope_tile(n_tokens, n_pairs); }
void paged(const prism_paged_attn_push* p, long long* out) {
    const PagedPlan r = paged_plan(*p);
    out[0] = r.many;
    out[1] = r.head_tiles;
    out[2] = r.waves;
    out[3] = r.splits;
    out[4] = r.grid;
    out[5] = paged_workspace(*p, r);
}
int tile_heads(int n_heads, int n_kv_heads) { return seq_tile_heads(n_heads, n_kv_heads); }
long long seq_tiles(long long n_q, long long n_seqs, int tile_q) { return prism::seq_tiles(n_q, n_seqs, tile_q); }
int grid_ok(long long grid, int threads) { return seq_grid_ok(grid, threads); }
void seq(const prism_seq_attn_push* p, long long* out) {
    const SeqPlan r = seq_plan(*p);
    out[0] = r.kind;
    out[1] = r.tile_heads;
    out[2] = r.tile_q;
    out[3] = r.grid;
}
void keys(int32_t p, int32_t n, int32_t left, int32_t right, int32_t sinks, int32_t* out) {
    const KeyRange r = key_range(p, n, left, right, sinks);
    out[0] = r.sink;
    out[1] = r.lo;
    out[2] = r.hi;
}
void rows(const int32_t* cu, int32_t s, int32_t n_seqs, int32_t n, int32_t* out) {
    const RowRange r = row_range(cu, s, n_seqs, n);
    out[0] = r.start;
    out[1] = r.end;
}
int page(int32_t entry, int32_t n_pages) { return page_ok(entry, n_pages); }
}
