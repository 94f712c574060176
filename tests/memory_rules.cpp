/* Checks of the 4-bit cache's and linear attention's arguments, and how they are launched
 * (csrc/engine/seq_rules.h) for ctypes. */
#include "../prism-inference_amd/csrc/engine/seq_rules.h"

using namespace prism;

extern "C" {
int rope_append_check(const prism_rope_append_push* p) { const char* w; return check_rope_append(*p, &w); }
int cache_read_check(const prism_cache_read_push* p) { const char* w; return check_cache_read(*p, &w); }
int linear_check(const prism_linear_attn_push* p) { const char* w; return check_linear(*p, &w); }
int linear_step_check(const prism_linear_attn_push* p) { const char* w; return check_linear_step(*p, &w); }
int append_tile_of(int64_t n, int64_t heads, int hd) { return append_tile(n, heads, hd); }
int append_tile_channels(void) { return APPEND_TILE_CHANNELS; }
/* out: many, head tiles, waves, splits, grid, keys of a wave, keys expected, workspace */
void paged4_of(const prism_paged_attn_push* p, int64_t* out) {
    const PagedPlan r = paged4_plan(*p);
    const int64_t v[] = {r.many, r.head_tiles, r.waves, r.splits, r.grid, paged4_each(*p, r), paged_keys(*p), paged_workspace(*p, r)};
    for (int i = 0; i < 8; ++i) out[i] = v[i];
}
/* out: segment, split, segments, workspace */
void linear_of(const prism_linear_attn_push* p, int64_t* out) {
    const LinearPlan r = linear_plan(*p);
    const int64_t v[] = {r.segment, r.split, r.segments, linear_workspace(*p, r)};
    for (int i = 0; i < 4; ++i) out[i] = v[i];
}
}
