/* Checks of the 4-bit cache's and linear attention's arguments
 * (csrc/engine/seq_rules.h) for ctypes. */
#include "../prism-inference_amd/csrc/engine/seq_rules.h"

using namespace prism;

extern "C" {
int rope_append_check(const prism_rope_append_push* p) { const char* w; return check_rope_append(*p, &w); }
int cache_read_check(const prism_cache_read_push* p) { const char* w; return check_cache_read(*p, &w); }
int linear_check(const prism_linear_attn_push* p) { const char* w; return check_linear(*p, &w); }
int linear_step_check(const prism_linear_attn_push* p) { const char* w; return check_linear_step(*p, &w); }
}
