/*
 * memory_kernels.hip - the kernels of the cache in 4 bits and of linear attention, linked
 * with prism_kernels.hip's into one code object (prism_kernels.hsaco).
 *
 *   prism_rope_append{,4}_{f16,bf16}_h{16,32,64,128}   turned queries and keys, keys and values into a cache of 16 or 4 bits
 *   prism_cache_read_h*, prism_cache_read4_{f16,bf16}_h*  rows of such a cache back
 *   prism_paged_attn4_{f16,bf16}_h{16,32}_{g1,g2}      one new token per sequence over its cache of 4 bits: few heads,
 *   prism_paged_attn4_{f16,bf16}_h{16,32,64,128}_many  ... by matrix products
 *   prism_paged_attn4_join_{f16,bf16}_h*               ... the splits of long sequences together
 *   prism_linear_attn_{f16,bf16}_h{16,32,64,128}       linear attention along sequences
 *   prism_linear_states_{f16,bf16}_h*                  ... before it, what segments of few long ones add to their state
 *   prism_linear_step_{f16,bf16}_h{16,32,64,128}       ... one new token per sequence
 */
#include "cache4.hpp"
#include "paged_attn4.hpp"
#include "linear_attn.hpp"
