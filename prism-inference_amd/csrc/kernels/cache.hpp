/*
 * cache.hpp - writes new tokens' keys and values into a paged cache.
 *
 * Token i goes to slot pos % page_size of page table[seq][pos / page_size], as
 * [page][head][slot][channel]. A token whose sequence, position or page is out
 * of range is skipped (the padding rows of a batch carry seq -1).
 */
#pragma once
#include "seq_types.hpp"

extern "C" __global__ void __launch_bounds__(256) prism_cache_append(AppendArgs a) {
    const int cpr = a.head_dim / 8; /* 16-byte chunks of a row */
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t per_token = (int64_t)a.n_kv_heads * cpr;
    if (id >= a.n_new * per_token) return;
    const int t = (int)(id / per_token), r = (int)(id % per_token), h = r / cpr, c = (r % cpr) * 8;
    const int s = a.seq_of[t], pos = a.pos_of[t];
    if ((uint32_t)s >= (uint32_t)a.n_seqs || pos < 0) return;
    const int slot_page = pos >> a.page_log2;
    if (slot_page >= a.table_pages) return;
    const int page = a.table[(int64_t)s * a.table_pages + slot_page];
    if (!page_ok(page, a.n_pages)) return;
    const int slot = pos & ((1 << a.page_log2) - 1);
    const int64_t to = ((((int64_t)page * a.n_kv_heads + h) << a.page_log2) + slot) * a.head_dim + c;
    st8<F16>(a.k_pages + to, ld8<F16>(a.k + t * a.k_token_stride + h * a.k_head_stride + c));
    st8<F16>(a.v_pages + to, ld8<F16>(a.v + t * a.v_token_stride + h * a.v_head_stride + c));
}
