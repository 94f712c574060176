/*
 * seq_index.h - index arithmetic of the sequence operators (rotary positions,
 * paged cache, attention along a sequence), shared by the kernels and by host
 * code: which keys a query sees, which page and slot hold a token, which
 * query tile a workgroup computes. Every value that comes from device memory
 * (a length, a table entry, a start) is brought into its range here.
 */
#ifndef PRISM_SEQ_INDEX_H
#define PRISM_SEQ_INDEX_H
#include <stdint.h>

#ifdef __HIP__
#define PRISM_HD __host__ __device__ inline __attribute__((always_inline))
#else
#define PRISM_HD inline
#endif

PRISM_HD int32_t seq_min(int32_t a, int32_t b) { return a < b ? a : b; }
PRISM_HD int32_t seq_max(int32_t a, int32_t b) { return a > b ? a : b; }
PRISM_HD int32_t seq_clamp(int32_t v, int32_t lo, int32_t hi) { return seq_max(lo, seq_min(v, hi)); }

/* a + b held to the 32-bit range (positions plus a window's width) */
PRISM_HD int32_t seq_add(int32_t a, int32_t b) {
    const int64_t s = (int64_t)a + b;
    return s > INT32_MAX ? INT32_MAX : s < INT32_MIN ? INT32_MIN : (int32_t)s;
}

/* The keys that a query at position p sees among n: j in [lo, hi) and j in
 * [0, sink). left, right: keys before and behind p, negative = all of them. */
struct KeyRange {
    int32_t sink, lo, hi;
};
PRISM_HD KeyRange key_range(int32_t p, int32_t n, int32_t left, int32_t right, int32_t sinks) {
    KeyRange r;
    r.hi = right < 0 ? n : seq_clamp(seq_add(seq_add(p, right), 1), 0, n);
    r.lo = left < 0 ? 0 : seq_clamp(seq_add(p, -left), 0, r.hi);
    r.sink = seq_min(sinks, r.lo);
    return r;
}

/* Rows [start, end) of sequence s of n_seqs among n rows. cu: n_seqs + 1 starts,
 * NULL = sequences of equal length. Starts out of range or out of order give
 * rows inside [0, n), possibly none. */
struct RowRange {
    int32_t start, end;
};
PRISM_HD RowRange row_range(const int32_t* cu, int32_t s, int32_t n_seqs, int32_t n) {
    RowRange r;
    if (!cu) {
        const int32_t each = n / n_seqs;
        r.start = s * each;
        r.end = r.start + each;
        return r;
    }
    r.start = seq_clamp(cu[s], 0, n);
    r.end = seq_clamp(cu[s + 1], r.start, n);
    return r;
}

/* A page-table entry that names a page of the pool. */
PRISM_HD bool page_ok(int32_t entry, int32_t n_pages) { return (uint32_t)entry < (uint32_t)n_pages; }

#endif
