// Index arithmetic of the paged key / value cache: plain integer functions, shared by the kernels (paged.hip, paged_attn.hip) and by the
// host-compiled check of their bounds (tests/test_paged_cpu.py builds this header with the host compiler).  Every value that comes from
// device memory -- lengths, page ids, counts, slots -- passes through one of these before it becomes an address.
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#define SPN_HD __host__ __device__ __forceinline__
#else
#define SPN_HD inline
#endif

namespace spn_paged {

constexpr int HEAD = 64;   // head width of every attention kernel of the library

SPN_HD bool page_ok(int id, int num_pages) { return (uint32_t)id < (uint32_t)num_pages; }

// pages that `len` rows occupy (0 for len <= 0); the sum is taken in 64 bits: len may be anything
SPN_HD long pages_of(long len, int shift) { return len > 0 ? (len + (1L << shift) - 1) >> shift : 0; }

// rows of a request that the attention walks: its length, cut to what its table row can hold
SPN_HD int rows_of(int len, int W, int shift) {
    const long cap = (long)W << shift;
    return len <= 0 ? 0 : (int)(len < cap ? len : cap);
}

// Pages a request needs for `fresh` more rows; -1: it cannot be served (a negative length, a count outside [0, width], a table row too
// short).  A served request gets exactly pages_of(len) .. pages_of(len + fresh) - 1 of its table row.
SPN_HD int pages_needed(int len, int fresh, int width, int W, int shift) {
    if (len < 0 || fresh < 0 || fresh > width) return -1;
    const long after = pages_of((long)len + fresh, shift);
    return after > W ? -1 : (int)(after - pages_of(len, shift));
}

// where row `pos` of a request lies, or -1 (page id outside the pool)
SPN_HD long slot_of(int id, long pos, int num_pages, int shift) {
    return page_ok(id, num_pages) ? ((long)id << shift) + (pos & ((1L << shift) - 1)) : -1;
}

SPN_HD bool slot_ok(long slot, int num_pages, int shift) { return slot >= 0 && slot < ((long)num_pages << shift); }

// element offset of (page, head, row of the page) in pages [num_pages, kvh, page, 64]: 64 bits, a pool passes 2^32 elements
SPN_HD long row_offset(long page, int head, long off, int kvh, int shift) { return (((page * kvh + head) << shift) + off) * HEAD; }

}  // namespace spn_paged
