// The paged K/V cache and its batch of new tokens, as the kernels see them.
//
// Cache row r of sequence b lies in row r % page_rows of page page_table[b][r / page_rows] of a pool
// [pages][page_rows][kv_heads][dim].  Sequence b's new tokens are rows token_start[b] ..
// token_start[b + 1] of the token-major tensors and the last of the cache_len[b] cache rows.
//
// All of it is device memory that the host never sees, so that a captured step can be replayed
// with other lengths.  What does not fit (a page outside the pool, tokens outside the tensors, a
// length beyond the page table) is clamped to what does and reported in the status words.
#ifndef QW_PAGED_CUH
#define QW_PAGED_CUH

#include <stdint.h>

#include "../qw_cuda.h"

namespace paged {

struct Cache {
    const uint32_t *page_table;
    const uint32_t *token_start;
    const uint32_t *cache_len;
    uint32_t batch, tokens, table_width;
    uint32_t page_shift;  // log2 of the rows of a page
    uint32_t pool_pages;
    uint32_t *status;
};

static __device__ __noinline__ void report(const Cache &c, uint32_t what, uint32_t sequence,
                                           uint32_t value) {
    if (atomicCAS(c.status, 0u, (uint32_t)QWCU_STATUS_BAD_CACHE) == 0u) {
        c.status[1] = what;
        c.status[2] = sequence;
        c.status[3] = value;
    }
    __threadfence_system();
}

struct Sequence {
    uint32_t start;  // first new token
    int fresh;       // new tokens
    int length;      // cache rows, the new tokens among them
};

__device__ __forceinline__ Sequence sequence(const Cache &c, uint32_t b) {
    const uint32_t start = __ldg(c.token_start + b), end = __ldg(c.token_start + b + 1);
    const uint32_t length = __ldg(c.cache_len + b), most = c.table_width << c.page_shift;
    if (start > end || end > c.tokens) report(c, QWCU_BAD_TOKEN_START, b, end);
    if (length > most) report(c, QWCU_BAD_CACHE_LEN, b, length);
    Sequence s;
    s.start = min(start, c.tokens);
    s.fresh = (int)(max(min(end, c.tokens), s.start) - s.start);
    s.length = (int)min(length, most);
    return s;
}

// The page of a sequence's cache rows [index << page_shift, ...).
__device__ __forceinline__ uint32_t page(const Cache &c, uint32_t b, uint32_t index) {
    const uint32_t p = __ldg(c.page_table + (size_t)b * c.table_width + index);
    if (p < c.pool_pages) return p;
    report(c, QWCU_BAD_PAGE, b, p);
    return 0;
}

// Row of the pool that holds cache row `row` of sequence b.
__device__ __forceinline__ size_t pool_row(const Cache &c, uint32_t b, uint32_t row) {
    return ((size_t)page(c, b, row >> c.page_shift) << c.page_shift) +
           (row & ((1u << c.page_shift) - 1u));
}

}  // namespace paged

#endif
