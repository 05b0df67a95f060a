// The paged K/V cache and its batch of new tokens, as the kernels see them.
//
// Cache row r of sequence b lies in row r % page_rows of page page_table[b][r / page_rows] of a pool
// [pages][page_rows][kv_heads][dim].  Sequence b's new tokens are rows token_start[b] ..
// token_start[b + 1] of the token-major tensors and the last of the cache_len[b] cache rows.
//
// All of it is device memory that the host never sees, so that a captured step can be replayed
// with other lengths.  What does not fit (a page outside the pool, tokens outside the tensors, a
// length beyond the page table) is reported in the status words.  Reads are clamped to what does fit;
// nothing is written for it, since the pools' rows may be another sequence's.
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
    bool fits;       // nothing of it was clamped
};

__device__ __forceinline__ Sequence sequence(const Cache &c, uint32_t b) {
    const uint32_t start = __ldg(c.token_start + b), end = __ldg(c.token_start + b + 1);
    const uint32_t length = __ldg(c.cache_len + b), most = c.table_width << c.page_shift;
    const bool in_tokens = start <= end && end <= c.tokens;
    if (!in_tokens) report(c, QWCU_BAD_TOKEN_START, b, end);
    if (length > most) report(c, QWCU_BAD_CACHE_LEN, b, length);
    Sequence s;
    s.fits = in_tokens && length <= most;
    s.start = min(start, c.tokens);
    s.fresh = (int)(max(min(end, c.tokens), s.start) - s.start);
    s.length = (int)min(length, most);
    return s;
}

// Row of the pool that holds cache row `row` of sequence b, or -1 where its page is outside the pool.
__device__ __forceinline__ long long pool_row_or_none(const Cache &c, uint32_t b, uint32_t row) {
    const uint32_t p = __ldg(c.page_table + (size_t)b * c.table_width + (row >> c.page_shift));
    if (p < c.pool_pages) return ((long long)p << c.page_shift) + (row & ((1u << c.page_shift) - 1u));
    report(c, QWCU_BAD_PAGE, b, p);
    return -1;
}

// The same for reads: a row of the first page there.
__device__ __forceinline__ size_t pool_row(const Cache &c, uint32_t b, uint32_t row) {
    const long long at = pool_row_or_none(c, b, row);
    return at >= 0 ? (size_t)at : (size_t)(row & ((1u << c.page_shift) - 1u));
}

}  // namespace paged

#endif
