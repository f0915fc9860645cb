// What the paged-cache kernels share: the call's sequences as the device sees
// them, and the search for a row's or a page's sequence.
#pragma once
#include <cstdint>

#include "lq_device.cuh"
#include "lq_host.h"

namespace lq {

enum : int {
    DEV_BAD_PAGE = 0x202,  // a page number outside the cache, or a position past max_pages pages
    DEV_BAD_ROWS = 0x203,  // a sequence's rows outside the call's, or more than max_rows
    DEV_BAD_POS = 0x204,   // a position past the rotation table, or past max_context
};

// rows [r0, r0 + n) of the call are positions [begin, ctx) of the sequence;
// rows [first, r0) would be at negative positions and are no tokens
struct SeqRows {
    int first, r0, n, begin, ctx;
};

__device__ __forceinline__ SeqRows seq_rows(const KVBatch& b, int s, int* err) {
    const int a = ld_after(b.row_start + s), e = ld_after(b.row_start + s + 1);
    SeqRows q;
    q.ctx = ld_after(b.context + s);
    q.first = q.r0 = a;
    q.n = e - a;
    if (a < 0 || e < a || e > b.n_rows || e - a > b.max_rows) {
        set_err(err, DEV_BAD_ROWS);
        q.n = 0;
    }
    if (q.ctx > b.max_context) {
        set_err(err, DEV_BAD_POS);
        q.n = 0;
        q.ctx = 0;
    }
    if (q.ctx < 0) q.ctx = 0;
    if (q.n > q.ctx) {
        q.r0 += q.n - q.ctx;
        q.n = q.ctx;
    }
    q.begin = q.ctx - q.n;
    return q;
}

// the physical page of logical page lp, or -1 (recorded) when there is none
__device__ __forceinline__ int64_t page_of(const PagedKV& c, const KVBatch& b, int s, int lp, int* err) {
    if (lp < b.max_pages) {
        const int p = ld_after(b.pages + (int64_t)s * b.max_pages + lp);
        if (p >= 0 && p < c.n_pages) return p;
    }
    set_err(err, DEV_BAD_PAGE);
    return -1;
}

}  // namespace lq
