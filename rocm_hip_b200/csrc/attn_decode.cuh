// attn_decode.cuh -- attention of one new token per sequence over a paged FP16 cache. Row t of sequence b is row
// (t & mask) of page pages[b][t >> kv_shift], a page of the block-major cache being kv_bstride values
// (kv_row in kv_store.cuh with the page in place of the block). Two kernels read the cache, attn_prefix.cuh the rows that
// the batch shares and attn_own.cuh each sequence's own, a third joins what they found.

#ifndef B200_ATTN_DECODE_CUH
#define B200_ATTN_DECODE_CUH

#include <limits.h>

#include "attn_rows.cuh"
#include "kv_store.cuh"

namespace b200 {

struct PagedKv {
    const __half* K;
    const __half* V;
    const int* pages;   // [B][max_pages]
    const int* lens;    // [B]
    long long kv_bstride;
    int kv_stride, kv_shift, n_pages, max_pages;
    static constexpr int MOST_ROWS = INT_MAX - 4096;      // of a sequence: whole tiles fit an int
    // rows of sequence b: lens[b] within what its page list can hold
    __device__ __forceinline__ int len(int b) const {
        const long long cap = min((long long)max_pages << kv_shift, (long long)MOST_ROWS);
        const long long n = max(lens[b], 0);
        return (int)(n < cap ? n : cap);
    }
    // offset of row t of sequence b in values, -1 where the page list holds no page of the cache
    __device__ __forceinline__ long long row(int b, int t) const {
        const int p = pages[(long long)b * max_pages + (t >> kv_shift)];
        return (unsigned)p < (unsigned)n_pages
                   ? p * kv_bstride + (long long)(t & ((1 << kv_shift) - 1)) * kv_stride : -1;
    }
};

}  // namespace b200

#endif  // B200_ATTN_DECODE_CUH
