// attn_decode.cuh -- attention of one new token per sequence over a paged FP16 cache. Row t of sequence b is row
// (t & mask) of page pages[b][t >> kv_shift], a page of the block-major cache being kv_bstride values
// (kv_row in kv_store.cuh with the page in place of the block).

#ifndef B200_ATTN_DECODE_CUH
#define B200_ATTN_DECODE_CUH

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
    // rows of sequence b: lens[b] within what its page list can hold
    __device__ __forceinline__ int len(int b) const {
        const long long cap = (long long)max_pages << kv_shift;
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

template <int D, typename T>
__global__ void __launch_bounds__(128)
k_attn_decode_rows(const T* q, PagedKv kv, T* out, int n_q, int G, int B, float scale2) {
    pdl_entry();
    constexpr int N = D / 32;
    const long long w = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int b = (int)(w / n_q), h = (int)(w % n_q), c = (threadIdx.x & 31) * N;
    if (b >= B) return;
    float qv[N], kr[N], vr[N];
    load_vals(q + w * D + c, qv);
    RowSoftmax<N> st;
    const int n = kv.len(b);
    for (int j = 0; j < n; ++j) {
        const long long r = kv.row(b, j);
        if (r < 0) continue;
        load_vals(kv.K + r + h / G * D + c, kr);
        load_vals(kv.V + r + h / G * D + c, vr);
        st.key(warp_dot(qv, kr) * scale2, vr);
    }
    const float inv = st.l > 0.0f ? 1.0f / st.l : (st.l == 0.0f ? 0.0f : st.l);
#pragma unroll
    for (int i = 0; i < N; ++i) st.o[i] *= inv;
    store_vals(out + w * D + c, st.o);
}

}  // namespace b200

#endif  // B200_ATTN_DECODE_CUH
