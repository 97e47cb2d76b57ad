// attn_prompt.cuh -- causal attention over packed prompts (several sequences one after another in the rows), grouped
// heads, 16-bit rows:
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp(scale q[t, h] . k[j, h / G]),  j in t's sequence, j <= t
// Sequence b is rows [seq_start[b], seq_start[b + 1]); rows in no sequence are not written.

#ifndef B200_ATTN_PROMPT_CUH
#define B200_ATTN_PROMPT_CUH

#include "attn_rows.cuh"

namespace b200 {

// The sequence of row t: the last b with seq_start[b] <= t, its borders clamped to the T rows there are. False if t
// lies in none.
__device__ __forceinline__ bool find_seq(const int* seq_start, int n_seqs, int T, int t, int* first, int* end) {
    int lo = 0, hi = n_seqs;
    if (!seq_start) { *first = 0; *end = T; return true; }
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (seq_start[mid] <= t) lo = mid + 1; else hi = mid;
    }
    if (lo == 0) return false;
    *first = max(seq_start[lo - 1], 0);
    *end = min(seq_start[lo], T);
    return t >= *first && t < *end;
}

template <int D, typename T>
__global__ void __launch_bounds__(128)
k_attn_prompt_rows(const T* q, const T* k, const T* v, T* out, const int* seq_start, int n_seqs, int rows, int n_q, int G,
                   long long q_stride, long long k_stride, long long v_stride, float scale2) {
    pdl_entry();
    const long long w = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int t = (int)(w / n_q), h = (int)(w % n_q);
    int first, end;
    if (t >= rows || !find_seq(seq_start, n_seqs, rows, t, &first, &end)) return;
    attn_row_prompt<D, T>(q + t * q_stride + h * D, k + first * k_stride + h / G * D, v + first * v_stride + h / G * D, k_stride,
                          v_stride, t - first + 1, scale2, out + (long long)t * n_q * D + h * D);
}

}  // namespace b200

#endif  // B200_ATTN_PROMPT_CUH
