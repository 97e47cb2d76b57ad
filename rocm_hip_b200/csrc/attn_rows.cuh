// attn_rows.cuh -- attention of one query row by one warp, in fp32 on the CUDA cores: the definition written out, for the
// rows that the tile kernels must not answer. A key is looked at only if the row may see it, so nothing in a masked place
// (an infinity, a NaN, memory never written) can reach the result.
//   s_j = scale (q . k_j),  m = max s_j,  p_j = 2^((s_j - m) log2 e),  out = sum_j p_j v_j / sum_j p_j
// with the running maximum: one pass over the keys, o and l rescaled when m grows. Lane i holds values
// [i D / 32, (i + 1) D / 32) of q, o and of every k and v row.

#ifndef B200_ATTN_ROWS_CUH
#define B200_ATTN_ROWS_CUH

#include <type_traits>

#include "common.cuh"

namespace b200 {

constexpr float LOG2E = 1.4426950408889634f;

// D / 32 = 2, 4 or 8 consecutive values as fp32
template <int N, typename T>
__device__ __forceinline__ void load_vals(const T* p, float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 f = *reinterpret_cast<const float2*>(p + i);
            v[i] = f.x;
            v[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(p + i);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                v[i] = bf16_lo(w);
                v[i + 1] = bf16_hi(w);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                v[i] = f.x;
                v[i + 1] = f.y;
            }
        }
    }
}

template <int N, typename T>
__device__ __forceinline__ void store_vals(T* p, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) Io<T>::store1(p + i, v[i]);
}

// The row's online softmax state
template <int N>
struct RowSoftmax {
    float m = -INFINITY, l = 0.0f, o[N];
    __device__ __forceinline__ RowSoftmax() {
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = 0.0f;
    }
    // one key: s2 = s_j log2 e, the same value in all lanes
    __device__ __forceinline__ void key(float s2, const float (&v)[N]) {
        const float mn = fmaxf(m, s2);
        if (mn == -INFINITY) return;              // a score of -inf before any other: weight 0
        const float a = exp2f(m - mn), p = exp2f(s2 - mn);
        m = mn;
        l = l * a + p;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * a + p * v[i];
    }
};

template <int N>
__device__ __forceinline__ float warp_dot(const float (&a)[N], const float (&b)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(a[i], b[i], s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    return s;
}

// Row of a prompt whose values in `out` came out non-finite and may owe that to keys the row does not see: query q, keys
// k0 + j k_stride, j < n. Lanes in `mine` look after their columns: the row is written anew unless all of its NaN turn out to
// be its own (found as soon as the keys that cause them have been met, so that inputs full of NaN do not cost a pass over
// all keys per row).
template <int D, typename T>
__device__ void attn_row_again(const T* q, const T* k0, const T* v0, long long k_stride, long long v_stride, int n, float scale2,
                               T* out, unsigned mine) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31, c = lane * N;
    const bool write = mine >> lane & 1;
    float qv[N], kv[N], vv[N], was[N];
    load_vals(q + c, qv);
    load_vals(out + c, was);
    RowSoftmax<N> st;
    for (int j = 0; j < n; ++j) {
        load_vals(k0 + j * k_stride + c, kv);
        load_vals(v0 + j * v_stride + c, vv);
        st.key(warp_dot(qv, kv) * scale2, vv);
        if ((j & 15) == 0) {
            bool open = false;      // a column of the row that is non-finite for a reason not yet met
#pragma unroll
            for (int i = 0; i < N; ++i) open |= !(fabsf(was[i]) < INFINITY) && st.o[i] == st.o[i] && st.l == st.l;
            if (!__any_sync(0xffffffffu, write && open)) return;
        }
    }
    const float r = st.l > 0.0f ? 1.0f / st.l : (st.l == 0.0f ? 0.0f : st.l);
#pragma unroll
    for (int i = 0; i < N; ++i) st.o[i] *= r;
    if (write) store_vals(out + c, st.o);
}

// Bit r of word r / 32: row r of a tile of 128 (of which `rows` exist) holds a value that is not finite
template <int D, typename T>
__device__ __forceinline__ void find_non_finite(const T* v, long long stride, int rows, unsigned (&bits)[4]) {
    constexpr int N = D / 32;
    const int c = (threadIdx.x & 31) * N;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        unsigned b = 0;
        for (int r = 0; r < 32 && w * 32 + r < rows; ++r) {
            float x[N];
            load_vals(v + (w * 32 + r) * stride + c, x);
            bool bad = false;
#pragma unroll
            for (int i = 0; i < N; ++i) bad |= !(fabsf(x[i]) < INFINITY);
            if (__any_sync(0xffffffffu, bad)) b |= 1u << r;
        }
        bits[w] = b;
    }
}

}  // namespace b200

#endif  // B200_ATTN_ROWS_CUH
