// attn_rows.cuh -- a warp's view of a row of D values, which the attention kernels share: lane i holds values
// [i D / 32, (i + 1) D / 32), as fp32.

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

}  // namespace b200

#endif  // B200_ATTN_ROWS_CUH
