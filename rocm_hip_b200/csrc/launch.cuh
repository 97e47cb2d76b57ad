// launch.cuh -- host-side launch helpers shared by the translation units that launch kernels (layer_ops.cu,
// attention.cu): SM count, resident grids, programmatic dependent launches.

#ifndef B200_LAUNCH_CUH
#define B200_LAUNCH_CUH

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace b200 {

// SM count of the current device, cached per device (atomics: launchers run on any thread)
inline int sm_count() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int next_pow2(int v) { int p = 1; while (p < v) p <<= 1; return p; }
inline int round_up(int v, int m) { return (v + m - 1) / m * m; }

// Resident CTAs of `block` threads a B200 SM holds when only the thread count limits it
inline long long resident_ctas(int block) { return (long long)sm_count() * (2048 / block > 0 ? 2048 / block : 1); }

// CTAs of this kernel that are resident on the whole device at once (registers and shared memory counted): the grid
// of a kernel whose CTAs walk their rows with a grid stride, so that no CTA waits for another to retire. Cached per
// kernel and launch shape (the occupancy query costs microseconds).
template <typename K>
long long persistent_grid(K kernel, int block, size_t smem) {
    struct Entry { const void* f; int block; size_t smem; int dev; int per_sm; };
    thread_local Entry cache[16];
    thread_local int used = 0;
    int dev = 0;
    (void)cudaGetDevice(&dev);
    const void* f = reinterpret_cast<const void*>(kernel);
    for (int i = 0; i < used; ++i)
        if (cache[i].f == f && cache[i].block == block && cache[i].smem == smem && cache[i].dev == dev)
            return (long long)cache[i].per_sm * sm_count();
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem) != cudaSuccess || per_sm < 1) {
        (void)cudaGetLastError();
        per_sm = 1;
    }
    cache[used % 16] = {f, block, smem, dev, per_sm};
    if (used < 16) ++used;
    return (long long)per_sm * sm_count();
}

// Launch with programmatic stream serialisation allowed: the kernels launched this way start with pdl_entry(), so
// they may be scheduled while the kernel before them in the stream drains (see common.cuh). A failed launch leaves its
// error for launched() to return.
template <typename... KA, typename... A>
inline void launch_pdl(void (*kernel)(KA...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, static_cast<KA>(args)...);
}

}  // namespace b200

#endif  // B200_LAUNCH_CUH
