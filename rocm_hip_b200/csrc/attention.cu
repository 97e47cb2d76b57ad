// attention.cu -- launchers of part 5 of include/b200_layer_ops.h: attention over packed prompts, attention of single
// tokens over a paged cache, and the pages of that cache.

#include "b200_layer_ops.h"

#include <limits.h>
#include <math.h>

#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <type_traits>

#include "attn_decode.cuh"
#include "attn_own.cuh"
#include "attn_prefix.cuh"
#include "attn_prompt.cuh"
#include "internal.h"
#include "kv_pages.cuh"
#include "launch.cuh"

using namespace b200;

namespace {

bool good_scale(float s) { return s > 0.0f && s < INFINITY; }
bool good_heads(int n_q, int n_kv, int D) {
    return n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && (D == 64 || D == 128 || D == 256) && n_q <= INT_MAX / D;
}

// ---------------------------------------------------------------- tensor maps

// cuTensorMapEncodeTiled by the runtime's entry point lookup: the library does not link the driver
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> cached{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 fn = cached.load(std::memory_order_acquire);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        cached.store(fn, std::memory_order_release);
    }
    return fn;
}

template <typename T>
constexpr CUtensorMapDataType map_type() {
    return std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// rows [T][heads * D] `stride` values apart, fetched as boxes of 128 rows x 64 values of one head
template <typename T>
bool row_map(CUtensorMap* m, const T* p, int D, int heads, long long rows, long long stride) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {CHUNK, 1, TILE_ROWS}, step[3] = {1, 1, 1};
    const auto fn = encode_fn();
    return fn && fn(m, map_type<T>(), 3, const_cast<T*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Lets a kernel have `bytes` of dynamic shared memory on the current device: asked once per kernel and device (`done`: a
// bit per device, the caller's static for that kernel), for the call costs as much as a launch
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t st = cudaGetDevice(&dev);
    if (st != cudaSuccess) return st;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (st == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return st;
}

// ---------------------------------------------------------------- prompts

template <typename T>
cudaError_t launch_prompt(const T* q, const T* k, const T* v, T* out, const int* seq_start, int n_seqs, long long rows, int n_q,
                          int n_kv, int D, long long q_stride, long long k_stride, long long v_stride, float scale,
                          cudaStream_t stream) {
    if (!q || !k || !v || !out || n_seqs < 1 || (!seq_start && n_seqs != 1) || rows < 1 || rows > (1 << 27) ||
        !good_heads(n_q, n_kv, D) || !good_scale(scale))
        return cudaErrorInvalidValue;
    if (q_stride == 0) q_stride = (long long)n_q * D;
    if (k_stride == 0) k_stride = (long long)n_kv * D;
    if (v_stride == 0) v_stride = (long long)n_kv * D;
    if (q_stride < (long long)n_q * D || k_stride < (long long)n_kv * D || v_stride < (long long)n_kv * D || q_stride % 8 ||
        k_stride % 8 || v_stride % 8 || !al16(q) || !al16(k) || !al16(v) || !al16(out) || out == q || out == k || out == v)
        return cudaErrorInvalidValue;
    // How a CTA's two query tiles come about (attn_prompt.cuh): two heads of an even group, else 256 rows; and, where those
    // would hardly fill the SMs once, one tile whose keys are shared between the two: half the steps for the block that takes
    // longest, for twice the K and V bytes a step (one sequence, 16 / 8 heads of 128: 512 rows, 32 blocks, 12.8 -> 9.9 us;
    // 1,024 rows, 64, 19.1 -> 13.7; 2,427 rows, 152, 39.8 -> 37.4; four of 1,024 rows, heads of 64, 288 blocks: 33 -> 42)
    const long long slots128 = seq_start ? rows / TILE_ROWS + n_seqs : (rows + TILE_ROWS - 1) / TILE_ROWS;
    const long long slots256 = seq_start ? rows / (2 * TILE_ROWS) + n_seqs : (rows + 2 * TILE_ROWS - 1) / (2 * TILE_ROWS);
    const bool even = n_q / n_kv % 2 == 0;
    int mode = D == 256 ? BY_ROWS : even ? BY_HEADS : BY_ROWS;
    if (D < 256 && (even ? slots128 * (n_q / 2) : slots256 * n_q) * 4 < 5LL * sm_count()) mode = BY_KEYS;
    const long long n_slots = D < 256 && mode == BY_ROWS ? slots256 : slots128, grid = n_slots * (mode == BY_HEADS ? n_q / 2 : n_q);
    if (grid > INT_MAX) return cudaErrorInvalidValue;
    if (!lib_ready()) return cudaErrorInvalidDeviceFunction;
    CUtensorMap mq, mk, mv;
    if (!row_map<T>(&mq, q, D, n_q, rows, q_stride) || !row_map<T>(&mk, k, D, n_kv, rows, k_stride) ||
        !row_map<T>(&mv, v, D, n_kv, rows, v_stride))
        return cudaErrorInvalidValue;
    cudaError_t st;
#define TILES(D_, MODE_)                                                                                                     \
    do {                                                                                                                     \
        using Ti = PromptTiles<D_, T>;                                                                                       \
        constexpr int SMEM = Ti::SMEM + PROMPT_OUT<D_>;                                                                      \
        static std::atomic<unsigned long long> done;                                                                         \
        st = allow_smem(k_attn_prompt<D_, T, MODE_>, SMEM, done);                                                                  \
        if (st != cudaSuccess) return st;                                                                                    \
        launch_pdl((k_attn_prompt<D_, T, MODE_>), (unsigned)grid, PROMPT_WARPS<D_> * 32, SMEM, stream, mq, mk, mv, v, out, seq_start,  \
                   n_seqs, (int)rows, n_q, n_q / n_kv, v_stride, scale * LOG2E, (int)n_slots);                               \
    } while (0)
#define MODES(D_)                                                                                                            \
    do {                                                                                                                     \
        if (mode == BY_KEYS) TILES(D_, BY_KEYS); else if (mode == BY_HEADS) TILES(D_, BY_HEADS); else TILES(D_, BY_ROWS);    \
    } while (0)
    if (D == 64) MODES(64); else if (D == 128) MODES(128); else TILES(256, BY_ROWS);
#undef MODES
#undef TILES
    return launched();
}

// ---------------------------------------------------------------- single tokens

// The pages of one half (K or V) of a layer, fetched as boxes of up to `rows` rows x 64 values of one head
bool page_map(CUtensorMap* m, const __half* p, int D, int heads, const PagedKv& kv, int rows) {
    const int in_page = 1 << kv.kv_shift;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)in_page, (cuuint64_t)kv.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)kv.kv_stride * 2,
                                   (cuuint64_t)(kv.n_pages > 1 ? kv.kv_bstride : kv.kv_stride) * 2};
    const cuuint32_t box[4] = {CHUNK, 1, (cuuint32_t)(in_page < rows ? in_page : rows), 1}, step[4] = {1, 1, 1, 1};
    const auto fn = encode_fn();
    return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(p), dims, strides, box, step,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a decode call launches and where its pieces lie in scratch: a function of the sizes the host knows. `bytes` covers what
// a call of either row type uses and grows with B and the prefix, so that the scratch of the largest call serves all smaller
// ones.
struct DecodePlan {
    int grid_own, nq, row_tiles, splits;     // splits 0: nothing is shared
    long long px_rows;
    size_t first, shares, own_ml, own_o, px_ml, px_o, bytes;

    DecodePlan(int n_q, int n_kv, int D, int B, int prefix, bool f32) {
        const int warps = D == 256 ? OwnShape<256>::WARPS : OwnShape<128>::WARPS, sms = sm_count();
        const OwnPlan own(n_q, n_kv, warps);
        grid_own = sms;
        const size_t pieces = ((size_t)grid_own + (size_t)B * own.groups) * warps * own.hg;
        splits = 0;
        nq = row_tiles = 0;
        px_rows = 0;
        const long long M = (long long)B * (n_q / n_kv);
        size_t px_most = 0;
        // One sequence shares nothing, and less than two tiles of rows are not worth a launch of their own
        if (B > 1 && prefix >= 2 * TILE_ROWS) {
            nq = D == 256 || M <= TILE_ROWS ? 1 : 2;
            row_tiles = (int)((M + nq * TILE_ROWS - 1) / (nq * TILE_ROWS));
            px_rows = (long long)row_tiles * nq * TILE_ROWS;
            // stretches of the prefix: as many as make the CTAs whole waves of the device, counting about four tiles' time
            // for what a CTA does once (its queries, its result and the pieces' way through scratch). For fp32 rows no
            // longer than six tiles: the tensor cores cut sums off where fp32 arithmetic rounds, a stretch of t tiles
            // (16 t additions) loses up to 2.5e-8 per addition, and joining stretches does not (against 64 bits: 8,192 rows,
            // heads of 256, 1.7e-6; 32,768 rows, heads of 128, 1.4e-6; stretches of nine and of 37 tiles, which the waves
            // alone would give, lost twice and eight times as much). Beyond that, CTAs for four waves or eight per query tile
            // at most, for scratch's sake (one in 180 of 40,000 drawn sizes would take more, by this count 11 % faster at best).
            const int tiles = ((prefix < PagedKv::MOST_ROWS ? prefix : PagedKv::MOST_ROWS) + TILE_ROWS - 1) / TILE_ROWS;
            const int six = (tiles + 5) / 6, least = f32 ? six : 1;
            const long long base = (long long)n_kv * row_tiles, ctas = 4LL * sms > 8 * base ? 4LL * sms : 8 * base;
            long long best = LLONG_MAX;
            if (prefix <= PagedKv::MOST_ROWS)      // (no sequence has more)
                for (int s = least; s <= tiles && s < least + 64 && (s == least || base * s <= ctas); ++s) {
                    const long long cost = ((base * s + sms - 1) / sms) * ((tiles + s - 1) / s + 4);
                    if (cost < best) { best = cost; splits = s; }
                }
            const long long longest = base * six > ctas ? base * six : ctas, all = base * tiles;
            px_most = (size_t)(longest < all ? longest : all) * nq * TILE_ROWS;
        }
        const auto put = [this](size_t n) {
            const size_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        bytes = 256;
        first = put(((size_t)B + 1) * 4);
        shares = put((size_t)B * 4);
        own_ml = put(pieces * 8);
        own_o = put(pieces * D * 4);
        px_ml = put(px_most * 8);
        px_o = put(px_most * D * 4);
    }
};

template <int D, typename T>
cudaError_t launch_decode_d(const T* q, const PagedKv& kv, int prefix, T* out, int n_q, int n_kv, int B, float scale2, char* scratch,
                            const DecodePlan& pl, cudaStream_t stream) {
    constexpr bool SPLIT = sizeof(T) == 4;
    const OwnPlan own(n_q, n_kv, OwnShape<D>::WARPS);
    // The copy engine takes the cache apart where pages are whole swizzle atoms (8 rows) and a tensor map can describe it;
    // else a prefix is read like every sequence's own rows, and those by the threads. It fetches 16 rows at a time, so a
    // sequence's last fetch may reach behind its rows, to the page's end at most: pages of more than 4,096 rows (a contiguous
    // cache is one of 2^30) need not be memory up to there.
    CUtensorMap mk, mv, ok, ov;
    const bool box = kv.kv_shift >= 3 && kv.kv_shift <= 12 && page_map(&ok, kv.K, D, n_kv, kv, 16) && page_map(&ov, kv.V, D, n_kv, kv, 16);
    const long long grid = (long long)n_kv * pl.row_tiles * pl.splits;
    const bool shared = grid > 0 && grid <= INT_MAX && kv.kv_shift >= 3 && page_map(&mk, kv.K, D, n_kv, kv, TILE_ROWS) &&
                        page_map(&mv, kv.V, D, n_kv, kv, TILE_ROWS);
    const PrefixScratch px{shared ? pl.splits : 0, pl.px_rows, reinterpret_cast<float*>(scratch + pl.px_ml),
                           reinterpret_cast<float*>(scratch + pl.px_o)};
    const int behind = shared ? prefix : 0;
    const OwnScratch sc{reinterpret_cast<int*>(scratch), reinterpret_cast<int*>(scratch + pl.first),
                        shared ? reinterpret_cast<int*>(scratch + pl.shares) : nullptr, reinterpret_cast<float*>(scratch + pl.own_ml),
                        reinterpret_cast<float*>(scratch + pl.own_o)};
    cudaError_t st;
    if (shared) {
        launch_pdl(k_attn_shares, (unsigned)B, SHARES_THREADS, 0, stream, kv, sc.shares, B, prefix);
        if ((st = launched()) != cudaSuccess) return st;
    }
#define OWN(BOX_)                                                                                                            \
    do {                                                                                                                     \
        static std::atomic<unsigned long long> done;                                                                         \
        if ((st = allow_smem(k_attn_own<D, T, BOX_>, OwnShape<D>::SMEM, done)) != cudaSuccess) return st;                         \
        launch_pdl((k_attn_own<D, T, BOX_>), (unsigned)pl.grid_own, OwnShape<D>::WARPS * 32, OwnShape<D>::SMEM, stream, ok, ov, q, kv, \
                   sc, own, n_q, n_q / n_kv, B, behind, scale2);                                                                       \
    } while (0)
    if (box) OWN(true); else OWN(false);
#undef OWN
    if ((st = launched()) != cudaSuccess) return st;
    if (shared) {
#define PREFIX(NQ_)                                                                                                       \
    do {                                                                                                                  \
        using Ti = typename PrefixShape<D, NQ_, SPLIT>::Ti;                                                               \
        static std::atomic<unsigned long long> done;                                                                      \
        if ((st = allow_smem(k_attn_prefix<D, NQ_, T>, Ti::SMEM, done)) != cudaSuccess) return st;                             \
        launch_pdl((k_attn_prefix<D, NQ_, T>), (unsigned)grid, Ti::WARPS * 32, Ti::SMEM, stream, mk, mv, q, kv, px, n_q, n_kv, B, prefix, scale2, \
                   pl.row_tiles);                                                                                         \
    } while (0)
        if constexpr (D < 256) {
            if (pl.nq == 2) PREFIX(2); else PREFIX(1);
        } else {
            PREFIX(1);
        }
#undef PREFIX
        if ((st = launched()) != cudaSuccess) return st;
    }
    launch_pdl((k_attn_join<D, T>), (unsigned)(((long long)B * n_q + 3) / 4), 128, 0, stream, sc, own, px, out, n_q, n_kv, B);
    return launched();
}

template <typename T>
cudaError_t launch_decode(const T* q, const uint16_t* K, const uint16_t* V, int kv_stride, int kv_shift, long long kv_bstride,
                          int n_pages, const int* pages, int max_pages, const int* lens, int prefix_len, T* out, int n_q, int n_kv,
                          int D, int B, float scale, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    if (!q || !K || !V || !pages || !lens || !out || !good_heads(n_q, n_kv, D) || !good_scale(scale) || B < 1 ||
        (long long)B * n_q > (1 << 28) || n_pages < 1 || max_pages < 1 || kv_shift < 0 || kv_shift > 30 ||
        kv_stride < (long long)n_kv * D || kv_stride % 8 || kv_bstride % 8 || kv_bstride < 0 || !al16(q) || !al16(K) || !al16(V) ||
        !al16(out) || (const void*)out == (const void*)q)
        return cudaErrorInvalidValue;
    if (prefix_len < 0 || prefix_len % (1 << kv_shift) || prefix_len > ((long long)max_pages << kv_shift)) return cudaErrorInvalidValue;
    const DecodePlan pl(n_q, n_kv, D, B, prefix_len, sizeof(T) == 4);
    if (scratch_bytes < pl.bytes || !scratch || !al16(scratch)) return cudaErrorInvalidValue;
    if (!lib_ready()) return cudaErrorInvalidDeviceFunction;
    const PagedKv kv{reinterpret_cast<const __half*>(K), reinterpret_cast<const __half*>(V), pages, lens, kv_bstride, kv_stride,
                     kv_shift, n_pages, max_pages};
#define CALL(D_) launch_decode_d<D_, T>(q, kv, prefix_len, out, n_q, n_kv, B, scale * LOG2E, static_cast<char*>(scratch), pl, stream)
    return D == 64 ? CALL(64) : D == 128 ? CALL(128) : CALL(256);
#undef CALL
}

// ---------------------------------------------------------------- pages

bool good_pages(const b200_kv_pages* kv) {
    return kv && kv->table && kv->lens && kv->refs && kv->info && kv->work && kv->pool && kv->n_seqs > 0 && kv->max_pages > 0 &&
           kv->n_pages > 0 && kv->page_shift >= 0 && kv->page_shift <= 30 &&
           ((long long)kv->n_pages << kv->page_shift) <= INT_MAX && kv->page_bytes > 0 && kv->page_bytes % 16 == 0 &&
           kv->page_bytes <= INT_MAX && kv->n_parts > 0 && (kv->n_parts == 1 || kv->part_stride >= kv->page_bytes * kv->n_pages) &&
           kv->part_stride % 16 == 0 && al16(kv->pool) && (long long)kv->n_seqs * kv->max_pages <= INT_MAX;
}

// How many CTAs the control kernel takes: one where its tables are small, so that the passes over them are separated by a
// CTA's barrier only, else a cluster of eight
bool small_pages(const b200_kv_pages* kv) { return (long long)kv->n_seqs * kv->max_pages <= 16384 && kv->n_pages <= 16384; }

// The control kernel, then the copies it listed
template <int CTAS, typename... KA, typename... A>
cudaError_t launch_pages(const b200_kv_pages* kv, cudaStream_t stream, void (*kernel)(KA...), A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CTAS, 1, 1);
    cfg.blockDim = dim3(KVP_THREADS, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, kernel, static_cast<KA>(args)...);
    const cudaError_t st = launched();
    if (st != cudaSuccess) return st;
    launch_pdl(k_kv_pages_copy, (unsigned)resident_ctas(256), 256, 0, stream, *kv);
    return launched();
}

}  // namespace

extern "C" {

cudaError_t gpu_attn_prompt_bf16(const uint16_t* q, const uint16_t* k, const uint16_t* v, uint16_t* out, const int* seq_start,
                                 int n_seqs, long long T, int n_q, int n_kv, int head_dim, long long q_stride, long long k_stride,
                                 long long v_stride, float scale, cudaStream_t stream) {
    using E = __nv_bfloat16;
    return launch_prompt(reinterpret_cast<const E*>(q), reinterpret_cast<const E*>(k), reinterpret_cast<const E*>(v),
                         reinterpret_cast<E*>(out), seq_start, n_seqs, T, n_q, n_kv, head_dim, q_stride, k_stride, v_stride, scale,
                         stream);
}

cudaError_t gpu_attn_prompt_f16(const uint16_t* q, const uint16_t* k, const uint16_t* v, uint16_t* out, const int* seq_start,
                                int n_seqs, long long T, int n_q, int n_kv, int head_dim, long long q_stride, long long k_stride,
                                long long v_stride, float scale, cudaStream_t stream) {
    using E = __half;
    return launch_prompt(reinterpret_cast<const E*>(q), reinterpret_cast<const E*>(k), reinterpret_cast<const E*>(v),
                         reinterpret_cast<E*>(out), seq_start, n_seqs, T, n_q, n_kv, head_dim, q_stride, k_stride, v_stride, scale,
                         stream);
}

int b200_attn_gave_up(void) {
    int n = 0;
    return cudaMemcpyFromSymbol(&n, attn_gave_up, sizeof n) == cudaSuccess ? n : -1;
}

size_t gpu_attn_decode_scratch_bytes(int n_q, int n_kv, int head_dim, int B, int prefix_len) {
    if (!good_heads(n_q, n_kv, head_dim) || B < 1 || (long long)B * n_q > (1 << 28) || prefix_len < 0) return 0;
    return DecodePlan(n_q, n_kv, head_dim, B, prefix_len, true).bytes;
}

cudaError_t gpu_attn_decode(const float* q, const uint16_t* K, const uint16_t* V, int kv_stride, int kv_shift, long long kv_bstride,
                            int n_pages, const int* pages, int max_pages, const int* lens, int prefix_len, float* out, int n_q,
                            int n_kv, int head_dim, int B, float scale, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
    return launch_decode(q, K, V, kv_stride, kv_shift, kv_bstride, n_pages, pages, max_pages, lens, prefix_len, out, n_q, n_kv,
                         head_dim, B, scale, scratch, scratch_bytes, stream);
}

cudaError_t gpu_attn_decode_bf16(const uint16_t* q, const uint16_t* K, const uint16_t* V, int kv_stride, int kv_shift,
                                 long long kv_bstride, int n_pages, const int* pages, int max_pages, const int* lens, int prefix_len,
                                 uint16_t* out, int n_q, int n_kv, int head_dim, int B, float scale, void* scratch,
                                 size_t scratch_bytes, cudaStream_t stream) {
    return launch_decode(reinterpret_cast<const __nv_bfloat16*>(q), K, V, kv_stride, kv_shift, kv_bstride, n_pages, pages, max_pages,
                         lens, prefix_len, reinterpret_cast<__nv_bfloat16*>(out), n_q, n_kv, head_dim, B, scale, scratch,
                         scratch_bytes, stream);
}

size_t gpu_kv_pages_work_ints(int n_seqs, int n_pages) {
    return n_seqs > 0 && n_pages > 0 ? KvPagesWork::ints(n_seqs, n_pages) : 0;
}

cudaError_t gpu_kv_pages_fork(const b200_kv_pages* kv, const int* parent, cudaStream_t stream) {
    if (!good_pages(kv) || !parent || parent == kv->lens) return cudaErrorInvalidValue;
    if (!lib_ready()) return cudaErrorInvalidDeviceFunction;
    return small_pages(kv) ? launch_pages<1>(kv, stream, k_kv_pages_fork<1>, *kv, parent)
                           : launch_pages<8>(kv, stream, k_kv_pages_fork<8>, *kv, parent);
}

cudaError_t gpu_kv_pages_resize(const b200_kv_pages* kv, const int* new_lens, int* slots, int n_slots, cudaStream_t stream) {
    if (!good_pages(kv) || !new_lens || new_lens == kv->lens || n_slots < 0) return cudaErrorInvalidValue;
    if (!lib_ready()) return cudaErrorInvalidDeviceFunction;
    return small_pages(kv) ? launch_pages<1>(kv, stream, k_kv_pages_resize<1>, *kv, new_lens, slots, n_slots)
                           : launch_pages<8>(kv, stream, k_kv_pages_resize<8>, *kv, new_lens, slots, n_slots);
}

cudaError_t gpu_kv_pages_compact(const b200_kv_pages* kv, cudaStream_t stream) {
    if (!good_pages(kv)) return cudaErrorInvalidValue;
    if (!lib_ready()) return cudaErrorInvalidDeviceFunction;
    return small_pages(kv) ? launch_pages<1>(kv, stream, k_kv_pages_compact<1>, *kv)
                           : launch_pages<8>(kv, stream, k_kv_pages_compact<8>, *kv);
}

}  // extern "C"
