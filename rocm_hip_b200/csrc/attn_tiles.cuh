// attn_tiles.cuh -- attention on the fifth-generation tensor cores, what the prompt and the shared-prefix kernels have in
// common. A CTA holds NQ query tiles of 128 rows and walks keys in tiles of 128:
//   S = Q K^T        tensor cores, 128 x 128 fp32 in tensor memory
//   P = 2^(S c - m)  a thread per row: registers, running maximum m and sum l; P goes back over S as 16-bit pairs
//   O += P V         tensor cores, A = P from tensor memory; O stays there until the last tile
// While one tile's rows are in the softmax the tensor cores work for the other tile (NQ = 2), or on the next S of the same
// tile (NQ = 1: 256-wide heads, whose O takes half of the 512 columns, or when there are no more than 128 query rows). O is
// rescaled only when a row's maximum has grown by more than 2^8 since it was last taken: P then stays within what
// 16-bit floats and the fp32 sums bear, and almost no tile after the first pays for reading and writing O. Rounding P to
// 16 bits is what the tensor cores take (SPLIT: P = hi + lo, 22 bits, two products; Q likewise); l sums unrounded values.

#ifndef B200_ATTN_TILES_CUH
#define B200_ATTN_TILES_CUH

#include "umma.cuh"

namespace b200 {

// CTAs that gave up on a wait since the library was loaded (b200_attn_gave_up): 0 unless the hardware or a caller's
// memory failed under a kernel
__device__ int attn_gave_up;

struct TileBars {
    unsigned long long q_full, s_full[2], p_full[2], o_full[2], o_part, full[8], empty[8];
    uint32_t tmem;
    int dead;
};

// A wait that gives up for the whole CTA: once one role is dead nobody waits or issues any more
__device__ __forceinline__ bool wait_or_die(unsigned long long* bar, unsigned parity, volatile int* dead) {
    if (*dead) return false;
    if (mbar_wait(bar, parity)) return true;
    *dead = 1;
    return false;
}

// SC: columns of a ring stage (a K or V tile is D / SC stages of 128 rows), ST: stages
template <int D, int NQ, int SC, int ST, bool SPLIT, typename T>
struct Tiles {
    static constexpr int STAGE = TILE_ROWS * SC * 2;
    static constexpr int PARTS = D / SC;
    static constexpr int QTILE = TILE_ROWS * D * 2;                        // one query tile, one half of a split one
    static constexpr int Q_BYTES = NQ * QTILE * (SPLIT ? 2 : 1);           // [NQ][hi, lo][D / 64][128 rows][64 values]
    static constexpr int SMEM = 1024 + Q_BYTES + ST * STAGE;
    static constexpr int WARPS = NQ == 2 ? 12 : 6;                         // softmax, tensor cores, copies (and two idle warps)
    static constexpr int P_SHIFT_T = std::is_same<T, __half>::value ? 7 : 0;   // fp16 weights are held times 2^7 (at most 2^15)

    // A softmax thread holds its row's 128 scores: 208 registers. Twelve warps start with 168 each (64,512 in all); the four
    // that compute nothing go down to 80 and the eight softmax warps up, 4 x 32 x 80 + 8 x 32 x 208 = 63,488. (Six warps
    // may have 255 from the start.)
    static __device__ __forceinline__ void few_registers() {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    }
    static __device__ __forceinline__ void many_registers() {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    }

    // Barriers and tensor memory; all threads. q_arrivals: who fills the query tiles.
    static __device__ __forceinline__ void setup(TileBars& bars, int q_arrivals) {
        const int warp = threadIdx.x >> 5;
        if (warp == NQ * 4) {
            tmem_alloc(&bars.tmem, 512);
            if ((threadIdx.x & 31) == 0) {
                mbar_init(&bars.q_full, q_arrivals);
                mbar_init(&bars.o_part, 1);
                for (int i = 0; i < 2; ++i) {
                    mbar_init(&bars.s_full[i], 1);
                    mbar_init(&bars.p_full[i], 4);
                    mbar_init(&bars.o_full[i], 1);
                }
                for (int i = 0; i < ST; ++i) {
                    mbar_init(&bars.full[i], 1);
                    mbar_init(&bars.empty[i], 1);
                }
                bars.dead = 0;
                mbar_fence_init();
            }
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }
    static __device__ __forceinline__ void teardown(TileBars& bars) {
        tc_fence_before();
        __syncthreads();
        if (threadIdx.x >> 5 == NQ * 4) tmem_free(bars.tmem, 512);
        if (threadIdx.x == 0 && bars.dead) atomicAdd(&attn_gave_up, 1);
    }

    // The ring as the copying warp sees it: `load(smem, part, bar)` issues the copies of one stage, each lane its share of
    // them. One lane waits, so that all of them go on or stop together.
    struct Ring {
        TileBars& bars;
        unsigned char* ring;
        int st = 0, ph = 0;
        template <typename F>
        __device__ __forceinline__ void put(F load) {
            for (int p = 0; p < PARTS; ++p) {
                int ok = 0;
                if ((threadIdx.x & 31) == 0) {
                    ok = wait_or_die(&bars.empty[st], ph ^ 1, &bars.dead);
                    if (ok) mbar_expect(&bars.full[st], STAGE);
                }
                if (!__shfl_sync(0xffffffffu, ok, 0)) return;
                load(ring + st * STAGE, p, &bars.full[st]);
                if (++st == ST) { st = 0; ph ^= 1; }
            }
        }
    };

    // One thread: everything the tensor cores do for n[0] / n[1] key tiles of the query tiles. The ring brings
    // K 0, K 1, V 0, K 2, V 1, ...
    static __device__ __forceinline__ void products(TileBars& bars, const unsigned char* qs, const unsigned char* ring, const int (&n)[2]) {
        const uint32_t tmem = bars.tmem, id_s = idesc_f16<T>(TILE_ROWS, false), id_o = idesc_f16<T>(SC, true);
        const int n_all = max(n[0], n[1]);
        int st = 0, ph = 0;                   // the next stage to be taken from the ring
        const auto take = [&](int* stage) {   // the stages of a tile
            for (int p = 0; p < PARTS; ++p) {
                stage[p] = st;
                wait_or_die(&bars.full[st], ph, &bars.dead);
                if (++st == ST) { st = 0; ph ^= 1; }
            }
            tc_fence_after();
        };
        const auto give = [&](const int* stage) {
            for (int p = 0; p < PARTS; ++p) mma_commit(&bars.empty[stage[p]]);
        };
        const auto score = [&](int i, int buf, const int* stage) {   // S[buf] = Q_i K^T
            if (bars.dead) return;
            for (int c = 0; c < D / CHUNK; ++c) {
                const uint64_t b = desc_k_major(smem_u32(ring) + stage[c / (SC / CHUNK)] * STAGE + c % (SC / CHUNK) * CHUNK_BYTES);
                for (int z = 0; z < (SPLIT ? 2 : 1); ++z) {
                    const uint64_t a = desc_k_major(smem_u32(qs) + (i * (SPLIT ? 2 : 1) + z) * QTILE + c * CHUNK_BYTES);
                    for (int e = 0; e < CHUNK / 16; ++e) mma_ss(tmem + buf * 128, a + e * 2, b + e * 2, id_s, c + e + z > 0);
                }
            }
            mma_commit(&bars.s_full[buf]);
        };
        const auto join = [&](int i, int buf, const int* stage, bool add) {   // O_i += P[buf] V
            if (bars.dead) return;
            for (int p = 0; p < PARTS; ++p) {
                const uint64_t b = desc_mn_major(smem_u32(ring) + stage[p] * STAGE);
                for (int z = 0; z < (SPLIT ? 2 : 1); ++z)
                    for (int e = 0; e < TILE_ROWS / 16; ++e)
                        mma_ts(tmem + 256 + i * D + p * SC, tmem + buf * 128 + z * 64 + e * 8, b + e * (16 * 128 >> 4), id_o, add || e + z > 0);
            }
        };
        wait_or_die(&bars.q_full, 0, &bars.dead);
        tc_fence_after();
        int ks[PARTS], vs[PARTS];
        take(ks);
        for (int i = 0; i < NQ; ++i)
            if (n[i] > 0) score(i, NQ == 1 ? 0 : i, ks);
        give(ks);
        for (int j = 0; j < n_all; ++j) {
            const bool more = j + 1 < n_all;
            if (more) take(ks);
            if (NQ == 1 && more) {
                score(0, (j + 1) & 1, ks);
                give(ks);
            }
            take(vs);
            for (int i = 0; i < NQ; ++i) {
                if (j >= n[i]) continue;
                const int buf = NQ == 1 ? j & 1 : i;
                wait_or_die(&bars.p_full[buf], NQ == 1 ? (j >> 1) & 1 : j & 1, &bars.dead);
                tc_fence_after();
                join(i, buf, vs, j > 0);
                if (j + 1 == n[i]) mma_commit(&bars.o_full[i]);
                else if (NQ == 1) mma_commit(&bars.o_part);
                if (NQ == 2 && j + 1 < n[i]) score(i, i, ks);
            }
            if (NQ == 2 && more) give(ks);
            give(vs);
        }
    }

    // A softmax thread: its row's scores against key tile j into x, once they are there
    static __device__ __forceinline__ bool scores(TileBars& bars, int i, int j, uint32_t (&x)[128]) {
        const int buf = NQ == 1 ? j & 1 : i;
        if (!wait_or_die(&bars.s_full[buf], NQ == 1 ? (j >> 1) & 1 : j & 1, &bars.dead)) return false;
        tc_fence_after();
        const uint32_t s_addr = bars.tmem + buf * 128 + ((uint32_t)(threadIdx.x & 96) << 16);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, x + c * 32);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_pin(x + c * 32);
        return true;
    }

    // ... and, masked scores (-inf) in x, from there to P in tensor memory; c > 0 turns scores into powers of two
    static __device__ __forceinline__ bool weights(TileBars& bars, int i, int j, uint32_t (&x)[128], float c, float& m, float& l) {
        const int buf = NQ == 1 ? j & 1 : i;
        const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
        const uint32_t s_addr = bars.tmem + buf * 128 + lanes, o_addr = bars.tmem + 256 + i * D + lanes;
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 128; ++e) mx = fmaxf(mx, __uint_as_float(x[e]));
        if (j == 0) m = mx;
        else if (__any_sync(0xffffffffu, (mx - m) * c > 8.0f)) {
            // O holds the tiles before this one. NQ = 2: their products were issued before this S, so they are done. NQ = 1:
            // the last of them comes behind this S.
            if (NQ == 1 && !wait_or_die(&bars.o_part, (j - 1) & 1, &bars.dead)) return false;
            tc_fence_after();
            const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : ex2((m - mn) * c);
            m = mn;
            l *= f;
            for (int e0 = 0; e0 < D; e0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + e0, o);
                tmem_ld_wait();
                tmem_pin(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(o_addr + e0, o);
            }
        }
        const float neg = m == -INFINITY ? 0.0f : P_SHIFT_T - m * c;
        const f2 neg2 = pk2(neg, neg), c2 = pk2(c, c);
        f2 sum = pk2(0.0f, 0.0f);
#pragma unroll
        for (int e0 = 0; e0 < 128; e0 += 64) {
            uint32_t p[32], lo[SPLIT ? 32 : 1];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                float a, b;
                upk2(fma2(pk2(__uint_as_float(x[e0 + 2 * e]), __uint_as_float(x[e0 + 2 * e + 1])), c2, neg2), a, b);
                a = ex2(a);
                b = ex2(b);
                sum = add2(sum, pk2(a, b));
                if constexpr (SPLIT) split16(a, b, &p[e], &lo[e]);
                else p[e] = pack16<T>(a, b);
            }
            tmem_st32(s_addr + e0 / 2, p);
            if constexpr (SPLIT) tmem_st32(s_addr + 64 + e0 / 2, lo);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&bars.p_full[buf]);
        float a, b;
        upk2(sum, a, b);
        l += a + b;
        return true;
    }
};

}  // namespace b200

#endif  // B200_ATTN_TILES_CUH
