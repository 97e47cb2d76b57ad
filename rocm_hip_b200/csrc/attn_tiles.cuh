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
//
// The methods are published ones: softmax with a running maximum and sum (Milakov and Gimelshein, 2018, "Online normalizer
// calculation for softmax"), two query tiles that take turns at the tensor cores, O rescaled only past a threshold, part of the
// exponentials by a polynomial after Cody and Waite's range reduction. The code and the coefficients are this library's own.

#ifndef B200_ATTN_TILES_CUH
#define B200_ATTN_TILES_CUH

#include "umma.cuh"

namespace b200 {

// CTAs that gave up on a wait since the library was loaded (b200_attn_gave_up): 0 unless the hardware or a caller's
// memory failed under a kernel
__device__ int attn_gave_up;

struct TileBars {
    unsigned long long q_full[2], s_full[2], p_half[2], p_full[2], o_full[2], o_part, quiet, full[8], empty[8];
    uint32_t tmem;
    int dead;
};

// Where a role stands: barriers count on over all the query tiles a CTA works through. steps: key tiles per query tile (NQ = 1:
// of the CTA, whose two S buffers take turns); items: query tiles; parts: products that were not a query tile's last.
struct TileFlow {
    int stage = 0, phase = 0;
    unsigned steps[2] = {0, 0}, items[2] = {0, 0}, parts = 0;
};

// A wait that gives up for the whole CTA: once one role is dead nobody waits or issues any more. `dead` is looked at only
// while the barrier is not there yet.
__device__ __forceinline__ bool wait_or_die(unsigned long long* bar, unsigned parity, volatile int* dead) {
    const unsigned b = smem_u32(bar);
    for (int i = 0; i < MBAR_POLLS; ++i) {
        unsigned ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(b), "r"(parity)
                     : "memory");
        if (ok) return true;
        if (*dead) return false;
    }
    *dead = 1;
    return false;
}

// The same for a whole warp: all lanes go on, or none. Such a wait is for one key tile's work of another role, microseconds;
// MBAR_POLLS are milliseconds at least.
__device__ __forceinline__ bool warp_wait(unsigned long long* bar, unsigned parity, volatile int* dead) {
    return __all_sync(0xffffffffu, wait_or_die(bar, parity, dead));
}

// A wait for another role's whole query tile, which takes two microseconds per 128 keys: a look every half microsecond after
// the first few thousand, for some eight seconds in all
__device__ __forceinline__ bool warp_wait_long(unsigned long long* bar, unsigned parity, volatile int* dead) {
    const unsigned b = smem_u32(bar);
    bool there = false;
    for (int i = 0; i < (1 << 24) && !there; ++i) {
        unsigned ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(b), "r"(parity)
                     : "memory");
        there = ok;
        if (!there && *dead) break;
        if (!there && i > 4096) __nanosleep(500);
    }
    if (!there) *dead = 1;
    return __all_sync(0xffffffffu, there);
}

// SC: columns of a ring stage (a K or V tile is D / SC stages of 128 rows), ST: stages
template <int D, int NQ, int SC, int ST, bool SPLIT, typename T>
struct Tiles {
    static constexpr int STAGE = TILE_ROWS * SC * 2, STAGES = ST;
    static constexpr int PARTS = D / SC;
    static constexpr int QTILE = TILE_ROWS * D * 2;                        // one query tile, one half of a split one
    static constexpr int Q_BYTES = NQ * QTILE * (SPLIT ? 2 : 1);           // [NQ][hi, lo][D / 64][128 rows][64 values]
    static constexpr int RING = ST * STAGE;
    static constexpr int SMEM = 1024 + Q_BYTES + RING;
    static constexpr int WARPS = NQ == 2 ? 12 : 7;                         // softmax, tensor cores, copies, two more (prompts: eight of one query tile)
    // NQ = 2: the products of a tile's first half of the keys begin while the second half is still in the softmax (8,192 rows,
    // 32 heads of 128: 1,246 -> 1,295 TFLOP/s). With one query tile the next S fills that time (heads of 256: 1,286 without,
    // 1,261 with).
    static constexpr bool HALVES = NQ == 2;
    // Weights are held times a power of two: fp16 ones 2^7 (at most 2^15, and normal for as long as they count), bf16 ones
    // 2^-24: m may lag by 2^8, so the sum of 65,536 of them is at most 1 and finite v of any size cannot make O overflow,
    // while v of 1e-30 still give normal products.
    static constexpr int P_SHIFT_T = std::is_same<T, __half>::value ? 7 : -24;

    // A softmax thread holds its row's 128 scores: 224 registers. Twelve warps start with 168 each (64,512 in all); the four
    // that compute nothing go down to 56 and the eight softmax warps up, 4 x 32 x 56 + 8 x 32 x 224 = 64,512. (Seven
    // warps may have 255 from the start.)
    static __device__ __forceinline__ void few_registers() {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    }
    static __device__ __forceinline__ void many_registers() {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    }

    // Barriers and tensor memory; all threads. q_arrivals: how many fill a query tile.
    static __device__ __forceinline__ void setup(TileBars& bars, int q_arrivals) {
        const int warp = threadIdx.x >> 5;
        if (warp == NQ * 4) {
            tmem_alloc(&bars.tmem, 512);
            if ((threadIdx.x & 31) == 0) {
                mbar_init(&bars.o_part, 1);
                mbar_init(&bars.quiet, 1);
                for (int i = 0; i < 2; ++i) {
                    mbar_init(&bars.q_full[i], q_arrivals);
                    mbar_init(&bars.s_full[i], 1);
                    mbar_init(&bars.p_half[i], 4);
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
    // them. One lane waits, so that all of them go on or stop together. The copies report to bars.full or, for tiles that
    // somebody looks at before the tensor cores may have them (and then arrives on bars.full), to `others`.
    struct Ring {
        TileBars& bars;
        unsigned char* ring;
        int st = 0, ph = 0;
        unsigned other = 0, turn = 0;     // bit s: stage s's last copies reported to the other barriers; parity of the next such
        template <typename F>
        __device__ __forceinline__ void put(F load, unsigned long long* others = nullptr) {
            unsigned long long* full = others ? others : bars.full;
            for (int p = 0; p < PARTS; ++p) {
                int ok = 0;
                if ((threadIdx.x & 31) == 0) {
                    ok = wait_or_die(&bars.empty[st], ph ^ 1, &bars.dead);
                    if (ok) mbar_expect(&full[st], STAGE);
                }
                if (!__shfl_sync(0xffffffffu, ok, 0)) return;
                load(ring + st * STAGE, p, &full[st]);
                const unsigned bit = 1u << st;
                if (others) { other |= bit; turn ^= bit; } else other &= ~bit;
                if (++st == ST) { st = 0; ph ^= 1; }
            }
        }
    };

    // The end of a role, also of one that gave up: nothing that it started is still under way when the CTA ends and its memory,
    // shared or tensor, becomes another's. Where all went well both are there already or about to be.
    static __device__ __forceinline__ void copies_done(TileBars& bars, const Ring& r, unsigned long long* others, const unsigned (&queries)[2]) {
#pragma unroll 1
        for (int i = 0; i < ST; ++i) {
            if (r.other >> i & 1) (void)mbar_wait(&others[i], (r.turn >> i & 1) ^ 1);
            else (void)mbar_wait(&bars.full[i], i < r.st ? r.ph : r.ph ^ 1);     // (a stage never used: the phase before the first)
        }
        for (int i = 0; i < 2; ++i)
            if (queries[i]) (void)mbar_wait(&bars.q_full[i], (queries[i] - 1) & 1);
    }
    static __device__ __forceinline__ void products_done(TileBars& bars) {
        if (elect_one()) mma_commit(&bars.quiet);
        (void)mbar_wait(&bars.quiet, 0);
    }

    static __device__ __forceinline__ int buffer(unsigned steps, int i) { return NQ == 1 ? steps & 1 : i; }
    static __device__ __forceinline__ unsigned parity(unsigned steps) { return NQ == 1 ? steps >> 1 & 1 : steps & 1; }

    // One warp: everything the tensor cores do for n0 / n1 key tiles of the query tiles. The ring brings
    // K 0, K 1, V 0, K 2, V 1, ...  q_empty: told when a query tile's last scores are done. False: given up.
    // KEYS: there is one query tile, and its n0 key tiles go to the two S and O in turn, as two query tiles' would; the ring
    // brings K 0, K 1, V 0, K 2, V 1, K 3, ...
    template <bool KEYS = false>
    static __device__ __forceinline__ bool products(TileBars& bars, const unsigned char* qs, const unsigned char* ring, int n0, int n1,
                                                    TileFlow& f, unsigned long long* q_empty = nullptr) {
        constexpr uint32_t id_s = idesc_f16<T>(TILE_ROWS, false), id_o = idesc_f16<T>(SC, true);
        constexpr int Z = SPLIT ? 2 : 1;
        const uint32_t tmem = bars.tmem, q_desc = desc_k_major(smem_u32(qs)), k_desc = desc_k_major(smem_u32(ring)),
                       v_desc = desc_mn_major(smem_u32(ring));
        const int n_all = max(n0, n1);
        bool dead = false;
        const auto after = [](int stage, int p) { return stage + p < ST ? stage + p : stage + p - ST; };
        const auto take = [&]() {             // the stages of a tile: the first one
            const int first = f.stage;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                dead = dead || !warp_wait(&bars.full[f.stage], f.phase, &bars.dead);
                if (++f.stage == ST) { f.stage = 0; f.phase ^= 1; }
            }
            tc_fence_after();
            return first;
        };
        const auto give = [&](int stage) {
            if (elect_one())
#pragma unroll
                for (int p = 0; p < PARTS; ++p) mma_commit(&bars.empty[after(stage, p)]);
        };
        const auto score = [&](int i, int buf, int stage) {   // S[buf] = Q_i K^T, Q_0 if KEYS
            const uint32_t d = tmem + buf * 128;
            if (elect_one()) {
                // (SPLIT: the low parts first, while the sum that each addition cuts off is still small)
#pragma unroll
                for (int z = Z - 1; z >= 0; --z)
#pragma unroll
                    for (int c = 0; c < D / CHUNK; ++c) {
                        const uint32_t b = k_desc + after(stage, c / (SC / CHUNK)) * (STAGE >> 4) + c % (SC / CHUNK) * (CHUNK_BYTES >> 4);
                        const uint32_t a = q_desc + ((KEYS ? 0 : i) * Z + z) * (QTILE >> 4) + c * (CHUNK_BYTES >> 4);
#pragma unroll
                        for (int e = 0; e < CHUNK / 16; ++e) mma_ss(d, a + e * 2, b + e * 2, id_s, z < Z - 1 || c + e > 0);
                    }
                mma_commit(&bars.s_full[buf]);
            }
        };
        // O_i += P[buf] V for the 16-key steps [e0, e1)
        const auto join = [&](int i, int buf, int stage, bool add, int e0, int e1) {
            if (elect_one()) {
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const uint32_t b = v_desc + after(stage, p) * (STAGE >> 4), d = tmem + 256 + i * D + p * SC;
#pragma unroll
                    for (int z = Z - 1; z >= 0; --z)
#pragma unroll
                        for (int e = e0; e < e1; ++e)
                            mma_ts(d, tmem + buf * 128 + z * 64 + e * 8, b + e * (16 * 128 >> 4), id_o, add || z < Z - 1 || e > e0);
                }
            }
        };
        int ks = take(), vs;
        if constexpr (KEYS) {
            static_assert(NQ == 2, "two S and two O");
            dead = dead || !warp_wait(&bars.q_full[0], f.items[0] & 1, &bars.dead);
            if (dead) return false;
            tc_fence_after();
            score(0, 0, ks);
            give(ks);
            if (n0 > 1) {
                ks = take();
                if (dead) return false;
                score(1, 1, ks);
                give(ks);
            }
            if (q_empty && n0 <= 2 && elect_one()) mma_commit(&q_empty[0]);
            for (int j = 0; j < n0; ++j) {
                const int i = j & 1;
                const unsigned par = (i ? f.steps[1] : f.steps[0]) & 1;
                vs = take();
                dead = dead || !warp_wait(&bars.p_half[i], par, &bars.dead);
                if (dead) return false;
                tc_fence_after();
                join(i, i, vs, j > 1, 0, 4);
                dead = dead || !warp_wait(&bars.p_full[i], par, &bars.dead);
                if (dead) return false;
                tc_fence_after();
                join(i, i, vs, true, 4, 8);
                if (i) ++f.steps[1]; else ++f.steps[0];
                if (j + 2 >= n0 && elect_one()) mma_commit(&bars.o_full[i]);
                give(vs);
                if (j + 2 < n0) {
                    ks = take();
                    if (dead) return false;
                    score(i, i, ks);
                    if (q_empty && j + 3 == n0 && elect_one()) mma_commit(&q_empty[0]);
                    give(ks);
                }
            }
            ++f.items[0];
            return true;
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            if ((i ? n1 : n0) == 0) continue;
            dead = dead || !warp_wait(&bars.q_full[i], f.items[i] & 1, &bars.dead);
            if (dead) return false;
            tc_fence_after();
            score(i, buffer(f.steps[i], i), ks);
            if (q_empty && (i ? n1 : n0) == 1 && elect_one()) mma_commit(&q_empty[i]);
        }
        give(ks);
        for (int j = 0; j < n_all; ++j) {
            const bool more = j + 1 < n_all;
            if (more) ks = take();
            if (dead) return false;
            if (NQ == 1 && more) {
                score(0, buffer(f.steps[0] + 1, 0), ks);
                if (q_empty && j + 2 == n_all && elect_one()) mma_commit(&q_empty[0]);
                give(ks);
            }
            vs = take();
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const int ni = i ? n1 : n0, buf = buffer(f.steps[i], i);
                if (j >= ni) continue;
                if (HALVES) {
                    dead = dead || !warp_wait(&bars.p_half[buf], parity(f.steps[i]), &bars.dead);
                    if (dead) return false;
                    tc_fence_after();
                    join(i, buf, vs, j > 0, 0, 4);
                }
                dead = dead || !warp_wait(&bars.p_full[buf], parity(f.steps[i]), &bars.dead);
                if (dead) return false;
                tc_fence_after();
                join(i, buf, vs, HALVES || j > 0, HALVES ? 4 : 0, 8);
                ++f.steps[i];
                if (NQ == 1 || j + 1 == ni) {
                    if (elect_one()) mma_commit(j + 1 == ni ? &bars.o_full[i] : &bars.o_part);
                }
                if (NQ == 2 && j + 1 < ni) {
                    score(i, i, ks);
                    if (q_empty && j + 2 == ni && elect_one()) mma_commit(&q_empty[i]);
                }
            }
            if (NQ == 2 && more) give(ks);
            give(vs);
        }
        if (n0 > 0) ++f.items[0];
        if (n1 > 0) ++f.items[1];
        return true;
    }

    // 64 scores of a row (columns 64 half ..) into weights: 16-bit pairs p (and lo, SPLIT), their sum added to `sum`.
    // Of every EMU pairs one takes the polynomial: the special-function unit gives 16 values a clock and SM, two query tiles
    // of 128-wide heads want 128 x 128 of them every 1,024 clocks, which is all of them (8,192 rows, 32 heads, EMU 0, 3, 4, 6:
    // 1,242, 1,272, 1,295 and 1,290 TFLOP/s), narrower heads more (64: 660, 731, 719 with 0, 3, 4); 256-wide heads half of
    // them, and the polynomial's instructions only cost (1,325, 1,249, 1,286 with 0, 3, 4).
    static constexpr int EMU = SPLIT || NQ == 1 ? 0 : D == 64 ? 3 : 4;
    static __device__ __forceinline__ void exps(const uint32_t (&x)[128], int half, f2 c2, f2 neg2, uint32_t (&p)[32],
                                                uint32_t (&lo)[SPLIT ? 32 : 1], f2 (&sum)[2]) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int at = half * 64 + 2 * e;
            f2 w = fma2(pk2(__uint_as_float(x[at]), __uint_as_float(x[at + 1])), c2, neg2);
            float a, b;
            if (EMU && e % (EMU + !EMU) == EMU - 1) {
                w = ex2_poly<std::is_same<T, __half>::value ? 4 : 3>(w);
                upk2(w, a, b);
            } else {
                upk2(w, a, b);
                a = ex2(a);
                b = ex2(b);
                w = pk2(a, b);
            }
            sum[e & 1] = add2(sum[e & 1], w);
            if constexpr (SPLIT) split16(a, b, &p[e], &lo[e]);
            else p[e] = pack16<T>(a, b);
        }
    }
    static __device__ __forceinline__ float row_max(const uint32_t (&x)[128]) {   // four chains of three-way maxima
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 128; e += 8)
#pragma unroll
            for (int t = 0; t < 4; ++t) top[t] = max3(top[t], __uint_as_float(x[e + 2 * t]), __uint_as_float(x[e + 2 * t + 1]));
        return fmaxf(max3(top[0], top[1], top[2]), top[3]);
    }

    // A softmax thread's part of one key tile: the row's scores, once they are there, masked (hide(x) sets what the row does not
    // see to -inf), turned into weights in tensor memory; c > 0 turns scores into powers of two; first / last: of the query
    // tile's key tiles. (f.steps[0] counts this role's steps whichever query tile it has.) False: given up.
    // (The first half's weights computed with the maximum so far, while the tile's own is still being found, and again in the
    // rare tile where it has grown by 2^8: 1,197 against 1,270 TFLOP/s for 8,192 rows, 32 heads of 128. The special-function
    // unit is what the two query tiles' warps share, and there is nothing to gain from being at it earlier.)
    template <typename Hide>
    static __device__ __forceinline__ bool softmax_step(TileBars& bars, int i, bool first, bool last, TileFlow& f, float c, float& m,
                                                        float& l, Hide hide) {
        const int buf = buffer(f.steps[0], i);
        if (!warp_wait(&bars.s_full[buf], parity(f.steps[0]), &bars.dead)) return false;
        tc_fence_after();
        const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
        const uint32_t s_addr = bars.tmem + buf * 128 + lanes, o_addr = bars.tmem + 256 + i * D + lanes;
        uint32_t x[128];
#pragma unroll
        for (int e = 0; e < 4; ++e) tmem_ld32(s_addr + e * 32, x + e * 32);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 4; ++e) tmem_pin(x + e * 32);
        hide(x);
        const float mx = row_max(x);
        if (first) m = mx;
        else if (__any_sync(0xffffffffu, (mx - m) * c > 8.0f)) {
            // O holds the tiles before this one. NQ = 2: their products were issued before this S, so they are done. NQ = 1:
            // the last of them comes behind this S.
            if (NQ == 1 && !warp_wait(&bars.o_part, (f.parts - 1) & 1, &bars.dead)) return false;
            tc_fence_after();
            const float mn = fmaxf(m, mx), k = mn == -INFINITY ? 1.0f : ex2((m - mn) * c);
            m = mn;
            l *= k;
            for (int e0 = 0; e0 < D; e0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + e0, o);
                tmem_ld_wait();
                tmem_pin(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * k);
                tmem_st32(o_addr + e0, o);
            }
        }
        const float neg = m == -INFINITY ? 0.0f : P_SHIFT_T - m * c;
        const f2 neg2 = pk2(neg, neg), c2 = pk2(c, c);
        f2 sum[2] = {pk2(0.0f, 0.0f), pk2(0.0f, 0.0f)};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t p[32], lo[SPLIT ? 32 : 1];
            exps(x, half, c2, neg2, p, lo, sum);
            tmem_st32(s_addr + half * 32, p);
            if constexpr (SPLIT) tmem_st32(s_addr + 64 + half * 32, lo);
            if (half == 1 || HALVES) {
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) mbar_arrive(half ? &bars.p_full[buf] : &bars.p_half[buf]);
            }
        }
        ++f.steps[0];
        if (!last) ++f.parts;
        float a, b;
        upk2(add2(sum[0], sum[1]), a, b);
        l += a + b;
        return true;
    }
};

}  // namespace b200

#endif  // B200_ATTN_TILES_CUH
