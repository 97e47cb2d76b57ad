// attn_own.cuh -- the part of single-token attention that no other sequence shares: each sequence's own cache rows, read
// once, a warp per key head and stretch of rows. Bound by the cache's bytes (2 D 2 per row and key head); the arithmetic
// is two small products per 16 rows, which mma.sync does in passing:
//   S^T [16 rows x 8 heads] = K Q^T          A = K as it lies in the cache, B = the group's queries, in registers
//   O^T [D x 8 heads]      += V^T P^T        A = V transposed by ldmatrix, B = P by movmatrix
// Query heads are the narrow side, so a group of up to 8 heads wastes nothing of the wide one (16 query rows as the wide
// side took twice the products and registers).
//
// Queries meet an FP16 cache, so they become fp16 too, without losing anything that counts: a row is scaled by the power
// of two that takes its largest value to [2^9, 2^10), and fp32 rows are split into q = hi + lo, two fp16 values with 22
// bits together; weights likewise (P = hi + lo, scaled by 2^P_SHIFT), for bf16 rows hi alone, whose 2^-12 is far below
// the rounding of the result.
//
// Work is dealt out evenly whatever the lengths are: all sequences' row tiles, one after another, are cut into equal
// shares, one per CTA, so that one long sequence is spread over the device and many short ones share a CTA. Each piece
// of a sequence leaves (m, l, o) in scratch, and k_attn_join puts the pieces together.

#ifndef B200_ATTN_OWN_CUH
#define B200_ATTN_OWN_CUH

#include <limits.h>

#include "attn_decode.cuh"
#include "attn_tiles.cuh"

namespace b200 {

constexpr int P_SHIFT = 7;        // weights are held as 2^(s - m + 7): at most 2^15 (m may lag by 2^8), fp16's lower end far away
// A CTA's share is two tiles at least: fewer pieces to join (five sequences of up to 700 rows, 8 key heads of 128, shares of at
// least 2, 3, 4 and 6 tiles: 13.2, 13.3, 13.9 and 15.7 us)
constexpr int OWN_LEAST = 2;
constexpr float P_LAG = 8.0f;     // how far a score may exceed m before everything is rescaled

template <int D>
struct OwnShape {
    static constexpr int WARPS = D == 256 ? 4 : 8;
    static constexpr int STAGES = D == 64 ? 6 : 3;
    static constexpr int STAGE = 2 * 16 * D * 2;                       // 16 rows of K, then 16 of V
    static constexpr int SMEM = 1024 + WARPS * STAGES * STAGE;         // 193 KB
};

// How query heads and rows are spread over a CTA's warps: `units` (key head, up to 8 of its query heads) take a warp each;
// where that leaves warps over, R row groups of 16 run side by side.
struct OwnPlan {
    int gt, units, groups, wh, R, hg;     // tiles of 8 query heads per key head; units; CTA-sized groups of them; units per CTA
    OwnPlan(int n_q, int n_kv, int warps) {
        const int G = n_q / n_kv;
        gt = (G + 7) / 8;
        hg = G < 8 ? G : 8;               // query heads a unit writes at most
        units = n_kv * gt;
        groups = (units + warps - 1) / warps;
        wh = (units + groups - 1) / groups;
        R = warps / wh;
    }
};

// Where the pieces lie in scratch. Slot = CTA + sequence * groups + group: both ascend along the work, so no two pieces
// share one; a slot holds `warps` pieces of hg heads.
struct OwnScratch {
    int* head;        // [0] tiles per CTA
    int* first;       // [B + 1] tiles before sequence b (of one group)
    int* shares;      // [B] whether sequence b begins with the batch's prefix (k_attn_shares); null: nothing is shared
    float* ml;        // [slot][warp][hg][2]
    float* o;         // [slot][warp][hg][D]
};

// A tile of 16 rows in shared memory: chunks of 64 values, [16 rows][128 bytes], 16-byte units swizzled as the copy engine
// does (unit ^ row mod 8), so that ldmatrix meets no bank twice
__device__ __forceinline__ uint32_t own_at(int row, int unit) { return unit / 8 * 2048 + row * 128 + ((unit & 7) ^ (row & 7)) * 16; }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ uint32_t mov_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes, or 16 zeros where `n` is 0
__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// The exponent e that takes a row's largest magnitude `top` to [2^9, 2^10) as top * 2^e (0 for a row of zeros or a
// non-finite one)
__device__ __forceinline__ int q_exponent(float top) {
    const int x = (__float_as_int(top) >> 23) & 255;
    return top > 0.0f && x < 255 ? 9 + 127 - (x ? x : 1) : 0;
}
// Rows of its own that sequence b has, and where they begin: behind the shared prefix if it has that
__device__ __forceinline__ int own_rows(const PagedKv& kv, const OwnScratch& sc, int b, int prefix, int* start) {
    *start = sc.shares && sc.shares[b] ? prefix : 0;
    return kv.len(b) - *start;
}

// QT: type of the queries (fp32: two fp16 values per query value and weight). BOX: tiles come by the copy engine, in boxes
// of 8 or 16 rows of a page, at four instructions a tile; a thread's own 16-byte copies, the other way, cost a third of
// all instructions (64 sequences of 1 .. 2,048 rows, 8 heads of 128: 62 us) and serve pages of fewer rows and caches that a
// tensor map cannot describe.
template <int D, typename QT, bool BOX>
__global__ void __launch_bounds__(OwnShape<D>::WARPS * 32, 1)
k_attn_own(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const QT* q, PagedKv kv, OwnScratch sc,
           OwnPlan pl, int n_q, int G, int B, int prefix, float scale2) {
    using Sh = OwnShape<D>;
    constexpr bool SPLIT = sizeof(QT) == 4;
    constexpr int W = Sh::WARPS, ST = Sh::STAGES, KS = D / 16, UNITS = D / 8, NT = W * 32;
    extern __shared__ unsigned char smem_raw[];
    __shared__ int part[NT / 32 + 1], at[4];
    __shared__ unsigned long long full[W][ST];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (BOX && lane == 0) {
        for (int i = 0; i < ST; ++i) mbar_init(&full[warp][i], 1);
        mbar_fence_init();
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    pdl_entry();
    const int tile = 16 * pl.R;

    // ---- the shares: every CTA sums the tiles of all sequences, then finds where its own share begins
    const auto tiles_of = [&](int b) {
        int s;
        return b < B ? (own_rows(kv, sc, b, prefix, &s) + tile - 1) / tile : 0;
    };
    const auto cta_scan = [&](int v, int* total) {
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) part[warp] = x;
        __syncthreads();
        int base = 0, all = 0;
        for (int i = 0; i < W; ++i) {
            base += i < warp ? part[i] : 0;
            all += part[i];
        }
        *total = all;
        return base + x - v;
    };
    int total = 0, n_mine = 0, before_mine = 0;      // (of the last round: the only one while B <= NT)
    for (int b0 = 0; b0 < B; b0 += NT) {
        int t;
        n_mine = tiles_of(b0 + tid);
        before_mine = total + cta_scan(n_mine, &t);
        if (blockIdx.x == 0 && b0 + tid < B) sc.first[b0 + tid] = before_mine;
        total += t;
    }
    if (blockIdx.x == 0 && tid == 0) sc.first[B] = total;
    const long long all = (long long)total * pl.groups;
    const long long per = max((all + gridDim.x - 1) / gridDim.x, (long long)OWN_LEAST);
    if (blockIdx.x == 0 && tid == 0) *reinterpret_cast<long long*>(sc.head) = per;
    long long t0 = blockIdx.x * per;
    const long long t_end = min(t0 + per, all);
    if (t0 >= t_end) return;
    if (tid == 0) at[0] = B;
    __syncthreads();
    const auto look = [&](int b, int n, int before) {
        if (n > 0 && t0 >= (long long)before * pl.groups && t0 < (long long)(before + n) * pl.groups) {
            at[0] = b;
            at[1] = (int)(t0 - (long long)before * pl.groups);
        }
    };
    if (B <= NT) look(tid, n_mine, before_mine);
    else {
        int done = 0;
        for (int b0 = 0; b0 < B; b0 += NT) {
            int t;
            const int n = tiles_of(b0 + tid), before = done + cta_scan(n, &t);
            look(b0 + tid, n, before);
            done += t;
        }
    }
    __syncthreads();
    int b = at[0], in_seq = at[1];          // the share begins with tile in_seq (counted over the groups) of sequence b
    if (warp >= pl.wh * pl.R) return;       // (no barrier of the whole CTA from here on)

    unsigned char* ring = smem + warp * ST * Sh::STAGE;
    unsigned phases = 0;                    // bit s: the parity stage s completes next
    const int wu = warp % pl.wh, rg = warp / pl.wh;
    const int g8 = lane >> 2, t4 = lane & 3;
    for (; t0 < t_end && b < B; ++b, in_seq = 0) {
        int start;
        const int own = own_rows(kv, sc, b, prefix, &start), n_tiles = (own + tile - 1) / tile;
        while (in_seq < n_tiles * pl.groups && t0 < t_end) {
            // ---- one piece: tiles [k0, k1) of group `grp` of sequence b
            const int grp = in_seq / n_tiles, k0 = in_seq - grp * n_tiles;
            const int k1 = (int)min((long long)n_tiles, k0 + (t_end - t0));
            in_seq += k1 - k0;
            t0 += k1 - k0;
            const int u = grp * pl.wh + wu;
            if (u >= pl.units) continue;
            const int kh = u / pl.gt, h0 = u % pl.gt * 8, heads = min(8, G - h0);

            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, o[KS][4];
#pragma unroll
            for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

            // Where tile k begins. BOX: lane 0 issues the copies, so every lane holds the same first page; the second one of
            // a tile over two 8-row pages is its neighbour in the list. Else lane r holds where row r lies. -1: not there.
            const auto where = [&](int k) -> long long {
                const int r = k * tile + rg * 16 + (BOX ? 0 : lane & 15);
                if (k >= k1 || r >= own) return -1;
                if constexpr (!BOX) return kv.row(b, start + r);
                const int* list = kv.pages + (long long)b * kv.max_pages + ((start + r) >> kv.kv_shift);
                const auto valid = [&](int p) { return (unsigned)p < (unsigned)kv.n_pages ? p : -1; };
                const int p0 = valid(list[0]), p1 = kv.kv_shift == 3 && r + 8 < own ? valid(list[1]) : -1;
                return ((long long)p1 << 32) | (unsigned)p0;
            };
            unsigned seen[ST];       // which rows of a stage hold a row of the sequence (indexed by unrolled stages only)
            const auto fetch = [&](int s, int k, long long at) -> unsigned {
                if constexpr (BOX) {
                    const int p0 = (int)at, p1 = (int)(at >> 32), r = k * tile + rg * 16, t = start + r;
                    if (lane == 0) {
                        fence_async_smem();      // the rows that a tail blanked in this stage
                        unsigned char* dst = ring + s * Sh::STAGE;
                        mbar_expect(&full[warp][s], Sh::STAGE);
                        const int in_page = t & ((1 << kv.kv_shift) - 1);
#pragma unroll
                        for (int c = 0; c < D / CHUNK; ++c) {
                            tma_4d(dst + c * 2048, &mk, c * CHUNK, kh, in_page, p0, &full[warp][s]);
                            tma_4d(dst + 16 * D * 2 + c * 2048, &mv, c * CHUNK, kh, in_page, p0, &full[warp][s]);
                            if (kv.kv_shift == 3) {
                                tma_4d(dst + c * 2048 + 1024, &mk, c * CHUNK, kh, 0, p1, &full[warp][s]);
                                tma_4d(dst + 16 * D * 2 + c * 2048 + 1024, &mv, c * CHUNK, kh, 0, p1, &full[warp][s]);
                            }
                        }
                    }
                    const unsigned rows = own - r >= 16 ? 0xffffu : own - r > 0 ? (1u << (own - r)) - 1 : 0;
                    const unsigned pages = kv.kv_shift == 3 ? (p0 >= 0 ? 0xffu : 0) | (p1 >= 0 ? 0xff00u : 0) : p0 >= 0 ? 0xffffu : 0;
                    return rows & pages;
                } else {
                    const uint32_t dst = smem_u32(ring + s * Sh::STAGE);
#pragma unroll
                    for (int i = 0; i < UNITS / 2; ++i) {
                        const int x = i * 32 + lane, r = x / UNITS, unit = x % UNITS;
                        const long long off = __shfl_sync(0xffffffffu, at, r);
                        const long long src = (off < 0 ? 0 : off) + kh * D + unit * 8;
                        const uint32_t d = dst + own_at(r, unit);
                        cp_async16z(d, kv.K + src, off < 0 ? 0 : 16);
                        cp_async16z(d + 16 * D * 2, kv.V + src, off < 0 ? 0 : 16);
                    }
                    return __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
                }
            };
            __syncwarp();            // the stages of the piece before have been read
            long long next = where(k0);
#pragma unroll
            for (int s = 0; s < ST - 1; ++s) {
                const long long at = next;
                next = where(k0 + s + 1);
                seen[s] = 0;
                if (k0 + s < k1) seen[s] = fetch(s, k0 + s, at);
                if (!BOX) cp_async_commit();
            }
            // queries: lane (g8, t4) holds values 16 k + 2 t4 + {0, 1, 8, 9} of head h0 + g8
            uint32_t qh[KS][2], ql[SPLIT ? KS : 1][2];
            const QT* qrow = q + ((long long)b * n_q + kh * G + h0 + g8) * D + t4 * 2;
            float top = 0.0f;
            if (g8 < heads)
                for (int i = 0; i < KS * 2; ++i) {
                    float v[2];
                    load_vals(qrow + i * 8, v);
                    top = fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1])));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = q_exponent(top);
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float v[2] = {0.0f, 0.0f};
                    if (g8 < heads) load_vals(qrow + i * 16 + p * 8, v);
                    v[0] = scale2e(v[0], e);
                    v[1] = scale2e(v[1], e);
                    uint32_t lo;
                    split16(v[0], v[1], &qh[i][p], &lo);
                    if constexpr (SPLIT) ql[i][p] = lo;
                }
            // score = S c in powers of two; this lane's columns of S^T are heads 2 t4 and 2 t4 + 1
            const float c_own = scale2e(scale2, -e);
            const float c0 = __shfl_sync(0xffffffffu, c_own, t4 * 8), c1 = __shfl_sync(0xffffffffu, c_own, t4 * 8 + 4);

            for (int k = k0; k < k1; k += ST) {
#pragma unroll
                for (int s = 0; s < ST; ++s) {       // stages by constant index
                    if (k + s < k1) {                // (uniform)
                        const int f = (s + ST - 1) % ST;
                        const long long at = next;
                        next = where(k + s + ST);
                        seen[f] = 0;
                        if (k + s + ST - 1 < k1) seen[f] = fetch(f, k + s + ST - 1, at);
                        unsigned char* Kt = ring + s * Sh::STAGE;
                        unsigned char* Vt = Kt + 16 * D * 2;
                        if constexpr (BOX) {
                            if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][s], phases >> s & 1))) goto gave_up;
                            phases ^= 1u << s;
                            if (seen[s] != 0xffffu) {   // a weight of 0 needs a finite v: what lies behind the sequence is blanked
                                for (int e = lane; e < 16 * UNITS; e += 32)
                                    if (!(seen[s] >> (e / UNITS) & 1)) *reinterpret_cast<uint4*>(Vt + own_at(e / UNITS, e % UNITS)) = make_uint4(0, 0, 0, 0);
                            }
                        } else {
                            cp_async_commit();
                            cp_async_wait<ST - 1>();
                        }
                        __syncwarp();
                        // two chains of products, so that one's latency hides the other's
                        float st[4] = {0.0f, 0.0f, 0.0f, 0.0f}, su[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sl[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < KS; i += 2) {
                            uint32_t a[4], c[4];
                            ldsm4(smem_u32(Kt) + own_at((lane & 7) + (lane >> 3 & 1) * 8, i * 2 + (lane >> 4)), a);
                            ldsm4(smem_u32(Kt) + own_at((lane & 7) + (lane >> 3 & 1) * 8, i * 2 + 2 + (lane >> 4)), c);
                            if constexpr (SPLIT) {
                                mma16(sl, a, ql[i][0], ql[i][1]);
                                mma16(sl, c, ql[i + 1][0], ql[i + 1][1]);
                            }
                            mma16(st, a, qh[i][0], qh[i][1]);
                            mma16(su, c, qh[i + 1][0], qh[i + 1][1]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) st[i] = (sl[i] + su[i]) + st[i];
                        const bool s0 = seen[s] >> g8 & 1, s1 = seen[s] >> (g8 + 8) & 1;
                        const float x0 = s0 ? st[0] * c0 : -INFINITY, x1 = s0 ? st[1] * c1 : -INFINITY;
                        const float x2 = s1 ? st[2] * c0 : -INFINITY, x3 = s1 ? st[3] * c1 : -INFINITY;
                        if (__any_sync(0xffffffffu, fmaxf(x0, x2) > m0 + P_LAG || fmaxf(x1, x3) > m1 + P_LAG)) {
                            float n0 = fmaxf(m0, fmaxf(x0, x2)), n1 = fmaxf(m1, fmaxf(x1, x3));
#pragma unroll
                            for (int off = 4; off < 32; off <<= 1) {
                                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, off));
                                n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, off));
                            }
                            const float f0 = n0 == -INFINITY ? 1.0f : ex2(m0 - n0), f1 = n1 == -INFINITY ? 1.0f : ex2(m1 - n1);
                            m0 = n0;
                            m1 = n1;
                            l0 *= f0;
                            l1 *= f1;
#pragma unroll
                            for (int i = 0; i < KS; ++i) {
                                o[i][0] *= f0;
                                o[i][1] *= f1;
                                o[i][2] *= f0;
                                o[i][3] *= f1;
                            }
                        }
                        const float e0 = m0 == -INFINITY ? 0.0f : P_SHIFT - m0, e1 = m1 == -INFINITY ? 0.0f : P_SHIFT - m1;
                        const float p0 = ex2(x0 + e0), p1 = ex2(x1 + e1), p2 = ex2(x2 + e0), p3 = ex2(x3 + e1);
                        l0 += p0 + p2;
                        l1 += p1 + p3;
                        uint32_t h01, h23, w01, w23;
                        split16(p0, p1, &h01, &w01);
                        split16(p2, p3, &h23, &w23);
                        const uint32_t b0 = mov_trans(h01), b1 = mov_trans(h23);
                        uint32_t d0 = 0, d1 = 0;
                        if constexpr (SPLIT) {
                            d0 = mov_trans(w01);
                            d1 = mov_trans(w23);
                        }
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            uint32_t a[4];
                            ldsm4t(smem_u32(Vt) + own_at((lane & 7) + (lane >> 4) * 8, i * 2 + (lane >> 3 & 1)), a);
                            if constexpr (SPLIT) {
                                // (the tensor cores cut a sum off where fp32 arithmetic rounds: over thousands of rows the sums
                                // shrink, 2.0e-6 after 4,000 against 5.9e-7. So only a tile's own products are summed there.)
                                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma16(y, a, d0, d1);
                                mma16(y, a, b0, b1);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[i][e] += y[e];
                            } else {
                                mma16(o[i], a, b0, b1);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, off);
                l1 += __shfl_xor_sync(0xffffffffu, l1, off);
            }
            const long long piece = ((long long)(blockIdx.x + (long long)b * pl.groups + grp) * W + warp) * pl.hg;
            if (g8 == 0) {
                if (2 * t4 < heads) { sc.ml[(piece + 2 * t4) * 2] = m0; sc.ml[(piece + 2 * t4) * 2 + 1] = l0; }
                if (2 * t4 + 1 < heads) { sc.ml[(piece + 2 * t4 + 1) * 2] = m1; sc.ml[(piece + 2 * t4 + 1) * 2 + 1] = l1; }
            }
            float* po = sc.o + piece * D;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const int d = i * 16 + g8;
                if (2 * t4 < heads) { po[2 * t4 * D + d] = o[i][0]; po[2 * t4 * D + d + 8] = o[i][2]; }
                if (2 * t4 + 1 < heads) { po[(2 * t4 + 1) * D + d] = o[i][1]; po[(2 * t4 + 1) * D + d + 8] = o[i][3]; }
            }
        }
    }
    if (!BOX) cp_async_wait_all();
    return;
gave_up:                                    // no copy may still be under way when the CTA ends and its memory becomes another's
    for (int i = 0; i < ST; ++i) (void)mbar_wait(&full[warp][i], phases >> i & 1);
    if (lane == 0) atomicAdd(&attn_gave_up, 1);
}

// The pieces the prefix kernel leaves: [split][key head][row b G + g]
struct PrefixScratch {
    int splits;       // 0: there is none
    long long rows;   // B G rounded up to whole tiles
    float* ml;        // [split][n_kv][rows][2]
    float* o;         // [split][n_kv][rows][D]
};

// out[b, h] = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the pieces i of the row, in the order of the rows they
// cover; a row without pieces, or with none that saw a key, is zero. A warp per row.
template <int D, typename QT>
__global__ void __launch_bounds__(128)
k_attn_join(OwnScratch sc, OwnPlan pl, PrefixScratch px, QT* out, int n_q, int n_kv, int B) {
    pdl_entry();
    constexpr int N = D / 32, W = OwnShape<D>::WARPS;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;     // (B n_q <= 2^28)
    if (row >= B * n_q) return;
    const int b = row / n_q, h = row - b * n_q, G = n_q / n_kv, kh = h / G, g = h - kh * G;
    const int u = kh * pl.gt + g / 8, grp = u / pl.wh, wu = u - grp * pl.wh;
    // (volatile loads, all four together: 13.1 us for five sequences of up to 700 rows, 13.3 as plain ones)
    const int before = *(const volatile int*)(sc.first + b), n_tiles = *(const volatile int*)(sc.first + b + 1) - before;
    const long long per = *(const volatile long long*)sc.head;
    const int n_px = px.splits && *(const volatile int*)(sc.shares + b) ? px.splits : 0;
    const long long t0 = (long long)before * pl.groups + (long long)grp * n_tiles, t1 = t0 + n_tiles - 1;
    int c0 = 0, n_own = 0;
    if (n_tiles > 0) {
        int c1;
        if (t1 < INT_MAX) {      // (a 64-bit division is a hundred instructions)
            c0 = (int)t0 / (int)per;
            c1 = (int)t1 / (int)per;
        } else {
            c0 = (int)(t0 / per);
            c1 = (int)(t1 / per);
        }
        n_own = (c1 - c0 + 1) * pl.R;
    }
    const int n = n_px + n_own;
    // piece i of the row -> its (m, l) and o
    const auto piece = [&](int i, const float** o) -> const float* {
        if (i < n_px) {
            const long long at = ((long long)i * n_kv + kh) * px.rows + (long long)b * G + g;
            *o = px.o + at * D;
            return px.ml + at * 2;
        }
        i -= n_px;
        const int k = pl.R == 1 ? i : i / pl.R;
        const long long slot = c0 + k + (long long)b * pl.groups + grp;
        const long long at = (slot * W + wu + (i - k * pl.R) * pl.wh) * pl.hg + g % 8;
        *o = sc.o + at * D;
        return sc.ml + at * 2;
    };
    // lane i takes piece i of every 32: its m, l and where its o lies
    float M = -INFINITY, l = 0.0f, acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const float* mine = nullptr;
        float mi = -INFINITY, li = 0.0f;
        if (i0 + lane < n) {
            const float* ml = piece(i0 + lane, &mine);
            mi = ml[0];
            li = ml[1];
        }
        float top = fmaxf(M, mi);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float old = M == -INFINITY ? 0.0f : ex2(M - top), f = mi == -INFINITY ? 0.0f : ex2(mi - top);
        float sum = f * li;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l = l * old + sum;
        M = top;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] *= old;
        const int count = min(32, n - i0);
        constexpr int F = N == 8 ? 8 : 16;       // rows in flight
        for (int i = 0; i < count; i += F) {
            float v[F][N];
#pragma unroll
            for (int t = 0; t < F; ++t) {
                const float* o = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)mine, i + t));
                if (i + t < count) load_vals(o + lane * N, v[t]);
            }
#pragma unroll
            for (int t = 0; t < F; ++t) {
                const float ft = __shfl_sync(0xffffffffu, f, i + t);
                if (i + t < count)
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[e] += ft * v[t][e];
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= inv;
    store_vals(out + (long long)row * D + lane * N, acc);
}

}  // namespace b200

#endif  // B200_ATTN_OWN_CUH
