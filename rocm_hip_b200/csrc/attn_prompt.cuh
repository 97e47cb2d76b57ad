// attn_prompt.cuh -- causal attention over packed prompts (several sequences one after another in the rows), grouped
// heads, 16-bit rows:
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp(scale q[t, h] . k[j, h / G]),  j in t's sequence, j <= t
// Sequence b is rows [seq_start[b], seq_start[b + 1]); rows in no sequence are not written.

#ifndef B200_ATTN_PROMPT_CUH
#define B200_ATTN_PROMPT_CUH

#include "attn_rows.cuh"
#include "umma.cuh"

namespace b200 {

// CTAs that gave up on a wait since the library was loaded (b200_attn_gave_up): 0 unless the hardware or a caller's
// memory failed under a kernel
__device__ int attn_gave_up;

// ---------------------------------------------------------------- the tile kernel
//
// A CTA holds NQ query tiles of 128 rows of one head and walks the keys in tiles of 128:
//   S = Q K^T        tensor cores, 128 x 128 fp32 in tensor memory
//   P = 2^(S c - m)  a thread per row: registers, running maximum m and sum l; P goes back over S as 16-bit pairs
//   O += P V         tensor cores, A = P from tensor memory; O stays there until the last tile
// While one tile's rows are in the softmax the tensor cores work for the other tile (NQ = 2), or on the next S of the same
// tile (NQ = 1, for the 256-wide heads, whose O takes half of the 512 columns). O is rescaled only when a row's maximum
// has grown by more than 2^8 since it was last taken: P then stays below 2^8, which 16-bit floats and the fp32 sums bear,
// and almost no tile after the first pays for reading and writing O. Rounding P to 16 bits is what the tensor cores take;
// l sums the unrounded values.
template <int D>
struct PromptShape {
    static constexpr int NQ = D == 256 ? 1 : 2;
    static constexpr int SC = D < 128 ? D : 128;               // columns of a ring stage
    static constexpr int STAGE = TILE_ROWS * SC * 2;
    static constexpr int PARTS = D / SC;                       // stages per K or V tile
    static constexpr int Q_BYTES = NQ * TILE_ROWS * D * 2;
    static constexpr int STAGES = D == 64 ? 8 : 5;
    static constexpr int WARPS = NQ == 2 ? 12 : 6;             // softmax, tensor cores, copies (and two idle warps, see below)
    static constexpr int SMEM = 1024 + Q_BYTES + STAGES * STAGE;
    static constexpr int ROWS = NQ * TILE_ROWS;                // query rows of a CTA
};

struct PromptBars {
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

template <int D, typename T>
__global__ void __launch_bounds__(PromptShape<D>::WARPS * 32, 1)
k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
              const T* q, const T* k, const T* v, T* out, const int* seq_start, int n_seqs, int rows, int n_q, int G,
              long long q_stride, long long k_stride, long long v_stride, float scale2, int n_slots) {
    using Sh = PromptShape<D>;
    constexpr int NQ = Sh::NQ, SC = Sh::SC, PARTS = Sh::PARTS, ST = Sh::STAGES;
    extern __shared__ unsigned char smem_raw[];
    __shared__ PromptBars bars;
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* ring = smem + Sh::Q_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == NQ * 4) {
        tmem_alloc(&bars.tmem, 512);
        if (lane == 0) {
            mbar_init(&bars.q_full, 1);
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
    } else if (warp == NQ * 4 + 1 && lane == 0) {
        tma_prefetch(&mq);
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    pdl_entry();

    // which rows: slot s of the packed batch is tile s - f(b) of sequence b, f(b) = floor(start(b) / ROWS) + b, the last b with
    // f(b) <= s; f(b + 1) - f(b) is at least the number of tiles b has. Slots are taken from the last one down, so that in a
    // long sequence the tiles with the most keys start first.
    const int h = blockIdx.x % n_q, slot = n_slots - 1 - blockIdx.x / n_q;
    int first = 0, end = rows, tile = slot;
    if (seq_start) {
        int lo = 0, hi = n_seqs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (min(max(seq_start[mid], 0), rows) / Sh::ROWS + mid <= slot) lo = mid + 1; else hi = mid;
        }
        const int b = max(lo - 1, 0);
        first = min(max(seq_start[b], 0), rows);
        end = min(seq_start[b + 1], rows);
        tile = slot - (first / Sh::ROWS + b);
    }
    const int q0 = tile < 0 || tile > (end - first) / Sh::ROWS ? end : first + tile * Sh::ROWS;   // (no overflow on bad borders)
    if (q0 < end) {
    // key tiles per query tile: those up to its last row's own place
    int n[2];
    for (int i = 0; i < 2; ++i) {
        const int a = q0 + i * TILE_ROWS;
        n[i] = i < NQ && a < end ? (min(a + TILE_ROWS, end) - 1 - first) / TILE_ROWS + 1 : 0;
    }
    const int n_all = max(n[0], n[1]);
    // A softmax thread holds its row's 128 scores: 208 registers. Twelve warps start with 168 each (64,512 in all); the four
    // that compute nothing go down to 80 and the eight softmax warps up, 4 x 32 x 80 + 8 x 32 x 208 = 63,488. (Six warps
    // may have 255 from the start.)

    if (warp == NQ * 4 + 1) {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // ---- copies: Q, then K and V tiles in the order the tensor cores take them
        if (lane == 0) {
            const int kh = h / G;
            mbar_expect(&bars.q_full, (n[1] ? 2 : 1) * TILE_ROWS * D * 2);
            for (int i = 0; i < (n[1] ? 2 : 1); ++i)
                for (int c = 0; c < D / CHUNK; ++c)
                    tma_3d(smem + (i * (D / CHUNK) + c) * CHUNK_BYTES, &mq, c * CHUNK, h, q0 + i * TILE_ROWS, &bars.q_full);
            int st = 0, ph = 0;
            const auto put = [&](const CUtensorMap* map, int j) {
                for (int p = 0; p < PARTS; ++p) {
                    if (!wait_or_die(&bars.empty[st], ph ^ 1, &bars.dead)) return;
                    mbar_expect(&bars.full[st], Sh::STAGE);
                    for (int c = 0; c < SC / CHUNK; ++c)
                        tma_3d(ring + st * Sh::STAGE + c * CHUNK_BYTES, map, p * SC + c * CHUNK, kh, first + j * TILE_ROWS, &bars.full[st]);
                    if (++st == ST) { st = 0; ph ^= 1; }
                }
            };
            put(&mk, 0);
            for (int j = 0; j < n_all; ++j) {
                if (j + 1 < n_all) put(&mk, j + 1);
                put(&mv, j);
            }
        }
    } else if (warp == NQ * 4) {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // ---- tensor cores
        if (lane == 0) {
            const uint32_t id_s = idesc_f16<T>(TILE_ROWS, false), id_o = idesc_f16<T>(SC, true);
            int st = 0, ph = 0;          // the next stage to be taken from the ring
            const auto take = [&](int* stage) {   // the PARTS stages of a tile
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
                    const uint64_t a = desc_k_major(smem_u32(smem) + (i * (D / CHUNK) + c) * CHUNK_BYTES);
                    const uint64_t b = desc_k_major(smem_u32(ring) + stage[c / (SC / CHUNK)] * Sh::STAGE + c % (SC / CHUNK) * CHUNK_BYTES);
                    for (int e = 0; e < CHUNK / 16; ++e) mma_ss(tmem + buf * 128, a + e * 2, b + e * 2, id_s, c + e > 0);
                }
                mma_commit(&bars.s_full[buf]);
            };
            const auto join = [&](int i, int buf, const int* stage, bool add) {   // O_i += P[buf] V
                if (bars.dead) return;
                for (int p = 0; p < PARTS; ++p) {
                    const uint64_t b = desc_mn_major(smem_u32(ring) + stage[p] * Sh::STAGE);
                    for (int e = 0; e < TILE_ROWS / 16; ++e)
                        mma_ts(tmem + 256 + i * D + p * SC, tmem + buf * 128 + e * 8, b + e * (16 * 128 >> 4), id_o, add || e > 0);
                }
            };
            wait_or_die(&bars.q_full, 0, &bars.dead);
            int ks[2], vs[2];
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
    } else if (warp < NQ * 4) {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax: thread = row
        const int i = warp >> 2, r = threadIdx.x & 127, row = q0 + i * TILE_ROWS + r;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_addr = tmem + 256 + i * D + lanes;
        float m = -INFINITY, l = 0.0f;
        const f2 c2 = pk2(scale2, scale2);
        for (int j = 0; j < n[i]; ++j) {
            const int buf = NQ == 1 ? j & 1 : i;
            const uint32_t s_addr = tmem + buf * 128 + lanes;
            if (!wait_or_die(&bars.s_full[buf], NQ == 1 ? (j >> 1) & 1 : j & 1, &bars.dead)) break;
            tc_fence_after();
            uint32_t x[128];
            for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, x + c * 32);
            tmem_ld_wait();
            for (int c = 0; c < 4; ++c) tmem_pin(x + c * 32);
            const int last = row - first - j * TILE_ROWS;   // the last key of this tile that the row sees
            if (j + 1 == n[i])   // (uniform) only a query tile's last key tile reaches past any of its rows
#pragma unroll
                for (int c = 0; c < 128; ++c)
                    if (c > last) x[c] = 0xff800000u;
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 128; ++c) mx = fmaxf(mx, __uint_as_float(x[c]));
            if (j == 0) m = mx;
            else if (__any_sync(0xffffffffu, (mx - m) * scale2 > 8.0f)) {
                // O holds the tiles before this one. NQ = 2: their products were issued before this S, so they are done. NQ = 1:
                // the last of them comes behind this S.
                if (NQ == 1 && !wait_or_die(&bars.o_part, (j - 1) & 1, &bars.dead)) break;
                tc_fence_after();
                const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : ex2((m - mn) * scale2);
                m = mn;
                l *= f;
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + c, o);
                    tmem_ld_wait();
                    tmem_pin(o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st32(o_addr + c, o);
                }
            }
            const float neg = m == -INFINITY ? 0.0f : -m * scale2;
            const f2 neg2 = pk2(neg, neg);
            f2 sum = pk2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 128; c += 64) {
                uint32_t p[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float a, b;
                    upk2(fma2(pk2(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])), c2, neg2), a, b);
                    a = ex2(a);
                    b = ex2(b);
                    sum = add2(sum, pk2(a, b));
                    p[e] = pack16<T>(a, b);
                }
                tmem_st32(s_addr + c / 2, p);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[buf]);
            float a, b;
            upk2(sum, a, b);
            l += a + b;
        }
        if (n[i] > 0 && wait_or_die(&bars.o_full[i], 0, &bars.dead)) {
            tc_fence_after();
            // O / l through the Q tile's shared memory (its last S is done), so that whole rows leave the warp together
            unsigned char* mine = smem + (i * TILE_ROWS + (warp & 3) * 32) * (D * 2);
            const float inv = 1.0f / l;
            bool bad = false;
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + c, o);
                tmem_ld_wait();
                tmem_pin(o);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    float f[8];
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        f[t] = __uint_as_float(o[e + t]) * inv;
                        bad |= !(fabsf(f[t]) < INFINITY);
                    }
                    const int u = (c + e) / 8;
                    *reinterpret_cast<uint4*>(mine + lane * (D * 2) + ((u ^ (lane & 7)) * 16)) = Io<T>::pack(f);
                }
            }
            __syncwarp();
            constexpr int UNITS = D / 8;
            for (int e = lane; e < 32 * UNITS; e += 32) {
                const int rr = e / UNITS, u = e % UNITS, t = q0 + i * TILE_ROWS + (warp & 3) * 32 + rr;
                if (t < end)
                    st_stream(reinterpret_cast<unsigned char*>(out + ((long long)t * n_q + h) * D) + u * 16,
                              *reinterpret_cast<const uint4*>(mine + rr * (D * 2) + ((u ^ (rr & 7)) * 16)));
            }
            // A weight of 0 times a non-finite v is not 0 on the tensor cores: rows that came out non-finite are computed again
            // from the keys they may see alone
            unsigned again = __ballot_sync(0xffffffffu, bad && row < end);
            __syncwarp();
            while (again) {
                const int rr = __ffs(again) - 1, t = q0 + i * TILE_ROWS + (warp & 3) * 32 + rr;
                again &= again - 1;
                attn_row_prompt<D, T>(q + t * q_stride + h * D, k + first * k_stride + h / G * D, v + first * v_stride + h / G * D,
                                      k_stride, v_stride, t - first + 1, scale2, out + ((long long)t * n_q + h) * D);
            }
        }
    } else {
        if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == NQ * 4) tmem_free(tmem, 512);
    if (threadIdx.x == 0 && bars.dead) atomicAdd(&attn_gave_up, 1);
}

}  // namespace b200

#endif  // B200_ATTN_PROMPT_CUH
