// attn_prompt.cuh -- causal attention over packed prompts (several sequences one after another in the rows), grouped
// heads, 16-bit rows:
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp(scale q[t, h] . k[j, h / G]),  j in t's sequence, j <= t
// Sequence b is rows [seq_start[b], seq_start[b + 1]); rows in no sequence are not written.

#ifndef B200_ATTN_PROMPT_CUH
#define B200_ATTN_PROMPT_CUH

#include "attn_rows.cuh"
#include "attn_tiles.cuh"

namespace b200 {

// Two query tiles per CTA, one for the 256-wide heads; K and V stages as large as shared memory allows beside them
template <int D, typename T>
using PromptTiles = Tiles<D, D == 256 ? 1 : 2, D < 128 ? D : 128, D == 64 ? 8 : 5, false, T>;
__host__ __device__ constexpr int prompt_rows(int D) { return D == 256 ? TILE_ROWS : 2 * TILE_ROWS; }   // query rows of a CTA

template <int D, typename T>
__global__ void __launch_bounds__(PromptTiles<D, T>::WARPS * 32, 1)
k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
              const T* q, const T* k, const T* v, T* out, const int* seq_start, int n_seqs, int rows, int n_q, int G,
              long long q_stride, long long k_stride, long long v_stride, float scale2, int n_slots) {
    using Ti = PromptTiles<D, T>;
    constexpr int NQ = D == 256 ? 1 : 2, SC = D < 128 ? D : 128, ROWS = prompt_rows(D);
    extern __shared__ unsigned char smem_raw[];
    __shared__ TileBars bars;
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* ring = smem + Ti::Q_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == NQ * 4 + 1 && lane == 0) {
        tma_prefetch(&mq);
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    Ti::setup(bars, 1);
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
            if (min(max(seq_start[mid], 0), rows) / ROWS + mid <= slot) lo = mid + 1; else hi = mid;
        }
        const int b = max(lo - 1, 0);
        first = min(max(seq_start[b], 0), rows);
        end = min(seq_start[b + 1], rows);
        tile = slot - (first / ROWS + b);
    }
    const int q0 = tile < 0 || tile > (end - first) / ROWS ? end : first + tile * ROWS;   // (no overflow on bad borders)
    if (q0 < end) {
    // key tiles per query tile: those up to its last row's own place
    int n[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int a = q0 + i * TILE_ROWS;
        n[i] = i < NQ && a < end ? (min(a + TILE_ROWS, end) - 1 - first) / TILE_ROWS + 1 : 0;
    }

    if (warp == NQ * 4 + 1) {
        Ti::few_registers();
        // ---- copies: Q, then K and V tiles in the order the tensor cores take them
        const int kh = h / G, n_all = max(n[0], n[1]);
        if (lane == 0) {
            mbar_expect(&bars.q_full, (n[1] ? 2 : 1) * Ti::QTILE);
            for (int i = 0; i < (n[1] ? 2 : 1); ++i)
                for (int c = 0; c < D / CHUNK; ++c)
                    tma_3d(smem + i * Ti::QTILE + c * CHUNK_BYTES, &mq, c * CHUNK, h, q0 + i * TILE_ROWS, &bars.q_full);
        }
        typename Ti::Ring r{bars, ring};
        const auto put = [&](const CUtensorMap* map, int j) {
            r.put([&](unsigned char* dst, int p, unsigned long long* bar) {
                if (lane < SC / CHUNK) tma_3d(dst + lane * CHUNK_BYTES, map, p * SC + lane * CHUNK, kh, first + j * TILE_ROWS, bar);
            });
        };
        put(&mk, 0);
        for (int j = 0; j < n_all; ++j) {
            if (j + 1 < n_all) put(&mk, j + 1);
            put(&mv, j);
        }
    } else if (warp == NQ * 4) {
        Ti::few_registers();
        if (lane == 0) Ti::products(bars, smem, ring, n);
    } else if (warp < NQ * 4) {
        Ti::many_registers();
        // ---- softmax: thread = row
        const int i = warp >> 2, r = threadIdx.x & 127, row = q0 + i * TILE_ROWS + r, tiles = i ? n[1] : n[0];
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < tiles; ++j) {
            uint32_t x[128];
            if (!Ti::scores(bars, i, j, x)) break;
            const int last = row - first - j * TILE_ROWS;   // the last key of this tile that the row sees
            if (j + 1 == tiles)   // (uniform) only a query tile's last key tile reaches past any of its rows
#pragma unroll
                for (int c = 0; c < 128; ++c)
                    if (c > last) x[c] = 0xff800000u;
            if (!Ti::weights(bars, i, j, x, scale2, m, l)) break;
        }
        if (tiles > 0 && wait_or_die(&bars.o_full[i], 0, &bars.dead)) {
            tc_fence_after();
            // O / l through the Q tile's shared memory (its last S is done), so that whole rows leave the warp together
            const uint32_t o_addr = bars.tmem + 256 + i * D + ((uint32_t)(threadIdx.x & 96) << 16);
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
        Ti::few_registers();
    }
    }
    Ti::teardown(bars);
}

}  // namespace b200

#endif  // B200_ATTN_PROMPT_CUH
