// attn_prefix.cuh -- the part of single-token attention that the whole batch shares: the prefix's rows, read once. The
// queries of all sequences that read one key head are the rows of a product, B G of them, and the kernel is the tile
// kernel of the prompts without its mask: CTA = (key head, 128 or 256 query rows, a stretch of the prefix), K and V tiles
// by TMA straight out of the cache's pages. Each CTA leaves (m, l, o) of its stretch for k_attn_join.
//
// Queries become fp16 as in attn_own.cuh: scaled by a power of two per row, fp32 ones as hi + lo.

#ifndef B200_ATTN_PREFIX_CUH
#define B200_ATTN_PREFIX_CUH

#include "attn_own.cuh"
#include "attn_tiles.cuh"

namespace b200 {

// The first sequence that is as long as the prefix, whose pages the prefix is read from; -1: none is. A warp.
__device__ __forceinline__ int prefix_owner(const PagedKv& kv, int B, int prefix) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const unsigned has = __ballot_sync(0xffffffffu, b0 + lane < B && kv.len(b0 + lane) >= prefix);
        if (has) return b0 + __ffs(has) - 1;
    }
    return -1;
}

// Which sequences share the prefix: those whose list begins with the pages of the first one that is long enough. One that has
// pages of its own in their place (it was cut back below the prefix and grew again, or comes from another prompt) reads
// all its rows itself. A CTA per sequence; bound by two memory latencies, so the sequence's own entries are on their way while
// the first one is looked for, and the next kernel while this one runs (64 sequences, 1,024 pages each: 71.6 -> 73.2 us for
// the call).
constexpr int SHARES_THREADS = 256;
__global__ void __launch_bounds__(SHARES_THREADS)
k_attn_shares(PagedKv kv, int* shares, int B, int prefix) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // (k_attn_own waits before it reads or writes anything)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b = blockIdx.x, n = prefix >> kv.kv_shift;
    const int* mine = kv.pages + (long long)b * kv.max_pages;
    constexpr int AHEAD = 4;
    int m[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) m[i] = threadIdx.x + i * SHARES_THREADS < n ? mine[threadIdx.x + i * SHARES_THREADS] : 0;
    const int owner = prefix_owner(kv, B, prefix);
    int same = owner >= 0 && kv.len(b) >= prefix;
    if (same && owner != b) {      // (uniform)
        const int* theirs = kv.pages + (long long)owner * kv.max_pages;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (threadIdx.x + i * SHARES_THREADS < n) same &= m[i] == theirs[threadIdx.x + i * SHARES_THREADS];
#pragma unroll 4
        for (int i = threadIdx.x + AHEAD * SHARES_THREADS; i < n; i += SHARES_THREADS) same &= mine[i] == theirs[i];
    }
    same = __syncthreads_and(same);
    if (threadIdx.x == 0) shares[b] = same;
}

template <int D, int NQ, bool SPLIT>
struct PrefixShape {
    // fp32 queries of 256-wide heads take 128 KB: stages of 64 columns, so that six of them fit beside
    static constexpr int SC = D == 64 || (D == 256 && SPLIT) ? 64 : 128;
    static constexpr int Q_BYTES = NQ * TILE_ROWS * D * 2 * (SPLIT ? 2 : 1);
    static constexpr int FIT = (230400 - 1024 - Q_BYTES) / (TILE_ROWS * SC * 2);
    static constexpr int ST = FIT < 8 ? FIT : 8;
    using Ti = Tiles<D, NQ, SC, ST, SPLIT, __half>;
};

template <int D, int NQ, typename QT>
__global__ void __launch_bounds__(PrefixShape<D, NQ, sizeof(QT) == 4>::Ti::WARPS * 32, 1)
k_attn_prefix(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const QT* q, PagedKv kv, PrefixScratch px,
              int n_q, int n_kv, int B, int prefix, float scale2, int row_tiles) {
    constexpr bool SPLIT = sizeof(QT) == 4;
    using Ti = typename PrefixShape<D, NQ, SPLIT>::Ti;
    constexpr int SC = PrefixShape<D, NQ, SPLIT>::SC;
    extern __shared__ unsigned char smem_raw[];
    __shared__ TileBars bars;
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* ring = smem + Ti::Q_BYTES;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, G = n_q / n_kv;
    if (warp == NQ * 4 + 1 && lane == 0) {
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    Ti::setup(bars, 4);
    // No wait for the kernel before this one (k_attn_own) here: it goes on only after its own predecessors are done, it writes
    // nothing that is read here, and this kernel starts only once all of its CTAs have gone on. The wait at the end makes
    // this kernel's completion stand for both.

    const int kh = blockIdx.x % n_kv, rt = blockIdx.x / n_kv % row_tiles, split = blockIdx.x / n_kv / row_tiles;
    const int tiles = (prefix + TILE_ROWS - 1) / TILE_ROWS;
    const int j0 = (int)((long long)tiles * split / px.splits), j1 = (int)((long long)tiles * (split + 1) / px.splits);
    const int M = B * G, r0 = rt * NQ * TILE_ROWS;
    const int owner = prefix_owner(kv, B, prefix);
    const int* pages = kv.pages + (long long)owner * kv.max_pages;
    if (owner >= 0) {   // else nobody reads what this kernel would write
    int n[2] = {j1 - j0, NQ == 2 && r0 + TILE_ROWS < M ? j1 - j0 : 0};
    const int n_all = n[0];

    if (warp == NQ * 4 + 1) {
        Ti::few_registers();
        // A tile is 128 / box boxes, lane a issues box a (box: the rows of a page, at most 128). The pages of a tile are looked
        // up two tiles ahead: one lane walking the list in line with its copies waited a memory latency per box (pages of 16
        // rows: 6 us a tile). Rows behind the prefix and pages outside the cache: page -1, which the copy fills with zeros.
        const int in_page = 1 << kv.kv_shift, box = min(in_page, TILE_ROWS), boxes = TILE_ROWS / box;
        const auto page_of = [&](int j) {
            const int t = (j0 + j) * TILE_ROWS + lane * box;
            if (lane >= boxes || j >= n_all || t >= prefix) return -1;
            const int p = pages[t >> kv.kv_shift];
            return (unsigned)p < (unsigned)kv.n_pages ? p : -1;
        };
        typename Ti::Ring r{bars, ring};
        const auto put = [&](const CUtensorMap* map, int j, int page) {
            const int row = ((j0 + j) * TILE_ROWS + lane * box) & (in_page - 1);
            r.put([&](unsigned char* dst, int p, unsigned long long* bar) {
                if (lane < boxes)
                    for (int c = 0; c < SC / CHUNK; ++c)
                        tma_4d(dst + c * CHUNK_BYTES + lane * box * 128, map, p * SC + c * CHUNK, kh, row, page, bar);
            });
        };
        int p0 = page_of(0), p1 = page_of(1), p2 = page_of(2);
        put(&mk, 0, p0);
        for (int j = 0; j < n_all; ++j) {
            const int p3 = page_of(j + 3);
            if (j + 1 < n_all) put(&mk, j + 1, p1);
            put(&mv, j, p0);
            p0 = p1;
            p1 = p2;
            p2 = p3;
        }
        Ti::copies_done(bars, r, nullptr, {0, 0});
    } else if (warp == NQ * 4) {
        Ti::few_registers();
        TileFlow f;
        Ti::products(bars, smem, ring, n[0], n[1], f);
        Ti::products_done(bars);
    } else if (warp < NQ * 4) {
        Ti::many_registers();
        const int i = warp >> 2, mine = r0 + warp * 32;     // this warp's 32 query rows
        // ---- queries to shared memory: four lanes to a row, eight rows at a time; K-major with 128-byte swizzle. (The whole warp
        // to a row, 32 rows one after another, was 15 us of a stretch's 27: one warp per scheduler issues an instruction every
        // few clocks, and it took five times as many.)
        float c_row = 0.0f;
        constexpr int VE = Io<QT>::VE, NV = D / 4 / VE;     // values in 16 bytes, and 16-byte loads of a lane
#pragma unroll 1
        for (int r8 = 0; r8 < 32; r8 += 8) {
            const int r = mine + r8 + (lane >> 2), in_tile = (warp & 3) * 32 + r8 + (lane >> 2);
            const QT* src = q + ((long long)(r / G) * n_q + kh * G + r % G) * D + (lane & 3) * VE;
            float v[NV][VE], top = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint4 raw = r < M ? __ldg(reinterpret_cast<const uint4*>(src + k * 4 * VE)) : make_uint4(0, 0, 0, 0);
                Io<QT>::unpack(raw, v[k]);
#pragma unroll
                for (int e = 0; e < VE; ++e) top = fmaxf(top, fabsf(v[k][e]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int x = q_exponent(top);
            // (c > 0 also for a row near the least float: a hidden score, -inf, times 0 would be NaN)
            const float k0 = pow2(x / 2), k1 = pow2(x - x / 2), c_own = fmaxf(scale2e(scale2, -x), 0x1p-126f);
            const float c = __shfl_sync(0xffffffffu, c_own, (lane & 7) * 4);
            if (lane >> 3 == r8 >> 3) c_row = c;
            unsigned char* row = smem + i * Ti::QTILE * (SPLIT ? 2 : 1) + in_tile * 128;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int col = (k * 4 + (lane & 3)) * VE;
                unsigned char* at = row + col / CHUNK * CHUNK_BYTES + ((col % CHUNK / 8 ^ (in_tile & 7)) * 16) + col % 8 * 2;
                uint32_t hi[VE / 2], lo[VE / 2];
#pragma unroll
                for (int e = 0; e < VE / 2; ++e) split16(v[k][2 * e] * k0 * k1, v[k][2 * e + 1] * k0 * k1, &hi[e], &lo[e]);
                if constexpr (SPLIT) {
                    *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(at + Ti::QTILE) = make_uint2(lo[0], lo[1]);
                } else {
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[VE / 2 - 2], hi[VE / 2 - 1]);
                }
            }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full[i]);

        float m = -INFINITY, l = 0.0f;
        const int tiles_i = i ? n[1] : n[0];
        // four neighbouring rows of a tile are in one page: lane k speaks for keys 4 k .. 4 k + 3
        const auto look = [&](int j) {
            const int t = (j0 + j) * TILE_ROWS + lane * 4;
            return j < tiles_i && t < prefix && (unsigned)pages[t >> kv.kv_shift] < (unsigned)kv.n_pages;
        };
        bool next = look(0);
        TileFlow f;
        for (int j = 0; j < tiles_i; ++j) {
            const unsigned seen = __ballot_sync(0xffffffffu, next);
            next = look(j + 1);
            if (!Ti::softmax_step(bars, i, j == 0, j + 1 == tiles_i, f, c_row, m, l, [&](uint32_t (&x)[128]) {
                    if (seen != 0xffffffffu)
#pragma unroll
                        for (int e = 0; e < 128; ++e)
                            if (!(seen >> (e / 4) & 1)) x[e] = 0xff800000u;
                }))
                break;
        }
        if (tiles_i > 0 && warp_wait(&bars.o_full[i], 0, &bars.dead)) {
            tc_fence_after();
            const uint32_t o_addr = bars.tmem + 256 + i * D + ((uint32_t)(threadIdx.x & 96) << 16);
            const long long at = ((long long)split * n_kv + kh) * px.rows + mine;
            px.ml[(at + lane) * 2] = m == -INFINITY ? -INFINITY : m * c_row;
            px.ml[(at + lane) * 2 + 1] = l;
            // through this warp's part of the query tile (32 rows of at least 128 bytes), 32 columns at a time
            float* buf = reinterpret_cast<float*>(smem + (i * TILE_ROWS + (warp & 3) * 32) * (D * 2 * (SPLIT ? 2 : 1)));
            static_assert(32 * 32 * 4 <= 32 * D * 2, "32 rows of 32 floats fit the warp's part");
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + c, o);
                tmem_ld_wait();
                tmem_pin(o);
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<uint4*>(buf + lane * 32 + ((e / 4 ^ (lane & 7)) * 4)) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int rr = e * 4 + (lane >> 3), u = lane & 7;
                    *reinterpret_cast<uint4*>(px.o + (at + rr) * D + c + u * 4) =
                        *reinterpret_cast<const uint4*>(buf + rr * 32 + ((u ^ (rr & 7)) * 4));
                }
                __syncwarp();
            }
        }
    } else {
        Ti::few_registers();
    }
    }
    Ti::teardown(bars);
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace b200

#endif  // B200_ATTN_PREFIX_CUH
