// attn_prompt.cuh -- causal attention over packed prompts (several sequences one after another in the rows), grouped
// heads, 16-bit rows:
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp(scale q[t, h] . k[j, h / G]),  j in t's sequence, j <= t
// Sequence b is rows [seq_start[b], seq_start[b + 1]); rows in no sequence are not written.

#ifndef B200_ATTN_PROMPT_CUH
#define B200_ATTN_PROMPT_CUH

#include "attn_rows.cuh"
#include "attn_tiles.cuh"

namespace b200 {

// Two query tiles per CTA, one for the 256-wide heads; K and V stages as large as shared memory allows beside them. The 64-wide
// heads leave room for a buffer through which finished rows leave (2 KB a warp), so that the next query tile can come as
// soon as the last scores against the old one are done (61 sequences of 200 rows: 82 -> 69 us); the others send their rows
// out through the query tile's memory (a buffer in the place of a ring stage cost 2 % of long prompts).
template <int D, typename T>
using PromptTiles = Tiles<D, D == 256 ? 1 : 2, D < 128 ? D : 128, D == 64 ? 8 : 5, false, T>;
template <int D>
constexpr int PROMPT_OUT = D == 64 ? 8 * 2048 : 0;

// What a CTA works on next. Two query tiles are 256 rows of one head (BY_ROWS), or the same rows of two heads that share a key
// head (BY_HEADS: the group has an even number of heads; both tiles then see the same keys). BY_KEYS there is one query tile,
// even and odd key tiles take the places of the two, and both softmax halves join what they found: half the way for a tile
// with many keys, for calls that have too few tiles to fill the device otherwise.
enum { BY_ROWS = 0, BY_HEADS = 1, BY_KEYS = 2 };
struct PromptItem {
    int h, first, q0, end;      // head; the sequence's first row; the first query row; the sequence's end
    int n[2];                   // key tiles per query tile; n[0] == 0: there is nothing more
};
struct PromptBars {
    unsigned long long item_full[2], item_empty[2], q_empty[2], asked, ml_full, o_read, raw[8], looked[4];
    uint4 answer;               // of the work distributor, 16 bytes
    PromptItem item[2];
    unsigned odd[4][2][4];      // of four items in turn, of their up to two tiles looked at: the keys whose v was blanked
};

// Softmax warps, tensor cores, copies, schedule, and one that looks at V tiles
template <int D>
constexpr int PROMPT_WARPS = D == 256 ? 8 : 12;

// A weight of 0 times a non-finite v is not 0 on the tensor cores, and a query tile's last key tile holds keys that some of its
// rows do not see: later ones, the next sequence's, rows in no sequence. So from the first query tile's last key tile on
// (one tile, or two where the query tiles are 256 rows of one head) the copies of V report to a warp of its own, which blanks
// what is not finite and then hands the tile to the tensor cores; rows get back what they do see of that with plain
// additions, an infinity or a NaN as it is. What a row does not see can then change no bit of its result, and what the
// hand-over costs is one packed multiply-add per pair of values (v 0 + 0 is NaN for them), while the tile's scores are in the
// softmax: 61 sequences of 64-wide heads 62.5 -> 66.9 us, one sequence of 2,427 rows 38.8 -> 37.9, 32,768 rows 2.78 -> 2.76 ms
// against rows that were computed again, key after key, when they came out non-finite, which took the softmax warps out of
// the CTA's pipeline for as long as a sequence has keys. (The tensor cores' warp asking for the look when it takes a tile:
// two more waits in its loop cost 11 % of long prompts. By mma.sync in place of the multiply-adds: no faster.)

// v 0 + acc for pairs: NaN from the first value on that is not finite
template <typename T>
__device__ __forceinline__ uint32_t mark_non_finite(uint32_t w, uint32_t acc) {
    uint32_t r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(acc));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(acc));
    return r;
}

// One warp: blanks what is not finite in BYTES of a V tile of 128 rows, [values / 64][128 rows][64 values], and sets the bits of
// its rows
template <typename T, int BYTES>
__device__ __forceinline__ void blank_non_finite(unsigned char* part, unsigned* odd) {
    constexpr uint32_t EXP = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    constexpr int AT_ONCE = 8;
    static_assert(BYTES % (AT_ONCE * 512) == 0, "whole rounds");
    const int lane = threadIdx.x & 31;
    uint32_t acc[4] = {0, 0, 0, 0};
    for (int at = lane * 16; at < BYTES; at += AT_ONCE * 512) {
        uint4 w[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) w[i] = *reinterpret_cast<const uint4*>(part + at + i * 512);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            acc[0] = mark_non_finite<T>(w[i].x, acc[0]);
            acc[1] = mark_non_finite<T>(w[i].y, acc[1]);
            acc[2] = mark_non_finite<T>(w[i].z, acc[2]);
            acc[3] = mark_non_finite<T>(w[i].w, acc[3]);
        }
    }
    // (the sums are +-0 or NaN)
    if (!__any_sync(0xffffffffu, (acc[0] | acc[1] | acc[2] | acc[3]) & 0x7fff7fffu)) return;
    for (int at = lane * 16; at < BYTES; at += 512) {
        uint4 w = *reinterpret_cast<const uint4*>(part + at);
        const auto blank = [](uint32_t x) {
            if ((x & EXP) == EXP) x &= 0xffff0000u;
            if ((x >> 16 & EXP) == EXP) x &= 0x0000ffffu;
            return x;
        };
        const uint4 b = make_uint4(blank(w.x), blank(w.y), blank(w.z), blank(w.w));
        if (b.x != w.x || b.y != w.y || b.z != w.z || b.w != w.w) {
            *reinterpret_cast<uint4*>(part + at) = b;
            const int row = at / 128 % TILE_ROWS;
            atomicOr(odd + row / 32, 1u << row % 32);
        }
    }
    fence_async_smem();          // the tensor cores read through the other proxy
}

// What blank_non_finite took from the rows of a warp that see it, added to them: `word` of lanes 0 .. 7 are the bits of the
// blanked keys, v0 the first of these keys, `from` that key's distance to the warp's first row, `rows` how many rows it has,
// out the first one. Lanes in `mine` look after their columns.
template <int D, typename T>
__device__ void give_non_finite(unsigned word, const T* v0, long long v_stride, int from, int rows, T* out, long long out_stride, unsigned mine) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31, c = lane * N;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int r = 0, k = 0; r < rows; ++r) {
        for (; k <= from + r; ++k) {            // the keys up to the row's own
            if (!(__shfl_sync(0xffffffffu, word, k >> 5) >> (k & 31) & 1)) continue;
            float x[N];
            load_vals(v0 + k * v_stride + c, x);
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += fabsf(x[i]) < INFINITY ? 0.0f : x[i];
        }
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i) any |= sum[i] != 0.0f;
        if (any && (mine >> lane & 1)) {
            float y[N];
            load_vals(out + r * out_stride + c, y);
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] += sum[i];
            store_vals(out + r * out_stride + c, y);
        }
    }
}

// The next block of the grid that has not begun, taken over by this CTA (the hardware's work distributor hands blocks to CTAs
// that ask as it hands them to SMs that are free): asks, and later reads the answer. One thread.
__device__ __forceinline__ void ask_for_block(PromptBars& pb) {
    mbar_expect(&pb.asked, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(&pb.answer)), "r"(smem_u32(&pb.asked))
                 : "memory");
}
__device__ __forceinline__ int block_answer(PromptBars& pb) {   // the block's index, -1: there is none
    int got, x;
    asm volatile("{\n\t.reg .b128 r;\n\t.reg .pred p;\n\tld.shared.b128 r, [%2];\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.s32 %0, 1, 0, p;\n\tmov.s32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
                 : "=r"(got), "=r"(x)
                 : "r"(smem_u32(&pb.answer))
                 : "memory");
    return got ? x : -1;
}

// The grid is all blocks of work, heaviest first as far as one pass over the batch knows; a CTA that has finished one takes
// the next that nobody has begun. Its roles run ahead of one another: while the softmax warps still write one block's rows,
// the schedule warp has looked up the next block, its first K and V tiles are on their way, and the tensor cores begin as
// soon as the query tile's memory is free and filled again. (One CTA per block: 61 sequences of 200 rows, 16 heads of 64, took 98 us, most of
// it the way from a CTA's start to its first product and from its last to its end.)
template <int D, typename T, int MODE>
__global__ void __launch_bounds__(PROMPT_WARPS<D> * 32, 1)
k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
              const T* v, T* out, const int* seq_start, int n_seqs, int rows, int n_q, int G, long long v_stride, float scale2, int n_slots) {
    using Ti = PromptTiles<D, T>;
    constexpr int NQ = D == 256 ? 1 : 2, SC = D < 128 ? D : 128;
    constexpr int ROWS = NQ == 2 && MODE == BY_ROWS ? 2 * TILE_ROWS : TILE_ROWS;                       // of a block
    constexpr int dh = MODE == BY_HEADS ? 1 : 0, dq = MODE == BY_ROWS ? TILE_ROWS : 0;                // from one query tile to the other
    const int n_heads = MODE == BY_HEADS ? n_q / 2 : n_q;
    extern __shared__ unsigned char smem_raw[];
    __shared__ TileBars bars;
    __shared__ PromptBars pb;
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* ring = smem + Ti::Q_BYTES;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (warp == NQ * 4 + 1 && lane == 0) {
        tma_prefetch(&mq);
        tma_prefetch(&mk);
        tma_prefetch(&mv);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&pb.item_full[i], 1);
            mbar_init(&pb.item_empty[i], NQ * 4 + 3);
            mbar_init(&pb.q_empty[i], PROMPT_OUT<D> ? 1 : MODE == BY_KEYS ? 8 : 4);
        }
        mbar_init(&pb.asked, 1);
        mbar_init(&pb.ml_full, 8);
        mbar_init(&pb.o_read, 8);
        for (int i = 0; i < Ti::STAGES; ++i) mbar_init(&pb.raw[i], 1);
        for (int i = 0; i < 4; ++i) mbar_init(&pb.looked[i], 1);
        mbar_fence_init();
    }
    Ti::setup(bars, 1);
    pdl_entry();

    // the consumers' side of the items: what to do next, until n[0] is 0
    unsigned taken = 0;
    const auto next_item = [&](PromptItem* it) {
        const int slot = taken & 1;
        if (!warp_wait_long(&pb.item_full[slot], taken >> 1 & 1, &bars.dead)) return false;
        *it = pb.item[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&pb.item_empty[slot]);
        ++taken;
        return it->n[0] > 0;
    };

    if (warp == NQ * 4 + 2) {
        Ti::few_registers();
        // ---- schedule: blocks of work, two ahead of the CTA's slowest role
        int block = blockIdx.x;
        unsigned made = 0, asked = 0;
        while (true) {
            // (the next answer is under way while this block is looked up)
            if (block >= 0 && lane == 0) ask_for_block(pb);
            PromptItem it = {0, 0, 0, 0, {0, 0}};
            if (block >= 0) {
                // slot s of the packed batch is tile s - f(b) of sequence b, f(b) = floor(start(b) / ROWS) + b, the last b with
                // f(b) <= s; f(b + 1) - f(b) is at least the number of tiles b has. Slots are taken from the last one down, so
                // that in a sequence the tiles with the most keys come first.
                const int slot = n_slots - 1 - block / n_heads;
                int first = 0, end = rows, tile = slot;
                if (seq_start) {
                    int lo = 0, hi = n_seqs;            // the last b with f(b) <= slot is in [lo - 1, hi): 32 probes a step
                    while (lo < hi) {
                        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
                        const bool yes = at < hi && min(max(seq_start[at], 0), rows) / ROWS + at <= slot;
                        const unsigned votes = __ballot_sync(0xffffffffu, yes);
                        const int k = votes ? 32 - __clz(votes) : 0;      // probes up to k - 1 hold
                        if (k == 0) { hi = lo; break; }
                        const int base = lo + (k - 1) * step;             // holds; the answer is in [base, base + step)
                        lo = base + 1;
                        hi = min(base + step, hi);
                    }
                    const int b = max(lo - 1, 0);
                    first = min(max(seq_start[b], 0), rows);
                    end = max(first, min(seq_start[b + 1], rows));
                    tile = slot - (first / ROWS + b);
                }
                if (tile >= 0 && tile <= (end - first) / ROWS && first + tile * ROWS < end) {   // (no overflow on bad borders)
                    it.h = block % n_heads << dh;
                    it.first = first;
                    it.q0 = first + tile * ROWS;
                    it.end = end;
#pragma unroll
                    for (int i = 0; i < (MODE == BY_KEYS ? 1 : NQ); ++i) {   // those up to the last row's own place
                        const int a = it.q0 + i * dq;
                        it.n[i] = a < end ? (min(a + TILE_ROWS, end) - 1 - first) / TILE_ROWS + 1 : 0;
                    }
                }
            }
            if (it.n[0] > 0 || block < 0) {
                const int s = made & 1;
                if (!warp_wait_long(&pb.item_empty[s], made >> 1 & 1 ^ 1, &bars.dead)) break;
                if (lane == 0) {
                    pb.item[s] = it;
                    mbar_arrive(&pb.item_full[s]);
                }
                ++made;
            }
            if (block < 0) break;
            if (!warp_wait(&pb.asked, asked & 1, &bars.dead)) break;
            ++asked;
            block = block_answer(pb);
            fence_async_smem();          // the answer has been read before the next one may arrive
            __syncwarp();
        }
        if (block >= 0) (void)mbar_wait(&pb.asked, asked & 1);      // (given up with a question open)
    } else if (warp == NQ * 4 + 1) {
        Ti::few_registers();
        // ---- copies: K and V tiles in the order the tensor cores take them, and Q as soon as its place is free
        typename Ti::Ring r{bars, ring};
        PromptItem it;
        unsigned items[2] = {0, 0};
        while (next_item(&it)) {
            const int kh = it.h / G, n_all = max(it.n[0], it.n[1]);
            const auto put = [&](const CUtensorMap* map, int j, bool look = false) {
                r.put([&](unsigned char* dst, int p, unsigned long long* bar) {
                    if (lane < SC / CHUNK) tma_3d(dst + lane * CHUNK_BYTES, map, p * SC + lane * CHUNK, kh, it.first + j * TILE_ROWS, bar);
                }, look ? pb.raw : nullptr);
            };
            put(&mk, 0);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                if (it.n[i] == 0) continue;
                if (!warp_wait(&pb.q_empty[i], items[i] & 1 ^ 1, &bars.dead)) break;
                ++items[i];
                if (lane == 0) mbar_expect(&bars.q_full[i], Ti::QTILE);
                __syncwarp();
                if (lane < D / CHUNK)
                    tma_3d(smem + i * Ti::QTILE + lane * CHUNK_BYTES, &mq, lane * CHUNK, it.h + i * dh, it.q0 + i * dq, &bars.q_full[i]);
            }
            if (MODE == BY_KEYS && n_all > 1) put(&mk, 1);
            for (int j = 0; j < n_all; ++j) {
                if (MODE != BY_KEYS && j + 1 < n_all) put(&mk, j + 1);
                put(&mv, j, j + 1 >= it.n[0]);
                if (MODE == BY_KEYS && j + 2 < n_all) put(&mk, j + 2);
            }
        }
        Ti::copies_done(bars, r, pb.raw, items);
    } else if (warp == NQ * 4) {
        Ti::few_registers();
        TileFlow f;
        PromptItem it;
        while (next_item(&it))
            if (!Ti::template products<MODE == BY_KEYS>(bars, smem, ring, it.n[0], it.n[1], f, PROMPT_OUT<D> ? pb.q_empty : nullptr)) break;
        Ti::products_done(bars);
    } else if (warp == NQ * 4 + 3) {
        Ti::few_registers();
        // ---- looks: V tiles in which a row may have unseen keys, where the ring has them (K 0, K 1, V 0, K 2, V 1, .., V n - 1)
        PromptItem it;
        unsigned parity = 0;      // bit s: of stage s's next copy that reports here
        int base = 0;             // the stage of the item's K 0
        bool ok = true;
        while (ok && next_item(&it)) {
            const int n_all = max(it.n[0], it.n[1]), slot = taken - 1 & 3;
            if (lane < 8) pb.odd[slot][lane >> 2][lane & 3] = 0;
            __syncwarp();
#pragma unroll 1
            for (int j = it.n[0] - 1; ok && j < n_all; ++j) {
                const int at = (base + (j + 1 < n_all ? 2 * j + 2 : 2 * n_all - 1) % Ti::STAGES * Ti::PARTS) % Ti::STAGES;
#pragma unroll 1
                for (int p = 0; ok && p < Ti::PARTS; ++p) {
                    const int st = at + p < Ti::STAGES ? at + p : at + p - Ti::STAGES;
                    ok = warp_wait_long(&pb.raw[st], parity >> st & 1, &bars.dead);
                    parity ^= 1u << st;
                    if (ok) blank_non_finite<T, Ti::STAGE>(ring + st * Ti::STAGE, pb.odd[slot][j - (it.n[0] - 1)]);
                    __syncwarp();
                    if (lane == 0) {
                        if (j + 1 == n_all && p + 1 == Ti::PARTS) mbar_arrive(&pb.looked[slot]);
                        mbar_arrive(&bars.full[st]);
                    }
                }
            }
            base = (base + 2 * n_all % Ti::STAGES * Ti::PARTS) % Ti::STAGES;
        }
    } else if (warp < NQ * 4) {
        Ti::many_registers();
        // ---- softmax: thread = row
        const int i = warp >> 2, r = threadIdx.x & 127;
        TileFlow f;
        PromptItem it;
        while (next_item(&it)) {
            const int h = it.h + i * dh, first = it.first, end = it.end, t0 = it.q0 + i * dq, row = t0 + r;
            // this half's key tiles: j0, j0 + dj, ... below `tiles`
            constexpr int dj = MODE == BY_KEYS ? 2 : 1;
            const int tiles = MODE != BY_KEYS && i ? it.n[1] : it.n[0], j0 = MODE == BY_KEYS ? i : 0;
            if (tiles == 0) continue;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int j = j0; j < tiles && ok; j += dj) {
                const int seen = row - first - j * TILE_ROWS;   // the last key of this tile that the row sees
                ok = Ti::softmax_step(bars, i, j == j0, j + dj >= tiles, f, scale2, m, l, [&](uint32_t (&x)[128]) {
                    if (j + 1 == tiles)   // (uniform) only a query tile's last key tile reaches past any of its rows
#pragma unroll
                        for (int e = 0; e < 128; ++e)
                            if (e > seen) x[e] = 0xff800000u;
                });
            }
            // (behind this item's last weights, where there is nothing else to do until their products are done)
            if (!ok || !warp_wait(&pb.looked[taken - 1 & 3], taken - 1 >> 2 & 1, &bars.dead)) break;
            const unsigned odd = lane < 8 ? pb.odd[taken - 1 & 3][lane >> 2][lane & 3] : 0;
            // the weights of the two halves' O, 1 / l included
            float w0 = 1.0f, w1 = 0.0f;
            if constexpr (MODE == BY_KEYS) {
                float2* ml = reinterpret_cast<float2*>(smem + Ti::QTILE);   // (where a second query tile would be)
                ml[i * TILE_ROWS + r] = make_float2(m, l);
                __syncwarp();
                if (lane == 0) mbar_arrive(&pb.ml_full);
                if (!warp_wait(&pb.ml_full, f.items[0] & 1, &bars.dead) || !warp_wait(&bars.o_full[0], f.items[0] & 1, &bars.dead)) break;
                if (tiles > 1 && !warp_wait(&bars.o_full[1], f.items[1] & 1, &bars.dead)) break;
                const float2 a = ml[r], b = ml[TILE_ROWS + r];
                const float top = fmaxf(a.x, b.x);
                w0 = a.x == -INFINITY ? 0.0f : ex2((a.x - top) * scale2);
                w1 = b.x == -INFINITY ? 0.0f : ex2((b.x - top) * scale2);
                const float inv = 1.0f / (w0 * a.y + w1 * b.y);
                w0 *= inv;
                w1 *= inv;
                if (tiles > 1) ++f.items[1];
            } else {
                if (!warp_wait(&bars.o_full[i], f.items[0] & 1, &bars.dead)) break;
                w0 = 1.0f / l;
            }
            ++f.items[0];
            tc_fence_after();
            // O / l through shared memory, CW columns at a time, so that the rows' stretches leave the warp together. BY_KEYS
            // each half writes half of the columns.
            constexpr bool BUF = PROMPT_OUT<D> > 0;
            constexpr int COLS = MODE == BY_KEYS ? D / 2 : D, CW = BUF ? 32 : COLS, UNITS = CW / 8, ROW = BUF ? CW * 2 : D * 2;
            const int at0 = MODE == BY_KEYS ? i * COLS : 0;
            const uint32_t o_addr = bars.tmem + 256 + (MODE == BY_KEYS ? 0 : i * D) + at0 + ((uint32_t)(threadIdx.x & 96) << 16);
            unsigned char* mine = BUF ? ring + Ti::RING + warp * 2048
                                      : smem + ((MODE == BY_KEYS ? 0 : i * TILE_ROWS) + (warp & 3) * 32) * (D * 2) + at0 * 2;
            for (int c0 = 0; c0 < COLS; c0 += CW) {
                for (int c = 0; c < CW; c += 32) {
                    uint32_t o[32], o1[MODE == BY_KEYS ? 32 : 1];
                    tmem_ld32(o_addr + c0 + c, o);
                    if constexpr (MODE == BY_KEYS) tmem_ld32(o_addr + D + c0 + c, o1);   // (of a single tile: anything)
                    tmem_ld_wait();
                    tmem_pin(o);
                    if constexpr (MODE == BY_KEYS) tmem_pin(o1);
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float y[8];
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            y[t] = __uint_as_float(o[e + t]) * w0;
                            if constexpr (MODE == BY_KEYS) {
                                const float both = fmaf(__uint_as_float(o1[e + t]), w1, y[t]);
                                y[t] = tiles > 1 ? both : y[t];
                            }
                        }
                        // (units of 16 bytes, stirred so that neither eight lanes' rows nor eight units share a bank)
                        const int u = (c + e) / 8, at = BUF ? u ^ (lane >> 1 & 3) : u ^ (lane & 7);
                        *reinterpret_cast<uint4*>(mine + lane * ROW + at * 16) = Io<T>::pack(y);
                    }
                }
                __syncwarp();
#pragma unroll 4
                for (int e = lane; e < 32 * UNITS; e += 32) {
                    const int rr = e / UNITS, u = e % UNITS, t = t0 + (warp & 3) * 32 + rr;
                    const int at = BUF ? u ^ (rr >> 1 & 3) : u ^ (rr & 7);
                    const uint4 y = *reinterpret_cast<const uint4*>(mine + rr * ROW + at * 16);
                    if (t < end) st_stream(reinterpret_cast<unsigned char*>(out + ((long long)t * n_q + h) * D + at0 + c0) + u * 16, y);
                }
                __syncwarp();
            }
            if (!BUF) {   // the query tile's memory may take the next one
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pb.q_empty[MODE == BY_KEYS ? 0 : i]);
            }
            if constexpr (MODE == BY_KEYS) {   // neither half may write the next O (nor its m and l) before both have read these
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pb.o_read);
            }
            // What was blanked in the tiles that were looked at goes to the rows that see it
            if (__any_sync(0xffffffffu, odd != 0)) {
                const int k0 = first + (it.n[0] - 1) * TILE_ROWS, t = t0 + (warp & 3) * 32;
                give_non_finite<D, T>(odd, v + k0 * v_stride + h / G * D, v_stride, t - k0, min(32, end - t),
                                      out + ((long long)t * n_q + h) * D, (long long)n_q * D,
                                      MODE != BY_KEYS ? 0xffffffffu : i ? 0xffff0000u : 0xffffu);
            }
            if constexpr (MODE == BY_KEYS) {
                if (!warp_wait(&pb.o_read, (f.items[0] - 1) & 1, &bars.dead)) break;
            }
        }
    }
    Ti::teardown(bars);
}

}  // namespace b200

#endif  // B200_ATTN_PROMPT_CUH
