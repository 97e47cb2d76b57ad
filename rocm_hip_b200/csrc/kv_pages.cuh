// kv_pages.cuh -- the pages of a paged KV cache: sequences forked, grown, cut back and freed, live pages moved to the
// front. The state is a page table, a length per sequence and a reference count per page; a page is free when its
// count is 0, and pages are always taken lowest id first, so the same calls give the same tables and a freed page needs
// no list of its own.
//
// A call is a control kernel and a copy kernel. The control kernel is one CTA or ONE cluster of eight (CTAS): it has little to
// do (a few words per sequence and page), what costs is the number of dependent passes over it, and a barrier of the CTA or
// the cluster orders those passes without a launch in between. It leaves a list of (from, to) pages; the copy kernel, on
// the whole device, moves them.

#ifndef B200_KV_PAGES_CUH
#define B200_KV_PAGES_CUH

#include <limits.h>

#include "b200_layer_ops.h"
#include "common.cuh"

namespace b200 {

constexpr int KVP_THREADS = 1024;
constexpr int KVP_HEAD = 64;    // ints at the start of the work memory (below)

// info[0]: what became of the call
enum { KVP_OK = 0, KVP_FULL = 1, KVP_BAD = 2 };

// Work memory: head [0 .. 15] free (or live) pages in each CTA's range, [16 .. 31] and [32 .. 47] holes and movers
// (compaction), [48] pages needed, [49] bad arguments, [50] new tokens, [51] copies, [56] pages to copy, [57] next tile of
// the copy; per sequence the rank of its first new page, of its first new token and of its copied page; per page the
// two sides of the list of copies and a third list.
struct KvPagesWork {
    int *head, *off, *soff, *coff, *from, *to, *list;
    __device__ __host__ KvPagesWork(int* w, int n_seqs, int n_pages)
        : head(w), off(w + KVP_HEAD), soff(off + n_seqs), coff(soff + n_seqs), from(coff + n_seqs), to(from + n_pages),
          list(to + n_pages) {}
    static size_t ints(int n_seqs, int n_pages) { return KVP_HEAD + 3 * (size_t)n_seqs + 3 * (size_t)n_pages; }
};

// All threads of the CTA or cluster; orders their global accesses too
template <int CTAS>
__device__ __forceinline__ void kvp_sync() {
    if constexpr (CTAS == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Exclusive sums over the CTA in thread order of N values at once, and their totals. Two barriers; part: N * 32 ints.
template <int N>
__device__ __forceinline__ void kvp_scan(int (&v)[N], int (&total)[N], int* part) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int own[N];
#pragma unroll
    for (int k = 0; k < N; ++k) own[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int y = __shfl_up_sync(0xffffffffu, v[k], o);
            if (lane >= o) v[k] += y;
        }
    __syncthreads();
    if (lane == 31)
#pragma unroll
        for (int k = 0; k < N; ++k) part[k * 32 + w] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {      // every warp sums the warps' totals
        const int mine = part[k * 32 + lane];
        int x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        total[k] = __shfl_sync(0xffffffffu, x, 31);
        v[k] += __shfl_sync(0xffffffffu, x - mine, w) - own[k];
    }
}
__device__ __forceinline__ int kvp_scan1(int v, int* total, int* part) {
    int a[1] = {v}, t[1];
    kvp_scan<1>(a, t, part);
    *total = t[0];
    return a[0];
}

// The CTA's share of the pages: [*a, *b)
template <int CTAS>
__device__ __forceinline__ void kvp_range(int n_pages, int cta, int* a, int* b) {
    const int per = (n_pages + CTAS - 1) / CTAS;
    *a = min(n_pages, cta * per);
    *b = min(n_pages, *a + per);
}

// How many pages of [a, b) satisfy test(page, refs[page]); the same value in every thread
template <typename F>
__device__ __forceinline__ int kvp_count(const int* refs, int a, int b, int* part, F test) {
    int n = 0, total;
    for (int p = a + threadIdx.x; p < b; p += KVP_THREADS) n += test(p, refs[p]) ? 1 : 0;
    kvp_scan1(n, &total, part);
    return total;
}

// list[base + r] = the r-th page of [a, b) that satisfies the test, as long as base + r < limit
template <typename F>
__device__ __forceinline__ void kvp_list(const int* refs, int a, int b, int base, int limit, int* list, int* part, F test) {
    for (int p0 = a; p0 < b && base < limit; p0 += KVP_THREADS) {   // uniform in the CTA
        const int p = p0 + threadIdx.x;
        const bool yes = p < b && test(p, refs[p]);
        int total;
        const int r = kvp_scan1(yes ? 1 : 0, &total, part);
        if (yes && base + r < limit) list[base + r] = p;
        base += total;
    }
}

template <int CTAS>
__device__ __forceinline__ int kvp_before(const int* counts, int cta, int* all) {
    int base = 0, sum = 0;
    for (int i = 0; i < CTAS; ++i) {
        base += i < cta ? counts[i] : 0;
        sum += counts[i];
    }
    *all = sum;
    return base;
}

__device__ __forceinline__ void kvp_tell(const b200_kv_pages& kv, int* head, int status, int n_free, int copies) {
    kv.info[0] = status;
    kv.info[1] = n_free;
    kv.info[2] = copies;
    head[56] = copies;
    head[57] = 0;
}

// A length the table can hold
__device__ __forceinline__ int kvp_len(const b200_kv_pages& kv, int s) {
    const long long cap = (long long)kv.max_pages << kv.page_shift;
    const int n = max(kv.lens[s], 0);
    return (int)min((long long)n, cap);
}

// Pages that n rows take
__device__ __forceinline__ int kvp_pages(int n, int shift) { return (int)(((long long)n + (1 << shift) - 1) >> shift); }

// parent[s] >= 0: the empty sequence s becomes a copy of parent[s]. Whole pages are shared, a last page that is only
// partly filled gets a copy of its own, so that both may grow.
template <int CTAS>
__global__ void __launch_bounds__(KVP_THREADS)
k_kv_pages_fork(b200_kv_pages kv, const int* parent) {
    __shared__ int part[96];
    pdl_entry();
    const int cta = blockIdx.x, mask = (1 << kv.page_shift) - 1;
    const KvPagesWork w(kv.work, kv.n_seqs, kv.n_pages);
    int a, b;
    kvp_range<CTAS>(kv.n_pages, cta, &a, &b);
    const auto is_free = [](int, int r) { return r == 0; };
    const int mine = kvp_count(kv.refs, a, b, part, is_free);
    if (threadIdx.x == 0) w.head[cta] = mine;
    if (cta == 0) {   // which forks need a page, and the rank of each among them
        int base = 0, bad = 0;
        for (int s0 = 0; s0 < kv.n_seqs; s0 += KVP_THREADS) {
            const int s = s0 + threadIdx.x;
            int need = 0;
            if (s < kv.n_seqs) {
                const int p = parent[s];
                int n = -1;
                if (p >= 0) {
                    if (p >= kv.n_seqs || p == s || kv.lens[s] != 0) bad = 1;
                    else {
                        n = kvp_len(kv, p);
                        need = (n & mask) != 0;
                    }
                }
                w.soff[s] = n;   // the parent's length, or -1
            }
            int total;
            const int r = kvp_scan1(need, &total, part);
            if (s < kv.n_seqs) w.off[s] = base + r;
            base += total;
        }
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0) { w.head[48] = base; w.head[49] = bad; }
    }
    kvp_sync<CTAS>();
    int n_free;
    const int before = kvp_before<CTAS>(w.head, cta, &n_free), need = w.head[48];
    const int status = w.head[49] ? KVP_BAD : need > n_free ? KVP_FULL : KVP_OK;
    if (status == KVP_OK) kvp_list(kv.refs, a, b, before, need, w.to, part, is_free);
    kvp_sync<CTAS>();
    if (cta == 0 && threadIdx.x == 0) kvp_tell(kv, w.head, status, n_free - (status == KVP_OK ? need : 0), status == KVP_OK ? need : 0);
    if (status != KVP_OK) return;
    const int lane = threadIdx.x & 31;
    for (int s = cta + CTAS * (threadIdx.x >> 5); s < kv.n_seqs; s += CTAS * (KVP_THREADS / 32)) {
        const int n = w.soff[s];
        if (n < 0) continue;
        const int* from = kv.table + (long long)parent[s] * kv.max_pages;
        int* row = kv.table + (long long)s * kv.max_pages;
        const int full = n >> kv.page_shift;
        for (int i = lane; i < kv.max_pages; i += 32) {
            int p = -1;
            if (i < full) {
                p = from[i];
                if ((unsigned)p < (unsigned)kv.n_pages) atomicAdd(kv.refs + p, 1);
            } else if (i == full && (n & mask)) {
                const int r = w.off[s];
                p = w.to[r];
                kv.refs[p] = 1;
                w.from[r] = from[i];
            }
            row[i] = p;
        }
        if (lane == 0) kv.lens[s] = n;
    }
}

// Sequence s gets the length to[s] (< 0: it keeps its own). First every sequence that gets shorter gives back what it
// no longer needs; then the others take the pages they lack, in the order of the sequences, and the cache rows of
// their new tokens go to slots. A last page that is partly filled and shared is replaced by a copy before it grows.
// Where the pages do not suffice, or a length exceeds the table, no sequence grows.
template <int CTAS>
__global__ void __launch_bounds__(KVP_THREADS)
k_kv_pages_resize(b200_kv_pages kv, const int* new_lens, int* slots, int n_slots) {
    __shared__ int part[96];
    pdl_entry();
    const int cta = blockIdx.x, mask = (1 << kv.page_shift) - 1, lane = threadIdx.x & 31;
    const long long cap = (long long)kv.max_pages << kv.page_shift;
    const KvPagesWork w(kv.work, kv.n_seqs, kv.n_pages);
    const int s_first = cta + CTAS * (threadIdx.x >> 5), s_step = CTAS * (KVP_THREADS / 32);
    for (int s = s_first; s < kv.n_seqs; s += s_step) {
        const int to = new_lens[s], n = kvp_len(kv, s);
        __syncwarp();   // every lane has read the length before lane 0 writes it
        if (to < 0 || to >= n) continue;
        int* row = kv.table + (long long)s * kv.max_pages;
        const int stay = kvp_pages(to, kv.page_shift), had = kvp_pages(n, kv.page_shift);
        for (int i = stay + lane; i < had; i += 32) {
            const int p = row[i];
            if ((unsigned)p < (unsigned)kv.n_pages) atomicSub(kv.refs + p, 1);
            row[i] = -1;
        }
        if (lane == 0) kv.lens[s] = to;
    }
    kvp_sync<CTAS>();
    int a, b;
    kvp_range<CTAS>(kv.n_pages, cta, &a, &b);
    const auto is_free = [](int, int r) { return r == 0; };
    const int mine = kvp_count(kv.refs, a, b, part, is_free);
    if (threadIdx.x == 0) w.head[cta] = mine;
    if (cta == 0) {
        int base = 0, sbase = 0, cbase = 0, bad = 0;
        for (int s0 = 0; s0 < kv.n_seqs; s0 += KVP_THREADS) {
            const int s = s0 + threadIdx.x;
            int need = 0, more = 0, cow = 0;
            if (s < kv.n_seqs) {
                const int to = new_lens[s], n = kvp_len(kv, s);
                if (to > cap) bad = 1;
                else if (to > n) {
                    more = to - n;
                    need = kvp_pages(to, kv.page_shift) - kvp_pages(n, kv.page_shift);
                    if (n & mask) {
                        const int p = kv.table[(long long)s * kv.max_pages + (n >> kv.page_shift)];
                        if ((unsigned)p >= (unsigned)kv.n_pages) bad = 1;
                        else cow = kv.refs[p] > 1;
                    }
                }
            }
            int rank[3] = {need + cow, more, cow}, total[3];
            kvp_scan<3>(rank, total, part);
            if (s < kv.n_seqs) {
                w.off[s] = base + rank[0];
                w.soff[s] = sbase + rank[1];
                w.coff[s] = cow ? cbase + rank[2] : -1;
            }
            base += total[0];
            sbase += total[1];
            cbase += total[2];
        }
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0) { w.head[48] = base; w.head[49] = bad; w.head[50] = sbase; w.head[51] = cbase; }
    }
    kvp_sync<CTAS>();
    int n_free;
    const int before = kvp_before<CTAS>(w.head, cta, &n_free), need = w.head[48], n_new = w.head[50], copies = w.head[51];
    const int status = w.head[49] ? KVP_BAD : need > n_free ? KVP_FULL : KVP_OK;
    if (status == KVP_OK) kvp_list(kv.refs, a, b, before, need, w.list, part, is_free);
    kvp_sync<CTAS>();
    if (status != KVP_OK) {
        if (cta == 0 && threadIdx.x == 0) kvp_tell(kv, w.head, status, n_free, 0);
        return;
    }
    for (int s = s_first; s < kv.n_seqs; s += s_step) {
        const int to = new_lens[s], n = kvp_len(kv, s);
        __syncwarp();   // every lane has read the length before lane 0 writes it
        if (to <= n) continue;
        int* row = kv.table + (long long)s * kv.max_pages;
        const int c = w.coff[s], had = kvp_pages(n, kv.page_shift), want = kvp_pages(to, kv.page_shift);
        const int* ids = w.list + w.off[s];
        if (c >= 0) {
            if (lane == 0) {
                const int old = row[had - 1];
                atomicSub(kv.refs + old, 1);
                w.from[c] = old;
                w.to[c] = ids[0];
                kv.refs[ids[0]] = 1;
                row[had - 1] = ids[0];
            }
            ++ids;
        }
        for (int i = had + lane; i < want; i += 32) {
            row[i] = ids[i - had];
            kv.refs[ids[i - had]] = 1;
        }
        if (lane == 0) kv.lens[s] = to;
    }
    kvp_sync<CTAS>();
    if (slots) {   // a thread per new token: its sequence is the last whose first new token is not behind it
        const int n_out = min(n_new, n_slots);
        for (int i = cta * KVP_THREADS + threadIdx.x; i < n_out; i += CTAS * KVP_THREADS) {
            int lo = 0, hi = kv.n_seqs;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (w.soff[mid] <= i) lo = mid + 1; else hi = mid;
            }
            const int s = lo - 1, next = s + 1 < kv.n_seqs ? w.soff[s + 1] : n_new;
            const int t = new_lens[s] - (next - i);
            slots[i] = (kv.table[(long long)s * kv.max_pages + (t >> kv.page_shift)] << kv.page_shift) + (t & mask);
        }
    }
    if (copies == 0) {
        if (cta == 0 && threadIdx.x == 0) kvp_tell(kv, w.head, KVP_OK, n_free - need, 0);
        return;
    }
    // pages whose last reader took a copy are free again: none of them was handed out by this call
    const int left = kvp_count(kv.refs, a, b, part, is_free);
    if (threadIdx.x == 0) w.head[16 + cta] = left;
    kvp_sync<CTAS>();
    if (cta == 0 && threadIdx.x == 0) {
        int all;
        kvp_before<CTAS>(w.head + 16, 0, &all);
        kvp_tell(kv, w.head, KVP_OK, all, copies);
    }
}

// The n_live pages in use become pages 0 .. n_live - 1: those at or behind n_live move, in ascending order, into the
// free ids before it. No page is both moved from and moved to.
template <int CTAS>
__global__ void __launch_bounds__(KVP_THREADS)
k_kv_pages_compact(b200_kv_pages kv) {
    __shared__ int part[96];
    pdl_entry();
    const int cta = blockIdx.x, lane = threadIdx.x & 31;
    const KvPagesWork w(kv.work, kv.n_seqs, kv.n_pages);
    int a, b, n_live, n_holes, n_move;
    kvp_range<CTAS>(kv.n_pages, cta, &a, &b);
    const int mine = kvp_count(kv.refs, a, b, part, [](int, int r) { return r > 0; });
    if (threadIdx.x == 0) w.head[cta] = mine;
    kvp_sync<CTAS>();
    kvp_before<CTAS>(w.head, cta, &n_live);
    const auto hole = [n_live](int p, int r) { return r <= 0 && p < n_live; };
    const auto mover = [n_live](int p, int r) { return r > 0 && p >= n_live; };
    const int h = kvp_count(kv.refs, a, b, part, hole), m = kvp_count(kv.refs, a, b, part, mover);
    if (threadIdx.x == 0) { w.head[16 + cta] = h; w.head[32 + cta] = m; }
    kvp_sync<CTAS>();
    const int hb = kvp_before<CTAS>(w.head + 16, cta, &n_holes), mb = kvp_before<CTAS>(w.head + 32, cta, &n_move);
    kvp_list(kv.refs, a, b, hb, kv.n_pages, w.to, part, hole);
    kvp_list(kv.refs, a, b, mb, kv.n_pages, w.from, part, mover);
    for (int p = max(a, n_live) + threadIdx.x; p < b; p += KVP_THREADS) w.list[p] = p;
    kvp_sync<CTAS>();
    for (int r = cta * KVP_THREADS + threadIdx.x; r < n_move; r += CTAS * KVP_THREADS) {
        w.list[w.from[r]] = w.to[r];
        kv.refs[w.to[r]] = kv.refs[w.from[r]];
        kv.refs[w.from[r]] = 0;
    }
    kvp_sync<CTAS>();
    for (int s = cta + CTAS * (threadIdx.x >> 5); s < kv.n_seqs; s += CTAS * (KVP_THREADS / 32)) {
        int* row = kv.table + (long long)s * kv.max_pages;
        const int used = kvp_pages(kvp_len(kv, s), kv.page_shift);
        for (int i = lane; i < used; i += 32) {
            const int p = row[i];
            if (p >= n_live && p < kv.n_pages) row[i] = w.list[p];
        }
    }
    if (cta == 0 && threadIdx.x == 0) kvp_tell(kv, w.head, KVP_OK, kv.n_pages - n_live, n_move);
}

// Copies the listed pages, part by part, in tiles of 16 KB: eight CTAs per SM, 64 bytes of each thread's in flight. How many
// pages there are is known on the device only, so the grid is what fits, and a CTA takes the next tile that nobody has
// taken: tiles are then under way in the order of memory, which this memory system rewards (a compaction that moves 4,870
// pages of 256 KB: 456 us with tiles dealt out in strides of the grid, 411 taken in order; forks that copy 320 pages of
// 1 MB: 121 and 108). Which CTA copies a tile changes nothing.
__global__ void __launch_bounds__(256)
k_kv_pages_copy(b200_kv_pages kv) {
    __shared__ int taken[2];
    pdl_entry();
    constexpr int TILE = 16384;
    const KvPagesWork w(kv.work, kv.n_seqs, kv.n_pages);
    const int n = w.head[56];
    const int per = (int)((kv.page_bytes + TILE - 1) / TILE);
    const long long total = (long long)n * kv.n_parts * per;
    const bool in_order = total < INT_MAX - (long long)gridDim.x;
    long long i = blockIdx.x;
    for (int turn = 0; i < total; turn ^= 1) {
        if (in_order && threadIdx.x == 0) taken[turn] = (int)gridDim.x + atomicAdd(w.head + 57, 1);   // (while this tile is copied)
        const int c = (int)(i % per);
        const long long u = i / per;
        const int part = (int)(u % kv.n_parts), r = (int)(u / kv.n_parts);
        const int from = w.from[r], to = w.to[r];
        const bool inside = (unsigned)from < (unsigned)kv.n_pages && (unsigned)to < (unsigned)kv.n_pages;
        const size_t at = part * kv.part_stride + (size_t)c * TILE;
        const char* src = (const char*)kv.pool + at + (size_t)from * kv.page_bytes;
        char* dst = (char*)kv.pool + at + (size_t)to * kv.page_bytes;
        const int bytes = inside ? (int)min((size_t)TILE, kv.page_bytes - (size_t)c * TILE) : 0;
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int o = (j * 256 + threadIdx.x) * 16;
            if (o < bytes) v[j] = ld_stream(src + o);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int o = (j * 256 + threadIdx.x) * 16;
            if (o < bytes) st_stream(dst + o, v[j]);
        }
        if (in_order) {
            __syncthreads();
            i = taken[turn];
        } else {
            i += gridDim.x;
        }
    }
}

}  // namespace b200

#endif  // B200_KV_PAGES_CUH
