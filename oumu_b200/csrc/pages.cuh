// Pages of a cache: handing them out, forking takes, giving pages back, packing a pool (include/oumu_attn.h). The
// pages' contents are bytes here; every layer has its own pool, one page table and one count per page serve them all.
//
// Whoever hands out or moves pages works in one block, in the order of takes and page numbers (prefix sums, no race
// decides), so the same state gives the same pages in every run; what copies bytes runs on the whole GPU. The counts
// and tables are a few KB, so these launches are bound by their latency, the copies by HBM. Measured on one B200: 64 takes
// forked from a prompt of 1000 positions in 36 layers and extended 18.0 us (47 MB written; the extend 2.1), freed 1.7 us,
// 248 of 1000 pages of 36 layers moved in 67.6 us (366 MB, 5.4 TB/s).
#pragma once
#include "common.cuh"
#include "kv4.cuh"

namespace pg {

constexpr int PAGE = kv4::PAGE;
constexpr int NT = 1024;      // threads of a planning block
constexpr int BMAX = 4096;    // takes at most (prefix sums in shared memory)

// Exclusive prefix sum of v over the block, and its total; every thread calls it.
struct ScanMem {
    int warp[NT / 32], total;
};
__device__ __forceinline__ int block_scan(int v, ScanMem &m, int *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) m.warp[w] = x;
    __syncthreads();
    if (w == 0) {
        const int y0 = m.warp[lane];
        int y = y0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        m.warp[lane] = y - y0;
        if (lane == 31) m.total = y;
    }
    __syncthreads();
    const int r = x - v + m.warp[w];
    *total = m.total;
    __syncthreads();
    return r;
}

// Free pages in ascending order: take(rank, page) for the first `want` of them; the number found. The counts are read
// past L1: atomics of this block may just have changed them.
template <class Take>
__device__ __forceinline__ int hand_out(const int *ref, int npages, int want, ScanMem &m, Take take) {
    int found = 0;
    for (int base = 0; base < npages && found < want; base += 4 * NT) {
        const int i0 = base + 4 * static_cast<int>(threadIdx.x);
        bool f[4];
        int c = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f[e] = i0 + e < npages && __ldcg(ref + i0 + e) == 0;
            c += f[e];
        }
        int total;
        int r = found + block_scan(c, m, &total);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (f[e]) {
                if (r < want) take(r, i0 + e);
                r++;
            }
        found += total;
    }
    return found < want ? found : want;
}

// Pages of the first `extra` positions past every take's length, for takes that hold any.
__global__ void __launch_bounds__(NT) k_pages_extend(int *table, int *ref, const int *lens, int extra, int *status,
                                                     int B, int npages, int maxpages) {
    __shared__ ScanMem m;
    __shared__ int base[BMAX], first[BMAX];  // a take's first rank among the pages handed out, its first missing entry
    int need_total = 0;
    for (int s0 = 0; s0 < B; s0 += NT) {
        const int s = s0 + threadIdx.x;
        int need = 0;
        if (s < B) {
            const long L = lens[s];
            long want = L > 0 ? (L + extra + PAGE - 1) / PAGE : 0;
            if (L < 0 || want > maxpages) {
                record_error(OUMU_DEVERR_LENGTH);
                want = L < 0 ? 0 : maxpages;
            }
            // rows are filled from the front: the first missing entry, most often none
            int k = static_cast<int>(want);
            const int *row = table + static_cast<long>(s) * maxpages;
            if (k > 0 && row[k - 1] < 0) {
                int lo = 0;
                k--;
                while (lo < k) {
                    const int mid = (lo + k) >> 1;
                    if (row[mid] < 0) k = mid; else lo = mid + 1;
                }
            }
            need = static_cast<int>(want) - k;
            first[s] = k;
        }
        int total;
        const int r = block_scan(need, m, &total);
        if (s < B) base[s] = need_total + r;
        need_total += total;
    }
    __syncthreads();
    int got = 0;
    if (need_total > 0)
        got = hand_out(ref, npages, need_total, m, [&](int r, int page) {
            int lo = 0, hi = B - 1;
            while (lo < hi) {  // the last take whose first rank is <= r: it needs at least one page
                const int mid = (lo + hi + 1) >> 1;
                if (base[mid] <= r) lo = mid; else hi = mid - 1;
            }
            table[static_cast<long>(lo) * maxpages + first[lo] + r - base[lo]] = page;
            ref[page] = 1;
        });
    if (threadIdx.x == 0) status[0] = need_total - got;
}

// Take s gives every page of its row back (each entry once, whoever else releases the same row); one warp.
__device__ __forceinline__ void release_row(int *table, int *ref, int s, int npages, int maxpages, int lane) {
    int *row = table + static_cast<long>(s) * maxpages;
    for (int k = 0; k < maxpages; k += 32) {
        int p = -1;
        if (k + lane < maxpages && row[k + lane] >= 0) p = atomicExch(row + k + lane, -1);
        if (p >= npages) record_error(OUMU_DEVERR_PAGE);
        else if (p >= 0) atomicSub(ref + p, 1);
        if (!__any_sync(0xffffffffu, p >= 0)) break;  // rows are filled from the front
    }
}

__global__ void __launch_bounds__(256) k_pages_free(int *table, int *ref, int *lens, const int *takes, int n, int B,
                                                    int npages, int maxpages) {
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= n) return;
    const int s = takes[i];
    if (s < 0 || s >= B) {
        if (lane == 0) record_error(OUMU_DEVERR_PAGE);
        return;
    }
    release_row(table, ref, s, npages, maxpages, lane);
    if (lane == 0) lens[s] = 0;
}

// Whether pair i of a fork is carried out: takes in range, no earlier pair fills the same take, and no pair fills the
// take it reads. Called by whole warps.
__device__ __forceinline__ bool pair_ok(const int *src, const int *dst, int n, int i, int B, int lane) {
    const int a = src[i], b = dst[i];
    bool ok = a >= 0 && a < B && b >= 0 && b < B && a != b;
    for (int j = lane; j < n; j += 32) {
        const int d = dst[j];
        ok = ok && !(d == a || (j < i && d == b));
    }
    return __all_sync(0xffffffffu, ok);
}

// Fork, the tables, a warp per pair: the target's row is given back and filled with the source's full pages in one pass
// (no other pair reads or writes it); then the lowest free pages go to the last, partly filled pages in the order of
// the pairs.
__global__ void __launch_bounds__(NT) k_pages_fork(int *table, int *ref, int *lens, const int *src, const int *dst,
                                                   int n, int *status, int B, int npages, int maxpages) {
    __shared__ ScanMem m;
    __shared__ int rank[BMAX];  // pair -> its rank among those that need a page; -1 needs none, -2 not carried out
    __shared__ int pair[BMAX];  // rank -> pair
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    for (int i = warp; i < n; i += NT / 32) {
        if (!pair_ok(src, dst, n, i, B, lane)) {
            if (lane == 0) {
                record_error(OUMU_DEVERR_PAGE);
                rank[i] = -2;
            }
            continue;
        }
        int L = lens[src[i]];
        if (L < 0 || L > static_cast<long>(maxpages) * PAGE) {
            if (lane == 0) record_error(OUMU_DEVERR_LENGTH);
            L = 0;
        }
        const int full = L / PAGE, all = (L + PAGE - 1) / PAGE;
        const int *from = table + static_cast<long>(src[i]) * maxpages;
        int *to = table + static_cast<long>(dst[i]) * maxpages;
        bool bad = false;
        for (int k0 = 0; k0 < maxpages; k0 += 32) {
            const int k = k0 + lane;
            const int old = k < maxpages ? to[k] : -1, p = k < all ? from[k] : -1;
            bad = bad || (k < all && (p < 0 || p >= npages));
            const bool share = k < full && p >= 0 && p < npages;
            if (old >= npages) record_error(OUMU_DEVERR_PAGE);
            else if (old >= 0) atomicSub(ref + old, 1);
            if (share) atomicAdd(ref + p, 1);
            if (k < maxpages) to[k] = share ? p : -1;
            // rows are filled from the front: nothing behind
            if (k0 + 32 >= all && !__any_sync(0xffffffffu, old >= 0)) break;
        }
        if (__any_sync(0xffffffffu, bad)) {  // the source lacks pages of its own positions: nothing to share
            if (lane == 0) record_error(OUMU_DEVERR_PAGE);
            __syncwarp();
            release_row(table, ref, dst[i], npages, maxpages, lane);
            L = 0;
        }
        if (lane == 0) {
            lens[dst[i]] = L;
            rank[i] = L % PAGE ? 0 : -1;
        }
    }
    __syncthreads();
    int want = 0;
    for (int i0 = 0; i0 < n; i0 += NT) {
        const int i = i0 + threadIdx.x;
        const int need = i < n && rank[i] == 0;
        int total;
        const int r = block_scan(need, m, &total);
        if (need) {
            rank[i] = want + r;
            pair[want + r] = i;
        }
        want += total;
    }
    __syncthreads();
    int got = 0;
    if (want > 0)
        got = hand_out(ref, npages, want, m, [&](int r, int page) {
            const int d = dst[pair[r]];
            table[static_cast<long>(d) * maxpages + lens[d] / PAGE] = page;
            ref[page] = 1;
        });
    if (got < want) {
        __syncthreads();
        for (int i = warp; i < n; i += NT / 32) {  // no page left for them: they end up empty
            if (rank[i] < got) continue;
            release_row(table, ref, dst[i], npages, maxpages, lane);
            if (lane == 0) lens[dst[i]] = 0;
        }
    }
    if (threadIdx.x == 0) status[0] = want - got;
}

// 16-byte copy of one page by a block of 256 threads.
__device__ __forceinline__ void copy_page(const uint4 *from, uint4 *to, int vecs) {
    int v = threadIdx.x;
    for (; v + 3 * 256 < vecs; v += 4 * 256) {
        const uint4 a = from[v], b = from[v + 256], c = from[v + 512], d = from[v + 768];
        to[v] = a;
        to[v + 256] = b;
        to[v + 512] = c;
        to[v + 768] = d;
    }
    for (; v < vecs; v += 256) to[v] = from[v];
}

// Fork, the bytes: the source's last, partly filled page into the targets' own. A block per layer and group of pairs, a
// warp of it finding out each pair's pages; pairs of one source, which follow one another in the usual call, read its
// page once. Bound by HBM: 64 takes, 36 layers of 20 KB pages, 47 MB written.
constexpr int PAIRS = 8;
__global__ void __launch_bounds__(256) k_pages_fork_copy(uint8_t *pools, long layer_stride, long page_bytes,
                                                         const int *table, const int *lens, const int *src,
                                                         const int *dst, int n, int B, int npages, int maxpages) {
    __shared__ int from[PAIRS], to[PAIRS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = blockIdx.x * PAIRS + warp;
    const bool ok = i < n && pair_ok(src, dst, n, i, B, lane);
    pdl_wait();
    int a = -1, b = -1;
    if (ok) {
        const int d = dst[i], L = lens[d];
        if (L > 0 && L % PAGE) {
            a = table[static_cast<long>(src[i]) * maxpages + L / PAGE];
            b = table[static_cast<long>(d) * maxpages + L / PAGE];
        }
    }
    if (lane == 0) {
        from[warp] = a >= 0 && a < npages && b >= 0 && b < npages ? a : -1;
        to[warp] = b;
    }
    __syncthreads();
    uint8_t *pool = pools + blockIdx.y * layer_stride;
    const int vecs = static_cast<int>(page_bytes / 16);
    constexpr int V = 5;  // 16-byte vectors a thread holds: a 20 KB page (2 kv heads of 128) at once
    for (int v0 = threadIdx.x; v0 < vecs; v0 += V * 256) {
        uint4 x[V];
        int have = -1;
#pragma unroll 1
        for (int k = 0; k < PAIRS; k++) {
            const int f = from[k];
            if (f < 0) continue;
            if (f != have) {
                const uint4 *p = reinterpret_cast<const uint4 *>(pool + f * page_bytes);
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (v0 + e * 256 < vecs) x[e] = p[v0 + e * 256];
                have = f;
            }
            uint4 *q = reinterpret_cast<uint4 *>(pool + to[k] * page_bytes);
#pragma unroll
            for (int e = 0; e < V; e++)
                if (v0 + e * 256 < vecs) __stcs(q + v0 + e * 256, x[e]);
        }
    }
}

// Packing a pool. Workspace: [moves][pages in use][pad 2] from[npages / 2 + 1] to[npages / 2 + 1] map[npages].
struct Plan {
    int *head, *from, *to, *map;
    __host__ __device__ Plan(void *ws, int npages)
        : head(static_cast<int *>(ws)), from(head + 4), to(from + npages / 2 + 1), map(to + npages / 2 + 1) {}
    static size_t bytes(int npages) { return 4 * (4 + 2 * (static_cast<size_t>(npages) / 2 + 1) + npages); }
};

// The k-th page in use at or past `live` (the number in use) goes to the k-th free page below it.
__global__ void __launch_bounds__(NT) k_pages_plan(int *ref, void *ws, int *status, int npages) {
    __shared__ ScanMem m;
    const Plan P(ws, npages);
    pdl_trigger();
    int live = 0;
    for (int i0 = 0; i0 < npages; i0 += 4 * NT) {
        int c = 0, total;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = i0 + 4 * static_cast<int>(threadIdx.x) + e;
            c += i < npages && ref[i] > 0;
        }
        block_scan(c, m, &total);
        live += total;
    }
    int holes = 0, moves = 0;
    for (int i0 = 0; i0 < npages; i0 += 4 * NT) {
        bool h[4], v[4];
        int c = 0, total;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = i0 + 4 * static_cast<int>(threadIdx.x) + e;
            const bool used = i < npages && ref[i] > 0;
            h[e] = i < live && !used;
            v[e] = i >= live && used;
            if (i < npages) P.map[i] = i < live ? i : -1;
            c += h[e] + (v[e] << 16);  // both counts of a chunk of 4096 fit 16 bits
        }
        const int r = block_scan(c, m, &total);
        int a = holes + (r & 0xffff), b = moves + (r >> 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = i0 + 4 * static_cast<int>(threadIdx.x) + e;
            if (h[e]) P.to[a++] = i;
            if (v[e]) P.from[b++] = i;
        }
        holes += total & 0xffff;
        moves += total >> 16;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += NT) {
        const int a = P.from[k], b = P.to[k];
        P.map[a] = b;
        ref[b] = ref[a];
        ref[a] = 0;
    }
    if (threadIdx.x == 0) {
        P.head[0] = moves;
        P.head[1] = live;
        status[0] = live;
        status[1] = moves;
    }
}

__global__ void __launch_bounds__(256) k_pages_move(uint8_t *pools, long layer_stride, int layers, long page_bytes,
                                                    int *table, void *ws, int B, int npages, int maxpages) {
    const Plan P(ws, npages);
    pdl_wait();
    const int moves = P.head[0];
    const long entries = static_cast<long>(B) * maxpages, step = static_cast<long>(gridDim.x) * 256;
    for (long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x; i < entries; i += step) {
        const int p = table[i];
        if (p < 0) continue;
        const int q = p < npages ? P.map[p] : -1;
        if (q < 0) record_error(OUMU_DEVERR_PAGE);  // a page that no count knows: left as it is
        else if (q != p) table[i] = q;
    }
    for (long k = blockIdx.x; k < static_cast<long>(moves) * layers; k += gridDim.x) {
        const int mv = static_cast<int>(k / layers);
        uint8_t *pool = pools + (k % layers) * layer_stride;
        copy_page(reinterpret_cast<const uint4 *>(pool + P.from[mv] * page_bytes),
                  reinterpret_cast<uint4 *>(pool + P.to[mv] * page_bytes), static_cast<int>(page_bytes / 16));
    }
}

}  // namespace pg
