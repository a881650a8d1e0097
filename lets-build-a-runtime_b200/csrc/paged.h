// paged.h -- what the paged-attention kernels share: how a call's work is cut
// into units and spread over the grid, and the layout of unfinished results.
//
// The rows of a sequence are its (new token, query head of a cache head)
// pairs, token-major, cut into tiles of R rows; an item is one row tile of one
// sequence and cache head, and its units are the key tiles of KT positions
// that at least one of its rows sees.  Lengths are known on the device only,
// so every block derives the same list from them: sequences in order, then row
// tiles, cache heads, key tiles.  Block c takes units [c * per, (c + 1) * per)
// of the whole list, so blocks finish together however unequal the sequences
// are.  An item that falls into several blocks leaves an unnormalised sum, a
// maximum and a weight sum per row in each (slot 2c + 1 from the block where
// it starts, slot 2c from the others); the join kernel adds them in block
// order, so results do not depend on timing.
#pragma once
#include "rt_internal.h"

namespace rt {

struct PagedArgs {
    RtPagedAttention a;
    float* part;       // [2 * blocks][R * DP + 2 * R]: sums, maxima (log2 units), weight sums
    int* err;
    int group;         // query heads per cache head
    int whole;         // 1: a block takes whole items (no join)
    int min_units;
    int page_shift;    // log2 of the page size, -1 when it is not a power of two
};

struct PagedSeq {
    int b, first, n, L;   // sequence, first row of q, new tokens, cached positions
};
struct PagedTiles {
    int t0, count;        // key tiles (at least one, also where nothing is seen)
    int lo, hi;           // positions that some row of the tile sees
};

#ifdef __CUDACC__
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& p, int b) {
    PagedSeq s;
    s.b = b;
    s.first = p.a.cu_new[b];
    s.n = p.a.cu_new[b + 1] - s.first;
    s.L = p.a.kv_lens[b];
    if (s.first < 0 || s.n < 0 || s.n > p.a.total_new - s.first) {
        atomicCAS(p.err, 0, KERR_LENGTH);
        s.first = s.n = 0;
    }
    const int64_t most = (int64_t)p.a.table_width * p.a.cache.page_size;
    if (s.L < 0 || s.L > most) {
        atomicCAS(p.err, 0, KERR_LENGTH);
        s.L = s.L < 0 ? 0 : (int)most;
    }
    return s;
}

template <int R, int KT>
__device__ __forceinline__ PagedTiles paged_tiles(const PagedArgs& p, const PagedSeq& s, int qt) {
    PagedTiles t;
    const int last = (min((qt + 1) * R, s.n * p.group) - 1) / p.group, first = qt * R / p.group;
    t.hi = p.a.causal ? min(s.L, s.L - s.n + last + 1) : s.L;
    t.lo = p.a.window > 0 ? max(0, s.L - s.n + first - p.a.window + 1) : 0;
    if (t.lo >= t.hi) t.lo = t.hi = 0;
    t.t0 = t.lo / KT;
    t.count = max(1, (t.hi + KT - 1) / KT - t.t0);
    return t;
}

template <int R>
__device__ __forceinline__ int paged_row_tiles(const PagedArgs& p, const PagedSeq& s) {
    return (int)(((int64_t)s.n * p.group + R - 1) / R);
}

template <int R, int KT>
__device__ __forceinline__ int paged_units(const PagedArgs& p, int b) {
    if (b >= p.a.n_seqs) return 0;
    const PagedSeq s = paged_seq(p, b);
    const int nq = paged_row_tiles<R>(p, s);
    if (p.whole) return nq * p.a.cache.n_heads;
    int sum = 0;
    for (int q = 0; q < nq; q++) sum += paged_tiles<R, KT>(p, s, q).count;
    return sum * p.a.cache.n_heads;
}

// Inclusive sum over the block's T threads; `total` gets the block's sum.
template <int T>
__device__ __forceinline__ int paged_scan(int x, int* sh, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < T / 32; w++) {
        if (w < warp) before += sh[w];
        all += sh[w];
    }
    *total = all;
    return x + before;
}

// Where a block stands in the list of units.
struct PagedCursor {
    PagedSeq s;
    PagedTiles t;
    int nq, qt, h, i;     // row tiles of the sequence; row tile, cache head, key tile inside the item

    template <int R, int KT>
    __device__ __forceinline__ void open(const PagedArgs& p, int b) {   // the first item at or after sequence b
        qt = h = i = 0;
        nq = 0;
        s.b = b;
        while (s.b < p.a.n_seqs) {
            s = paged_seq(p, s.b);
            nq = paged_row_tiles<R>(p, s);
            if (nq > 0) break;
            s.b++;
        }
        if (nq > 0) t = paged_tiles<R, KT>(p, s, 0);
    }
    template <int R, int KT>
    __device__ __forceinline__ void next_item(const PagedArgs& p) {
        i = 0;
        if (++h < p.a.cache.n_heads) return;
        h = 0;
        if (++qt < nq) t = paged_tiles<R, KT>(p, s, qt);
        else open<R, KT>(p, s.b + 1);
    }
};

// The units of this call and the block's share.  `unit`: the first unit to
// look at (c * per).  False when the block has none.  sh: T / 32 + 2 ints.
template <int T, int R, int KT>
__device__ __forceinline__ bool paged_schedule(const PagedArgs& p, int block, int blocks, int* sh, PagedCursor& c, int& u,
                                               int& per, int& total) {
    int mine = paged_units<R, KT>(p, threadIdx.x), all;
    int incl = paged_scan<T>(mine, sh, &all);
    total = all;
    for (int base = T; base < p.a.n_seqs; base += T) {
        int part;
        paged_scan<T>(paged_units<R, KT>(p, base + threadIdx.x), sh, &part);
        total += part;
    }
    per = max(p.min_units, (total + blocks - 1) / blocks);
    u = (int)min((int64_t)block * per, (int64_t)0x7fffffff);
    if (u >= total) return false;
    int carry = 0;
    for (int base = 0;; base += T) {
        if (base) {
            mine = paged_units<R, KT>(p, base + threadIdx.x);
            incl = paged_scan<T>(mine, sh, &all);
        }
        const int first = carry + incl - mine;
        if (first <= u && u < first + mine) {
            sh[T / 32] = base + threadIdx.x;
            sh[T / 32 + 1] = first;
        }
        carry += all;
        if (u < carry) break;
    }
    __syncthreads();
    const int b = sh[T / 32];
    int r = u - sh[T / 32 + 1];
    __syncthreads();
    c.open<R, KT>(p, b);
    while (true) {   // row tile, then head and key tile
        const int per_head = p.whole ? 1 : c.t.count, n = per_head * p.a.cache.n_heads;
        if (r < n) {
            c.h = r / per_head;
            c.i = r % per_head;
            return true;
        }
        r -= n;
        c.t = paged_tiles<R, KT>(p, c.s, ++c.qt);
    }
}

// Position -> page and slot in it.
__device__ __forceinline__ void paged_split(const PagedArgs& p, int pos, int& page, int& slot) {
    if (p.page_shift >= 0) {
        page = pos >> p.page_shift;
        slot = pos & (p.a.cache.page_size - 1);
    } else {
        page = pos / p.a.cache.page_size;
        slot = pos - page * p.a.cache.page_size;
    }
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
#endif

// One launch (and the join, when items can be split): k_paged_few.cu for
// tiles of 8 or 16 rows on the warp-level matrix instructions.
size_t paged_few_workspace(const RtPagedAttention& p);
Status launch_paged_few(PagedArgs& p, void* ws, cudaStream_t st);

}  // namespace rt
