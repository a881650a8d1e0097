// paged.h -- what the paged-attention kernels share: how a call's work is cut
// into units and spread over the grid, and the layout of unfinished results.
//
// The rows of a sequence are its (new token, query head of a cache head)
// pairs, token-major, cut into tiles of R rows; an item is one row tile of one
// sequence and one group of cache heads, and its units are the key tiles of 2^key_shift
// positions that at least one of its rows sees.  Lengths are known on the device only,
// so every block derives the same list from them: sequences in order, then row
// tiles, cache heads, key tiles.  Block c takes units [c * per, (c + 1) * per)
// of the whole list, so blocks finish together however unequal the sequences
// are.  An item that falls into several blocks leaves an unnormalised sum, a
// maximum and a weight sum per row in each (slot 2c + 1 from the block where
// it starts, slot 2c from the others); the join kernel adds them in block
// order, so results do not depend on timing.
#pragma once
#include <cuda_bf16.h>

#include "rt_internal.h"

namespace rt {

struct PagedNote;
struct PagedArgs {
    RtPagedAttention a;
    float* part;       // [2 * blocks][heads of a group][R * DP + 2 * R]: sums, maxima (log2 units), weight sums
    PagedNote* notes;  // per block: the item to be joined there
    int* err;
    int group;         // query heads per cache head
    int whole;         // 1: a block takes whole items (no join)
    int min_units;
    int key_shift;     // log2 of the positions of a key tile
    int head_group;    // cache heads of an item
    int head_groups;
    int page_shift;    // log2 of the page size, -1 when it is not a power of two
    bool vec_q, vec_out;   // every row of q / out starts on 16 bytes
};
// Workspace: the notes, then the slots.
inline size_t paged_workspace(int blocks, int head_group, int slot_floats) {
    return (((size_t)blocks * 32 + 255) & ~(size_t)255) + (size_t)blocks * 2 * head_group * slot_floats * sizeof(float);
}
inline void paged_set_workspace(PagedArgs& p, void* ws, int blocks) {
    p.notes = static_cast<PagedNote*>(ws);
    p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + (((size_t)blocks * 32 + 255) & ~(size_t)255));
}
inline bool paged_rows16(const void* p, const int64_t st[2], int dtype) {
    return aligned16(p) && (st[0] * dtype_bytes(dtype)) % 16 == 0 && (st[1] * dtype_bytes(dtype)) % 16 == 0;
}

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

// The first position that a token at `at` sees (at < 0: before the first; windows of any size).
__device__ __forceinline__ int paged_lo(const PagedArgs& p, int at) {
    return p.a.window > 0 && at >= p.a.window ? at - p.a.window + 1 : 0;
}

template <int R>
__device__ __forceinline__ PagedTiles paged_tiles(const PagedArgs& p, const PagedSeq& s, int qt) {
    PagedTiles t;
    const int last = (min((qt + 1) * R, s.n * p.group) - 1) / p.group, first = qt * R / p.group;
    t.hi = p.a.causal ? min(s.L, s.L - s.n + last + 1) : s.L;
    t.lo = paged_lo(p, s.L - s.n + first);
    if (t.lo >= t.hi) t.lo = t.hi = 0;
    t.t0 = t.lo >> p.key_shift;
    t.count = max(1, ((t.hi + (1 << p.key_shift) - 1) >> p.key_shift) - t.t0);
    return t;
}

template <int R>
__device__ __forceinline__ int paged_row_tiles(const PagedArgs& p, const PagedSeq& s) {
    return (int)(((int64_t)s.n * p.group + R - 1) / R);
}

template <int R>
__device__ __forceinline__ int paged_units(const PagedArgs& p, const PagedSeq& s) {
    const int nq = paged_row_tiles<R>(p, s);
    if (p.whole) return nq * p.head_groups;
    int sum = 0;
    for (int q = 0; q < nq; q++) sum += paged_tiles<R>(p, s, q).count;
    return sum * p.head_groups;
}

// `refused`: set where the sequence's offsets are refused.
template <int R>
__device__ __forceinline__ int paged_units(const PagedArgs& p, int b, bool& refused) {
    if (b >= p.a.n_seqs) return 0;
    const PagedSeq s = paged_seq(p, b);
    if (s.n == 0 && p.a.cu_new[b] != p.a.cu_new[b + 1]) refused = true;
    return paged_units<R>(p, s);
}

// Zeros, and a log-sum-exp of -inf, for the rows of q that no sequence owns: padding before the
// first and after the last sequence's, rows of a refused one.  A warp per row.
template <int T>
__device__ __forceinline__ void paged_rest(const PagedArgs& p) {
    const int lane = threadIdx.x & 31, total = p.a.total_new, D = p.a.cache.head_dim;
    for (int64_t row = (int64_t)blockIdx.x * (T / 32) + (threadIdx.x >> 5); row < total; row += (int64_t)gridDim.x * (T / 32)) {
        bool owned = false;
        for (int b = lane; b - lane < p.a.n_seqs && !owned; b += 32) {
            bool mine = false;
            if (b < p.a.n_seqs) {
                const int first = p.a.cu_new[b], n = p.a.cu_new[b + 1] - first;
                mine = first >= 0 && n >= 0 && n <= total - first && row >= first && row - first < n;
            }
            owned = __any_sync(0xffffffffu, mine);
        }
        if (owned) continue;
        for (int h = 0; h < p.a.n_q_heads; h++) {
            const int64_t at = row * p.a.out_stride[0] + h * p.a.out_stride[1];
            for (int d = lane; d < D; d += 32) {
                if (p.a.dtype == RT_BF16) static_cast<__nv_bfloat16*>(p.a.out)[at + d] = __float2bfloat16_rn(0.0f);
                else static_cast<float*>(p.a.out)[at + d] = 0.0f;
            }
            if (p.a.lse && lane == 0) p.a.lse[row * p.a.n_q_heads + h] = -INFINITY;
        }
    }
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
    int nq, qt, h, i;     // row tiles of the sequence; row tile, head group, key tile inside the item

    template <int R>
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
        if (nq > 0) t = paged_tiles<R>(p, s, 0);
    }
    template <int R>
    __device__ __forceinline__ void next_item(const PagedArgs& p) {
        i = 0;
        if (++h < p.head_groups) return;
        h = 0;
        if (++qt < nq) t = paged_tiles<R>(p, s, qt);
        else open<R>(p, s.b + 1);
    }
};

// The units of this call and the block's share.  `u`: the first unit to
// look at (c * per).  False when the block has none.  `rest`: some rows of q
// belong to no sequence.  sh: T / 32 + 2 ints.
template <int T, int R>
__device__ __forceinline__ bool paged_schedule(const PagedArgs& p, int block, int blocks, int* sh, PagedCursor& c, int& u,
                                               int& per, int& total, bool& rest) {
    auto settle = [&](int r) {   // row tile, then head group and key tile, from units after the sequence's first
        while (true) {
            const int per_head = p.whole ? 1 : c.t.count, n = per_head * p.head_groups;
            if (r < n) {
                c.h = r / per_head;
                c.i = r % per_head;
                return;
            }
            r -= n;
            c.t = paged_tiles<R>(p, c.s, ++c.qt);
        }
    };
    if (p.a.n_seqs <= 32) {   // every warp for itself, a lane per sequence: no barrier, every length read once
        const int lane = threadIdx.x & 31;
        PagedSeq s = {lane, 0, 0, 0};
        if (lane < p.a.n_seqs) s = paged_seq(p, lane);
        const int mine = s.n > 0 ? paged_units<R>(p, s) : 0;
        rest = __reduce_add_sync(0xffffffffu, s.n) != p.a.total_new;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        total = __shfl_sync(0xffffffffu, incl, 31);
        per = max(p.min_units, (total + blocks - 1) / blocks);
        u = (int)min((int64_t)block * per, (int64_t)0x7fffffff);
        if (u >= total) return false;
        const int from = __ffs(__ballot_sync(0xffffffffu, u < incl)) - 1;
        c.s.b = from;
        c.s.first = __shfl_sync(0xffffffffu, s.first, from);
        c.s.n = __shfl_sync(0xffffffffu, s.n, from);
        c.s.L = __shfl_sync(0xffffffffu, s.L, from);
        const int r = u - __shfl_sync(0xffffffffu, incl - mine, from);
        c.qt = c.h = c.i = 0;
        c.nq = paged_row_tiles<R>(p, c.s);
        c.t = paged_tiles<R>(p, c.s, 0);
        settle(r);
        return true;
    }
    bool left = p.a.cu_new[0] != 0 || p.a.cu_new[p.a.n_seqs] != p.a.total_new;
    int mine = paged_units<R>(p, (int)threadIdx.x, left), all;
    int incl = paged_scan<T>(mine, sh, &all);
    total = all;
    for (int base = T; base < p.a.n_seqs; base += T) {
        int part;
        paged_scan<T>(paged_units<R>(p, base + (int)threadIdx.x, left), sh, &part);
        total += part;
    }
    rest = __syncthreads_or(left);
    per = max(p.min_units, (total + blocks - 1) / blocks);
    u = (int)min((int64_t)block * per, (int64_t)0x7fffffff);
    if (u >= total) return false;
    int carry = 0;
    for (int base = 0;; base += T) {
        if (base) {
            mine = paged_units<R>(p, base + (int)threadIdx.x, left);
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
    const int r = u - sh[T / 32 + 1];
    __syncthreads();
    c.open<R>(p, b);
    settle(r);
    return true;
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

// Where row `row` (of the sequence's rows under cache head h) goes, and its
// log-sum-exp from its maximum (log2 units) and weight sum.
__device__ __forceinline__ int64_t paged_out_at(const PagedArgs& p, const PagedSeq& s, int h, int row) {
    return (int64_t)(s.first + row / p.group) * p.a.out_stride[0] + (h * p.group + row % p.group) * p.a.out_stride[1];
}
// Four features from d on (d a multiple of 4), as one store where rows allow it.
__device__ __forceinline__ void paged_store4(const PagedArgs& p, const PagedSeq& s, int h, int row, int d, float a, float b, float c, float e) {
    const int64_t at = paged_out_at(p, s, h, row) + d;
    if (p.a.dtype == RT_BF16) {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out) + at;
        if (p.vec_out) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, e);
            *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
        } else {
            out[0] = __float2bfloat16_rn(a);
            out[1] = __float2bfloat16_rn(b);
            out[2] = __float2bfloat16_rn(c);
            out[3] = __float2bfloat16_rn(e);
        }
    } else {
        float* out = static_cast<float*>(p.a.out) + at;
        if (p.vec_out) {
            *reinterpret_cast<float4*>(out) = make_float4(a, b, c, e);
        } else {
            out[0] = a;
            out[1] = b;
            out[2] = c;
            out[3] = e;
        }
    }
}
__device__ __forceinline__ void paged_store_lse(const PagedArgs& p, const PagedSeq& s, int h, int row, float m, float l) {
    if (p.a.lse)
        p.a.lse[(int64_t)(s.first + row / p.group) * p.a.n_q_heads + h * p.group + row % p.group] =
            l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// A block that starts inside an item leaves a note for the join kernel if it is
// the first one to do so: what is to be added up there.  Every block writes one.
struct PagedNote {
    int first, n, L, b;        // the sequence
    int qt, h, from, count;    // row tile, head group; blocks the item lies in
};
template <int R>
__device__ __forceinline__ void paged_note(const PagedArgs& p, bool some, const PagedCursor& c, int u, int per) {
    if (p.whole || threadIdx.x) return;
    PagedNote x = {0, 0, 0, 0, 0, 0, 0, 0};
    if (some && c.i > 0) {
        const int first = u - c.i, from = first / per;
        if (from == (int)blockIdx.x - 1) x = {c.s.first, c.s.n, c.s.L, c.s.b, c.qt, c.h, from, (first + c.t.count - 1) / per - from + 1};
    }
    p.notes[blockIdx.x] = x;
}

// Adds up the items that fell into several blocks: block (c, y, z) takes what
// block c + 1 of the main kernel noted, some rows of the item, head z of its
// group.  An item of a long sequence may lie in hundreds of blocks: their
// maxima are read side by side, and the sums by several threads per feature,
// each with several loads under way; the order of additions is fixed.
constexpr int JOIN_THREADS = 256;
template <int DP, int R>
struct Join {
    static constexpr int ROWS = R <= 32 ? R / 4 : 16;                  // rows of a block
    static constexpr int ITEMS = ROWS * DP / 4;                        // 4 features of a row each
    static constexpr int PARTS = ITEMS >= JOIN_THREADS ? 1 : JOIN_THREADS / ITEMS;   // threads that share an item
};
template <int DP, int R>
__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(const __grid_constant__ PagedArgs p, int blocks) {
    using J = Join<DP, R>;
    __shared__ float top[J::ROWS][JOIN_THREADS / J::ROWS], sums[J::PARTS > 1 ? JOIN_THREADS : 1][4];
    extern __shared__ float factor[];                      // [blocks of the item][ROWS]
    asm volatile("griddepcontrol.wait;" ::: "memory");     // (launched while the main kernel runs)
    const PagedNote note = p.notes[blockIdx.x + 1];
    if (note.count == 0) return;
    const int c0 = note.from, n = note.count;
    constexpr int SLOT = R * DP + 2 * R;
    const int z = blockIdx.z, h = note.h * p.head_group + z;
    auto slot_of = [&](int k) { return p.part + ((int64_t)(2 * (c0 + k) + (k == 0)) * p.head_group + z) * SLOT; };
    const PagedSeq s = {note.b, note.first, note.n, note.L};
    const int row0 = note.qt * R, rows = min(R, s.n * p.group - row0);
    for (int first_row = blockIdx.y * J::ROWS; first_row < rows; first_row += gridDim.y * J::ROWS) {
        __syncthreads();
        // ---- the rows' maxima and weight sums ----
        const int tid = threadIdx.x, lr = tid % J::ROWS, lane = tid / J::ROWS;
        constexpr int LANES = JOIN_THREADS / J::ROWS;
        const bool mine = first_row + lr < rows;
        float m = -INFINITY;
        if (mine)
            for (int k = lane; k < n; k += LANES) {
                const float x = slot_of(k)[R * DP + first_row + lr];
                factor[k * J::ROWS + lr] = x;
                m = fmaxf(m, x);
            }
        top[lr][lane] = m;
        __syncthreads();
        for (int k = 0; k < LANES; k++) m = fmaxf(m, top[lr][k]);
        __syncthreads();
        float ls = 0.0f;
        if (mine)
            for (int k = lane; k < n; k += LANES) {
                // a share that saw nothing has no weight and is left out; one whose scores are all
                // NaN has no maximum, but a weight sum of NaN, which goes into the result
                const float l = slot_of(k)[R * DP + R + first_row + lr];
                const float f = l == 0.0f ? -1.0f : l == l ? exp2_fast(factor[k * J::ROWS + lr] - m) : l;
                factor[k * J::ROWS + lr] = f;
                ls += f < 0.0f ? 0.0f : l * f;
            }
        top[lr][lane] = ls;
        __syncthreads();
        ls = 0.0f;
        for (int k = 0; k < LANES; k++) ls += top[lr][k];
        if (mine && lane == 0) paged_store_lse(p, s, h, row0 + first_row + lr, m, ls);
        __syncthreads();
        if (lane == 0) top[lr][0] = ls == 0.0f ? 0.0f : 1.0f / ls;
        __syncthreads();
        // ---- the sums ----
        for (int e0 = 0; e0 < J::ITEMS; e0 += JOIN_THREADS) {
            const int e = e0 + tid % (JOIN_THREADS / J::PARTS), part = tid / (JOIN_THREADS / J::PARTS);
            const int r = e / (DP / 4), d = e % (DP / 4) * 4;
            float sum[4] = {0, 0, 0, 0};
            if (first_row + r < rows) {
#pragma unroll 8
                for (int k = part; k < n; k += J::PARTS) {
                    const float f = factor[k * J::ROWS + r];
                    const float4 x = f < 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *reinterpret_cast<const float4*>(slot_of(k) + (first_row + r) * DP + d);
                    sum[0] += x.x * f; sum[1] += x.y * f; sum[2] += x.z * f; sum[3] += x.w * f;
                }
            }
            if constexpr (J::PARTS > 1) {
#pragma unroll
                for (int j = 0; j < 4; j++) sums[tid][j] = sum[j];
                __syncthreads();
                if (part == 0) {
#pragma unroll
                    for (int k = 1; k < J::PARTS; k++)
#pragma unroll
                        for (int j = 0; j < 4; j++) sum[j] += sums[tid + k * (JOIN_THREADS / J::PARTS)][j];
                }
            }
            if (part == 0 && first_row + r < rows && d < p.a.cache.head_dim) {
                const float inv = top[r][0];
                paged_store4(p, s, h, row0 + first_row + r, d, sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
            }
        }
    }
}
template <int DP, int R>
Status launch_paged_join(const PagedArgs& p, int blocks, cudaStream_t st) {
    using J = Join<DP, R>;
    cudaLaunchConfig_t cfg = {};
    const int64_t most = (int64_t)(p.a.max_new < p.a.total_new ? p.a.max_new : p.a.total_new) * p.group;   // (a bound of the host's: blocks loop)
    const int tall = (int)(most < 1 ? 1 : most < R ? most : R);
    cfg.gridDim = dim3(blocks - 1, (tall + J::ROWS - 1) / J::ROWS, p.head_group);
    cfg.blockDim = dim3(JOIN_THREADS);
    cfg.dynamicSmemBytes = (size_t)blocks * J::ROWS * sizeof(float);   // an item in every block at most
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    RT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_join_kernel<DP, R>, p, blocks));
    return Status::ok();
}
#endif

// One launch (and the join, when items can be split): k_paged_few.cu for
// tiles of 8, 16 or 32 rows on the warp-level matrix instructions.
size_t paged_few_workspace(const RtPagedAttention& p);
Status launch_paged_few(PagedArgs& p, void* ws, cudaStream_t st);
// k_paged_tiles.cu for tiles of 128 rows on the tensor cores (tcgen05).
bool paged_tiles_takes(const RtPagedAttention& p);
size_t paged_tiles_workspace(const RtPagedAttention& p);
Status launch_paged_tiles(PagedArgs& p, void* ws, cudaStream_t st);

}  // namespace rt
