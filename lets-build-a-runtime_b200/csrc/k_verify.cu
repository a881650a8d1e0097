// k_verify.cu -- verification of drafted tokens (speculative sampling).
//
// A draft x proposed with probability q(x) is kept with probability
// min(1, p(x) / q(x)): u q(x) < p(x) for a given uniform u.  After the first
// refusal the next token comes from max(p - q, 0), normalised; together the
// sequence is distributed as if the target had sampled every token.
//
// Sampling is by inversion: the lowest token whose running sum of weights
// exceeds u times their total.  The weights are fixed-point integers (2^-40),
// so sums are exact, independent of the order and of how the vocabulary is
// split, and the token is a function of the inputs alone.
//
// Only the row where a sequence stops is read, once: 8 bytes per entry of the
// vocabulary in fp32, bound by HBM for many sequences and by latency for few.
// A cluster of up to 8 blocks takes a sequence, each a slice of the row: a
// block settles the drafts by itself (a few loads), sums its slice, sends its
// sum to the others, and the one in whose slice the running sum crosses finds
// the token there.  A slice streams through a ring in shared memory that bulk
// copies fill (rows of any alignment: what lies before the first and after the
// last 16-byte boundary is loaded and stored by threads).  Sums are kept for
// every piece, so only the piece with the token is looked at again.
//
// A warp copies, the others sum: what a block has under way is then bound by
// the ring alone, and one block of 16 + 1 warps per SM with six slots of 2 x 16
// KB does better than several smaller ones (128 rows of 131071 entries, fp32
// target and draft, 134 MB: 26 us = 5.2 TB/s; two blocks with 5 x 16 KB 30,
// three with 3 x 16 KB 35; loads into registers without a ring 50).  One
// sequence of 32000 entries takes 7.2 us, of which the loads that follow from
// one another (lengths, drafts, their probabilities, the row) are the most.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "rt_internal.h"
#include "sm100_ptx.h"

namespace rt {
namespace {

constexpr int VT = 512, MAX_CLUSTER = 8, BLOCKS_PER_SM = 1;   // VT threads that sum, and a warp that copies
constexpr int PIECE = 16384, SLOTS = 6;          // bytes of a row in a slot; slots
constexpr int ROW_SLOT = PIECE + 16;             // (a piece may start anywhere in its first 16 bytes)
constexpr int GROUPS = 128;                      // sums kept per slice, each of 2^k pieces
constexpr int RING_BYTES = SLOTS * 2 * ROW_SLOT;
constexpr int KERR_WAIT = 0x351;
constexpr uint64_t WAIT_NS = 200000000ull;

// w = a - b, clamped to [0, 1] (NaN: 0), in units of 2^-40, truncated: the
// steps of 2^-20 below it by adding 8 with rounding toward zero (whose last
// place is 2^-20), then the steps of 2^-40 of what is left, which is exact.
// Two 32-bit counts instead of a 64-bit integer: conversions to 64 bits run at
// a fraction of the rate, and the counts of a warp's entries in a group fit
// (2^20 per entry, at most 2^11 entries).
__device__ __forceinline__ void weight(float a, float b, uint32_t& hi, uint32_t& lo) {
    float w;
    asm("sub.sat.f32 %0, %1, %2;" : "=f"(w) : "f"(a), "f"(b));
    const float t = __fadd_rz(w, 8.0f);
    const float r = __fmaf_rz(w - (t - 8.0f), 1048576.0f, 8.0f);
    hi = __float_as_uint(t) - 0x41000000u;
    lo = __float_as_uint(r) - 0x41000000u;
}
__device__ __forceinline__ float load_prob(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_prob(const __nv_bfloat16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ unsigned long long warp_scan(unsigned long long x, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// A wait of a whole warp: all its lanes go on, or none.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
    return __all_sync(0xffffffffu, ptx::wait_short(bar, parity, abort_flag, err, KERR_WAIT, WAIT_NS));
}

// Entries [0, size) of a row from `base` (any alignment) as pieces in a ring.
template <class T>
struct RowPieces {
    static constexpr int C = PIECE / (int)sizeof(T);   // entries of a piece
    uint64_t base, end;
    uint32_t off;   // of the first entry in its 16 bytes
    __device__ RowPieces(const T* p, int size)
        : base(reinterpret_cast<uint64_t>(p)), end(base + (uint64_t)size * sizeof(T)), off((uint32_t)base & 15) {}
    // The 16-byte parts of piece c that lie within the row.
    __device__ __forceinline__ void bounds(int c, uint64_t& from, uint32_t& bytes) const {
        const uint64_t a = base + (uint64_t)c * PIECE, b = a + PIECE;
        from = c ? a & ~15ull : (a + 15) & ~15ull;
        const uint64_t to = min((b + 15) & ~15ull, end & ~15ull);
        bytes = to > from ? (uint32_t)(to - from) : 0;
    }
    // Its place in the slot is that of the row, so every piece starts at `off`.
    __device__ __forceinline__ uint32_t copy(int c, uint8_t* slot, uint64_t* bar) const {
        uint64_t from;
        uint32_t bytes;
        bounds(c, from, bytes);
        if (bytes) ptx::bulk_load(slot + (uint32_t)(from - (base - off + (uint64_t)c * PIECE)), reinterpret_cast<const void*>(from), bytes, bar);
        return bytes;
    }
    // The rest of piece c, an entry for each of 32 / sizeof(T) lanes: what lies before the copied
    // part and after it (less than 16 bytes each), or all of the piece if that is less than 32.
    __device__ __forceinline__ void edges(int c, uint8_t* slot, int e) const {
        constexpr int HALF = 16 / (int)sizeof(T);
        uint64_t from;
        uint32_t bytes;
        bounds(c, from, bytes);
        const uint64_t first = base + (uint64_t)c * PIECE, last = min(end, first + PIECE);
        const bool after = bytes && e >= HALF;
        const uint64_t at = after ? from + bytes + (e - HALF) * sizeof(T) : first + e * sizeof(T);
        if (at >= (after || !bytes ? last : from)) return;
        *reinterpret_cast<T*>(slot + (uint32_t)(at - (base - off + (uint64_t)c * PIECE))) = *reinterpret_cast<const T*>(at);
        ptx::fence_proxy_async_smem();   // a later piece's copy writes here
    }
};

template <class T>
__global__ void __launch_bounds__(VT + 32, BLOCKS_PER_SM) verify_kernel(const __grid_constant__ RtVerifyDraft v, int blocks, int slice, int group_shift, int* err) {
    constexpr int C = RowPieces<T>::C, PER = C / VT;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ unsigned long long parts[GROUPS][VT / 32], group_sums[GROUPS], sums[VT / 32], share[2][MAX_CLUSTER];
    __shared__ uint64_t full[SLOTS], empty[SLOTS];
    __shared__ int first, abort_flag;
    const int b = blockIdx.y, rank = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int N = v.n_drafts, V = v.vocab;
    const T* target = static_cast<const T*>(v.target) + b * v.target_stride[0];
    const T* draft = v.draft ? static_cast<const T*>(v.draft) + b * v.draft_stride[0] : nullptr;

    if (blocks > 1) ptx::cluster_started_arrive();

    // ---- how many drafts stand ----
    if (t == 0) {
        first = N;
        abort_flag = 0;
        for (int i = 0; i < SLOTS; i++) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], VT / 32);
        }
        ptx::fence_mbar_init();
    }
    int limit = v.draft_lens ? v.draft_lens[b] : N;
    const float u = v.sample_u[b];
    __syncthreads();
    for (int i = t; i < N; i += VT + 32) {   // (what lies beyond the limit is loaded along with it and not looked at)
        const int x = v.draft_tokens[b * N + i];
        const float au = v.accept_u[b * N + i];
        const bool known = x >= 0 && x < V;
        float p = 0.0f, q = 1.0f;
        if (known) {
            p = load_prob(target + i * v.target_stride[1] + x);
            if (draft) q = load_prob(draft + i * v.draft_stride[1] + x);
        }
        if (i < limit) {
            if (!known && rank == 0) atomicCAS(err, 0, KERR_TOKEN);
            if (!known || !(__fmul_rn(au, q) < p)) atomicMin(&first, i);
        }
    }
    if (limit < 0 || limit > N) {
        if (t == 0) atomicCAS(err, 0, KERR_LENGTH);
        limit = limit < 0 ? 0 : N;
    }
    __syncthreads();
    const int n = min(first, limit);
    bool residual = n < limit;
    const T* row = target + n * v.target_stride[1];
    const T* qrow = draft && residual ? draft + n * v.draft_stride[1] : nullptr;
    int point = !draft && residual ? v.draft_tokens[b * N + n] : -1;   // a certain draft: q is 1 there
    const int lo = min(V, rank * slice), size = min(V, lo + slice) - lo, pieces = (size + C - 1) / C;
    row += lo;
    if (qrow) qrow += lo;
    const RowPieces<T> ps(row, size), qs(qrow ? qrow : row, size);

    // ---- the slice's sum, and everybody's ----
    unsigned long long total = 0;
    const int group_mask = (1 << group_shift) - 1;
    int slot = 0, phase = 0, slot0 = 0;   // slot0: the pass's first
    int filled = 0;                       // slots filled so far, over both passes
    for (int pass = 0; pass < 2; pass++) {
        const bool two = residual && qrow;
        slot0 = slot;
        if (warp == VT / 32) {
            for (int c = 0; c < pieces; c++) {
                uint8_t* at = ring + slot * 2 * ROW_SLOT;
                // (a slot's n-th filling waits for its (n - 1)-th emptying; the first for none)
                if (!wait_warp(&empty[slot], phase ^ 1, &abort_flag, err)) break;
                uint32_t bytes = 0;
                if (lane == 0) {
                    bytes = ps.copy(c, at, &full[slot]);
                    if (two) bytes += qs.copy(c, at + ROW_SLOT, &full[slot]);
                }
                if (c == 0 || c >= pieces - 2) {
                    if (lane < 32 / sizeof(T)) ps.edges(c, at, lane);
                    if (two && lane < 32 / sizeof(T)) qs.edges(c, at + ROW_SLOT, lane);
                    __syncwarp();
                }
                if (lane == 0) ptx::mbar_expect_tx(&full[slot], bytes);
                filled++;
                if (++slot == SLOTS) slot = 0, phase ^= 1;
            }
        } else {
            uint32_t hi = 0, lo20 = 0;
            for (int c = 0; c < pieces; c++) {
                if (!wait_warp(&full[slot], phase, &abort_flag, err)) break;
                const T* p = reinterpret_cast<const T*>(ring + slot * 2 * ROW_SLOT + ps.off) + t;
                const T* q = reinterpret_cast<const T*>(ring + slot * 2 * ROW_SLOT + ROW_SLOT + qs.off) + t;
                auto sum = [&](auto whole, auto with_q) {
#pragma unroll
                    for (int k = 0; k < PER; k++) {
                        const int i = c * C + k * VT + t;
                        uint32_t h = 0, l = 0;
                        if (decltype(whole)::value || i < size)
                            weight(to_float(p[k * VT]), decltype(with_q)::value ? to_float(q[k * VT]) : lo + i == point ? 1.0f : 0.0f, h, l);
                        hi += h;
                        lo20 += l;
                    }
                };
                const bool whole = (c + 1) * C <= size;
                if (two) whole ? sum(std::true_type(), std::true_type()) : sum(std::false_type(), std::true_type());
                else whole ? sum(std::true_type(), std::false_type()) : sum(std::false_type(), std::false_type());
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&empty[slot]);
                if (++slot == SLOTS) slot = 0, phase ^= 1;
                if ((c & group_mask) == group_mask || c == pieces - 1) {
                    hi = __reduce_add_sync(0xffffffffu, hi);
                    lo20 = __reduce_add_sync(0xffffffffu, lo20);
                    if (lane == 0) parts[c >> group_shift][warp] = ((unsigned long long)hi << 20) + lo20;
                    hi = lo20 = 0;
                }
            }
        }
        const int groups = (pieces + group_mask) >> group_shift;
        __syncthreads();
        if (t < groups) {
            unsigned long long x = 0;
#pragma unroll
            for (int k = 0; k < VT / 32; k++) x += parts[t][(k + t) % (VT / 32)];
            group_sums[t] = x;
        }
        __syncthreads();
        if (pass == 0 && blocks > 1) ptx::cluster_started_wait();   // (before the stores to other blocks)
        if (warp == 0) {
            unsigned long long mine = 0;
            for (int i = lane; i < groups; i += 32) mine += group_sums[i];
            mine = warp_sum(mine);
            if (lane < blocks) {   // to the same place in every block of the cluster
                const uint32_t dst = ptx::mapa_shared(ptx::smem_u32(&share[pass][rank]), lane);
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst), "l"(mine) : "memory");
            }
        }
        if (blocks > 1) ptx::cluster_sync();
        else __syncthreads();
        total = 0;
        for (int r = 0; r < blocks; r++) total += share[pass][r];
        if (total || !residual) {
            unsigned long long before = 0;
            for (int r = 0; r < rank; r++) before += share[pass][r];
            const unsigned long long m = (unsigned long long)fminf(fmaxf(u, 0.0f) * 16777216.0f, 16777215.0f);
            const unsigned long long cut = m * (total >> 24) + ((m * (total & 0xffffffull)) >> 24);
            // ---- the token, in the slice where the sum crosses ----
            if (total && before <= cut && cut < before + share[pass][rank]) {
                // the group of pieces (every warp finds it for itself) ...
                int group = 0;
                for (int i = 0; i < groups; i += 32) {
                    unsigned long long x = i + lane < groups ? group_sums[i + lane] : 0ull;
                    const unsigned long long own = x;
                    x = warp_scan(x, lane);
                    const uint32_t over = __ballot_sync(0xffffffffu, before + x > cut);
                    if (over) {
                        const int at = __ffs(over) - 1;
                        group = i + at;
                        before += __shfl_sync(0xffffffffu, x - own, at);
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, x, 31);
                }
                // ... a lane takes EACH consecutive entries of it, a warp 32 times that (often
                // enough for longer groups); then the lane's entries in order
                constexpr int EACH = PER;
                const int g_from = group * C << group_shift, g_to = min(size, g_from + (C << group_shift));
                const bool in_ring = pieces <= SLOTS;
                float p[EACH], q[EACH];
                auto load = [&](int from) {   // this lane's entries, zeros past the end
#pragma unroll
                    for (int k = 0; k < EACH; k++) {
                        const int i = from + k;
                        p[k] = 0.0f;
                        q[k] = lo + i == point ? 1.0f : 0.0f;
                        if (i >= g_to) continue;
                        if (in_ring) {
                            const uint8_t* at = ring + (slot0 + i / C) % SLOTS * 2 * ROW_SLOT;
                            p[k] = to_float(reinterpret_cast<const T*>(at + ps.off)[i % C]);
                            if (two) q[k] = to_float(reinterpret_cast<const T*>(at + ROW_SLOT + qs.off)[i % C]);
                        } else {   // (from L2)
                            p[k] = load_prob(row + i);
                            if (two) q[k] = load_prob(qrow + i);
                        }
                    }
                };
                auto sum = [&] {
                    uint32_t hi = 0, lo20 = 0, h, l;
#pragma unroll
                    for (int k = 0; k < EACH; k++) {
                        weight(p[k], q[k], h, l);
                        hi += h;
                        lo20 += l;
                    }
                    return ((unsigned long long)hi << 20) + lo20;
                };
                const int steps = 1 << group_shift, w_from = g_from + warp * 32 * EACH * steps + lane * EACH;
                unsigned long long part = 0, x = 0;
                if (warp < VT / 32) {
                    for (int i = 0; i < steps; i++) {
                        load(w_from + i * 32 * EACH);
                        x = warp_scan(sum(), lane);
                        part += __shfl_sync(0xffffffffu, x, 31);
                    }
                    if (lane == 0) sums[warp] = part;
                }
                __syncthreads();
                for (int k = 0; k < warp; k++) before += sums[k];
                if (before <= cut && cut < before + part) {
                    for (int i = 0; i < steps; i++) {
                        if (steps > 1) {
                            load(w_from + i * 32 * EACH);
                            x = warp_scan(sum(), lane);
                        }
                        const uint32_t over = __ballot_sync(0xffffffffu, before + x > cut);
                        if (over) {
                            before += __shfl_up_sync(0xffffffffu, x, 1) * (lane > 0);
                            if (lane == __ffs(over) - 1) {
                                int token = w_from + i * 32 * EACH;
#pragma unroll
                                for (int k = 0; k < EACH - 1; k++) {
                                    uint32_t h, l;
                                    weight(p[k], q[k], h, l);
                                    before += ((unsigned long long)h << 20) + l;
                                    token += before <= cut;
                                }
                                v.tokens[b * (N + 1) + n] = lo + token;
                            }
                            break;
                        }
                        before += __shfl_sync(0xffffffffu, x, 31);
                    }
                }
            }
            break;
        }
        residual = false;   // nothing left of the residual: the target's own row
        point = -1;
    }
    if (rank == 0) {
        for (int i = t; i <= N; i += VT + 32)
            if (i != n || !total) v.tokens[b * (N + 1) + i] = i < n ? v.draft_tokens[b * N + i] : -1;
        if (t == 0) v.accepted[b] = n;
    }
    // after an abandoned wait the results mean nothing, but no copy may land here once the block is gone
    if (warp == VT / 32 && lane == 0 && *static_cast<volatile int*>(&abort_flag))
        for (int i = max(0, filled - SLOTS); i < filled; i++) {
            volatile int no_abort = 0;
            ptx::wait_bounded(&full[i % SLOTS], (i / SLOTS) & 1, &no_abort, err, KERR_WAIT, WAIT_NS);
        }
}

template <class T>
Status verify_as(const RtVerifyDraft& v, cudaStream_t st) {
    static const cudaError_t set = cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES);
    RT_CUDA_CHECK(set);
    // as many blocks a sequence as are resident at once, of two loads a thread at least
    int blocks = std::max(1, std::min(MAX_CLUSTER, BLOCKS_PER_SM * g_num_sms / v.n_seqs));
    while (blocks > 1 && v.vocab < blocks * 1024) blocks--;
    const int slice = (v.vocab + blocks - 1) / blocks;
    int group_shift = 0;
    while (((slice + RowPieces<T>::C - 1) / RowPieces<T>::C) > GROUPS << group_shift) group_shift++;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, v.n_seqs);
    cfg.blockDim = dim3(VT + 32);
    // (a call's two passes over a short slice use a slot a piece each)
    cfg.dynamicSmemBytes = std::min(SLOTS, 2 * ((slice + RowPieces<T>::C - 1) / RowPieces<T>::C)) * 2 * ROW_SLOT;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = blocks;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    RT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T>, v, blocks, slice, group_shift, serving_error_flag()));
    return Status::ok();
}

}  // namespace

Status launch_verify_draft(const RtVerifyDraft& v, cudaStream_t st) {
    return v.dtype == RT_BF16 ? verify_as<__nv_bfloat16>(v, st) : verify_as<float>(v, st);
}

}  // namespace rt
