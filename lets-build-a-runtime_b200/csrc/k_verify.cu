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
// block settles the drafts by itself (a few loads), sums its slice while it
// keeps the weights in shared memory, sends its sum to the others, and the one
// in whose slice the running sum crosses finds the token there.
#include <cuda_bf16.h>

#include <algorithm>

#include "rt_internal.h"
#include "sm100_ptx.h"

namespace rt {
namespace {

constexpr int VT = 512, MAX_CLUSTER = 8;
constexpr int STAGED = 4096;   // weights of a slice kept in shared memory; the one longer slice that holds the token is read again (L2)

// w = a - b, clamped to [0, 1] (NaN: 0), in units of 2^-40, truncated: the
// steps of 2^-20 below it by adding 8 with rounding toward zero (whose last
// place is 2^-20), then the steps of 2^-40 of what is left, which is exact.
// Two 32-bit counts instead of a 64-bit integer: conversions to 64 bits run at
// a fraction of the rate, and a thread's counts fit (2^20 per entry, at most
// 2^22 / 512 entries).
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

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <class T>
__global__ void __launch_bounds__(VT, 3) verify_kernel(RtVerifyDraft v, int blocks, int slice, int* err) {
    extern __shared__ float kept[];                       // weights of the slice, before fixed point
    __shared__ unsigned long long sums[VT / 32], share[2][MAX_CLUSTER];
    __shared__ int first;
    const int b = blockIdx.y, rank = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int N = v.n_drafts, V = v.vocab;
    const T* target = static_cast<const T*>(v.target) + b * v.target_stride[0];
    const T* draft = v.draft ? static_cast<const T*>(v.draft) + b * v.draft_stride[0] : nullptr;

    // ---- how many drafts stand ----
    int limit = v.draft_lens ? v.draft_lens[b] : N;
    if (limit < 0 || limit > N) {
        if (t == 0) atomicCAS(err, 0, KERR_LENGTH);
        limit = limit < 0 ? 0 : N;
    }
    if (t == 0) first = limit;
    __syncthreads();
    for (int i = t; i < limit; i += VT) {
        const int x = v.draft_tokens[b * N + i];
        const float u = v.accept_u[b * N + i];
        bool keep = false;
        if (x < 0 || x >= V) {
            if (rank == 0) atomicCAS(err, 0, KERR_TOKEN);
        } else {
            const float p = load_prob(target + i * v.target_stride[1] + x);
            const float q = draft ? load_prob(draft + i * v.draft_stride[1] + x) : 1.0f;
            keep = __fmul_rn(u, q) < p;
        }
        if (!keep) atomicMin(&first, i);
    }
    __syncthreads();
    const int n = first;
    const T* row = target + n * v.target_stride[1];
    bool residual = n < limit;
    const T* qrow = draft && residual ? draft + n * v.draft_stride[1] : nullptr;
    const int point = !draft && residual ? v.draft_tokens[b * N + n] : -1;   // a certain draft: q is 1 there
    const int lo = min(V, rank * slice), size = min(V, lo + slice) - lo;
    const bool keep_all = slice <= STAGED;
    const float u = v.sample_u[b];
    row += lo;
    if (qrow) qrow += lo;
    // What is taken off the target at entry i of the slice.
    auto taken = [&](int i) -> float {
        if (!residual) return 0.0f;
        return qrow ? load_prob(qrow + i) : (lo + i == point ? 1.0f : 0.0f);
    };

    // ---- the slice's sum, and everybody's ----
    unsigned long long total = 0;
    for (int pass = 0; pass < 2; pass++) {
        uint32_t hi = 0, lo20 = 0;
        for (int i0 = t; i0 < size; i0 += 8 * VT) {
            float p[8], q[8];
#pragma unroll
            for (int k = 0; k < 8; k++) p[k] = i0 + k * VT < size ? load_prob(row + i0 + k * VT) : 0.0f;
            if (residual && qrow) {
#pragma unroll
                for (int k = 0; k < 8; k++) q[k] = i0 + k * VT < size ? load_prob(qrow + i0 + k * VT) : 0.0f;
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) q[k] = taken(i0 + k * VT);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                uint32_t h, l;
                weight(p[k], q[k], h, l);
                hi += h;
                lo20 += l;
                if (keep_all && i0 + k * VT < size) kept[i0 + k * VT] = p[k] - q[k];
            }
        }
        unsigned long long mine = ((unsigned long long)hi << 20) + lo20;
        mine = warp_sum(mine);
        __syncthreads();
        if (lane == 0) sums[warp] = mine;
        __syncthreads();
        if (warp == 0) {
            mine = warp_sum(lane < VT / 32 ? sums[lane] : 0ull);
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
                // a warp takes consecutive entries, a lane every 32nd of them; then one warp's
                // entries again, in order
                const int per = ((size + VT / 32 - 1) / (VT / 32) + 31) & ~31, w0 = min(size, warp * per), w1 = min(size, w0 + per);
                auto again = [&](int i) -> unsigned long long {
                    uint32_t h, l;
                    if (keep_all) weight(kept[i], 0.0f, h, l);
                    else weight(load_prob(row + i), taken(i), h, l);
                    return ((unsigned long long)h << 20) + l;
                };
                unsigned long long part = 0;
                for (int i = w0 + lane; i < w1; i += 32) part += again(i);
                part = warp_sum(part);
                if (lane == 0) sums[warp] = part;
                __syncthreads();
                for (int k = 0; k < warp; k++) before += sums[k];
                if (before <= cut && cut < before + part) {
                    for (int i = w0; i < w1; i += 32) {
                        unsigned long long x = i + lane < w1 ? again(i + lane) : 0ull;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
                            if (lane >= o) x += y;
                        }
                        const uint32_t over = __ballot_sync(0xffffffffu, before + x > cut);
                        if (over) {
                            if (lane == 0) v.tokens[b * (N + 1) + n] = lo + i + __ffs(over) - 1;
                            break;
                        }
                        before += __shfl_sync(0xffffffffu, x, 31);
                    }
                }
            }
            break;
        }
        residual = false;   // nothing left of the residual: the target's own row
    }
    if (rank == 0) {
        for (int i = t; i <= N; i += VT)
            if (i != n || !total) v.tokens[b * (N + 1) + i] = i < n ? v.draft_tokens[b * N + i] : -1;
        if (t == 0) v.accepted[b] = n;
    }
}

template <class T>
Status verify_as(const RtVerifyDraft& v, cudaStream_t st) {
    static const cudaError_t set = cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, STAGED * 4);
    RT_CUDA_CHECK(set);
    int blocks = MAX_CLUSTER;
    while (blocks > 1 && v.vocab < blocks * 1024) blocks /= 2;   // a slice of less than two loads a thread is not worth a block
    const int slice = (v.vocab + blocks - 1) / blocks;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, v.n_seqs);
    cfg.blockDim = dim3(VT);
    cfg.dynamicSmemBytes = slice <= STAGED ? slice * 4 : 0;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = blocks;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    RT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T>, v, blocks, slice, kernel_error_flag()));
    return Status::ok();
}

}  // namespace

Status launch_verify_draft(const RtVerifyDraft& v, cudaStream_t st) {
    return v.dtype == RT_BF16 ? verify_as<__nv_bfloat16>(v, st) : verify_as<float>(v, st);
}

}  // namespace rt
