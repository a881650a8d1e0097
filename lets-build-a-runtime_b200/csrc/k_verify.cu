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
// split over threads, and the token is a function of the inputs alone.
#include <cuda_bf16.h>

#include "rt_internal.h"

namespace rt {
namespace {

constexpr int VT = 1024;   // threads

template <class T> __device__ __forceinline__ float as_float(T x) { return (float)x; }

// w in units of 2^-40, truncated; NaN and negative weights count nothing.
__device__ __forceinline__ unsigned long long weight(float w) {
    return w > 0.0f ? (unsigned long long)(fminf(w, 1.0f) * 1099511627776.0f) : 0ull;
}

// Sum over the block, to every thread.
__device__ unsigned long long block_sum(unsigned long long x, unsigned long long* sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
    for (int i = 0; i < VT / 32; i++) x += sh[i];
    return x;
}

template <class T>
__global__ void __launch_bounds__(VT) verify_simple_kernel(RtVerifyDraft v, int* err) {
    __shared__ unsigned long long sh[VT / 32];
    __shared__ int first;
    const int b = blockIdx.x, N = v.n_drafts, V = v.vocab, t = threadIdx.x;
    const T* target = static_cast<const T*>(v.target) + b * v.target_stride[0];
    const T* draft = v.draft ? static_cast<const T*>(v.draft) + b * v.draft_stride[0] : nullptr;
    int n = v.draft_lens ? v.draft_lens[b] : N;
    if (n < 0 || n > N) {
        if (t == 0) atomicCAS(err, 0, KERR_LENGTH);
        n = n < 0 ? 0 : N;
    }
    if (t == 0) first = n;
    __syncthreads();
    if (t < n) {
        const int x = v.draft_tokens[b * N + t];
        bool keep = false;
        if (x < 0 || x >= V) {
            atomicCAS(err, 0, KERR_TOKEN);
        } else {
            const float p = as_float(target[t * v.target_stride[1] + x]);
            const float q = draft ? as_float(draft[t * v.draft_stride[1] + x]) : 1.0f;
            keep = __fmul_rn(v.accept_u[b * N + t], q) < p;
        }
        if (!keep) atomicMin(&first, t);
    }
    __syncthreads();
    n = first;
    const int limit = v.draft_lens ? min(max(v.draft_lens[b], 0), N) : N;
    const T* row = target + n * v.target_stride[1];
    const T* qrow = draft && n < limit ? draft + n * v.draft_stride[1] : nullptr;
    const int point = !draft && n < limit ? v.draft_tokens[b * N + n] : -1;
    bool residual = n < limit;
    auto at = [&](int i) {
        const float p = as_float(row[i]);
        if (!residual) return weight(p);
        return weight(qrow ? p - as_float(qrow[i]) : (i == point ? p - 1.0f : p));
    };
    // thread t owns the consecutive entries [t * per, t * per + per)
    const int per = (V + VT - 1) / VT, lo = min(V, t * per), hi = min(V, lo + per);
    unsigned long long mine = 0, total = 0;
    for (int pass = 0; pass < 2; pass++) {
        mine = 0;
        for (int i = lo; i < hi; i++) mine += at(i);
        total = block_sum(mine, sh);
        if (total || !residual) break;
        residual = false;   // nothing left of the residual: the target's own row
    }
    const float u = v.sample_u[b];
    const unsigned long long m = (unsigned long long)fminf(fmaxf(u, 0.0f) * 16777216.0f, 16777215.0f);
    const unsigned long long cut = m * (total >> 24) + ((m * (total & 0xffffffull)) >> 24);
    __shared__ unsigned long long sums[VT];
    __shared__ int token;
    sums[t] = mine;
    if (t == 0) token = -1;
    __syncthreads();
    unsigned long long before = 0;
    for (int i = 0; i < t; i++) before += sums[i];
    if (total && before <= cut && before + mine > cut) {
        int i = lo;
        for (; i < hi; i++) {
            before += at(i);
            if (before > cut) break;
        }
        token = i;
    }
    __syncthreads();
    for (int i = t; i <= N; i += VT)
        v.tokens[b * (N + 1) + i] = i < n ? v.draft_tokens[b * N + i] : i == n ? token : -1;
    if (t == 0) v.accepted[b] = n;
}

}  // namespace

Status launch_verify_draft(const RtVerifyDraft& v, cudaStream_t st) {
    if (v.dtype == RT_BF16) verify_simple_kernel<__nv_bfloat16><<<v.n_seqs, VT, 0, st>>>(v, kernel_error_flag());
    else verify_simple_kernel<float><<<v.n_seqs, VT, 0, st>>>(v, kernel_error_flag());
    RT_LAUNCH_CHECK();
    return Status::ok();
}

}  // namespace rt
