// k_paged_attention.cu -- attention of new tokens over a paged cache.
//
// For the new token at position P of its sequence, with the visible positions
// lo <= j < hi (hi = P + 1 when causal, lo = P - window + 1 with a window):
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = q . k_j * scale,
// computed in one pass with the running maximum m: when m grows, what has
// been summed so far is multiplied by exp(m_old - m_new).
//
// One warp per (token, query head), lanes over the features, one key at a
// time: every sum is fp32 in registers.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "rt_internal.h"

namespace rt {
namespace {

template <int CT>
__device__ __forceinline__ float cache_at(const void* base, int64_t off) {
    if constexpr (CT == RT_F32) return static_cast<const float*>(base)[off];
    if constexpr (CT == RT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[off]);
    if constexpr (CT == RT_I8) return (float)static_cast<const int8_t*>(base)[off];
    if constexpr (CT == RT_F8E4M3) return (float)static_cast<const __nv_fp8_e4m3*>(base)[off];
    return 0.0f;
}

template <class A, int CT>
__global__ void __launch_bounds__(128) paged_simple_kernel(RtPagedAttention p, int* err) {
    const RtKvCache& c = p.cache;
    const int lane = threadIdx.x & 31, D = c.head_dim;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)p.total_new * p.n_q_heads) return;
    const int token = (int)(row / p.n_q_heads), h = (int)(row % p.n_q_heads), kh = h / (p.n_q_heads / c.n_heads);
    int b = 0, end = p.n_seqs;
    while (end - b > 1) {
        const int mid = (b + end) >> 1;
        if (p.cu_new[mid] <= token) b = mid;
        else end = mid;
    }
    const int n = p.cu_new[b + 1] - p.cu_new[b], i = token - p.cu_new[b];
    if (i < 0 || i >= n) return;   // a row that belongs to no sequence
    int L = p.kv_lens[b];
    if (L < 0 || (L + c.page_size - 1) / c.page_size > p.table_width) {
        if (lane == 0) atomicCAS(err, 0, KERR_LENGTH);
        L = L < 0 ? 0 : p.table_width * c.page_size;
    }
    const int at = L - n + i;
    const int hi = p.causal ? min(L, at + 1) : L;
    const int lo = p.window > 0 ? max(0, at - p.window + 1) : 0;
    const A* q = static_cast<const A*>(p.q) + token * p.q_stride[0] + h * p.q_stride[1];
    float qv[4], acc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; j++) qv[j] = lane + 32 * j < D ? (float)q[lane + 32 * j] * p.scale : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int k = lo; k < hi; k++) {
        const int page = p.page_table[b * p.table_stride + k / c.page_size];
        if (page < 0 || page >= c.n_pages) {
            if (lane == 0) atomicCAS(err, 0, KERR_PAGE);
            continue;
        }
        const int off = k % c.page_size;
        const int64_t e = page * c.stride[0] + off * c.stride[1] + kh * c.stride[2];
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (lane + 32 * j < D) s = fmaf(qv[j], cache_at<CT>(c.k, e + lane + 32 * j), s);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        float vs = 1.0f;
        if constexpr (CT == RT_I8 || CT == RT_F8E4M3) {
            const int64_t se = page * c.scale_stride[0] + off * c.scale_stride[1] + kh * c.scale_stride[2];
            s *= c.k_scale[se];
            vs = c.v_scale[se];
        }
        const float mn = fmaxf(m, s), corr = m == mn ? 1.0f : expf(m - mn), w = s == -INFINITY ? 0.0f : expf(s - mn);
        l = l * corr + w;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (lane + 32 * j < D) acc[j] = fmaf(w * vs, cache_at<CT>(c.v, e + lane + 32 * j), acc[j] * corr);
        m = mn;
    }
    A* out = static_cast<A*>(p.out) + token * p.out_stride[0] + h * p.out_stride[1];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (lane + 32 * j < D) out[lane + 32 * j] = (A)(acc[j] * inv);
    if (p.lse && lane == 0) p.lse[row] = l == 0.0f ? -INFINITY : m + logf(l);
}

template <class A>
Status launch_simple(const RtPagedAttention& p, cudaStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)p.total_new * p.n_q_heads + 3) / 4);
    int* err = kernel_error_flag();
    switch (p.cache.dtype) {
        case RT_F32: paged_simple_kernel<A, RT_F32><<<grid, 128, 0, st>>>(p, err); break;
        case RT_BF16: paged_simple_kernel<A, RT_BF16><<<grid, 128, 0, st>>>(p, err); break;
        case RT_F8E4M3: paged_simple_kernel<A, RT_F8E4M3><<<grid, 128, 0, st>>>(p, err); break;
        default: paged_simple_kernel<A, RT_I8><<<grid, 128, 0, st>>>(p, err); break;
    }
    RT_LAUNCH_CHECK();
    return Status::ok();
}

}  // namespace

size_t paged_attention_workspace(const RtPagedAttention&) { return 0; }

Status launch_paged_attention(const RtPagedAttention& p, void*, cudaStream_t st) {
    return p.dtype == RT_BF16 ? launch_simple<__nv_bfloat16>(p, st) : launch_simple<float>(p, st);
}

}  // namespace rt
