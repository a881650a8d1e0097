// k_paged_attention.cu -- attention of new tokens over a paged cache: which
// kernel takes a call.
#include "paged.h"

namespace rt {

size_t paged_attention_workspace(const RtPagedAttention& p) { return paged_few_workspace(p); }

Status launch_paged_attention(const RtPagedAttention& a, void* ws, cudaStream_t st) {
    PagedArgs p{};
    p.a = a;
    p.err = kernel_error_flag();
    p.group = a.n_q_heads / a.cache.n_heads;
    p.page_shift = -1;
    for (int i = 0; i < 31; i++)
        if (a.cache.page_size == 1 << i) p.page_shift = i;
    return launch_paged_few(p, ws, st);
}

}  // namespace rt
