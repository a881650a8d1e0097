// k_paged_attention.cu -- attention of new tokens over a paged cache: which
// kernel takes a call.
//
// The few-rows kernel takes up to 32 rows (new tokens x query heads of a cache
// head), more fill a tensor core tile of 128 well enough.  Measured on 32
// sequences of up to 4096 positions with 20 rows, few / tiles: int8 with bf16
// activations 130 / 205 us, with fp32 ones 161 / 185, fp32 cache 475 / 603.  A bf16
// cache with bf16 activations needs no conversion on its way to a tile, and
// goes there from 17 rows on (184 / 143).
// Head dims other than 64 and 128 have no such tiles and take the few-rows kernel
// whatever their rows.
#include "paged.h"

namespace rt {
namespace {

bool use_tiles(const RtPagedAttention& p) {
    const int64_t rows = (int64_t)(p.max_new < p.total_new ? p.max_new : p.total_new) * (p.n_q_heads / p.cache.n_heads);
    return rows > (p.dtype == RT_BF16 && p.cache.dtype == RT_BF16 ? 16 : 32) && paged_tiles_takes(p);
}

}  // namespace

size_t paged_attention_workspace(const RtPagedAttention& p) {
    return use_tiles(p) ? paged_tiles_workspace(p) : paged_few_workspace(p);
}

Status launch_paged_attention(const RtPagedAttention& a, void* ws, cudaStream_t st) {
    PagedArgs p{};
    p.a = a;
    p.err = serving_error_flag();
    p.group = a.n_q_heads / a.cache.n_heads;
    p.vec_q = paged_rows16(a.q, a.q_stride, a.dtype);
    p.vec_out = paged_rows16(a.out, a.out_stride, a.dtype);
    p.page_shift = -1;
    for (int i = 0; i < 31; i++)
        if (a.cache.page_size == 1 << i) p.page_shift = i;
    return use_tiles(a) ? launch_paged_tiles(p, ws, st) : launch_paged_few(p, ws, st);
}

}  // namespace rt
