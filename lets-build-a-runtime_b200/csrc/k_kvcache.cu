// k_kvcache.cu -- storing new keys and values in a paged cache (quantising
// them for 8-bit caches) and reading cached rows back.
//
// Both move every byte once: bound by HBM for many tokens, by latency for a
// few.  A row is one (token, head) of K or V, D <= 128 features; it is taken
// by 2^k lanes of one warp, each with one 16-byte unit of the dense side (4
// fp32 or 8 bf16 features), so dense loads and stores of neighbouring lanes
// join into whole lines and a row's maximum is a few shuffles.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "rt_internal.h"

namespace rt {
namespace {

template <class A> struct Unit;   // one lane's features of the dense side
template <> struct Unit<float> { static constexpr int N = 4; };
template <> struct Unit<__nv_bfloat16> { static constexpr int N = 8; };

__device__ __forceinline__ void load_unit(const float* p, bool vec, float (&x)[4]) {
    if (vec) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = p[i];
    }
}
__device__ __forceinline__ void load_unit(const __nv_bfloat16* p, bool vec, float (&x)[8]) {
    if (vec) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __bfloat162float(p[i]);
    }
}
__device__ __forceinline__ uint32_t bf16_two(float a, float b) {   // a in the low half
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void store_unit(float* p, bool vec, const float (&x)[4]) {
    if (vec) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = x[i];
    }
}
__device__ __forceinline__ void store_unit(__nv_bfloat16* p, bool vec, const float (&x)[8]) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(bf16_two(x[0], x[1]), bf16_two(x[2], x[3]), bf16_two(x[4], x[5]),
                                                  bf16_two(x[6], x[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = __float2bfloat16_rn(x[i]);
    }
}

// N consecutive features into / out of the cache at feature offset `off`
// (N * element size divides the alignment the entry point checks).
template <int N, int CT>
__device__ __forceinline__ void put_cache(void* base, int64_t off, const float (&x)[N]) {
    if constexpr (CT == RT_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + off);
#pragma unroll
        for (int i = 0; i < N / 4; i++) p[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else if constexpr (CT == RT_BF16) {
        uint32_t* p = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(base) + off);
        if constexpr (N == 8)
            *reinterpret_cast<uint4*>(p) = make_uint4(bf16_two(x[0], x[1]), bf16_two(x[2], x[3]), bf16_two(x[4], x[5]),
                                                      bf16_two(x[6], x[7]));
        else
            *reinterpret_cast<uint2*>(p) = make_uint2(bf16_two(x[0], x[1]), bf16_two(x[2], x[3]));
    } else {
        uint32_t w[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            if constexpr (CT == RT_I8) {
                w[i] = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) w[i] |= ((uint32_t)__float2int_rn(x[4 * i + j]) & 0xffu) << (8 * j);
            } else {   // satfinite, to the nearest, ties to even
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
                w[i] = lo | (hi << 16);
            }
        }
        uint32_t* p = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(base) + off);
        if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *p = w[0];
    }
}
template <int N, int CT>
__device__ __forceinline__ void get_cache(const void* base, int64_t off, float (&x)[N]) {
    if constexpr (CT == RT_F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const float4 v = p[i];
            x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
        }
    } else if constexpr (CT == RT_BF16) {
        const uint2* p = reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + off);
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint2 v = p[i];
            x[4 * i] = __uint_as_float(v.x << 16);
            x[4 * i + 1] = __uint_as_float(v.x & 0xffff0000u);
            x[4 * i + 2] = __uint_as_float(v.y << 16);
            x[4 * i + 3] = __uint_as_float(v.y & 0xffff0000u);
        }
    } else {
        uint32_t w[N / 4];
        const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + off);
        if constexpr (N == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[1] = v.y;
        } else {
            w[0] = *p;
        }
#pragma unroll
        for (int i = 0; i < N / 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (CT == RT_I8) {
                    x[4 * i + j] = (float)(int8_t)(w[i] >> (8 * j));
                } else {
                    __nv_fp8_e4m3 v;
                    v.__x = (__nv_fp8_storage_t)(w[i] >> (8 * j));
                    x[4 * i + j] = (float)v;
                }
            }
    }
}

struct RowMap {
    int lanes_log2;   // lanes of a row
    int units;        // lanes of a row that hold features
    int rows_per_token;
};

template <class A, int CT>
__global__ void __launch_bounds__(256) kv_write_kernel(RtKvWrite w, RowMap m, bool vec, int* err) {
    constexpr int N = Unit<A>::N;
    const RtKvCache& c = w.cache;
    const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t rows = (int64_t)w.n_tokens * m.rows_per_token;
    const int64_t row = tid >> m.lanes_log2;
    const int unit = (int)(tid & ((1 << m.lanes_log2) - 1));
    if (row >= rows) return;   // whole rows leave together
    const int token = (int)(row / m.rows_per_token), r = (int)(row % m.rows_per_token);
    const int is_v = r >= c.n_heads, head = is_v ? r - c.n_heads : r;
    const int64_t slot = w.slots[token];
    const bool live = unit < m.units;
    float x[N];
    const int64_t* st = is_v ? w.v_stride : w.k_stride;
    const A* src = static_cast<const A*>(is_v ? w.v : w.k) + token * st[0] + head * st[1] + unit * N;
    if (live) {
        load_unit(src, vec, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = 0.0f;
    }
    if (slot < 0) return;
    if (slot >= (int64_t)c.n_pages * c.page_size) {
        if (unit == 0) atomicCAS(err, 0, KERR_SLOT);
        return;
    }
    const int64_t page = slot / c.page_size, off = slot % c.page_size;
    void* dst = is_v ? c.v : c.k;
    const int64_t at = page * c.stride[0] + off * c.stride[1] + head * c.stride[2] + unit * N;
    if constexpr (CT == RT_I8 || CT == RT_F8E4M3) {
        constexpr float MAX_CODE = CT == RT_I8 ? 127.0f : 448.0f;
        // the maximum over the bits of |x|: NaN and infinity come out on top
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        const uint32_t group = m.lanes_log2 == 5 ? 0xffffffffu
                                                 : ((1u << (1 << m.lanes_log2)) - 1) << ((threadIdx.x & 31) >> m.lanes_log2 << m.lanes_log2);
        top = __reduce_max_sync(group, top);
        const float a = __uint_as_float(top);
        // scale = a (1/M) and code = round(x ((1/a) M)), each step rounded to fp32:
        // a function of the row that any fp32 arithmetic reproduces bit for bit
        float scale = __fmul_rn(a, 1.0f / MAX_CODE), inv = __fmul_rn(__frcp_rn(a), MAX_CODE);
        if (a < 7.888609052210118e-31f) scale = inv = 0.0f;                   // 2^-100: M / a overflows further down
        if (top >= 0x7f800000u) { scale = __uint_as_float(0x7fc00000u); inv = 0.0f; }
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = inv == 0.0f ? 0.0f : __fmul_rn(x[i], inv);
        if (unit == 0)
            (is_v ? c.v_scale : c.k_scale)[page * c.scale_stride[0] + off * c.scale_stride[1] + head * c.scale_stride[2]] = scale;
    }
    if (live) put_cache<N, CT>(dst, at, x);
}

// 16 tokens a block: their places in the cache are looked up once, then the
// block's threads take the tokens' rows.
constexpr int READ_TOKENS = 16;
template <class A, int CT>
__global__ void __launch_bounds__(256) kv_read_kernel(RtKvRead r, RowMap m, bool vec, int* err) {
    constexpr int N = Unit<A>::N;
    const RtKvCache& c = r.cache;
    __shared__ int64_t place[READ_TOKENS], scale_place[READ_TOKENS];
    const int t0 = blockIdx.x * READ_TOKENS;
    if (threadIdx.x < READ_TOKENS) {
        const int row = t0 + threadIdx.x;
        int64_t p = -1, sp = 0;
        if (row < r.n_rows && row < r.cu[r.n_seqs]) {
            int lo = 0, hi = r.n_seqs;   // the sequence whose rows hold this one: cu[lo] <= row < cu[lo + 1]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (r.cu[mid] <= row) lo = mid;
                else hi = mid;
            }
            const int64_t pos = (r.start ? r.start[lo] : 0) + (int64_t)(row - r.cu[lo]);
            const int64_t ip = pos / c.page_size, off = pos % c.page_size;
            if (pos < 0 || ip >= r.table_width || row < r.cu[lo]) {
                atomicCAS(err, 0, KERR_LENGTH);
            } else {
                const int page = r.page_table[lo * r.table_stride + ip];
                if (page < 0 || page >= c.n_pages) {
                    atomicCAS(err, 0, KERR_PAGE);
                } else {
                    p = page * c.stride[0] + off * c.stride[1];
                    sp = page * c.scale_stride[0] + off * c.scale_stride[1];
                }
            }
        }
        place[threadIdx.x] = p;
        scale_place[threadIdx.x] = sp;
    }
    __syncthreads();
    const int n_here = min(READ_TOKENS, r.n_rows - t0);
    const int per_token = m.rows_per_token << m.lanes_log2;
#pragma unroll 4
    for (int i = threadIdx.x; i < n_here * per_token; i += 256) {
        const int token = i / per_token, u = i % per_token;
        const int row = u >> m.lanes_log2, unit = u & ((1 << m.lanes_log2) - 1);
        if (unit >= m.units) continue;
        const int is_v = row >= c.n_heads, head = is_v ? row - c.n_heads : row;
        float x[N];
        if (place[token] >= 0) {
            get_cache<N, CT>(is_v ? c.v : c.k, place[token] + head * c.stride[2] + unit * N, x);
            if constexpr (CT == RT_I8 || CT == RT_F8E4M3) {
                const float s = (is_v ? c.v_scale : c.k_scale)[scale_place[token] + head * c.scale_stride[2]];
#pragma unroll
                for (int j = 0; j < N; j++) x[j] *= s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) x[j] = 0.0f;
        }
        const int64_t* st = is_v ? r.v_stride : r.k_stride;
        store_unit(static_cast<A*>(is_v ? r.v_out : r.k_out) + (t0 + token) * st[0] + head * st[1] + unit * N, vec, x);
    }
}

template <class A>
RowMap row_map(const RtKvCache& c) {
    RowMap m;
    m.units = c.head_dim / Unit<A>::N;
    m.lanes_log2 = 0;
    while ((1 << m.lanes_log2) < m.units) m.lanes_log2++;
    m.rows_per_token = 2 * c.n_heads;
    return m;
}
// Whether every row of a dense operand starts on a 16-byte boundary.
bool vector_rows(const void* p, const int64_t st[2], int dtype) {
    return aligned16(p) && (st[0] * dtype_bytes(dtype)) % 16 == 0 && (st[1] * dtype_bytes(dtype)) % 16 == 0;
}

template <class A, int CT>
Status write_as(const RtKvWrite& w, cudaStream_t st) {
    const RowMap m = row_map<A>(w.cache);
    const int64_t threads = ((int64_t)w.n_tokens * m.rows_per_token) << m.lanes_log2;
    const bool vec = vector_rows(w.k, w.k_stride, w.dtype) && vector_rows(w.v, w.v_stride, w.dtype);
    if ((threads + 255) / 256 > 0x7fffffff) return Status::err(RT_ERR_UNSUPPORTED, "kv_write: too many rows");
    kv_write_kernel<A, CT><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(w, m, vec, kernel_error_flag());
    RT_LAUNCH_CHECK();
    return Status::ok();
}
template <class A, int CT>
Status read_as(const RtKvRead& r, cudaStream_t st) {
    const RowMap m = row_map<A>(r.cache);
    const bool vec = vector_rows(r.k_out, r.k_stride, r.dtype) && vector_rows(r.v_out, r.v_stride, r.dtype);
    kv_read_kernel<A, CT><<<(unsigned)((r.n_rows + READ_TOKENS - 1) / READ_TOKENS), 256, 0, st>>>(r, m, vec, kernel_error_flag());
    RT_LAUNCH_CHECK();
    return Status::ok();
}

}  // namespace

#define DISPATCH(F, X, st)                                                  \
    const bool bf = (X).dtype == RT_BF16;                                   \
    switch ((X).cache.dtype) {                                              \
        case RT_F32: return bf ? F<__nv_bfloat16, RT_F32>(X, st) : F<float, RT_F32>(X, st);       \
        case RT_BF16: return bf ? F<__nv_bfloat16, RT_BF16>(X, st) : F<float, RT_BF16>(X, st);    \
        case RT_F8E4M3: return bf ? F<__nv_bfloat16, RT_F8E4M3>(X, st) : F<float, RT_F8E4M3>(X, st); \
        default: return bf ? F<__nv_bfloat16, RT_I8>(X, st) : F<float, RT_I8>(X, st);             \
    }

Status launch_kv_write(const RtKvWrite& w, cudaStream_t st) { DISPATCH(write_as, w, st) }
Status launch_kv_read(const RtKvRead& r, cudaStream_t st) { DISPATCH(read_as, r, st) }

}  // namespace rt
