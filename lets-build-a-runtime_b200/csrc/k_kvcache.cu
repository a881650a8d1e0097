// k_kvcache.cu -- storing new keys and values in a paged cache (quantising
// them for 8-bit caches) and reading cached rows back.
//
// Both move every byte once: bound by HBM for many tokens, by latency for a
// few.  A row is one (token, head) of K or V, D <= 128 features; it is taken
// by 2^k lanes of one warp, each with one 16-byte unit of the dense side (4
// fp32 or 8 bf16 features), so dense loads and stores of neighbouring lanes
// join into whole lines and a row's maximum is a few shuffles.
//
// Measured: reading 12 sequences of up to 8192 positions from fp8 to fp32, 843
// MB, 138 us = 6.1 TB/s (a look-up and a division per row and thread: 200);
// writing 12 K tokens of 8 heads of 128 from bf16 to fp8, 74 MB, 20.2 us = 3.7
// TB/s, 60 K tokens 373 MB, 87.7 us = 4.3 TB/s. The quantisation bounds that:
// the same 60 K tokens into a bf16 cache, 492 MB with the same loads under way,
// take 77.3 us = 6.4 TB/s. (4 loads a batch or a whole look-up per thread: 41 -
// 51 us for the 12 K tokens written and read back, against 34.) One token of 8
// sequences is written in 2.3 us, a prefix of 100 positions read in 2.7.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "rt_internal.h"

namespace rt {
namespace {

template <class A> struct Unit;   // one lane's features of the dense side
template <> struct Unit<float> { static constexpr int N = 4; };
template <> struct Unit<__nv_bfloat16> { static constexpr int N = 8; };

// Both are 16 bytes: loaded as they are, and given their values later.
__device__ __forceinline__ uint4 load_unit(const float* p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
    return make_uint4(__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3]));
}
__device__ __forceinline__ uint4 load_unit(const __nv_bfloat16* p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}
__device__ __forceinline__ void unit_values(uint4 v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unit_values(uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
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
                // to the nearest, ties to even, by adding 1.5 * 2^23: the low byte is the code (|x| <= 128)
                uint32_t b[4];
#pragma unroll
                for (int j = 0; j < 4; j++) b[j] = __float_as_uint(__fadd_rn(x[4 * i + j], 12582912.0f));
                w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
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
// The same the other way, in two steps: the loads of several rows go first.
template <int N, int CT>
struct Raw {
    static constexpr int WORDS = CT == RT_F32 ? N : CT == RT_BF16 ? N / 2 : N / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = 0;
    }
    __device__ __forceinline__ void load(const void* base, int64_t off) {
        const uint8_t* p = static_cast<const uint8_t*>(base) + off * (CT == RT_F32 ? 4 : CT == RT_BF16 ? 2 : 1);
        if constexpr (WORDS == 1) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (WORDS == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            w[0] = x.x; w[1] = x.y;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(p + i * 4);
                w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
            }
        }
    }
    __device__ __forceinline__ void values(float (&x)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (CT == RT_F32) {
                x[i] = __uint_as_float(w[i]);
            } else if constexpr (CT == RT_BF16) {
                x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
            } else if constexpr (CT == RT_I8) {
                x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i & 3)));
            } else if (i % 2 == 0) {
                uint32_t h;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w[i / 4] >> (8 * (i & 2)))));
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                x[i] = f.x;
                x[i + 1] = f.y;
            }
        }
    }
};
// A block takes threadIdx.x = part of a token's rows (K's heads, then V's; a
// token of more than 256 parts has several blocks, blockIdx.y), threadIdx.y =
// one of the tokens it takes side by side.  A thread has the same part of
// every token it takes, so that what belongs to the part is worked out once.
constexpr int KV_THREADS = 256;
struct RowMap {
    int lanes_log2;   // lanes of a row
    int units;        // lanes of a row that hold features
    int per_token;    // lanes of a token's rows
    int tokens;       // of a block
    uint32_t page_mul, page_shift;   // x / page_size = (x + mulhi(x, page_mul)) >> page_shift for x < 2^31
};
struct Part {
    bool is_v, live;  // live: holds features
    int head, unit;
};
__device__ __forceinline__ Part part_of(const RowMap& m, int n_heads) {
    const int u = blockIdx.y * blockDim.x + threadIdx.x, row = u >> m.lanes_log2;
    Part x;
    x.unit = u & ((1 << m.lanes_log2) - 1);
    x.is_v = row >= n_heads;
    x.head = x.is_v ? row - n_heads : row;
    x.live = x.unit < m.units && u < m.per_token;
    return x;
}
// Where a token's slot begins in the cache and among the scales; `at` < 0: nowhere.
struct Place {
    int64_t at, scale;
};
__device__ __forceinline__ Place place_of(const RtKvCache& c, int64_t page, int off) {
    return {page * c.stride[0] + off * c.stride[1], page * c.scale_stride[0] + off * c.scale_stride[1]};
}

// The largest |x| of a unit, as bits: NaN and infinity come out on top.
__device__ __forceinline__ uint32_t unit_top(uint4 v, float) {
    return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
}
__device__ __forceinline__ uint32_t unit_top(uint4 v, __nv_bfloat16) {
    const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
}

// A lane of every warp looks one of the block's tokens up, and hands its place
// to the others as they come to it (no barrier; a look-up by every thread for
// itself cost as much as the rest of its work).  A thread loads its part of
// WRITE_BATCH tokens while it works on those before.
constexpr int WRITE_TOKENS = 8, WRITE_BATCH = 2;
template <class A, int CT>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const __grid_constant__ RtKvWrite w, const __grid_constant__ RowMap m, bool vec, int* err) {
    constexpr int N = Unit<A>::N;
    constexpr bool SCALED = CT == RT_I8 || CT == RT_F8E4M3;
    const RtKvCache& c = w.cache;
    const Part x = part_of(m, c.n_heads);
    const int64_t* st = x.is_v ? w.v_stride : w.k_stride;
    const int t0 = blockIdx.x * m.tokens, n = min(m.tokens, w.n_tokens - t0);
    const A* src = static_cast<const A*>(x.is_v ? w.v : w.k) + (t0 + (int)threadIdx.y) * st[0] + x.head * st[1] + x.unit * N;
    const int64_t step = blockDim.y * st[0];
    void* dst = x.is_v ? c.v : c.k;
    float* scales = x.is_v ? c.v_scale : c.k_scale;
    const int64_t at = x.head * c.stride[2] + x.unit * N, scale_at = x.head * c.scale_stride[2];
    const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
    const int64_t slot = lane < n ? w.slots[t0 + lane] : -1;
    uint4 next[WRITE_BATCH];
    auto load = [&](int b) {
#pragma unroll
        for (int i = 0; i < WRITE_BATCH; i++) {
            next[i] = make_uint4(0, 0, 0, 0);
            if (x.live && b + i * (int)blockDim.y < n) next[i] = load_unit(src, vec);
            src += step;
        }
    };
    load(threadIdx.y);
    Place mine = {-1, 0};
    if (slot >= (int64_t)c.n_pages * c.page_size) {
        atomicCAS(err, 0, KERR_SLOT);
    } else if (slot >= 0) {
        const uint32_t page = ((uint32_t)slot + __umulhi((uint32_t)slot, m.page_mul)) >> m.page_shift;
        mine = place_of(c, page, (int)((uint32_t)slot - page * c.page_size));
    }
    for (int b0 = 0; b0 < n; b0 += WRITE_BATCH * blockDim.y) {   // (all lanes of a warp alike, for the shuffles)
        uint4 now[WRITE_BATCH];
#pragma unroll
        for (int i = 0; i < WRITE_BATCH; i++) now[i] = next[i];
        load(b0 + threadIdx.y + WRITE_BATCH * blockDim.y);
#pragma unroll
        for (int i = 0; i < WRITE_BATCH; i++) {
            const int token = b0 + threadIdx.y + i * blockDim.y;   // (a lane past the last holds "nowhere")
            Place p = {__shfl_sync(0xffffffffu, mine.at, token), 0};
            if constexpr (SCALED) p.scale = __shfl_sync(0xffffffffu, mine.scale, token);
            if (token >= n) p.at = -1;
            float v[N], scale = 0.0f, inv = 1.0f;
            if constexpr (SCALED) {
                constexpr float MAX_CODE = CT == RT_I8 ? 127.0f : 448.0f;
                uint32_t top = unit_top(now[i], A());
                for (int o = 1 << m.lanes_log2 >> 1; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float a = __uint_as_float(top);
                // scale = a (1/M) and code = round(x ((1/a) M)), each step rounded to fp32:
                // a function of the row that any fp32 arithmetic reproduces bit for bit
                inv = __fmul_rn(__frcp_rn(a), MAX_CODE);
                scale = __fmul_rn(a, 1.0f / MAX_CODE);
                if (a < 7.888609052210118e-31f) scale = inv = 0.0f;                   // 2^-100: M / a overflows further down
                if (top >= 0x7f800000u) { scale = __uint_as_float(0x7fc00000u); inv = 0.0f; }
                if (inv == 0.0f) now[i] = make_uint4(0, 0, 0, 0);
            }
            unit_values(now[i], v);
            if constexpr (SCALED) {
#pragma unroll
                for (int j = 0; j < N; j++) v[j] = __fmul_rn(v[j], inv);
            }
            if (p.at < 0 || !x.live) continue;
            if constexpr (SCALED)
                if (x.unit == 0) scales[p.scale + scale_at] = scale;
            put_cache<N, CT>(dst, p.at + at, v);
        }
    }
}

// A block looks its tokens' places up once (offsets, starts and pages are a
// chain of loads), then its threads take them READ_BATCH at a time.
constexpr int READ_TOKENS = 16, READ_BATCH = 8;
template <class A, int CT>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const __grid_constant__ RtKvRead r, const __grid_constant__ RowMap m, bool vec, int* err) {
    constexpr int N = Unit<A>::N;
    const RtKvCache& c = r.cache;
    __shared__ Place place[READ_TOKENS];
    const int t0 = blockIdx.x * m.tokens, n = min(m.tokens, r.n_rows - t0);
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < n; i += blockDim.x * blockDim.y) {
        const int row = t0 + i;
        Place p = {-1, 0};
        // the sequence whose rows hold this one: cu[lo] <= row < cu[lo + 1]
        int lo = 0;
        if (r.n_seqs <= 32) {   // their offsets side by side: one trip to memory, not one per halving
#pragma unroll 8
            for (int b = 1; b < r.n_seqs; b++) lo += r.cu[b] <= row;
        } else {
            int hi = r.n_seqs;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (r.cu[mid] <= row) lo = mid;
                else hi = mid;
            }
        }
        const int first = r.cu[lo];
        if (r.n_seqs > 0 && row < r.cu[r.n_seqs]) {
            const int64_t pos = (r.start ? r.start[lo] : 0) + (int64_t)(row - first);
            if (pos < 0 || pos >= min((int64_t)r.table_width * c.page_size, (int64_t)0x7fffffff) || row < first) {
                atomicCAS(err, 0, KERR_LENGTH);
            } else {
                const uint32_t ip = ((uint32_t)pos + __umulhi((uint32_t)pos, m.page_mul)) >> m.page_shift;
                const int page = r.page_table[lo * r.table_stride + ip];
                if (page < 0 || page >= c.n_pages) atomicCAS(err, 0, KERR_PAGE);
                else p = place_of(c, page, (int)pos - (int)ip * c.page_size);
            }
        }
        place[i] = p;
    }
    __syncthreads();
    const Part x = part_of(m, c.n_heads);
    if (!x.live) return;
    const int64_t* st = x.is_v ? r.v_stride : r.k_stride;
    A* dst = static_cast<A*>(x.is_v ? r.v_out : r.k_out) + x.head * st[1] + x.unit * N;
    const void* src = x.is_v ? c.v : c.k;
    const float* scales = x.is_v ? c.v_scale : c.k_scale;
    const int64_t at = x.head * c.stride[2] + x.unit * N, scale_at = x.head * c.scale_stride[2];
    for (int b = threadIdx.y; b < n; b += READ_BATCH * blockDim.y) {
        Raw<N, CT> raw[READ_BATCH];
        float s[READ_BATCH];
#pragma unroll
        for (int i = 0; i < READ_BATCH; i++) {
            const int token = b + i * blockDim.y;
            s[i] = 0.0f;
            raw[i].clear();
            if (token < n && place[token].at >= 0) {
                raw[i].load(src, place[token].at + at);
                if constexpr (CT == RT_I8 || CT == RT_F8E4M3) s[i] = scales[place[token].scale + scale_at];
            }
        }
#pragma unroll
        for (int i = 0; i < READ_BATCH; i++) {
            const int token = b + i * blockDim.y;
            if (token >= n) break;
            float y[N];
            raw[i].values(y);
            if constexpr (CT == RT_I8 || CT == RT_F8E4M3) {
#pragma unroll
                for (int j = 0; j < N; j++) y[j] *= s[i];
            }
            store_unit(dst + (t0 + token) * st[0], vec, y);
        }
    }
}

// Division by the page size as a product (Granlund and Montgomery): with 2^s
// >= d, floor(x / d) = (x + floor(x mul / 2^32)) >> s for mul = floor(2^32 (2^s -
// d) / d) + 1; the sum fits 32 bits while x < 2^31.
template <class A>
RowMap row_map(const RtKvCache& c, int n_tokens, int most, dim3& grid, dim3& block) {
    RowMap m;
    m.units = c.head_dim / Unit<A>::N;
    m.lanes_log2 = 0;
    while ((1 << m.lanes_log2) < m.units) m.lanes_log2++;
    m.per_token = (2 * c.n_heads) << m.lanes_log2;
    const int chunks = (m.per_token + KV_THREADS - 1) / KV_THREADS;
    int x = chunks == 1 ? m.per_token : ((m.per_token + chunks - 1) / chunks + 31) / 32 * 32;
    int side = std::min(KV_THREADS / x, most);
    // whole warps: by rows of threads without a token, or lanes without a part (5 heads of 16 in bf16
    // are 20 lanes a token; the last warp of 5 tokens would have 4 lanes, and a token's place is
    // fetched from the lane of the token's number)
    int step = 1;
    while (x * step % 32) step *= 2;
    if ((side + step - 1) / step * step * x > KV_THREADS) {
        x = (x + 31) / 32 * 32;
        step = 1;
        side = std::min(KV_THREADS / x, most);
    }
    // `most` tokens a block for long calls, fewer when that would leave SMs without a block
    const int64_t fill = (int64_t)n_tokens * chunks / (2 * g_num_sms);
    m.tokens = std::max(side, (int)std::min<int64_t>(most, fill) / side * side);
    grid = dim3((unsigned)(((int64_t)n_tokens + m.tokens - 1) / m.tokens), chunks);
    block = dim3(x, (std::min(side, n_tokens) + step - 1) / step * step);
    m.page_shift = 0;
    while (((uint64_t)1 << m.page_shift) < (uint64_t)c.page_size) m.page_shift++;
    m.page_mul = (uint32_t)(((uint64_t)((((uint64_t)1 << m.page_shift) - c.page_size)) << 32) / c.page_size + 1);
    return m;
}
// Whether every row of a dense operand starts on a 16-byte boundary.
bool vector_rows(const void* p, const int64_t st[2], int dtype) {
    return aligned16(p) && (st[0] * dtype_bytes(dtype)) % 16 == 0 && (st[1] * dtype_bytes(dtype)) % 16 == 0;
}

template <class A, int CT>
Status write_as(const RtKvWrite& w, cudaStream_t st) {
    dim3 grid, block;
    const RowMap m = row_map<A>(w.cache, w.n_tokens, WRITE_TOKENS, grid, block);
    const bool vec = vector_rows(w.k, w.k_stride, w.dtype) && vector_rows(w.v, w.v_stride, w.dtype);
    if (grid.y > 65535) return Status::err(RT_ERR_UNSUPPORTED, "kv_write: too many heads");
    kv_write_kernel<A, CT><<<grid, block, 0, st>>>(w, m, vec, serving_error_flag());
    RT_LAUNCH_CHECK();
    return Status::ok();
}
template <class A, int CT>
Status read_as(const RtKvRead& r, cudaStream_t st) {
    dim3 grid, block;
    const RowMap m = row_map<A>(r.cache, r.n_rows, READ_TOKENS, grid, block);
    const bool vec = vector_rows(r.k_out, r.k_stride, r.dtype) && vector_rows(r.v_out, r.v_stride, r.dtype);
    if (grid.y > 65535) return Status::err(RT_ERR_UNSUPPORTED, "kv_read: too many heads");
    kv_read_kernel<A, CT><<<grid, block, 0, st>>>(r, m, vec, serving_error_flag());
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
