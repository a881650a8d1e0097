// k_paged_few.cu -- paged attention for few rows per cache head: single
// tokens, drafted runs.
//
// out = sum_j w_j v_j / sum_j w_j over the visible positions j, w_j =
// 2^(s_j - m), s_j = q.k_j * scale * log2(e), m a running reference that is
// moved (and what has been summed rescaled) only when a score exceeds it by
// 2^8.  With R rows sharing one pass over the keys and values the call does
// 4 R operations per cached feature and reads it once: it is bound by HBM.
//
// So the work is laid out for loads in flight, not for the matrix rate: every
// warp runs alone over blocks of 32 positions and keeps STAGES - 1 pieces of
// 8 KB under way with cp.async.  The order of features and of positions inside
// a product is free, so each thread's mma.sync fragment is made of whole
// 16-byte pieces of a row: a thread copies exactly the bytes that it will use,
// to places of its own, and reads them back without a conflict or a barrier.
// No warp waits for another before the end of its share.
//
// Precision: products must be as good as fp32 for fp32 activations.  Operands
// are split x = hi + lo and, with at most 8 rows, the hi and lo parts of one
// row take rows r and r + 8 of the same 16-row instruction, so the split costs
// nothing; more rows take two instructions.
//   8-bit caches: codes are exact in fp16; q is scaled per row by a power of
//     two, weights times value scales by the largest value scale seen (22
//     significant bits each).  bf16 activations need one part (11 bits
//     against the 8 of the output).
//   bf16 cache, bf16 activations: bf16 products, exact for q.k; the weights
//     as hi + lo (16 bits).
//   the rest: tf32 products, q, weights and an fp32 cache's K and V as hi + lo
//     (22 bits); bf16 K and V are exact in tf32.
// Scores, maxima, weight sums and outputs are fp32.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "dev_math.h"
#include "paged.h"

namespace rt {
namespace {

constexpr int FT = 128, FW = FT / 32;   // threads, warps
constexpr int FKT = 32 * FW;            // positions per unit: a block of 32 for each warp
constexpr int M_F16 = 0, M_BF16 = 1, M_TF32 = 2;
constexpr float RAISE = 8.0f;           // the reference moves when a score passes it by this (log2)
constexpr float W_SCALE = 64.0f;        // fp16 weights reach 2^8 * 2^6, far from both ends of the type

template <int CT, bool F32ACT>
struct Mode {
    static constexpr int value = (CT == RT_I8 || CT == RT_F8E4M3) ? M_F16 : (CT == RT_BF16 && !F32ACT) ? M_BF16 : M_TF32;
};

template <int CT, bool F32ACT, int DP, int R>
struct Few {
    static constexpr int MODE = Mode<CT, F32ACT>::value;
    static constexpr bool Q8 = CT == RT_I8 || CT == RT_F8E4M3;
    static constexpr int ES = CT == RT_F32 ? 4 : CT == RT_BF16 ? 2 : 1;
    static constexpr bool PACK = R == 8;                               // hi / lo in rows r / r + 8
    static constexpr int RT = R <= 16 ? 1 : R / 16;                    // row tiles of 16
    static constexpr int NR = PACK ? 1 : 2 * RT;                       // rows of a thread
    static constexpr int NQ = PACK ? 1 : (F32ACT ? 2 : 1);             // instructions per query fragment
    static constexpr int NP = PACK ? 1 : (MODE == M_F16 && !F32ACT ? 1 : 2);
    static constexpr int KSTEP = MODE == M_TF32 ? 8 : 16;              // features per instruction
    static constexpr int KS = DP / KSTEP;
    static constexpr int SB = 32 / ES < 8 ? 8 : 32 / ES;               // positions per piece: 32, 16, 8
    static constexpr int SUBS = 32 / SB;
    static constexpr int NT = SB / 8;                                  // score tiles of 8 positions
    static constexpr int KC = DP * ES / 64;                            // 16-byte parts of a K row per thread
    static constexpr int VB = DP * ES / 8 < 16 ? DP * ES / 8 : 16;     // bytes of a V part
    static constexpr int VC = DP * ES / (8 * VB);                      // parts of a V row per thread
    static constexpr int VK = SB / 4;                                  // V rows per thread
    static constexpr int VE = VB / ES;                                 // features per part
    static constexpr int NO = DP / 8;                                  // output tiles of 8 features
    static constexpr int SLOT = R * DP + 2 * R;                        // floats of an unfinished result
    static constexpr int Q_BYTES = RT * NQ * KS * 32 * 16;
    static constexpr int K_BYTES = NT * KC * 512, V_BYTES = VK * VC * 32 * VB;
    static constexpr int STAGE = K_BYTES + V_BYTES + (Q8 ? 256 : 0) + 16;   // K, V, scales, existing positions
    static constexpr int STAGES = 2;
    static constexpr int RS = DP == 128 ? 152 : 72;                    // words of a row in the join: 9 per output tile, 8 (mod 16) in all
    static constexpr int JOIN = FW * R * (RS + 2) * 4;                 // sums of the warps, over the stages
    static constexpr int BODY = FW * STAGES * STAGE > JOIN ? FW * STAGES * STAGE : JOIN;
    static constexpr int SMEM = Q_BYTES + BODY + R * 4 + 64;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int MODE>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (MODE == M_F16) mma_f16(c, a, b0, b1);
    else if constexpr (MODE == M_BF16) mma_bf16(c, a, b0, b1);
    else mma_tf32(c, a, b0, b1);
}

// Four codes of a register as two fp16 pairs.
template <int CT>
__device__ __forceinline__ void codes_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if constexpr (CT == RT_I8) {
        // byte + 128 into the mantissa of 1024: 1024 + 128 + code, minus 1152
        x ^= 0x80808080u;
        const uint32_t bias = 0x64806480u;
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(bias));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(bias));
    } else {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)x));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(x >> 16)));
    }
}
__device__ __forceinline__ uint32_t tf32_hi(uint32_t x) { return (x + 0x1000u) & 0xffffe000u; }   // to the nearest
__device__ __forceinline__ uint32_t tf32_lo(uint32_t x) {
    return __float_as_uint(__uint_as_float(x) - __uint_as_float(tf32_hi(x)));
}
__device__ __forceinline__ uint32_t pair_bf16(float a, float b) {   // a in the low half, to the nearest
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// hi and lo parts of two weights as fragment registers.
template <int MODE>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
    if constexpr (MODE == M_F16) {
        hi = f16x2_rn(a, b);
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        lo = f16x2_rn(a - h.x, b - h.y);
    } else {
        hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);   // truncated: what is left is exact
        lo = pair_bf16(a - __uint_as_float(__float_as_uint(a) & 0xffff0000u),
                       b - __uint_as_float(__float_as_uint(b) & 0xffff0000u));
    }
}
__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

template <int BYTES>
__device__ __forceinline__ void copy_part(uint32_t dst, const uint8_t* src, bool live) {
    const int n = live ? BYTES : 0;   // 0: zeros
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES) : "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void read_part(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void read_part(uint32_t (&r)[2], uint32_t at) {
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
}

// Where feature f of a query fragment goes: step and thread-in-quad, matching
// the parts K is copied in (features of a thread per step: 4 for the 16-bit
// products, 2 for tf32).
template <class F>
struct QMap {
    static constexpr int PER = F::MODE == M_TF32 ? 2 : 4;
    static constexpr int STEPS = 16 / F::ES / PER;          // steps per 16-byte part
    static __device__ __forceinline__ int step(int f) { return f / (64 / F::ES) * STEPS + f % (16 / F::ES) / PER; }
    static __device__ __forceinline__ int quad(int f) { return f % (64 / F::ES) / (16 / F::ES); }
};

template <int CT, bool F32ACT, int DP, int R>
__global__ void __launch_bounds__(FT, R == 32 ? 2 : 3) paged_few_kernel(const __grid_constant__ PagedArgs p) {
    using F = Few<CT, F32ACT, DP, R>;
    constexpr int MODE = F::MODE, NR = F::NR, RT = F::RT;
    extern __shared__ __align__(16) uint8_t smem[];
    uint4* qs = reinterpret_cast<uint4*>(smem);                             // [RT][NQ][KS][32]
    float* os = reinterpret_cast<float*>(smem + F::Q_BYTES);                // [FW][R][RS], over the stages
    float* ml = os + FW * R * F::RS;                                        // [FW][2][R]
    float* qscale = reinterpret_cast<float*>(smem + F::Q_BYTES + F::BODY);  // [R]
    int* sched = reinterpret_cast<int*>(qscale + R);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const stages = smem + F::Q_BYTES + warp * F::STAGES * F::STAGE;
    const uint32_t stages_at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
    const RtKvCache& c = p.a.cache;
    const int D = c.head_dim;
    const bool act_bf16 = p.a.dtype == RT_BF16;

    asm volatile("griddepcontrol.launch_dependents;");
    PagedCursor cur;
    int u, per, total;
    if (!paged_schedule<FT, R, FKT>(p, blockIdx.x, gridDim.x, sched, cur, u, per, total)) return;
    const int u_end = (int)min((int64_t)u + per, (int64_t)total);

    while (u < u_end) {
        const int seg = p.whole ? cur.t.count : min(cur.t.count - cur.i, u_end - u);
        const PagedSeq& s = cur.s;
        const int row0 = cur.qt * R, rows = min(R, s.n * p.group - row0);
        const int k_begin = (cur.t.t0 + cur.i) * FKT, k_end = min((cur.t.t0 + cur.i + seg) * FKT, cur.t.hi);
        const uint8_t* kb = static_cast<const uint8_t*>(c.k) + cur.h * c.stride[2] * F::ES;
        const uint8_t* vb = static_cast<const uint8_t*>(c.v) + cur.h * c.stride[2] * F::ES;
        const int* table = p.a.page_table + s.b * p.a.table_stride;
        const int first = k_begin + warp * 32;                               // of this warp's blocks
        const int pieces = first < k_end ? (k_end - first + FKT - 1) / FKT * F::SUBS : 0;

        // ---- copies: a lane looks up one position of a block, a block ahead ----
        int copied = 0, page_next = -1;
        uint32_t off = ~0u;                                                  // this lane's row, units of 16 bytes
        auto page_of = [&](int pos) -> int {
            if (pos >= k_end || pos < cur.t.lo) return -1;
            int ip, slot;
            paged_split(p, pos, ip, slot);
            const int page = table[ip];
            return page < 0 ? 0x7fffffff : page;
        };
        auto copy_piece = [&]() {
            if (copied < pieces) {
                const int sub = copied % F::SUBS, pos = first + copied / F::SUBS * FKT + lane;
                const uint32_t at = stages_at + copied % F::STAGES * F::STAGE;
                if (sub == 0) {
                    off = ~0u;
                    int64_t sp = 0;
                    if (page_next >= c.n_pages) {
                        atomicCAS(p.err, 0, KERR_PAGE);
                    } else if (page_next >= 0) {
                        int ip, slot;
                        paged_split(p, pos, ip, slot);
                        off = (uint32_t)((page_next * c.stride[0] + slot * c.stride[1]) * F::ES >> 4);
                        if constexpr (F::Q8) sp = page_next * c.scale_stride[0] + slot * c.scale_stride[1] + cur.h * c.scale_stride[2];
                    }
                    page_next = page_of(pos + FKT);
                    if constexpr (F::Q8) {
                        copy_part<4>(at + F::K_BYTES + F::V_BYTES + lane * 4, reinterpret_cast<const uint8_t*>(c.k_scale + sp), off != ~0u);
                        copy_part<4>(at + F::K_BYTES + F::V_BYTES + 128 + lane * 4, reinterpret_cast<const uint8_t*>(c.v_scale + sp), off != ~0u);
                    }
                }
                const uint32_t there = __ballot_sync(0xffffffffu, off != ~0u);
                if (lane == 0) *reinterpret_cast<uint32_t*>(stages + copied % F::STAGES * F::STAGE + F::STAGE - 16) = there;
                // a row's address once, its parts at constant distances; rows that no one sees
                // give zeros
                auto rows_of = [&](auto whole) {
#pragma unroll
                    for (int n = 0; n < F::NT; n++) {
                        const uint32_t o = __shfl_sync(0xffffffffu, off, sub * F::SB + n * 8 + g);
                        const bool live = o != ~0u;
                        const uint8_t* row = kb + (live ? ((uint64_t)o << 4) + t * 16 : 0);
#pragma unroll
                        for (int i = 0; i < F::KC; i++) {
                            const bool in = decltype(whole)::value || i * 64 + t * 16 < D * F::ES;
                            copy_part<16>(at + ((n * F::KC + i) * 32 + lane) * 16, in ? row + i * 64 : kb, live && in);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < F::VK; n++) {   // 16-bit products: rows 2t, 2t+1, 2t+8, 2t+9 of each 16; tf32: 2t, 2t+1 of each 8
                        const int key = MODE == M_TF32 ? (n >> 1) * 8 + 2 * t + (n & 1) : (n >> 2) * 16 + ((n >> 1) & 1) * 8 + 2 * t + (n & 1);
                        const uint32_t o = __shfl_sync(0xffffffffu, off, sub * F::SB + key);
                        const bool live = o != ~0u;
                        const uint8_t* row = vb + (live ? ((uint64_t)o << 4) + g * F::VB : 0);
#pragma unroll
                        for (int i = 0; i < F::VC; i++) {
                            const bool in = decltype(whole)::value || i * 8 * F::VB + g * F::VB < D * F::ES;
                            copy_part<F::VB>(at + F::K_BYTES + ((n * F::VC + i) * 32 + lane) * F::VB, in ? row + i * 8 * F::VB : vb, live && in);
                        }
                    }
                };
                if (D == DP) rows_of(std::true_type());
                else rows_of(std::false_type());
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            copied++;
        };
        page_next = page_of(first + lane);
#pragma unroll
        for (int i = 0; i < F::STAGES - 1; i++) copy_piece();

        // ---- query fragments (the first pieces are on their way): 8 features a thread ----
        const float base = p.a.scale * 1.4426950408889634f;
        constexpr int LQ = DP / 8;                          // threads of a row
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += FT / LQ) {
            const int r = r0 + tid / LQ, d = tid % LQ * 8;
            if (R < FT / LQ && r >= R) break;               // (whole rows, which lie in whole half warps)
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = 0.0f;
            if (r < rows && d < D) {
                const int rr = row0 + r, tok = rr / p.group, hq = cur.h * p.group + rr - tok * p.group;
                const int64_t at = (int64_t)(s.first + tok) * p.a.q_stride[0] + hq * p.a.q_stride[1] + d;
                if (act_bf16) {
                    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.a.q) + at;
                    if (p.vec_q) {
                        const uint4 v = *reinterpret_cast<const uint4*>(q);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[2 * i] = __uint_as_float(w[i] << 16);
                            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = __bfloat162float(q[i]);
                    }
                } else {
                    const float* q = static_cast<const float*>(p.a.q) + at;
                    if (p.vec_q) {
                        const float4 v = *reinterpret_cast<const float4*>(q), w = *reinterpret_cast<const float4*>(q + 4);
                        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
                        x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = q[i];
                    }
                }
            }
            if constexpr (MODE == M_F16) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
                const uint32_t mates = (LQ == 16 ? 0xffffu : 0xffu) << (lane / LQ * LQ);
                m = __uint_as_float(__reduce_max_sync(mates, __float_as_uint(m)));
                const float up = pow2i(f16_scale_exp(m));
                if (tid % LQ == 0) qscale[r] = up;
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= up;
            }
            using M = QMap<F>;
            uint32_t* q = reinterpret_cast<uint32_t*>(qs + r / 16 * F::NQ * F::KS * 32);
#pragma unroll
            for (int i = 0; i < 8; i += M::PER) {
                uint32_t hi[2], lo[2];
                if constexpr (MODE == M_TF32) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        hi[j] = tf32_hi(__float_as_uint(x[i + j]));
                        lo[j] = tf32_lo(__float_as_uint(x[i + j]));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; j++) split_pair<MODE>(x[i + 2 * j], x[i + 2 * j + 1], hi[j], lo[j]);
                }
                uint32_t* e = q + (M::step(d + i) * 32 + r % 8 * 4 + M::quad(d + i)) * 4;
                if constexpr (F::PACK) {
                    *reinterpret_cast<uint4*>(e) = make_uint4(hi[0], lo[0], hi[1], lo[1]);
                } else {
                    const int half = r >> 3 & 1;
                    e[half] = hi[0];
                    e[half + 2] = hi[1];
                    if constexpr (F::NQ == 2) {
                        e[F::KS * 128 + half] = lo[0];
                        e[F::KS * 128 + half + 2] = lo[1];
                    }
                }
            }
        }
        __syncthreads();

        // ---- this thread's rows: g (+ 8, + 16, ...) ----
        float c_row[NR], m_ref[NR], l[NR];
        int lo_row[NR], hi_row[NR];
        bool mixed = false;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int r = g + 8 * i, tok = (row0 + r) / p.group, at = s.L - s.n + tok;
            c_row[i] = MODE == M_F16 ? base / qscale[r] : base;
            m_ref[i] = -INFINITY;
            l[i] = 0.0f;
            lo_row[i] = p.a.window > 0 ? max(0, at - p.a.window + 1) : 0;
            hi_row[i] = r < rows ? (p.a.causal ? min(s.L, at + 1) : s.L) : 0;
            mixed |= r < rows && (lo_row[i] > cur.t.lo || hi_row[i] < cur.t.hi);
        }
        mixed = __any_sync(0xffffffffu, mixed);   // rows that see different positions share this tile
        float o[RT][F::NO][4];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int i = 0; i < F::NO; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[rt][i][j] = 0.0f;
        float vs_max = 0.0f;   // 8-bit: the value scale that weights are expressed in

#pragma unroll 1
        for (int piece = 0; piece < pieces; piece++) {
            copies_wait<F::STAGES - 2>();
            __syncwarp();                       // scales and notes of other lanes; all are done with the stage that is refilled
            copy_piece();
            const uint8_t* stage = stages + piece % F::STAGES * F::STAGE;
            const uint32_t at = stages_at + piece % F::STAGES * F::STAGE;
            const int sub = piece % F::SUBS, pos = first + piece / F::SUBS * FKT + sub * F::SB;
            const uint32_t ok = *reinterpret_cast<const uint32_t*>(stage + F::STAGE - 16) >> (sub * F::SB);
            constexpr uint32_t ALL = F::SB == 32 ? 0xffffffffu : (1u << F::SB) - 1;
            const bool masked = mixed || (ok & ALL) != ALL;
            const float* k_scale = reinterpret_cast<const float*>(stage + F::K_BYTES + F::V_BYTES);
            const float* v_scale = k_scale + 32;
            float to_w = 0.0f;
            if constexpr (F::Q8) {
                const float mine = v_scale[lane];
                const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, mine > 0.0f && mine < INFINITY ? __float_as_uint(mine) : 0u));
                if (top > vs_max) {   // with room for four times more, so that it seldom moves
                    const float to = 4.0f * top, f = vs_max / to;
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int i = 0; i < F::NO; i++)
#pragma unroll
                            for (int j = 0; j < 4; j++) o[rt][i][j] *= f;
                    vs_max = to;
                }
                to_w = vs_max > 0.0f ? W_SCALE / vs_max : 0.0f;
            }
            // ---- scores ----
            float sc[RT][F::NT][4];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int n = 0; n < F::NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[rt][n][j] = 0.0f;
            constexpr int PER = F::KS / F::KC;          // steps per 16-byte part
#pragma unroll
            for (int i = 0; i < F::KC; i++) {
                uint32_t kr[F::NT][4];
#pragma unroll
                for (int n = 0; n < F::NT; n++) read_part(kr[n], at + ((n * F::KC + i) * 32 + lane) * 16);
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    uint32_t a[RT][F::NQ][4];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int k = 0; k < F::NQ; k++) {
                            const uint4 x = qs[((rt * F::NQ + k) * F::KS + i * PER + e) * 32 + lane];
                            a[rt][k][0] = x.x; a[rt][k][1] = x.y; a[rt][k][2] = x.z; a[rt][k][3] = x.w;
                        }
#pragma unroll
                    for (int n = 0; n < F::NT; n++) {
                        uint32_t b0, b1;
                        if constexpr (MODE == M_F16) {
                            codes_to_f16<CT>(kr[n][e], b0, b1);
                        } else if constexpr (MODE == M_BF16 || CT == RT_F32) {
                            b0 = kr[n][2 * e];
                            b1 = kr[n][2 * e + 1];
                        } else {
                            b0 = kr[n][e] << 16;
                            b1 = kr[n][e] & 0xffff0000u;
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int k = 0; k < F::NQ; k++) {
                                if constexpr (CT == RT_F32) {
                                    mma<MODE>(sc[rt][n], a[rt][k], tf32_hi(b0), tf32_hi(b1));
                                    mma<MODE>(sc[rt][n], a[rt][k], tf32_lo(b0), tf32_lo(b1));
                                } else {
                                    mma<MODE>(sc[rt][n], a[rt][k], b0, b1);
                                }
                            }
                    }
                }
            }

            // ---- weights ----
            float w[F::NT][2 * NR], mx[NR];
#pragma unroll
            for (int i = 0; i < NR; i++) mx[i] = -INFINITY;
#pragma unroll
            for (int n = 0; n < F::NT; n++) {
                float2 ks = make_float2(1.0f, 1.0f);
                if constexpr (F::Q8) ks = *reinterpret_cast<const float2*>(k_scale + n * 8 + 2 * t);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int key = n * 8 + 2 * t + j;
#pragma unroll
                    for (int i = 0; i < NR; i++) {
                        float x = F::PACK ? sc[0][n][j] + sc[0][n][2 + j] : sc[i / 2][n][2 * (i & 1) + j];
                        x *= F::Q8 ? (j ? ks.y : ks.x) * c_row[i] : c_row[i];
                        if (masked && !((ok >> key & 1) && pos + key >= lo_row[i] && pos + key < hi_row[i])) x = -INFINITY;
                        w[n][2 * i + j] = x;
                        mx[i] = fmaxf(mx[i], x);
                    }
                }
            }
            bool raise = false;
#pragma unroll
            for (int i = 0; i < NR; i++) raise |= mx[i] > m_ref[i] + RAISE;
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    float m = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    m = fmaxf(m, m_ref[i]);
                    const float f = m == m_ref[i] ? 1.0f : exp2_fast(m_ref[i] - m);
                    m_ref[i] = m;
                    l[i] *= f;
#pragma unroll
                    for (int k = 0; k < F::NO; k++) {
                        if constexpr (F::PACK) {
#pragma unroll
                            for (int j = 0; j < 4; j++) o[0][k][j] *= f;
                        } else {
                            o[i / 2][k][2 * (i & 1)] *= f;
                            o[i / 2][k][2 * (i & 1) + 1] *= f;
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < F::NT; n++) {
                float2 vs = make_float2(1.0f, 1.0f);
                if constexpr (F::Q8) {
                    vs = *reinterpret_cast<const float2*>(v_scale + n * 8 + 2 * t);
                    vs.x *= to_w;
                    vs.y *= to_w;
                }
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int i = 0; i < NR; i++) {
                        float& x = w[n][2 * i + j];
                        const bool out = masked && x == -INFINITY;
                        x = out ? 0.0f : exp2_fast(x - m_ref[i]);
                        l[i] += x;
                        if constexpr (F::Q8) x = out ? 0.0f : x * (j ? vs.y : vs.x);
                    }
            }

            // ---- values ----
            constexpr int PN = MODE == M_TF32 ? 1 : 2, VR = MODE == M_TF32 ? 2 : 4;   // score tiles, V rows per product step
            // Rows that do not see a position give it weight 0, but 0 times a value that is
            // not finite is NaN.  Where rows differ, such values are taken out of the product,
            // and rows that do see one get NaN from a product of "sees" and "is not finite".
            bool strange = false;
            if constexpr (!F::Q8) {
                if (mixed) {
#pragma unroll 1
                    for (int i = 0; i < F::VK * F::VC; i++) {
                        uint32_t x[4];
                        read_part(x, at + F::K_BYTES + (i * 32 + lane) * 16);
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            strange |= (x[r] & 0x7f800000u) == 0x7f800000u || (CT == RT_BF16 && (x[r] & 0x7f80u) == 0x7f80u);
                    }
                    strange = __any_sync(0xffffffffu, strange);
                }
            }
#pragma unroll
            for (int st = 0; st < F::NT / PN; st++) {
                uint32_t a[RT][F::NP][4];
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if constexpr (MODE == M_TF32) {
                            const uint32_t x = __float_as_uint(w[st][4 * rt + j]);
                            a[rt][0][2 * j] = tf32_hi(x);
                            if constexpr (F::PACK) {
                                a[rt][0][2 * j + 1] = tf32_lo(x);
                            } else {
                                const uint32_t y = __float_as_uint(w[st][4 * rt + 2 + j]);
                                a[rt][0][2 * j + 1] = tf32_hi(y);
                                a[rt][F::NP - 1][2 * j] = tf32_lo(x);
                                a[rt][F::NP - 1][2 * j + 1] = tf32_lo(y);
                            }
                        } else {
                            const float* x = w[2 * st + j] + 4 * rt;
                            uint32_t hi, lo;
                            split_pair<MODE>(x[0], x[1], hi, lo);
                            a[rt][0][2 * j] = hi;
                            if constexpr (F::PACK) {
                                a[rt][0][2 * j + 1] = lo;
                            } else {
                                uint32_t hi2, lo2;
                                split_pair<MODE>(x[2], x[3], hi2, lo2);
                                a[rt][0][2 * j + 1] = hi2;
                                if constexpr (F::NP == 2) {
                                    a[rt][1][2 * j] = lo;
                                    a[rt][1][2 * j + 1] = lo2;
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < F::VC; i++) {
                    uint32_t vr[VR][F::VB / 4];
#pragma unroll
                    for (int n = 0; n < VR; n++) read_part(vr[n], at + F::K_BYTES + (((st * VR + n) * F::VC + i) * 32 + lane) * F::VB);
                    if constexpr (MODE == M_F16) {
#pragma unroll
                        for (int r = 0; r < F::VB / 4; r++) {
                            // features 4r .. 4r+3 of rows (2t, 2t+1) and (2t+8, 2t+9), paired by row
                            uint32_t b0[4], b1[4];
                            codes_to_f16<CT>(__byte_perm(vr[0][r], vr[1][r], 0x5140), b0[0], b0[1]);
                            codes_to_f16<CT>(__byte_perm(vr[0][r], vr[1][r], 0x7362), b0[2], b0[3]);
                            codes_to_f16<CT>(__byte_perm(vr[2][r], vr[3][r], 0x5140), b1[0], b1[1]);
                            codes_to_f16<CT>(__byte_perm(vr[2][r], vr[3][r], 0x7362), b1[2], b1[3]);
#pragma unroll
                            for (int e = 0; e < 4; e++)
#pragma unroll
                                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                                    for (int k = 0; k < F::NP; k++) mma<MODE>(o[rt][i * F::VE + 4 * r + e], a[rt][k], b0[e], b1[e]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < F::VE; e++) {
                            uint32_t b0, b1;   // as the product takes them
                            float f[4];        // the values, for the check
                            if constexpr (MODE == M_BF16) {
                                const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
                                b0 = __byte_perm(vr[0][e / 2], vr[1][e / 2], sel);
                                b1 = __byte_perm(vr[2][e / 2], vr[3][e / 2], sel);
                                f[0] = __uint_as_float(b0 << 16); f[1] = __uint_as_float(b0 & 0xffff0000u);
                                f[2] = __uint_as_float(b1 << 16); f[3] = __uint_as_float(b1 & 0xffff0000u);
                            } else {
                                if constexpr (CT == RT_BF16) {
                                    b0 = e & 1 ? vr[0][e / 2] & 0xffff0000u : vr[0][e / 2] << 16;
                                    b1 = e & 1 ? vr[1][e / 2] & 0xffff0000u : vr[1][e / 2] << 16;
                                } else {
                                    b0 = vr[0][e];
                                    b1 = vr[1][e];
                                }
                                f[0] = f[1] = __uint_as_float(b0); f[2] = f[3] = __uint_as_float(b1);
                            }
                            if (strange) {
                                uint32_t one0 = 0, one1 = 0;
                                if constexpr (MODE == M_BF16) {
                                    one0 = (not_finite(f[0]) ? 0x3f80u : 0u) | (not_finite(f[1]) ? 0x3f800000u : 0u);
                                    one1 = (not_finite(f[2]) ? 0x3f80u : 0u) | (not_finite(f[3]) ? 0x3f800000u : 0u);
                                    b0 &= ~((one0 & 0xffffu ? 0xffffu : 0u) | (one0 >> 16 ? 0xffff0000u : 0u));
                                    b1 &= ~((one1 & 0xffffu ? 0xffffu : 0u) | (one1 >> 16 ? 0xffff0000u : 0u));
                                } else {
                                    if (not_finite(f[0])) one0 = 0x3f800000u, b0 = 0;
                                    if (not_finite(f[2])) one1 = 0x3f800000u, b1 = 0;
                                }
#pragma unroll
                                for (int rt = 0; rt < RT; rt++) {
                                    // [row sees position] x [value is not finite], in the layout of the product
                                    uint32_t sees[4];
#pragma unroll
                                    for (int j = 0; j < 2; j++)
#pragma unroll
                                        for (int i2 = 0; i2 < 2; i2++) {
                                            const int q = F::PACK ? 0 : 2 * rt + i2;
                                            const int k0 = MODE == M_TF32 ? pos + st * 8 + 2 * t + j : pos + (2 * st + j) * 8 + 2 * t;
                                            const bool s0 = k0 >= lo_row[q] && k0 < hi_row[q], s1 = k0 + 1 >= lo_row[q] && k0 + 1 < hi_row[q];
                                            sees[2 * j + i2] = MODE == M_TF32 ? (s0 ? 0x3f800000u : 0u) : (s0 ? 0x3f80u : 0u) | (s1 ? 0x3f800000u : 0u);
                                        }
                                    float hit[4] = {0, 0, 0, 0};
                                    mma<MODE>(hit, sees, one0, one1);
#pragma unroll
                                    for (int j = 0; j < 4; j++)
                                        if (hit[j] != 0.0f) o[rt][i * F::VE + e][j] = __uint_as_float(0x7fc00000u);
                                }
                            }
#pragma unroll
                            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                                for (int k = 0; k < F::NP; k++) {
                                    float(&acc)[4] = o[rt][i * F::VE + e];
                                    if constexpr (CT == RT_F32) {
                                        mma<MODE>(acc, a[rt][k], tf32_hi(b0), tf32_hi(b1));
                                        mma<MODE>(acc, a[rt][k], tf32_lo(b0), tf32_lo(b1));
                                    } else {
                                        mma<MODE>(acc, a[rt][k], b0, b1);
                                    }
                                }
                        }
                    }
                }
            }
        }

        // ---- join the warps ----
        copies_wait<0>();
        __syncthreads();                        // nobody needs the stages any more
        const float fo = F::Q8 ? vs_max / W_SCALE : 1.0f;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) {
                ml[warp * 2 * R + g + 8 * i] = m_ref[i];
                ml[warp * 2 * R + R + g + 8 * i] = l[i];
            }
        }
#pragma unroll
        for (int i = 0; i < F::VC; i++)
#pragma unroll
            for (int e = 0; e < F::VE; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    // word n * 9 + column of the row: a warp's stores and loads meet few conflicts
#pragma unroll
                    for (int k = 0; k < NR; k++) {
                        const float* x = o[k / 2][i * F::VE + e];
                        os[(warp * R + g + 8 * k) * F::RS + (i * F::VE + e) * 9 + 2 * t + j] = (F::PACK ? x[j] + x[2 + j] : x[2 * (k & 1) + j]) * fo;
                    }
                }
        __syncthreads();
        const bool done = cur.i == 0 && seg == cur.t.count;
        float* part = p.part + (int64_t)(2 * blockIdx.x + (cur.i == 0)) * F::SLOT;
        for (int e = tid; e < rows * (DP / 4); e += FT) {   // 4 features of a row a thread
            const int r = e / (DP / 4), d = e % (DP / 4) * 4;
            float f[FW], m = -INFINITY, ls = 0.0f, sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < FW; k++) {
                f[k] = ml[k * 2 * R + r];
                m = fmaxf(m, f[k]);
            }
#pragma unroll
            for (int k = 0; k < FW; k++) {
                f[k] = f[k] == -INFINITY ? 0.0f : exp2_fast(f[k] - m);   // (a warp without positions)
                if (f[k] == 0.0f) continue;
                ls += ml[k * 2 * R + R + r] * f[k];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int n = (d + j) / (8 * F::VE) * F::VE + (d + j) % F::VE, col = (d + j) / F::VE % 8;
                    sum[j] += os[(k * R + r) * F::RS + n * 9 + col] * f[k];
                }
            }
            if (!done) {
                *reinterpret_cast<float4*>(part + r * DP + d) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                if (d == 0) part[R * DP + r] = m, part[R * DP + R + r] = ls;
            } else if (d < D) {
                const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                paged_store4(p, s, cur.h, row0 + r, d, sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
                if (d == 0) paged_store_lse(p, s, cur.h, row0 + r, m, ls);
            }
        }
        __syncthreads();
        u += p.whole ? 1 : seg;
        cur.next_item<R, FKT>(p);
    }
}

// Calls whose longest sequence fits this many positions run as one launch,
// every item in one block: the join would cost more than it spreads.
constexpr int WHOLE_KEYS = 512;
constexpr int MIN_UNITS = 2;

template <int CT, bool F32ACT, int DP, int R>
int few_blocks_per_sm() {
    using F = Few<CT, F32ACT, DP, R>;
    static int n = [] {
        int k = 0;
        cudaFuncSetAttribute(paged_few_kernel<CT, F32ACT, DP, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&k, paged_few_kernel<CT, F32ACT, DP, R>, FT, F::SMEM) != cudaSuccess || k < 1) {
            cudaGetLastError();
            k = 1;
        }
        return k;
    }();
    return n;
}
constexpr int MAX_BLOCKS_PER_SM = 4;

// Blocks of a call: no more than fit the GPU at once, no more than it has work for.
int few_blocks(const RtPagedAttention& p, int R, int per_sm, bool whole) {
    const int64_t group = p.n_q_heads / p.cache.n_heads;
    const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(p.max_new, p.total_new)) * group;
    const int64_t items = (int64_t)p.n_seqs * p.cache.n_heads * ((rows + R - 1) / R);
    const int64_t units = whole ? items : items * ((p.max_kv + FKT - 1) / FKT);
    return (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)g_num_sms * per_sm, whole ? units : (units + MIN_UNITS - 1) / MIN_UNITS));
}

template <int CT, bool F32ACT, int DP, int R>
Status few_as(PagedArgs& p, void* ws, cudaStream_t st) {
    using F = Few<CT, F32ACT, DP, R>;
    const int per_sm = std::min(MAX_BLOCKS_PER_SM, few_blocks_per_sm<CT, F32ACT, DP, R>());
    const int blocks = few_blocks(p.a, R, per_sm, p.whole);
    p.part = static_cast<float*>(ws);
    p.min_units = p.whole ? 1 : MIN_UNITS;
    paged_few_kernel<CT, F32ACT, DP, R><<<blocks, FT, F::SMEM, st>>>(p);
    RT_LAUNCH_CHECK();
    if (p.whole || blocks == 1) return Status::ok();
    return launch_paged_join<DP, R, FKT>(p, blocks, st);
}

// Rows of a tile: 8 when that covers a call's rows and the hi / lo parts need
// the other 8; single-part products take 16 at the same cost, and two tiles of
// 16 over the same keys when there are more.
int few_rows(const RtPagedAttention& p) {
    const bool q8 = p.cache.dtype == RT_I8 || p.cache.dtype == RT_F8E4M3, bf = p.dtype == RT_BF16;
    const int64_t rows = (int64_t)std::min(p.max_new, p.total_new) * (p.n_q_heads / p.cache.n_heads);
    if (bf && rows > 16 && p.cache.dtype != RT_F32) return 32;
    return rows <= 8 && !(q8 && bf) ? 8 : 16;
}

template <int CT, bool F32ACT, int R>
Status few_dim(PagedArgs& p, void* ws, cudaStream_t st) {
    return p.a.cache.head_dim > 64 ? few_as<CT, F32ACT, 128, R>(p, ws, st) : few_as<CT, F32ACT, 64, R>(p, ws, st);
}
template <int CT, bool F32ACT>
Status few_sizes(PagedArgs& p, void* ws, cudaStream_t st) {
    constexpr bool Q8 = CT == RT_I8 || CT == RT_F8E4M3;
    const int rows = few_rows(p.a);
    if constexpr (!F32ACT)
        if (rows == 32) return few_dim<CT, F32ACT, 32>(p, ws, st);
    if constexpr (!Q8 || F32ACT)
        if (rows == 8) return few_dim<CT, F32ACT, 8>(p, ws, st);
    return few_dim<CT, F32ACT, 16>(p, ws, st);
}

bool few_whole(const RtPagedAttention& p) { return p.max_kv <= WHOLE_KEYS; }

}  // namespace

size_t paged_few_workspace(const RtPagedAttention& p) {
    if (few_whole(p)) return 0;
    const int R = few_rows(p), DP = p.cache.head_dim > 64 ? 128 : 64;
    return (size_t)few_blocks(p, R, MAX_BLOCKS_PER_SM, false) * 2 * (R * DP + 2 * R) * sizeof(float);
}

Status launch_paged_few(PagedArgs& p, void* ws, cudaStream_t st) {
    p.whole = few_whole(p.a);
    const bool f32 = p.a.dtype == RT_F32;
    switch (p.a.cache.dtype) {
        case RT_F32: return few_sizes<RT_F32, true>(p, ws, st);   // (bf16 activations need the same products)
        case RT_BF16: return f32 ? few_sizes<RT_BF16, true>(p, ws, st) : few_sizes<RT_BF16, false>(p, ws, st);
        case RT_F8E4M3: return f32 ? few_sizes<RT_F8E4M3, true>(p, ws, st) : few_sizes<RT_F8E4M3, false>(p, ws, st);
        default: return f32 ? few_sizes<RT_I8, true>(p, ws, st) : few_sizes<RT_I8, false>(p, ws, st);
    }
}

}  // namespace rt
