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
// warp runs alone over blocks of 32 positions, K and V go from global memory
// straight into the registers of mma.sync fragments (the order of features and
// of positions inside a product is free, so each thread's fragment is made of
// whole 16-byte pieces of a row), V of a block is on its way while its scores
// are computed and the next block's K while its values are summed.  Nothing
// is staged in shared memory but the query fragments, and no warp waits for
// another before the end of its share.
//
// Precision: products must be as good as fp32 for fp32 activations.  Operands
// are split x = hi + lo and, with at most 8 rows, the hi and lo parts of one
// row take rows r and r + 8 of the same 16-row instruction, so the split costs
// nothing; 9 to 16 rows take two instructions.
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
    static constexpr int NQ = PACK ? 1 : (F32ACT ? 2 : 1);             // instructions per query fragment
    static constexpr int NP = PACK ? 1 : (MODE == M_F16 && !F32ACT ? 1 : 2);
    static constexpr int KSTEP = MODE == M_TF32 ? 8 : 16;              // features per instruction
    static constexpr int KS = DP / KSTEP;
    static constexpr int SB = 32 / ES < 8 ? 8 : 32 / ES;               // positions per register block: 32, 16, 8
    static constexpr int SUBS = 32 / SB;
    static constexpr int NT = SB / 8;                                  // score tiles of 8 positions
    static constexpr int KC = DP * ES / 64;                            // 16-byte pieces of a K row per thread
    static constexpr int VB = DP * ES / 8 < 16 ? DP * ES / 8 : 16;     // bytes of a V piece
    static constexpr int VC = DP * ES / (8 * VB);                      // pieces of a V row per thread
    static constexpr int VK = SB / 4;                                  // V rows per thread
    static constexpr int VE = VB / ES;                                 // features per piece
    static constexpr int NO = DP / 8;                                  // output tiles of 8 features
    static constexpr int SLOT = R * DP + 2 * R;                        // floats of an unfinished result
    static constexpr int Q_BYTES = NQ * KS * 32 * 16;
    static constexpr int SMEM = Q_BYTES + FW * R * (DP + 2) * 4 + 16 * 4 + 64;
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
__device__ __forceinline__ void load_piece(uint32_t (&r)[BYTES / 4], const uint8_t* p, bool live) {
#pragma unroll
    for (int i = 0; i < BYTES / 4; i++) r[i] = 0;
    if (live) {
        if constexpr (BYTES == 16)
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
        else
            asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
    }
}

// Feature of a query fragment: step ks, thread-in-quad t, element e (of 4 for
// the 16-bit products, of 2 for tf32), matching the pieces K is loaded in.
template <class F>
__device__ __forceinline__ int frag_feature(int ks, int t, int e) {
    constexpr int PER = F::MODE == M_TF32 ? 2 : 4;          // features of a thread per step
    constexpr int STEPS = 16 / F::ES / PER;                 // steps per 16-byte piece
    return (ks / STEPS) * (64 / F::ES) + t * (16 / F::ES) + (ks % STEPS) * PER + e;
}

template <int CT, bool F32ACT, int DP, int R>
__global__ void __launch_bounds__(FT) paged_few_kernel(const __grid_constant__ PagedArgs p) {
    using F = Few<CT, F32ACT, DP, R>;
    constexpr int MODE = F::MODE;
    extern __shared__ __align__(16) uint8_t smem[];
    uint4* qs = reinterpret_cast<uint4*>(smem);                             // [NQ][KS][32]
    float* os = reinterpret_cast<float*>(smem + F::Q_BYTES);                // [FW][R][DP]
    float* ml = os + FW * R * DP;                                           // [FW][2][R]
    float* qscale = ml + FW * 2 * R;                                        // [16]
    int* sched = reinterpret_cast<int*>(qscale + 16);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
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
        const int k_begin = max((cur.t.t0 + cur.i) * FKT, 0), k_end = min((cur.t.t0 + cur.i + seg) * FKT, cur.t.hi);
        const uint8_t* kb = static_cast<const uint8_t*>(c.k) + cur.h * c.stride[2] * F::ES;
        const uint8_t* vb = static_cast<const uint8_t*>(c.v) + cur.h * c.stride[2] * F::ES;
        const int* table = p.a.page_table + s.b * p.a.table_stride;

        // place of position pos (a lane each): units of 16 bytes, ~0 where no row sees it
        auto place = [&](int pos, float& ks, float& vs) -> uint32_t {
            ks = vs = 0.0f;
            if (pos >= k_end || pos < cur.t.lo) return ~0u;
            int ip, slot;
            paged_split(p, pos, ip, slot);
            const int page = table[ip];
            if (page < 0 || page >= c.n_pages) {
                atomicCAS(p.err, 0, KERR_PAGE);
                return ~0u;
            }
            if constexpr (F::Q8) {
                const int64_t sp = page * c.scale_stride[0] + slot * c.scale_stride[1] + cur.h * c.scale_stride[2];
                ks = __ldg(c.k_scale + sp);
                vs = __ldg(c.v_scale + sp);
            }
            return (uint32_t)((page * c.stride[0] + slot * c.stride[1]) * F::ES >> 4);
        };
        uint32_t kr[F::NT][F::KC][4], vr[F::VK][F::VC][F::VB / 4];
        auto load_k = [&](uint32_t off, int sub) {
#pragma unroll
            for (int n = 0; n < F::NT; n++) {
                const uint32_t o = __shfl_sync(0xffffffffu, off, sub * F::SB + n * 8 + g);
                const uint8_t* row = kb + ((uint64_t)o << 4) + t * 16;
#pragma unroll
                for (int i = 0; i < F::KC; i++) load_piece<16>(kr[n][i], row + i * 64, o != ~0u && i * 64 + t * 16 < D * F::ES);
            }
        };
        auto load_v = [&](uint32_t off, int sub) {
#pragma unroll
            for (int n = 0; n < F::VK; n++) {   // 16-bit products: rows 2t, 2t+1, 2t+8, 2t+9 of each 16; tf32: 2t, 2t+1 of each 8
                const int key = MODE == M_TF32 ? (n >> 1) * 8 + 2 * t + (n & 1) : (n >> 2) * 16 + ((n >> 1) & 1) * 8 + 2 * t + (n & 1);
                const uint32_t o = __shfl_sync(0xffffffffu, off, sub * F::SB + key);
                const uint8_t* row = vb + ((uint64_t)o << 4) + g * F::VB;
#pragma unroll
                for (int i = 0; i < F::VC; i++)
                    load_piece<F::VB>(vr[n][i], row + i * 8 * F::VB, o != ~0u && i * 8 * F::VB + g * F::VB < D * F::ES);
            }
        };

        int pos = k_begin + warp * 32;
        float ks_l, vs_l, ks_n = 0.0f, vs_n = 0.0f;
        uint32_t off = place(pos + lane, ks_l, vs_l), off_n = ~0u;
        load_k(off, 0);

        // ---- query fragments (the first K is on its way) ----
        auto q_at = [&](int r, int d) -> float {
            if (r >= rows || d >= D) return 0.0f;
            const int rr = row0 + r, tok = rr / p.group, hq = cur.h * p.group + rr % p.group;
            const int64_t at = (int64_t)(s.first + tok) * p.a.q_stride[0] + hq * p.a.q_stride[1] + d;
            return act_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.a.q)[at]) : static_cast<const float*>(p.a.q)[at];
        };
        const float base = p.a.scale * 1.4426950408889634f;
        if constexpr (MODE == M_F16) {
            for (int r = warp; r < R; r += FW) {
                float m = 0.0f;
                for (int d = lane; d < D; d += 32) m = fmaxf(m, fabsf(q_at(r, d)));
#pragma unroll
                for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                if (lane == 0) qscale[r] = pow2i(f16_scale_exp(m));
            }
            __syncthreads();
        }
        for (int e = tid; e < F::KS * 32; e += FT) {
            const int st = e >> 5, ln = e & 31, gg = ln >> 2, tt = ln & 3;
            uint32_t hi[2][2], lo[2][2];   // [row half][register]
#pragma unroll
            for (int half = 0; half < (F::PACK ? 1 : 2); half++) {
                const int r = gg + 8 * half;
                const float sc = MODE == M_F16 ? qscale[r] : 1.0f;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if constexpr (MODE == M_TF32) {
                        const uint32_t x = __float_as_uint(q_at(r, frag_feature<F>(st, tt, j)));
                        hi[half][j] = tf32_hi(x);
                        lo[half][j] = tf32_lo(x);
                    } else {
                        split_pair<MODE>(q_at(r, frag_feature<F>(st, tt, 2 * j)) * sc, q_at(r, frag_feature<F>(st, tt, 2 * j + 1)) * sc,
                                         hi[half][j], lo[half][j]);
                    }
                }
            }
            if constexpr (F::PACK) {
                qs[e] = make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1]);
            } else {
                qs[e] = make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
                if constexpr (F::NQ == 2) qs[F::KS * 32 + e] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
            }
        }
        __syncthreads();

        // ---- this thread's rows: g, and g + 8 when not packed ----
        constexpr int NR = F::PACK ? 1 : 2;
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
        float o[F::NO][4];
#pragma unroll
        for (int i = 0; i < F::NO; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][j] = 0.0f;
        float vs_max = 0.0f;   // 8-bit: the value scale that weights are expressed in

        for (; pos < k_end; pos += FKT) {
            const uint32_t ok = __ballot_sync(0xffffffffu, off != ~0u);
            const bool masked = mixed || ok != 0xffffffffu;
            off_n = place(pos + FKT + lane, ks_n, vs_n);
            if constexpr (F::Q8) {
                float top = vs_l;
#pragma unroll
                for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                if (top > vs_max) {   // with room for four times more, so that it seldom moves
                    const float to = 4.0f * top, f = vs_max / to;
#pragma unroll
                    for (int i = 0; i < F::NO; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) o[i][j] *= f;
                    vs_max = to;
                }
            }
            const float to_w = F::Q8 && vs_max > 0.0f ? W_SCALE / vs_max : 0.0f;
#pragma unroll
            for (int sub = 0; sub < F::SUBS; sub++) {
                load_v(off, sub);
                // ---- scores ----
                float sc[F::NT][4];
#pragma unroll
                for (int n = 0; n < F::NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[n][j] = 0.0f;
#pragma unroll
                for (int st = 0; st < F::KS; st++) {
                    uint32_t a[F::NQ][4];
#pragma unroll
                    for (int i = 0; i < F::NQ; i++) {
                        const uint4 x = qs[i * F::KS * 32 + st * 32 + lane];
                        a[i][0] = x.x; a[i][1] = x.y; a[i][2] = x.z; a[i][3] = x.w;
                    }
#pragma unroll
                    for (int n = 0; n < F::NT; n++) {
                        if constexpr (MODE == M_F16) {
                            uint32_t b0, b1;
                            codes_to_f16<CT>(kr[n][st / 4][st % 4], b0, b1);
#pragma unroll
                            for (int i = 0; i < F::NQ; i++) mma<MODE>(sc[n], a[i], b0, b1);
                        } else if constexpr (MODE == M_BF16) {
#pragma unroll
                            for (int i = 0; i < F::NQ; i++) mma<MODE>(sc[n], a[i], kr[n][st / 2][st % 2 * 2], kr[n][st / 2][st % 2 * 2 + 1]);
                        } else if constexpr (CT == RT_BF16) {
                            const uint32_t x = kr[n][st / 4][st % 4];
#pragma unroll
                            for (int i = 0; i < F::NQ; i++) mma<MODE>(sc[n], a[i], x << 16, x & 0xffff0000u);
                        } else {
                            const uint32_t x = kr[n][st / 2][st % 2 * 2], y = kr[n][st / 2][st % 2 * 2 + 1];
#pragma unroll
                            for (int i = 0; i < F::NQ; i++) {
                                mma<MODE>(sc[n], a[i], tf32_hi(x), tf32_hi(y));
                                mma<MODE>(sc[n], a[i], tf32_lo(x), tf32_lo(y));
                            }
                        }
                    }
                }
                // the next K block, while this one's weights and sums are made
                if (sub + 1 < F::SUBS) load_k(off, sub + 1);
                else load_k(off_n, 0);

                // ---- weights ----
                float w[F::NT][2 * NR], mx[NR];
#pragma unroll
                for (int i = 0; i < NR; i++) mx[i] = -INFINITY;
#pragma unroll
                for (int n = 0; n < F::NT; n++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int key = sub * F::SB + n * 8 + 2 * t + j;
                        const float ks = F::Q8 ? __shfl_sync(0xffffffffu, ks_l, key) : 1.0f;
#pragma unroll
                        for (int i = 0; i < NR; i++) {
                            float x = F::PACK ? sc[n][j] + sc[n][2 + j] : sc[n][2 * i + j];
                            x *= F::Q8 ? ks * c_row[i] : c_row[i];
                            if (masked && !((ok >> key & 1) && pos + key >= lo_row[i] && pos + key < hi_row[i])) x = -INFINITY;
                            w[n][2 * i + j] = x;
                            mx[i] = fmaxf(mx[i], x);
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
                                for (int j = 0; j < 4; j++) o[k][j] *= f;
                            } else {
                                o[k][2 * i] *= f;
                                o[k][2 * i + 1] *= f;
                            }
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < F::NT; n++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float vs = F::Q8 ? __shfl_sync(0xffffffffu, vs_l, sub * F::SB + n * 8 + 2 * t + j) * to_w : 1.0f;
#pragma unroll
                        for (int i = 0; i < NR; i++) {
                            float& x = w[n][2 * i + j];
                            const bool out = masked && x == -INFINITY;
                            x = out ? 0.0f : exp2_fast(x - m_ref[i]);
                            l[i] += x;
                            if constexpr (F::Q8) x = out ? 0.0f : x * vs;
                        }
                    }

                // ---- values ----
                constexpr int PN = MODE == M_TF32 ? 1 : 2;          // score tiles per product step
                // Rows that do not see a position give it weight 0, but 0 times a value that is
                // not finite is NaN.  Where rows differ, such values are taken out of the product,
                // and rows that do see one get NaN from a product of "sees" and "is not finite".
                bool strange = false;
                if constexpr (!F::Q8) {
                    if (mixed) {
#pragma unroll
                        for (int n = 0; n < F::VK; n++)
#pragma unroll
                            for (int i = 0; i < F::VC; i++)
#pragma unroll
                                for (int r = 0; r < F::VB / 4; r++) {
                                    const uint32_t x = vr[n][i][r];
                                    strange |= (x & 0x7f800000u) == 0x7f800000u || (CT == RT_BF16 && (x & 0x7f80u) == 0x7f80u);
                                }
                        strange = __any_sync(0xffffffffu, strange);
                    }
                }
#pragma unroll
                for (int st = 0; st < F::NT / PN; st++) {
                    uint32_t a[F::NP][4];
                    if constexpr (MODE == M_TF32) {
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t x = __float_as_uint(w[st][j]);
                            a[0][2 * j] = tf32_hi(x);
                            if constexpr (F::PACK) {
                                a[0][2 * j + 1] = tf32_lo(x);
                            } else {
                                const uint32_t y = __float_as_uint(w[st][2 + j]);
                                a[0][2 * j + 1] = tf32_hi(y);
                                a[F::NP - 1][2 * j] = tf32_lo(x);
                                a[F::NP - 1][2 * j + 1] = tf32_lo(y);
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            uint32_t hi, lo;
                            split_pair<MODE>(w[2 * st + j][0], w[2 * st + j][1], hi, lo);
                            a[0][2 * j] = hi;
                            if constexpr (F::PACK) {
                                a[0][2 * j + 1] = lo;
                            } else {
                                uint32_t hi2, lo2;
                                split_pair<MODE>(w[2 * st + j][2], w[2 * st + j][3], hi2, lo2);
                                a[0][2 * j + 1] = hi2;
                                if constexpr (F::NP == 2) {
                                    a[1][2 * j] = lo;
                                    a[1][2 * j + 1] = lo2;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < F::VC; i++) {
                        if constexpr (MODE == M_F16) {
#pragma unroll
                            for (int r = 0; r < F::VB / 4; r++) {
                                // features 4r .. 4r+3 of rows (2t, 2t+1) and (2t+8, 2t+9), paired by row
                                const uint32_t x0 = vr[4 * st][i][r], x1 = vr[4 * st + 1][i][r];
                                const uint32_t y0 = vr[4 * st + 2][i][r], y1 = vr[4 * st + 3][i][r];
                                uint32_t b0[4], b1[4];
                                codes_to_f16<CT>(__byte_perm(x0, x1, 0x5140), b0[0], b0[1]);
                                codes_to_f16<CT>(__byte_perm(x0, x1, 0x7362), b0[2], b0[3]);
                                codes_to_f16<CT>(__byte_perm(y0, y1, 0x5140), b1[0], b1[1]);
                                codes_to_f16<CT>(__byte_perm(y0, y1, 0x7362), b1[2], b1[3]);
#pragma unroll
                                for (int e = 0; e < 4; e++)
#pragma unroll
                                    for (int k = 0; k < F::NP; k++) mma<MODE>(o[i * F::VE + 4 * r + e], a[k], b0[e], b1[e]);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < F::VE; e++) {
                                uint32_t b0, b1;   // as the product takes them
                                float f[4];        // the values, for the check
                                if constexpr (MODE == M_BF16) {
                                    const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
                                    b0 = __byte_perm(vr[4 * st][i][e / 2], vr[4 * st + 1][i][e / 2], sel);
                                    b1 = __byte_perm(vr[4 * st + 2][i][e / 2], vr[4 * st + 3][i][e / 2], sel);
                                    f[0] = __uint_as_float(b0 << 16); f[1] = __uint_as_float(b0 & 0xffff0000u);
                                    f[2] = __uint_as_float(b1 << 16); f[3] = __uint_as_float(b1 & 0xffff0000u);
                                } else if constexpr (CT == RT_BF16) {
                                    const uint32_t x = vr[2 * st][i][e / 2], y = vr[2 * st + 1][i][e / 2];
                                    b0 = e & 1 ? x & 0xffff0000u : x << 16;
                                    b1 = e & 1 ? y & 0xffff0000u : y << 16;
                                    f[0] = f[1] = __uint_as_float(b0); f[2] = f[3] = __uint_as_float(b1);
                                } else {
                                    b0 = vr[2 * st][i][e];
                                    b1 = vr[2 * st + 1][i][e];
                                    f[0] = f[1] = __uint_as_float(b0); f[2] = f[3] = __uint_as_float(b1);
                                }
                                float(&acc)[4] = o[i * F::VE + e];
                                if (strange) {
                                    // [row sees position] x [value is not finite], in the same layout
                                    uint32_t sees[4], one0 = 0, one1 = 0;
                                    if constexpr (MODE == M_BF16) {
#pragma unroll
                                        for (int j = 0; j < 2; j++) {
#pragma unroll
                                            for (int i2 = 0; i2 < 2; i2++) {
                                                const int k0 = pos + sub * F::SB + (2 * st + j) * 8 + 2 * t, q = F::PACK ? 0 : i2;
                                                sees[2 * j + i2] = (k0 >= lo_row[q] && k0 < hi_row[q] ? 0x3f80u : 0u) |
                                                                   (k0 + 1 >= lo_row[q] && k0 + 1 < hi_row[q] ? 0x3f800000u : 0u);
                                            }
                                        }
                                        one0 = (not_finite(f[0]) ? 0x3f80u : 0u) | (not_finite(f[1]) ? 0x3f800000u : 0u);
                                        one1 = (not_finite(f[2]) ? 0x3f80u : 0u) | (not_finite(f[3]) ? 0x3f800000u : 0u);
                                        b0 &= ~((one0 & 0xffffu ? 0xffffu : 0u) | (one0 >> 16 ? 0xffff0000u : 0u));
                                        b1 &= ~((one1 & 0xffffu ? 0xffffu : 0u) | (one1 >> 16 ? 0xffff0000u : 0u));
                                    } else {
#pragma unroll
                                        for (int j = 0; j < 2; j++)
#pragma unroll
                                            for (int i2 = 0; i2 < 2; i2++) {
                                                const int k0 = pos + sub * F::SB + st * 8 + 2 * t + j, q = F::PACK ? 0 : i2;
                                                sees[2 * j + i2] = k0 >= lo_row[q] && k0 < hi_row[q] ? 0x3f800000u : 0u;
                                            }
                                        if (not_finite(f[0])) one0 = 0x3f800000u, b0 = 0;
                                        if (not_finite(f[2])) one1 = 0x3f800000u, b1 = 0;
                                    }
                                    float hit[4] = {0, 0, 0, 0};
                                    mma<MODE>(hit, sees, one0, one1);
#pragma unroll
                                    for (int j = 0; j < 4; j++)
                                        if (hit[j] != 0.0f) acc[j] = __uint_as_float(0x7fc00000u);
                                }
#pragma unroll
                                for (int k = 0; k < F::NP; k++) {
                                    if constexpr (MODE == M_TF32 && CT == RT_F32) {
                                        mma<MODE>(acc, a[k], tf32_hi(b0), tf32_hi(b1));
                                        mma<MODE>(acc, a[k], tf32_lo(b0), tf32_lo(b1));
                                    } else {
                                        mma<MODE>(acc, a[k], b0, b1);
                                    }
                                }
                            }
                        }
                    }
                }
            }
            off = off_n;
            ks_l = ks_n;
            vs_l = vs_n;
        }

        // ---- join the warps ----
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
                    const int d = i * 8 * F::VE + (2 * t + j) * F::VE + e;
                    const float* x = o[i * F::VE + e];
                    if constexpr (F::PACK) {
                        os[(warp * R + g) * DP + d] = (x[j] + x[2 + j]) * fo;
                    } else {
                        os[(warp * R + g) * DP + d] = x[j] * fo;
                        os[(warp * R + g + 8) * DP + d] = x[2 + j] * fo;
                    }
                }
        __syncthreads();
        const bool done = cur.i == 0 && seg == cur.t.count;
        float* part = p.part + (int64_t)(2 * blockIdx.x + (cur.i == 0)) * F::SLOT;
        for (int e = tid; e < R * DP; e += FT) {
            const int r = e / DP, d = e % DP;
            if (r >= rows) break;
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < FW; k++) m = fmaxf(m, ml[k * 2 * R + r]);
            float sum = 0.0f, ls = 0.0f;
            if (m != -INFINITY) {
#pragma unroll
                for (int k = 0; k < FW; k++) {
                    const float f = exp2_fast(ml[k * 2 * R + r] - m);
                    if (f == 0.0f) continue;                       // (a warp without positions)
                    sum += os[(k * R + r) * DP + d] * f;
                    ls += ml[k * 2 * R + R + r] * f;
                }
            }
            if (!done) {
                part[e] = sum;
                if (d == 0) part[R * DP + r] = m, part[R * DP + R + r] = ls;
            } else if (d < D) {
                paged_store(p, s, cur.h, row0 + r, d, ls == 0.0f ? 0.0f : sum / ls);
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
// the other 8; single-part products take 16 at the same cost.
int few_rows(const RtPagedAttention& p) {
    const bool q8 = p.cache.dtype == RT_I8 || p.cache.dtype == RT_F8E4M3;
    if (q8 && p.dtype == RT_BF16) return 16;
    return (int64_t)std::min(p.max_new, p.total_new) * (p.n_q_heads / p.cache.n_heads) <= 8 ? 8 : 16;
}

template <int CT, bool F32ACT>
Status few_sizes(PagedArgs& p, void* ws, cudaStream_t st) {
    constexpr bool ONLY16 = (CT == RT_I8 || CT == RT_F8E4M3) && !F32ACT;
    const bool wide = p.a.cache.head_dim > 64;
    if constexpr (!ONLY16)
        if (few_rows(p.a) == 8) return wide ? few_as<CT, F32ACT, 128, 8>(p, ws, st) : few_as<CT, F32ACT, 64, 8>(p, ws, st);
    return wide ? few_as<CT, F32ACT, 128, 16>(p, ws, st) : few_as<CT, F32ACT, 64, 16>(p, ws, st);
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
