// k_paged_few.cu -- paged attention for few rows per cache head: single
// tokens, drafted runs.
//
// out = sum_j w_j v_j / sum_j w_j over the visible positions j, w_j =
// 2^(s_j - m), s_j = q.k_j * scale * log2(e), m a running reference that is
// moved (and what has been summed rescaled) only when a score exceeds it by
// 2^8.  With R rows sharing one pass over the keys and values the call does
// 4 R operations per cached feature and reads it once: it is bound by HBM.
//
// So the work is laid out for loads in flight, not for the matrix rate (128 KB
// under way per SM reach 6.4 TB/s of rows of 128 bytes, 64 KB 4.4 TB/s): every
// warp runs alone over blocks of 32 positions of one cache head, with a ring of
// its own that cp.async fills, K and V of a piece in slots of their own so that
// all but the one in use are under way.  The order of features and of positions
// inside a product is free, so each thread's mma.sync fragment is made of whole
// 16-byte parts of a row, read back without a conflict or a transpose.  A copy
// instruction takes whole rows of K (2 x 131072 positions in bf16: 236 -> 209 us
// against threads that copy their own parts, 64 bytes of each of 8 rows);
// for 8-bit rows of 128 bytes, with a look-up for every 4 of them, the latter
// is the faster one (64 sequences over int8: 164 against 177 us).
// The warps of a block take heads of the same positions (neighbours in memory)
// when there is enough work for that, blocks of positions of one head otherwise;
// only then is there something to add up between them, at the end of an item.
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
//
// Measured: 64 sequences of up to 8192 positions, one token each, 8 heads of
// 128: int8 164 us = 3.9 TB/s, bf16 262 = 4.8, fp32 625 = 4.0; two of 131072
// in bf16 210 us = 5.1 TB/s.  8-bit caches are bound by the chain of dependent
// instructions of three warps a scheduler (issue slots 44 % busy, DRAM 47 %;
// the registers allow no fourth warp), and half of what is issued is the
// copies: a look-up and an address for each 128 bytes, scales 4 bytes at a time;
// the others are bound by loads in flight.  Drafted runs of 5 tokens x 4 heads
// (32 rows) over fp8 126 us: the rows' weights and fragments are 4 times those
// of 8 rows.  One token over 200 positions in fp32 takes 14 us, a chain of 4300
// instructions a warp.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "dev_math.h"
#include "paged.h"

namespace rt {
namespace {

constexpr int FT = 128, FW = FT / 32;   // threads, warps
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
    // The tensor core's sum truncates (toward zero, in steps of 2^-24 of it): over a few thousand
    // positions of an fp32 cache the output fell short by 1.2e-6 of its value.  With fp32 outputs
    // products are summed from zero every 8 positions, and added up in fp32 registers.
    static constexpr bool FOLD = MODE == M_TF32 && F32ACT;
    static constexpr int KSTEP = MODE == M_TF32 ? 8 : 16;              // features per instruction
    static constexpr int KS = DP / KSTEP;
    static constexpr int SB = 32 / ES;                                 // positions per piece: 32, 16, 8
    static constexpr int SUBS = 32 / SB;
    static constexpr int NT = SB / 8;                                  // score tiles of 8 positions
    static constexpr int KC = DP * ES / 64;                            // 16-byte parts of a K row per thread
    static constexpr int K_LANES = DP * ES / 16 < 32 ? DP * ES / 16 : 32, K_ROWS = 32 / K_LANES;   // of a copy
    static constexpr bool K_PRIVATE = ES == 1;                         // a thread copies its own parts of K
    static constexpr int VB = DP * ES / 8 < 16 ? DP * ES / 8 : 16;     // bytes of a V part
    static constexpr int VC = DP * ES / (8 * VB);                      // parts of a V row per thread
    static constexpr int VK = SB / 4;                                  // V rows per thread
    static constexpr int VE = VB / ES;                                 // features per part
    static constexpr int NO = DP / 8;                                  // output tiles of 8 features
    static constexpr int SLOT = R * DP + 2 * R;                        // floats of an unfinished result
    static constexpr bool Q_REGS = MODE != M_TF32 && RT * NQ == 1;     // query fragments in registers (32 of them)
    // otherwise in shared memory, a thread's own: tf32 as the values themselves
    // (hi and lo are made again for each use), 16 bits as the fragments
    static constexpr int Q_BYTES = Q_REGS ? 0 : MODE == M_TF32 ? KS * (PACK ? 1 : 2) * 32 * 8 : RT * NQ * KS * 32 * 16;
    static constexpr int HALF = NT * KC * 512;                         // K, or V, of a piece
    static_assert(HALF == VK * VC * 32 * VB, "K and V alike");
    static constexpr int SLOT_BYTES = HALF + (Q8 ? 128 : 0) + 16;       // and scales, and which positions exist
    static constexpr int SLOTS = 16 * 1024 / HALF < 8 ? 16 * 1024 / HALF : 8;
    static constexpr int RS = DP == 128 ? 152 : 72;                    // words of a row in the join: 9 per output tile, 8 (mod 16) in all
    static constexpr int JOIN = FW * R * (RS + 2) * 4;                 // sums of the warps, over the rings
    static constexpr int BODY = FW * SLOTS * SLOT_BYTES > JOIN ? FW * SLOTS * SLOT_BYTES : JOIN;
    static constexpr int SMEM = FW * Q_BYTES + BODY + 64;
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

template <int CT, bool F32ACT, int DP, int R>
__global__ void __launch_bounds__(FT, R == 32 ? 2 : 3) paged_few_kernel(const __grid_constant__ PagedArgs p) {
    using F = Few<CT, F32ACT, DP, R>;
    constexpr int MODE = F::MODE, NR = F::NR, RT = F::RT;
    extern __shared__ __align__(16) uint8_t smem[];
    float* os = reinterpret_cast<float*>(smem + FW * F::Q_BYTES);           // [FW][R][RS], over the rings
    float* ml = os + FW * R * F::RS;                                        // [FW][2][R]
    int* sched = reinterpret_cast<int*>(smem + FW * F::Q_BYTES + F::BODY);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const my_q = smem + warp * F::Q_BYTES;
    uint8_t* const ring = smem + FW * F::Q_BYTES + warp * F::SLOTS * F::SLOT_BYTES;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    const RtKvCache& c = p.a.cache;
    const int D = c.head_dim;
    const bool act_bf16 = p.a.dtype == RT_BF16;
    const int key_warps = FW / p.head_group, w_head = warp & (p.head_group - 1), w_key = warp / p.head_group;
    const int stride = 32 * key_warps;                                      // positions of a key tile

    asm volatile("griddepcontrol.launch_dependents;");
    PagedCursor cur;
    int u, per, total;
    bool rest;
    const bool some = paged_schedule<FT, R>(p, blockIdx.x, gridDim.x, sched, cur, u, per, total, rest);
    paged_note<R>(p, some, cur, u, per);
    const int u_end = some ? (int)min((int64_t)u + per, (int64_t)total) : u;

    while (u < u_end) {
        const int seg = p.whole ? cur.t.count : min(cur.t.count - cur.i, u_end - u);
        const PagedSeq& s = cur.s;
        const int row0 = cur.qt * R, rows = min(R, s.n * p.group - row0), head = cur.h * p.head_group + w_head;
        const int k_begin = (cur.t.t0 + cur.i) << p.key_shift, k_end = min((cur.t.t0 + cur.i + seg) << p.key_shift, cur.t.hi);
        const uint8_t* kb = static_cast<const uint8_t*>(c.k) + head * c.stride[2] * F::ES;
        const uint8_t* vb = static_cast<const uint8_t*>(c.v) + head * c.stride[2] * F::ES;
        const int* table = p.a.page_table + s.b * p.a.table_stride;
        const int first = k_begin + w_key * 32;                              // of this warp's blocks
        const int pieces = first < k_end ? (k_end - first + stride - 1) / stride * F::SUBS : 0;

        // ---- copies: K and V of piece after piece; a lane looks up one position of a block, a block ahead ----
        int copied = 0, slot_c = 0, page_next = -1, sp = 0;                  // sp: this lane's scale
        uint32_t off = ~0u;                                                  // this lane's row, units of 16 bytes
        auto page_of = [&](int pos) -> int {
            if (pos >= k_end || pos < cur.t.lo) return -1;
            int ip, slot;
            paged_split(p, pos, ip, slot);
            const int page = table[ip];
            return page < 0 ? 0x7fffffff : page;
        };
        auto copy_half = [&]() {
            if (copied < 2 * pieces) {
                const int sub = (copied >> 1) % F::SUBS, pos = first + (copied >> 1) / F::SUBS * stride + lane;
                const bool is_v = copied & 1;
                const uint32_t at = ring_at + slot_c * F::SLOT_BYTES;
                if (sub == 0 && !is_v) {
                    off = ~0u;
                    if (page_next >= c.n_pages) {
                        atomicCAS(p.err, 0, KERR_PAGE);
                    } else if (page_next >= 0) {
                        int ip, slot;
                        paged_split(p, pos, ip, slot);
                        off = (uint32_t)((page_next * c.stride[0] + slot * c.stride[1]) * F::ES >> 4);
                        if constexpr (F::Q8) sp = (int)(page_next * c.scale_stride[0] + slot * c.scale_stride[1] + head * c.scale_stride[2]);
                    }
                    page_next = page_of(pos + stride);
                }
                if constexpr (F::Q8)
                    copy_part<4>(at + F::HALF + lane * 4, reinterpret_cast<const uint8_t*>((is_v ? c.v_scale : c.k_scale) + sp), off != ~0u);
                if (!is_v) {
                    const uint32_t there = __ballot_sync(0xffffffffu, off != ~0u) >> (sub * F::SB);
                    if (lane == 0) *reinterpret_cast<uint32_t*>(ring + slot_c * F::SLOT_BYTES + F::SLOT_BYTES - 16) = there;
                }
                // a row's address once, its parts at constant distances; rows that no one sees
                // give zeros
                auto rows_of = [&](auto whole) {
                    if (!is_v && F::K_PRIVATE) {
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
                    } else if (!is_v) {   // whole rows by neighbouring lanes; odd rows' halves of 128 bytes change places
#pragma unroll
                        for (int i = 0; i < F::HALF / 512; i++) {
                            const int r = i * F::K_ROWS + lane / F::K_LANES, unit = lane % F::K_LANES;
                            const uint32_t o = __shfl_sync(0xffffffffu, off, sub * F::SB + r);
                            const bool live = o != ~0u && (decltype(whole)::value || unit * 16 < D * F::ES);
                            copy_part<16>(at + r * DP * F::ES + ((unit ^ (r & 1) << 2) << 4), live ? kb + ((uint64_t)o << 4) + unit * 16 : kb, live);
                        }
                    } else {
#pragma unroll
                        for (int n = 0; n < F::VK; n++) {   // 16-bit products: rows 2t, 2t+1, 2t+8, 2t+9 of each 16; tf32: 2t, 2t+1 of each 8
                            const int key = MODE == M_TF32 ? (n >> 1) * 8 + 2 * t + (n & 1) : (n >> 2) * 16 + ((n >> 1) & 1) * 8 + 2 * t + (n & 1);
                            const uint32_t o = __shfl_sync(0xffffffffu, off, sub * F::SB + key);
                            const bool live = o != ~0u;
                            const uint8_t* row = vb + (live ? ((uint64_t)o << 4) + g * F::VB : 0);
#pragma unroll
                            for (int i = 0; i < F::VC; i++) {
                                const bool in = decltype(whole)::value || i * 8 * F::VB + g * F::VB < D * F::ES;
                                copy_part<F::VB>(at + ((n * F::VC + i) * 32 + lane) * F::VB, in ? row + i * 8 * F::VB : vb, live && in);
                            }
                        }
                    }
                };
                if (D == DP) rows_of(std::true_type());
                else rows_of(std::false_type());
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            copied++;
            slot_c = slot_c + 1 == F::SLOTS ? 0 : slot_c + 1;
        };
        page_next = page_of(first + lane);
#pragma unroll 1
        for (int i = 0; i < F::SLOTS - 1; i++) copy_half();

        // ---- query fragments (the first pieces are on their way): a thread reads the features that it uses ----
        const float base = p.a.scale * 1.4426950408889634f;
        float up[NR];
        uint4 qr[F::Q_REGS ? F::KS : 1];
        {
            constexpr int PF = 16 / F::ES, CH = DP / (4 * PF);   // consecutive features of a thread, and how often
            float x[NR][CH * PF];
#pragma unroll
            for (int k = 0; k < NR; k++) {
                const int r = g + 8 * k, rr = row0 + r, tok = rr / p.group, hq = head * p.group + rr - tok * p.group;
                const int64_t at = (int64_t)(s.first + tok) * p.a.q_stride[0] + hq * p.a.q_stride[1];
#pragma unroll
                for (int i = 0; i < CH * PF; i += 4) {
                    const int d = i / PF * 4 * PF + t * PF + i % PF;
                    float* v = x[k] + i;
                    v[0] = v[1] = v[2] = v[3] = 0.0f;
                    if (r < rows && d < D) {
                        if (act_bf16) {
                            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.a.q) + at + d;
                            if (p.vec_q) {
                                const uint2 w = *reinterpret_cast<const uint2*>(q);
                                v[0] = __uint_as_float(w.x << 16);
                                v[1] = __uint_as_float(w.x & 0xffff0000u);
                                v[2] = __uint_as_float(w.y << 16);
                                v[3] = __uint_as_float(w.y & 0xffff0000u);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++) v[j] = __bfloat162float(q[j]);
                            }
                        } else {
                            const float* q = static_cast<const float*>(p.a.q) + at + d;
                            if (p.vec_q) {
                                const float4 w = *reinterpret_cast<const float4*>(q);
                                v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++) v[j] = q[j];
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < NR; k++) {
                up[k] = 1.0f;
                if constexpr (MODE == M_F16) {
                    float m = 0.0f;
#pragma unroll
                    for (int i = 0; i < CH * PF; i++) m = fmaxf(m, fabsf(x[k][i]));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    up[k] = pow2i(f16_scale_exp(m));
#pragma unroll
                    for (int i = 0; i < CH * PF; i++) x[k][i] *= up[k];
                }
            }
            if constexpr (MODE == M_TF32) {
#pragma unroll
                for (int st = 0; st < F::KS; st++)
#pragma unroll
                    for (int k = 0; k < NR; k++)
                        *reinterpret_cast<float2*>(my_q + ((st * NR + k) * 32 + lane) * 8) = make_float2(x[k][2 * st], x[k][2 * st + 1]);
            } else {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int st = 0; st < F::KS; st++) {
                        uint32_t hi[2][2], lo[2][2];   // [row half][register]
#pragma unroll
                        for (int h = 0; h < (F::PACK ? 1 : 2); h++)
#pragma unroll
                            for (int j = 0; j < 2; j++) split_pair<MODE>(x[2 * rt + h][4 * st + 2 * j], x[2 * rt + h][4 * st + 2 * j + 1], hi[h][j], lo[h][j]);
                        const uint4 first_part = F::PACK ? make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1])
                                                         : make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
                        if constexpr (F::Q_REGS) {
                            qr[st] = first_part;
                        } else {
                            uint4* q = reinterpret_cast<uint4*>(my_q) + (rt * F::NQ * F::KS + st) * 32 + lane;
                            *q = first_part;
                            if constexpr (F::NQ == 2) q[F::KS * 32] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
                        }
                    }
            }
        }

        // ---- this thread's rows: g (+ 8, + 16, ...) ----
        float c_row[NR], m_ref[NR], l[NR];
        int lo_row[NR], hi_row[NR];
        int all_lo = 0, all_hi = 0x7fffffff;   // positions that every row of the tile sees
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int r = g + 8 * i, tok = (row0 + r) / p.group, at = s.L - s.n + tok;
            c_row[i] = base / up[i];
            m_ref[i] = -INFINITY;
            l[i] = 0.0f;
            lo_row[i] = paged_lo(p, at);
            hi_row[i] = p.a.causal ? max(0, min(s.L, at + 1)) : s.L;
            if (r < rows) {
                all_lo = max(all_lo, lo_row[i]);
                all_hi = min(all_hi, hi_row[i]);
            }
        }
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        float o[RT][F::NO][4];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int i = 0; i < F::NO; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[rt][i][j] = 0.0f;
        float vs_max = 0.0f;   // 8-bit: the value scale that weights are expressed in
        int slot = 0;

#pragma unroll 1
        for (int piece = 0; piece < pieces; piece++) {
            copies_wait<F::SLOTS - 2>();
            __syncwarp();                       // scales and notes of other lanes; all are done with the slot that is refilled
            copy_half();
            const int sub = piece % F::SUBS, pos = first + piece / F::SUBS * stride + sub * F::SB;
            const uint32_t k_at = ring_at + slot * F::SLOT_BYTES;
            const float* k_scale = reinterpret_cast<const float*>(ring + slot * F::SLOT_BYTES + F::HALF);
            const uint32_t ok = *reinterpret_cast<const uint32_t*>(ring + slot * F::SLOT_BYTES + F::SLOT_BYTES - 16);
            slot = slot + 1 == F::SLOTS ? 0 : slot + 1;
            constexpr uint32_t ALL = F::SB == 32 ? 0xffffffffu : (1u << (F::SB & 31)) - 1;
            const bool mixed = pos < all_lo || pos + F::SB > all_hi;           // rows see different positions of the piece
            const bool masked = mixed || (ok & ALL) != ALL;
            // ---- scores ----
            float sc[RT][F::NT][4], sc_lo[RT][F::NT][4];   // sc_lo: tf32, products with a lower part
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int n = 0; n < F::NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[rt][n][j] = sc_lo[rt][n][j] = 0.0f;
            constexpr int PER = F::KS / F::KC;          // steps per 16-byte part
#pragma unroll
            for (int i = 0; i < F::KC; i++) {
                uint32_t kr[F::NT][4];
#pragma unroll
                for (int n = 0; n < F::NT; n++) read_part(kr[n], k_at + (F::K_PRIVATE ? ((n * F::KC + i) * 32 + lane) << 4 : (n * 8 + g) * DP * F::ES + ((i ^ (g & 1)) * 4 + t << 4)));
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    const int st = i * PER + e;
                    uint32_t a[RT][F::NQ][4];
                    if constexpr (MODE == M_TF32) {
#pragma unroll
                        for (int k = 0; k < NR; k++) {
                            const float2 x = *reinterpret_cast<const float2*>(my_q + ((st * NR + k) * 32 + lane) * 8);
                            const uint32_t v[2] = {__float_as_uint(x.x), __float_as_uint(x.y)};
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                a[0][0][2 * j + (F::PACK ? 0 : k)] = tf32_hi(v[j]);
                                if constexpr (F::PACK) a[0][0][2 * j + 1] = tf32_lo(v[j]);
                                else a[0][F::NQ - 1][2 * j + k] = tf32_lo(v[j]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int k = 0; k < F::NQ; k++) {
                                const uint4 x = F::Q_REGS ? qr[F::Q_REGS ? st : 0]
                                                          : reinterpret_cast<const uint4*>(my_q)[((rt * F::NQ + k) * F::KS + st) * 32 + lane];
                                a[rt][k][0] = x.x; a[rt][k][1] = x.y; a[rt][k][2] = x.z; a[rt][k][3] = x.w;
                            }
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
                                float(&to)[4] = MODE == M_TF32 && k > 0 ? sc_lo[rt][n] : sc[rt][n];
                                if constexpr (CT == RT_F32) {
                                    mma<MODE>(to, a[rt][k], tf32_hi(b0), tf32_hi(b1));
                                    mma<MODE>(sc_lo[rt][n], a[rt][k], tf32_lo(b0), tf32_lo(b1));
                                } else {
                                    mma<MODE>(to, a[rt][k], b0, b1);
                                }
                            }
                    }
                }
            }

            if constexpr (MODE == M_TF32) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int n = 0; n < F::NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) sc[rt][n][j] += sc_lo[rt][n][j];
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
            // V of the piece; K's slot is free once its scales are used
            copies_wait<F::SLOTS - 2>();
            __syncwarp();
            copy_half();
            const uint32_t v_at = ring_at + slot * F::SLOT_BYTES;
            float* v_scale = reinterpret_cast<float*>(ring + slot * F::SLOT_BYTES + F::HALF);
            if constexpr (CT == RT_F8E4M3) {
                // Codes 0x7f and 0xff are NaN, and so is 0 times them. Where rows see different
                // positions such a row of values becomes zeros with a scale of NaN.
                if (mixed) {
#pragma unroll 1
                    for (int i = 0; i < F::VK * F::VC; i++) {
                        uint32_t x[F::VB / 4], top = 0;
                        const uint32_t at = (i * 32 + lane) * F::VB;
                        read_part(x, v_at + at);
#pragma unroll
                        for (int k = 0; k < F::VB / 4; k++) top |= (x[k] & 0x7f7f7f7fu) + 0x01010101u;
                        if (top & 0x80808080u) {
                            const int n = i / F::VC;   // as the copies place rows
#pragma unroll
                            for (int k = 0; k < F::VB / 4; k++) reinterpret_cast<uint32_t*>(ring + slot * F::SLOT_BYTES + at)[k] = 0;
                            v_scale[(n >> 2) * 16 + ((n >> 1) & 1) * 8 + 2 * t + (n & 1)] = __uint_as_float(0x7fc00000u);
                        }
                    }
                    __syncwarp();
                }
            }
            slot = slot + 1 == F::SLOTS ? 0 : slot + 1;
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
                        read_part(x, v_at + (i * 32 + lane) * 16);
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
                    for (int n = 0; n < VR; n++) read_part(vr[n], v_at + (((st * VR + n) * F::VC + i) * 32 + lane) * F::VB);
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
                            for (int rt = 0; rt < RT; rt++) {
                                float(&to)[4] = o[rt][i * F::VE + e];
                                float acc[4];
#pragma unroll
                                for (int j = 0; j < 4; j++) acc[j] = F::FOLD ? 0.0f : to[j];
#pragma unroll
                                for (int k = F::NP - 1; k >= 0; k--) {   // the small products first: they are truncated to their own size
                                    if constexpr (CT == RT_F32) {
                                        mma<MODE>(acc, a[rt][k], tf32_lo(b0), tf32_lo(b1));
                                        mma<MODE>(acc, a[rt][k], tf32_hi(b0), tf32_hi(b1));
                                    } else {
                                        mma<MODE>(acc, a[rt][k], b0, b1);
                                    }
                                }
#pragma unroll
                                for (int j = 0; j < 4; j++) to[j] = F::FOLD ? to[j] + acc[j] : acc[j];
                            }
                        }
                    }
                }
            }
        }

        copies_wait<0>();
        const float fo = F::Q8 ? vs_max / W_SCALE : 1.0f;
        const bool done = cur.i == 0 && seg == cur.t.count;
        float* parts = p.part + (int64_t)(2 * blockIdx.x + (cur.i == 0)) * p.head_group * F::SLOT;   // (heads of the group)
#pragma unroll
        for (int i = 0; i < NR; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        if (key_warps == 1) {
            // ---- a warp has its head to itself: VE consecutive features of a row at a time ----
#pragma unroll
            for (int k = 0; k < NR; k++) {
                const int r = g + 8 * k;
                if (r >= rows) continue;
                const float f = done ? (l[k] == 0.0f ? 0.0f : fo / l[k]) : fo;
                float* part = parts + w_head * F::SLOT + r * DP;
#pragma unroll
                for (int i = 0; i < F::VC; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int e = 0; e < F::VE; e += 4) {
                            const int d = i * 8 * F::VE + (2 * t + j) * F::VE + e;
                            float x[4];
#pragma unroll
                            for (int v = 0; v < 4; v++) {
                                const float* y = o[k / 2][i * F::VE + e + v];
                                x[v] = (F::PACK ? y[j] + y[2 + j] : y[2 * (k & 1) + j]) * f;
                            }
                            if (!done) *reinterpret_cast<float4*>(part + d) = make_float4(x[0], x[1], x[2], x[3]);
                            else if (d < D) paged_store4(p, s, head, row0 + r, d, x[0], x[1], x[2], x[3]);
                        }
                if (t == 0) {
                    if (!done) parts[w_head * F::SLOT + R * DP + r] = m_ref[k], parts[w_head * F::SLOT + R * DP + R + r] = l[k];
                    else paged_store_lse(p, s, head, row0 + r, m_ref[k], l[k]);
                }
            }
        } else {
            // ---- add up the warps of a head ----
            __syncthreads();                    // nobody needs the rings any more
            if (t == 0) {
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    ml[warp * 2 * R + g + 8 * i] = m_ref[i];
                    ml[warp * 2 * R + R + g + 8 * i] = l[i];
                }
            }
#pragma unroll
            for (int n = 0; n < F::NO; n++)
#pragma unroll
                for (int j = 0; j < 2; j++)   // word n * 9 + column of the row: a warp's stores and loads meet few conflicts
#pragma unroll
                    for (int k = 0; k < NR; k++) {
                        const float* x = o[k / 2][n];
                        os[(warp * R + g + 8 * k) * F::RS + n * 9 + 2 * t + j] = (F::PACK ? x[j] + x[2 + j] : x[2 * (k & 1) + j]) * fo;
                    }
            __syncthreads();
            for (int e = tid; e < p.head_group * rows * (DP / 4); e += FT) {   // 4 features of a row a thread
                const int h = e / (rows * (DP / 4)), r = e / (DP / 4) - h * rows, d = e % (DP / 4) * 4;
                float m = -INFINITY, ls = 0.0f, sum[4] = {0, 0, 0, 0};
                for (int k = h; k < FW; k += p.head_group) m = fmaxf(m, ml[k * 2 * R + r]);
                for (int k = h; k < FW; k += p.head_group) {
                    const float lk = ml[k * 2 * R + R + r];
                    if (lk == 0.0f) continue;                                  // (a warp that saw nothing)
                    const float f = lk == lk ? exp2_fast(ml[k * 2 * R + r] - m) : lk;   // NaN scores: no maximum, a sum of NaN
                    ls += lk * f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int n = (d + j) / (8 * F::VE) * F::VE + (d + j) % F::VE, col = (d + j) / F::VE % 8;
                        sum[j] += os[(k * R + r) * F::RS + n * 9 + col] * f;
                    }
                }
                float* part = parts + h * F::SLOT;
                if (!done) {
                    *reinterpret_cast<float4*>(part + r * DP + d) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                    if (d == 0) part[R * DP + r] = m, part[R * DP + R + r] = ls;
                } else if (d < D) {
                    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                    paged_store4(p, s, cur.h * p.head_group + h, row0 + r, d, sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
                    if (d == 0) paged_store_lse(p, s, cur.h * p.head_group + h, row0 + r, m, ls);
                }
            }
            __syncthreads();
        }
        u += p.whole ? 1 : seg;
        cur.next_item<R>(p);
    }
    // (here, and not above, the code is no longer on the way of a cold call: one token over 200
    // positions 14.6 us against 15.4)
    if (rest) paged_rest<FT>(p);
}

constexpr int MAX_BLOCKS_PER_SM = 3;
// How a call is spread.  Calls whose longest sequence fits WHOLE_KEYS positions
// run as one launch, every item in one block: the join would cost more than it
// spreads.  Blocks take a group of heads when there are enough items even then
// (heads of the same positions lie next to each other, and warps have nothing
// to add up: 64 sequences over int8 193 -> 166 us), one head when items have to
// be cut into many parts (2 x 65536 positions over int8: 75 -> 58 us).
constexpr int WHOLE_KEYS = 512;
constexpr int MIN_POSITIONS = 128;   // of a block's share (4 sequences of 2000 positions over int8: 20.1 us with 256, 17.1 with 128)
struct Spread {
    int rows, head_group, key_shift, blocks;
    bool whole;
};
// Rows of a tile: 8 when that covers a call's rows (a thread then has the
// weights of one row to make, not of two), 16, or two tiles of 16 over the
// same keys for one-part products.
int few_rows(const RtPagedAttention& p) {
    const bool bf = p.dtype == RT_BF16;
    const int64_t rows = (int64_t)std::min(p.max_new, p.total_new) * (p.n_q_heads / p.cache.n_heads);
    if (bf && rows > 16 && p.cache.dtype != RT_F32) return 32;
    return rows <= 8 ? 8 : 16;
}
Spread few_spread(const RtPagedAttention& p, int per_sm) {
    Spread s;
    s.rows = few_rows(p);
    s.whole = p.max_kv <= WHOLE_KEYS;
    const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(p.max_new, p.total_new)) * (p.n_q_heads / p.cache.n_heads);
    const int64_t tiles = (int64_t)p.n_seqs * ((rows + s.rows - 1) / s.rows), positions = std::max(p.max_kv, 1);
    s.head_group = 1;
    while (!s.whole && s.head_group < FW && p.cache.n_heads % (2 * s.head_group) == 0 &&
           tiles * (p.cache.n_heads / (2 * s.head_group)) * 6 >= (int64_t)g_num_sms * (s.rows == 32 ? 2 : MAX_BLOCKS_PER_SM))
        s.head_group *= 2;
    s.key_shift = s.head_group == 1 ? 7 : s.head_group == 2 ? 6 : 5;
    const int64_t items = tiles * (p.cache.n_heads / s.head_group);
    const int64_t shares = s.whole ? items : (items * positions + MIN_POSITIONS - 1) / MIN_POSITIONS;
    s.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)g_num_sms * per_sm, shares));
    return s;
}

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
        return std::min(k, MAX_BLOCKS_PER_SM);
    }();
    return n;
}

template <int CT, bool F32ACT, int DP, int R>
Status few_as(PagedArgs& p, void* ws, cudaStream_t st) {
    using F = Few<CT, F32ACT, DP, R>;
    const Spread s = few_spread(p.a, few_blocks_per_sm<CT, F32ACT, DP, R>());
    paged_set_workspace(p, ws, s.blocks);
    p.whole = s.whole;
    p.key_shift = s.key_shift;
    p.head_group = s.head_group;
    p.head_groups = p.a.cache.n_heads / s.head_group;
    p.min_units = s.whole ? 1 : MIN_POSITIONS >> s.key_shift;
    paged_few_kernel<CT, F32ACT, DP, R><<<s.blocks, FT, F::SMEM, st>>>(p);
    RT_LAUNCH_CHECK();
    return s.whole || s.blocks == 1 ? Status::ok() : launch_paged_join<DP, R>(p, s.blocks, st);
}

template <int CT, bool F32ACT, int R>
Status few_dim(PagedArgs& p, void* ws, cudaStream_t st) {
    return p.a.cache.head_dim > 64 ? few_as<CT, F32ACT, 128, R>(p, ws, st) : few_as<CT, F32ACT, 64, R>(p, ws, st);
}
template <int CT, bool F32ACT>
Status few_sizes(PagedArgs& p, void* ws, cudaStream_t st) {
    const int rows = few_rows(p.a);
    if constexpr (!F32ACT)
        if (rows == 32) return few_dim<CT, F32ACT, 32>(p, ws, st);
    if (rows == 8) return few_dim<CT, F32ACT, 8>(p, ws, st);
    return few_dim<CT, F32ACT, 16>(p, ws, st);
}

}  // namespace

size_t paged_few_workspace(const RtPagedAttention& p) {
    const Spread s = few_spread(p, MAX_BLOCKS_PER_SM);
    if (s.whole) return 0;
    const int DP = p.cache.head_dim > 64 ? 128 : 64;
    return paged_workspace(s.blocks, s.head_group, s.rows * DP + 2 * s.rows);
}

Status launch_paged_few(PagedArgs& p, void* ws, cudaStream_t st) {
    const bool f32 = p.a.dtype == RT_F32;
    switch (p.a.cache.dtype) {
        case RT_F32: return few_sizes<RT_F32, true>(p, ws, st);   // (bf16 activations need the same products)
        case RT_BF16: return f32 ? few_sizes<RT_BF16, true>(p, ws, st) : few_sizes<RT_BF16, false>(p, ws, st);
        case RT_F8E4M3: return f32 ? few_sizes<RT_F8E4M3, true>(p, ws, st) : few_sizes<RT_F8E4M3, false>(p, ws, st);
        default: return f32 ? few_sizes<RT_I8, true>(p, ws, st) : few_sizes<RT_I8, false>(p, ws, st);
    }
}

}  // namespace rt
