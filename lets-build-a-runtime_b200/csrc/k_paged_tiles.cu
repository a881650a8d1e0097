// k_paged_tiles.cu -- paged attention for chunks of new tokens, on the 5th
// generation tensor cores.
//
// Tiles of 128 rows (new token x query head of one cache head) x 128 cached
// positions: S = Q.K^T into TMEM, weights P = 2^(S c - m) back into TMEM over
// S, O = P.V with A from TMEM.  Two chains of tiles run in every block, so that
// one chain's softmax works while the tensor cores run the other's products:
//   more than 128 rows: chain t takes rows 128 t .. of the item's 256, both go
//     over all key tiles;
//   up to 128 rows: both chains have the same rows and take alternate key
//     tiles, each with its own maximum; they are added up at the end of the item.
// 512 threads: warps 0-3 fetch K and V from the pages into a ring of shared
// memory tiles (128-byte swizzle; K as [position][64 features], which is
// K-major for Q.K^T, V the same, which is MN-major for P.V -- nothing is
// transposed), warp 4 issues the MMAs, warps 8-11 and 12-15 are the softmax of
// chains 0 and 1, a thread per row.
//
// Operands.  bf16 activations over a bf16 cache: cp.async straight from the
// pages, bf16 products.  Everything else becomes fp16 on the way to shared
// memory: 8-bit codes are exact in fp16 and keep their scale per position; an
// fp32 or bf16 row is scaled by a power of two of its own (its maximum in
// [2^14, 2^15)), which then is such a scale too.  The scores of a position are
// multiplied by its key scale, its weights by its value scale; the running
// reference m carries the largest value scale seen, so weights stay in fp16's
// range.  fp32 activations: Q and P as fp16 hi + lo (22 bits), an fp32 cache's
// K and V as well: 2 or 3 products for one.  bf16 activations: one part each.
// The tensor core's own sum truncates, so O is folded into fp32 registers
// after every key tile.
//
// Bound: tensor pipe and exponentials for long chunks (a 128 x 128 tile pair
// of products is 1024 cycles at D = 128, its 16384 exponentials 1024 as well),
// HBM for few rows.
#include <cuda_fp16.h>

#include <algorithm>
#include <utility>

#include "dev_math.h"
#include "paged.h"
#include "sm100_ptx.h"

namespace rt {
namespace {

constexpr int TT = 512, TKT = 128;
constexpr int REG_LOAD = 72, REG_MMA = 40, REG_SOFT = 200;
static_assert(REG_LOAD + REG_MMA + 2 * REG_SOFT <= 512, "four warpgroups share 512 registers a thread");
constexpr uint64_t WAIT_NS = 2000000000ull;
constexpr int ERR_P_LOAD = 0x501, ERR_P_MMA = 0x502, ERR_P_SOFT = 0x503, ERR_P_SMEM = 0x505;
constexpr float RAISE = 8.0f;      // the reference moves when a score passes it by this (log2)
constexpr float W_LOG2 = 6.0f;     // fp16 weights reach 2^8 * 2^6

template <int CT, bool F32ACT, int D>
struct Tile {
    static constexpr int ES = CT == RT_F32 ? 4 : CT == RT_BF16 ? 2 : 1;
    static constexpr bool Q8 = ES == 1;
    static constexpr bool DIRECT = CT == RT_BF16 && !F32ACT;     // bf16 all the way
    static constexpr int CHAINS = CT == RT_F32 ? 1 : 2;
    static constexpr int R = 128 * CHAINS;
    static constexpr int QP = F32ACT ? 2 : 1;                    // parts of Q and of P
    static constexpr int VP = CT == RT_F32 ? 2 : 1;              // parts of K and of V
    static constexpr int PLANE = 128 * D * 2;                    // one part of a 128-row tile
    static constexpr int SLOT = VP * PLANE;                      // ring slot
    static constexpr int SLOTS = DIRECT ? 5 : F32ACT ? 2 : 3;
    static constexpr int RB = 4, RAW_PIECE = RB * 128 * 16;      // raw ring: RB loads of 16 bytes a thread
    static constexpr int NRAW = DIRECT ? 0 : F32ACT ? 3 : 6;
    // Scales are written with their tile and read by its softmax, which may be
    // behind the loads: V_j is still held while K_{j+2} (2 or 3 slots) and
    // V_{j+1} (3 slots) may be written.
    static constexpr int KSD = DIRECT ? 0 : 3, VSD = DIRECT ? 0 : 2;
    static constexpr int OFF_RING = CHAINS * QP * PLANE;
    static constexpr int OFF_RAW = OFF_RING + SLOTS * SLOT;
    static constexpr int OFF_RAW_SCALE = OFF_RAW + NRAW * RAW_PIECE;   // by load & 7
    static constexpr int OFF_KS = OFF_RAW_SCALE + (Q8 ? 4096 : 0);
    static constexpr int OFF_VS = OFF_KS + KSD * 512;
    static constexpr int OFF_BAR = OFF_VS + VSD * 512;
    static constexpr int SMEM = OFF_BAR + 1024;
    static constexpr uint32_t COL_S = 0, COL_O = 256;            // + 128 per chain
    static constexpr int OUT = R * D + 2 * R;                    // floats of an unfinished result
    static_assert(SMEM <= 232448, "shared memory");
};

struct Bars {
    uint64_t full[5], empty[5];
    uint64_t s_full[2], p_full[2], q_full[2], v_notes[4], join, drain;
    uint32_t tmem;
    int abort_flag;
    uint32_t ok[8][4];        // tile T & 7: positions that exist (bit per position)
    float vmax[4][4];         // tile T & 3: largest value scale of each 32 positions
    uint32_t strange[8][4];   // bf16 all the way: positions with values that are not finite
    uint32_t meta[4][8], there[4][8];   // a loading warp's notes on its loads under way
};
static_assert(sizeof(Bars) <= 1024, "barrier area");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    const int n = live ? 16 : 0;   // 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
    const int n = live ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ld_shared16(uint32_t a, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void st_shared8(uint32_t a, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
// Byte b of row r of a 128-row tile of 2-byte elements: blocks of 64 features
// (128 bytes), each [128 rows][128 bytes] in the 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_at(int r, int b) {
    return (uint32_t)(b >> 7) * 16384u + (uint32_t)r * 128u + ((((uint32_t)b >> 4 & 7u) ^ ((uint32_t)r & 7u)) << 4) + (b & 15);
}
template <int CT>
__device__ __forceinline__ void codes_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if constexpr (CT == RT_I8) {   // byte + 128 into the mantissa of 1024, minus 1152
        x ^= 0x80808080u;
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
    } else {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)x));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(x >> 16)));
    }
}
__device__ __forceinline__ uint32_t bf16_pair_rn(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// One product over all K steps.  P lies over S: per 16 positions 8 columns of
// hi pairs, then 8 of lo pairs.
template <class T, int D, int... I>
__device__ __forceinline__ void issue_scores(uint32_t d, uint32_t q, uint32_t k, uint32_t kind, std::integer_sequence<int, I...>) {
    (([&] {
         constexpr uint32_t o = ((I / 4) * 16384 + (I % 4) * 32) >> 4, part = T::PLANE >> 4;
         ptx::mma_f16_ss<o, o>(d, q, k, kind, I ? 1u : 0u);
         if constexpr (T::QP == 2) ptx::mma_f16_ss<o + part, o>(d, q, k, kind, 1u);
         if constexpr (T::VP == 2) ptx::mma_f16_ss<o, o + part>(d, q, k, kind, 1u);
     }()),
     ...);
}
template <class T, int... I>
__device__ __forceinline__ void issue_values(uint32_t d, uint32_t a, uint32_t v, uint32_t kind, std::integer_sequence<int, I...>) {
    (([&] {
         constexpr uint32_t o = I * 2048 >> 4, part = T::PLANE >> 4;
         ptx::mma_f16_ts<I * 16, o>(d, a, v, kind, I ? 1u : 0u);
         if constexpr (T::QP == 2) ptx::mma_f16_ts<I * 16 + 8, o>(d, a, v, kind, 1u);
         if constexpr (T::VP == 2) ptx::mma_f16_ts<I * 16, o + part>(d, a, v, kind, 1u);
     }()),
     ...);
}

// A wait of a whole warp: all its lanes go on, or none.
__device__ __forceinline__ bool wait_warp(uint64_t* b, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    return __all_sync(0xffffffffu, ptx::wait_bounded(b, parity, abort_flag, err, code, WAIT_NS));
}

// What every role walks through: the block's segments.
struct Segment {
    int tiles, k0;        // key tiles, first position of the first
    int row0, rows;       // rows of the item
    bool two;             // chains have rows of their own
};
template <class T>
__device__ __forceinline__ Segment segment_of(const PagedArgs& p, const PagedCursor& c, int u, int u_end) {
    Segment g;
    g.tiles = min(c.t.count - c.i, u_end - u);
    g.k0 = (c.t.t0 + c.i) * TKT;
    g.row0 = c.qt * T::R;
    g.rows = min(T::R, c.s.n * p.group - g.row0);
    g.two = T::CHAINS == 2 && g.rows > 128;
    return g;
}

template <int CT, bool F32ACT, int D>
__global__ void __launch_bounds__(TT, 1) paged_tiles_kernel(const __grid_constant__ PagedArgs p, const bool vec_q, const bool vec_out) {
    using T = Tile<CT, F32ACT, D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars& bar = *reinterpret_cast<Bars*>(smem + T::OFF_BAR);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RtKvCache& c = p.a.cache;
    volatile int* abort_flag = &bar.abort_flag;
    if ((ptx::smem_u32(smem) & 1023) != 0) {   // the swizzle needs tiles on 1024 bytes
        if (tid == 0) atomicCAS(p.err, 0, ERR_P_SMEM);
        return;
    }
    asm volatile("griddepcontrol.launch_dependents;");
    PagedCursor cur;
    int u, per, total;
    if (!paged_schedule<TT, T::R, TKT>(p, blockIdx.x, gridDim.x, reinterpret_cast<int*>(smem), cur, u, per, total)) return;
    const int u_end = (int)min((int64_t)u + per, (int64_t)total);

    if (tid == 0) {
        for (int i = 0; i < T::SLOTS; i++) {
            ptx::mbar_init(&bar.full[i], 128);
            ptx::mbar_init(&bar.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            ptx::mbar_init(&bar.s_full[i], 1);
            ptx::mbar_init(&bar.p_full[i], 128);
            ptx::mbar_init(&bar.q_full[i], 128);
            ptx::mbar_init(&bar.v_notes[i], 128);
            ptx::mbar_init(&bar.v_notes[2 + i], 128);
        }
        ptx::mbar_init(&bar.join, 256);
        ptx::mbar_init(&bar.drain, 1);
        bar.abort_flag = 0;
        for (int i = 0; i < 8; i++)
            for (int j = 0; j < 4; j++) bar.strange[i][j] = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 4) ptx::tmem_alloc(&bar.tmem, 512);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = bar.tmem;

    if (warp < 4) {
        // ------------------------------------------------ K and V from the pages
        // A lane looks up one position of the warp's 32, all lanes then copy rows:
        // cp.async, straight into the ring (bf16 all the way) or, in pieces of RB
        // loads a lane, into a raw ring from which the same thread converts its own
        // bytes.  Copies run AHEAD pieces in front of what is handed over.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_LOAD));
        bool ok = true;
        const uint32_t ring = ptx::smem_u32(smem + T::OFF_RING), raw = ptx::smem_u32(smem + T::OFF_RAW) + tid * 16;
        constexpr int LANES = D * T::ES / 16, ROWS = 32 / LANES;          // lanes of a row, rows of a warp's load
        constexpr int LOADS = 32 / ROWS;                                  // loads of a warp's 32 rows
        constexpr int PIECES = T::DIRECT ? 1 : LOADS / T::RB, PER = LOADS / PIECES;
        constexpr int AHEAD = T::DIRECT ? T::SLOTS - 2 : T::NRAW - 1;
        const int sub_row = lane / LANES, piece16 = lane % LANES;
        volatile uint32_t* meta = bar.meta[warp];                         // by load & 7: is_v | mixed << 1 | tile << 2
        volatile uint32_t* there = bar.there[warp];                       // by load & 7: positions that exist

        // ---- the copies ----
        Segment g = segment_of<T>(p, cur, u, u_end);
        int idx = 0, tile_base = 0, n_copy = 0, part = 0;   // load of the segment, tiles before it, loads begun, piece
        uint32_t off0 = ~0u, off1 = ~0u, off_now = ~0u;     // this lane's row of even / odd tiles, units of 16 bytes
        int sp0 = 0, sp1 = 0, sp_now = 0, page_next = 0;    // its scale; the page of the next key tile
        bool is_v = false;
        auto page_of = [&](int j) -> int {
            const int pos = g.k0 + j * TKT + warp * 32 + lane;
            if (pos < cur.t.lo || pos >= cur.t.hi) return -1;
            int ip, slot;
            paged_split(p, pos, ip, slot);
            const int page = p.a.page_table[cur.s.b * p.a.table_stride + ip];
            return page < 0 ? 0x7fffffff : page;
        };
        auto begin_load = [&]() {
            const int a = (T::CHAINS == 2 && !g.two) ? 2 : 1, n = g.tiles, head = min(a, n), r = idx - head, both = max(0, n - a);
            int j;   // K0 (K1) | V0 K(a) | V1 K(a+1) | ... | the last V
            if (r < 0) is_v = false, j = idx;
            else if (r < 2 * both) is_v = !(r & 1), j = (r >> 1) + (r & 1 ? a : 0);
            else is_v = true, j = both + r - 2 * both;
            if (idx == 0) page_next = page_of(0);
            if (!is_v) {
                const int pos = g.k0 + j * TKT + warp * 32 + lane;
                uint32_t off = ~0u;
                int sp = 0;
                if (page_next >= c.n_pages) {
                    atomicCAS(p.err, 0, KERR_PAGE);
                } else if (page_next >= 0) {
                    int ip, slot;
                    paged_split(p, pos, ip, slot);
                    off = (uint32_t)((page_next * c.stride[0] + slot * c.stride[1] + cur.h * c.stride[2]) * T::ES >> 4);
                    if constexpr (T::Q8) sp = (int)(page_next * c.scale_stride[0] + slot * c.scale_stride[1] + cur.h * c.scale_stride[2]);
                }
                if (j + 1 < n) page_next = page_of(j + 1);
                if (j & 1) off1 = off, sp1 = sp;
                else off0 = off, sp0 = sp;
            }
            off_now = j & 1 ? off1 : off0;
            sp_now = j & 1 ? sp1 : sp0;
            const uint32_t live = __ballot_sync(0xffffffffu, off_now != ~0u);
            bool mixed = false;
            if constexpr (T::DIRECT) {   // does every row of the item see all of this tile?
                const int tok0 = g.row0 / p.group, tok1 = (g.row0 + g.rows - 1) / p.group, at0 = cur.s.L - cur.s.n, k = g.k0 + j * TKT;
                mixed = is_v && tok1 > tok0 && ((p.a.causal && k + TKT > at0 + tok0 + 1) || (p.a.window > 0 && k < at0 + tok1 - p.a.window + 1));
            }
            if (lane == 0) {
                meta[n_copy & 7] = (is_v ? 1u : 0u) | (mixed ? 2u : 0u) | (uint32_t)(tile_base + j) << 2;
                there[n_copy & 7] = live;
            }
        };
        auto copy_piece = [&]() {
            if (part == 0) begin_load();
            uint32_t dst;
            if constexpr (T::DIRECT) {
                const int s = n_copy % T::SLOTS;
                if (n_copy >= T::SLOTS)
                    ok = wait_warp(&bar.empty[s], (n_copy / T::SLOTS - 1) & 1, abort_flag, p.err, ERR_P_LOAD);
                if (!ok) return;
                dst = ring + (uint32_t)s * T::SLOT;
            } else {
                dst = raw + (uint32_t)((n_copy * PIECES + part) % T::NRAW) * T::RAW_PIECE;
            }
            const uint8_t* base = static_cast<const uint8_t*>(is_v ? c.v : c.k);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int r = (part * PER + i) * ROWS + sub_row;
                const uint32_t o = __shfl_sync(0xffffffffu, off_now, r);
                const uint8_t* src = base + ((uint64_t)(o == ~0u ? 0 : o) << 4) + piece16 * 16;
                cp_async16(T::DIRECT ? dst + tile_at(warp * 32 + r, piece16 * 16) : dst + i * 2048, src, o != ~0u);
            }
            if constexpr (T::Q8)
                if (part == 0)
                    cp_async4(ptx::smem_u32(smem + T::OFF_RAW_SCALE) + ((n_copy & 7) * 128 + tid) * 4, (is_v ? c.v_scale : c.k_scale) + sp_now,
                              off_now != ~0u);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (++part == PIECES) {
                part = 0;
                n_copy++;
                if (++idx == 2 * g.tiles) {
                    idx = 0;
                    tile_base += g.tiles;
                    u += g.tiles;
                    cur.next_item<T::R, TKT>(p);
                    if (u < u_end) g = segment_of<T>(p, cur, u, u_end);
                }
            }
        };
        // ---- handing over ----
        int n_done = 0, done_part = 0;
        uint32_t top_all = 0;   // own scales: the largest of this lane's rows (bits)
        auto hand_piece = [&]() {
            const uint32_t what = meta[n_done & 7], live = there[n_done & 7];
            const bool v = what & 1;
            const int tile_no = (int)(what >> 2), s = n_done % T::SLOTS;
            const uint32_t dst = ring + (uint32_t)s * T::SLOT;
            if (!v && done_part == 0 && lane == 0) bar.ok[tile_no & 7][warp] = live;
            if constexpr (T::DIRECT) {
                if (v && warp == 0 && lane < 4) bar.strange[(tile_no + 4) & 7][lane] = 0;   // four tiles ahead of its use
                if (what & 2) {
                    // Rows of the item see this tile differently: values that are not finite
                    // leave it (0 times them is not 0) and their positions are noted.
#pragma unroll 1
                    for (int i = 0; i < LOADS; i++) {
                        const int r = warp * 32 + i * ROWS + sub_row;
                        const uint32_t at = dst + tile_at(r, piece16 * 16);
                        uint32_t w[4];
                        ld_shared16(at, w);
                        bool found = false;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if ((w[j] & 0x7f80u) == 0x7f80u) w[j] &= 0xffff0000u, found = true;
                            if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] &= 0xffffu, found = true;
                        }
                        if (found) {
                            st_shared16(at, w[0], w[1], w[2], w[3]);
                            atomicOr(&bar.strange[tile_no & 7][r >> 5], 1u << (r & 31));
                        }
                    }
                }
            } else {
                float* scales = v ? reinterpret_cast<float*>(smem + T::OFF_VS) + tile_no % T::VSD * 128
                                  : reinterpret_cast<float*>(smem + T::OFF_KS) + tile_no % T::KSD * 128;
                if (done_part == 0) {
                    if (n_done >= T::SLOTS)
                        ok = wait_warp(&bar.empty[s], (n_done / T::SLOTS - 1) & 1, abort_flag, p.err, ERR_P_LOAD);
                    if (!ok) return;
                    top_all = 0;
                    if constexpr (T::Q8) {
                        const float scale = *reinterpret_cast<const volatile float*>(smem + T::OFF_RAW_SCALE + ((n_done & 7) * 128 + tid) * 4);
                        scales[tid] = scale;
                        if (scale > 0.0f && scale < INFINITY) top_all = __float_as_uint(scale);
                    }
                }
                const uint32_t src = raw + (uint32_t)((n_done * PIECES + done_part) % T::NRAW) * T::RAW_PIECE;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int r = warp * 32 + (done_part * PER + i) * ROWS + sub_row;
                    uint32_t w[4];
                    ld_shared16(src + i * 2048, w);
                    if constexpr (T::Q8) {
                        uint32_t h[8];
#pragma unroll
                        for (int k = 0; k < 4; k++) codes_f16<CT>(w[k], h[2 * k], h[2 * k + 1]);
                        st_shared16(dst + tile_at(r, piece16 * 32), h[0], h[1], h[2], h[3]);
                        st_shared16(dst + tile_at(r, piece16 * 32 + 16), h[4], h[5], h[6], h[7]);
                    } else {
                        constexpr int N = 16 / T::ES;
                        float x[N];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if constexpr (CT == RT_BF16) {
                                x[2 * k] = __uint_as_float(w[k] << 16);
                                x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                            } else {
                                x[k] = __uint_as_float(w[k]);
                            }
                        }
                        uint32_t top = 0;   // over the bits of |x|: what is not finite comes out on top
#pragma unroll
                        for (int k = 0; k < N; k++) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
#pragma unroll
                        for (int o = LANES / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const int e = f16_scale_exp(__uint_as_float(top));
                        const bool finite = top < 0x7f800000u;
                        const float up = finite ? pow2i(e) : 0.0f;
                        const float down = finite ? pow2i(-e) : __uint_as_float(0x7fc00000u);
#pragma unroll
                        for (int k = 0; k < N; k++) x[k] = finite ? x[k] * up : 0.0f;
                        if (piece16 == 0) scales[r] = down;
                        if (finite && top) top_all = max(top_all, __float_as_uint(down));
                        if constexpr (T::VP == 1) {
                            st_shared16(dst + tile_at(r, piece16 * 16), f16x2_rn(x[0], x[1]), f16x2_rn(x[2], x[3]),
                                        f16x2_rn(x[4 % N], x[5 % N]), f16x2_rn(x[6 % N], x[7 % N]));
                        } else {
                            float h[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) h[k] = round11(x[k]);
                            const uint32_t at = dst + tile_at(r, piece16 * 8);
                            st_shared8(at, f16x2_rn(h[0], h[1]), f16x2_rn(h[2], h[3]));
                            st_shared8(at + T::PLANE, f16x2_rn(x[0] - h[0], x[1] - h[1]), f16x2_rn(x[2] - h[2], x[3] - h[3]));
                        }
                    }
                }
                if (v && done_part == PIECES - 1) {
                    const uint32_t top = __reduce_max_sync(0xffffffffu, top_all);
                    if (lane == 0) bar.vmax[tile_no & 3][warp] = __uint_as_float(top);
                }
            }
            if (++done_part == PIECES) {
                done_part = 0;
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(&bar.full[s]);
                if (v) ptx::mbar_arrive(&bar.v_notes[tile_no & 3]);
                n_done++;
            }
        };
        int ahead = 0;
        while (ok && u < u_end) {
            copy_piece();
            if (!ok) break;
            if (++ahead > AHEAD) {
                cp_wait<AHEAD>();
                __syncwarp();
                hand_piece();
                ahead--;
            }
        }
        cp_wait<0>();
        __syncwarp();
        for (; ok && ahead > 0; ahead--) hand_piece();
    } else if (warp < 8) {
        // ------------------------------------------------ MMA issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_MMA));
        if (warp == 4 && lane == 0) {
            constexpr uint32_t kind_s = T::DIRECT ? ptx::idesc_bf16(128, TKT) : ptx::idesc_f16(128, TKT);
            constexpr uint32_t kind_o = (T::DIRECT ? ptx::idesc_bf16(128, D) : ptx::idesc_f16(128, D)) | ptx::IDESC_B_MN;
            const uint32_t q_desc = ptx::desc_lo(smem), k_desc = ptx::desc_lo(smem + T::OFF_RING);
            const uint32_t v_desc = ptx::desc_lo(smem + T::OFF_RING, 16384);
            int n_use = 0, n_p[2] = {0, 0}, n_q[2] = {0, 0};
            bool ok = true;
            auto wait_load = [&](int n) {
                if (ok) ok = ptx::wait_bounded(&bar.full[n % T::SLOTS], (n / T::SLOTS) & 1, abort_flag, p.err, ERR_P_MMA, WAIT_NS);
                ptx::tc_fence_after();
            };
            auto release = [&](int n) { ptx::mma_commit(&bar.empty[n % T::SLOTS]); };
            auto scores = [&](int chain, int q_tile, int load) {   // S = Q.K^T: all features, hi.hi then the cross terms
                issue_scores<T, D>(tmem + T::COL_S + chain * 128, q_desc + (uint32_t)(q_tile * (T::QP * T::PLANE >> 4)),
                                   k_desc + (uint32_t)(load % T::SLOTS * (T::SLOT >> 4)), kind_s, std::make_integer_sequence<int, D / 16>());
            };
            auto values = [&](int chain, int load) {   // O = P.V over 128 positions
                issue_values<T>(tmem + T::COL_O + chain * 128, tmem + T::COL_S + chain * 128,
                                v_desc + (uint32_t)(load % T::SLOTS * (T::SLOT >> 4)), kind_o, std::make_integer_sequence<int, TKT / 16>());
            };
            auto wait_p = [&](int chain) {
                if (ok) ok = ptx::wait_bounded(&bar.p_full[chain], n_p[chain]++ & 1, abort_flag, p.err, ERR_P_MMA, WAIT_NS);
                ptx::tc_fence_after();
            };
            auto wait_q = [&](int chain) {
                if (ok) ok = ptx::wait_bounded(&bar.q_full[chain], n_q[chain]++ & 1, abort_flag, p.err, ERR_P_MMA, WAIT_NS);
                ptx::tc_fence_after();
            };
            while (ok && u < u_end) {
                const Segment g = segment_of<T>(p, cur, u, u_end);
                wait_q(0);
                if (g.two) wait_q(1);
                if (T::CHAINS == 2 && !g.two) {
                    // alternate key tiles: K0 K1 | V0 K2 | V1 K3 | ...
                    for (int j = 0; j < min(2, g.tiles) && ok; j++) {
                        wait_load(n_use);
                        if (!ok) break;
                        scores(j, 0, n_use);
                        release(n_use++);
                        ptx::mma_commit(&bar.s_full[j]);
                    }
                    for (int j = 0; j < g.tiles && ok; j++) {
                        const int t = j & 1;
                        wait_load(n_use);
                        wait_p(t);
                        if (!ok) break;
                        values(t, n_use);
                        release(n_use++);
                        if (j + 2 < g.tiles) {
                            wait_load(n_use);
                            if (!ok) break;
                            scores(t, 0, n_use);
                            release(n_use++);
                        }
                        ptx::mma_commit(&bar.s_full[t]);
                    }
                } else {
                    // every key tile for both: K0 | V0 K1 | V1 K2 | ...
                    wait_load(n_use);
                    if (!ok) break;
                    scores(0, 0, n_use);
                    ptx::mma_commit(&bar.s_full[0]);
                    if (g.two) {
                        scores(1, 1, n_use);
                        ptx::mma_commit(&bar.s_full[1]);
                    }
                    release(n_use++);
                    for (int j = 0; j < g.tiles && ok; j++) {
                        const int v = n_use, k = n_use + 1;
                        const bool more = j + 1 < g.tiles;
                        wait_load(v);
                        wait_p(0);
                        if (!ok) break;
                        values(0, v);
                        if (!g.two) release(v);
                        if (more) {
                            wait_load(k);
                            if (!ok) break;
                            scores(0, 0, k);
                            if (!g.two) release(k);
                        }
                        ptx::mma_commit(&bar.s_full[0]);
                        if (g.two) {
                            wait_p(1);
                            if (!ok) break;
                            values(1, v);
                            release(v);
                            if (more) {
                                scores(1, 1, k);
                                release(k);
                            }
                            ptx::mma_commit(&bar.s_full[1]);
                        }
                        n_use += more ? 2 : 1;
                    }
                }
                u += g.tiles;
                cur.next_item<T::R, TKT>(p);
            }
            ptx::mma_commit(&bar.drain);   // nothing in flight when TMEM is given back
            volatile int no_abort = 0;
            ptx::wait_bounded(&bar.drain, 0, &no_abort, p.err, ERR_P_MMA, WAIT_NS);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ softmax, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_SOFT));
        const int chain = (warp - 8) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_at = tmem + lanes + T::COL_S + chain * 128, o_at = tmem + lanes + T::COL_O + chain * 128;
        const float base = p.a.scale * 1.4426950408889634f;
        int n_s = 0, n_join = 0, tile_base = 0;
        bool ok = true, was_two = false;
        auto wait_s = [&]() {
            ok = wait_warp(&bar.s_full[chain], n_s++ & 1, abort_flag, p.err, ERR_P_SOFT);
            ptx::tc_fence_after();
        };
        auto meet = [&]() {   // both chains' softmax threads
            ptx::mbar_arrive(&bar.join);
            ok = wait_warp(&bar.join, n_join++ & 1, abort_flag, p.err, ERR_P_SOFT);
        };
        while (ok && u < u_end) {
            const Segment g = segment_of<T>(p, cur, u, u_end);
            const PagedSeq& s = cur.s;
            const bool split_keys = T::CHAINS == 2 && !g.two;
            const int my_row = g.row0 + row + (g.two ? chain * 128 : 0);
            const bool live = my_row < g.row0 + g.rows && (T::CHAINS == 2 || chain == 0);
            if (split_keys && was_two) {   // chain 1's products have read its own Q, whose place is used below
                meet();
                if (!ok) break;
            }
            was_two = g.two;
            // ---- the rows of Q into shared memory ----
            float c_row = base;
            uint8_t* q1 = smem + T::QP * T::PLANE;   // free when both chains share their rows
            if (chain == 0 || g.two) {
                const uint32_t dst = ptx::smem_u32(smem) + (uint32_t)(g.two ? chain : 0) * T::QP * T::PLANE;
                const int64_t at = live ? (int64_t)(s.first + my_row / p.group) * p.a.q_stride[0] +
                                              (cur.h * p.group + my_row % p.group) * p.a.q_stride[1] : 0;
                const bool bf = p.a.dtype == RT_BF16;
                const float* qf = static_cast<const float*>(p.a.q) + at;
                const __nv_bfloat16* qh = static_cast<const __nv_bfloat16*>(p.a.q) + at;
                auto get8 = [&](int d, float (&x)[8]) {
                    if (!live) {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = 0.0f;
                    } else if (bf && vec_q) {
                        const uint4 v = *reinterpret_cast<const uint4*>(qh + d);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[2 * i] = __uint_as_float(w[i] << 16);
                            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                        }
                    } else if (vec_q) {
                        const float4 a = *reinterpret_cast<const float4*>(qf + d), b = *reinterpret_cast<const float4*>(qf + d + 4);
                        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = bf ? __bfloat162float(qh[d + i]) : qf[d + i];
                    }
                };
                float up = 1.0f;
                if constexpr (!T::DIRECT) {
                    float m = 0.0f;
#pragma unroll 4
                    for (int d = 0; d < D; d += 8) {
                        float x[8];
                        get8(d, x);
#pragma unroll
                        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
                    }
                    const int e = f16_scale_exp(m);
                    up = pow2i(e);
                    c_row = base * pow2i(-e);
                }
#pragma unroll 4
                for (int d = 0; d < D; d += 8) {
                    float x[8];
                    get8(d, x);
                    const uint32_t a = dst + tile_at(row, d * 2);
                    if constexpr (T::DIRECT) {
                        st_shared16(a, bf16_pair_rn(x[0], x[1]), bf16_pair_rn(x[2], x[3]), bf16_pair_rn(x[4], x[5]), bf16_pair_rn(x[6], x[7]));
                    } else {
                        float h[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            x[i] *= up;
                            h[i] = T::QP == 2 ? round11(x[i]) : x[i];
                        }
                        st_shared16(a, f16x2_rn(h[0], h[1]), f16x2_rn(h[2], h[3]), f16x2_rn(h[4], h[5]), f16x2_rn(h[6], h[7]));
                        if constexpr (T::QP == 2)
                            st_shared16(a + T::PLANE, f16x2_rn(x[0] - h[0], x[1] - h[1]), f16x2_rn(x[2] - h[2], x[3] - h[3]),
                                        f16x2_rn(x[4] - h[4], x[5] - h[5]), f16x2_rn(x[6] - h[6], x[7] - h[7]));
                    }
                }
                if (split_keys && !T::DIRECT) reinterpret_cast<float*>(q1)[row] = c_row;
                ptx::fence_proxy_async_smem();
                if (T::CHAINS == 2 || chain == 0) ptx::mbar_arrive(&bar.q_full[g.two ? chain : 0]);
            }
            // ---- tiles ----
            const int at_pos = s.L - s.n + my_row / p.group;
            const int lo_row = p.a.window > 0 ? max(0, at_pos - p.a.window + 1) : 0;
            const int hi_row = live ? (p.a.causal ? min(s.L, at_pos + 1) : s.L) : 0;
            const bool any_live = __any_sync(0xffffffffu, live);
            float m = -INFINITY, l = 0.0f, ref = 0.0f, v_top = 0.0f;   // ref: what exponents are taken against
            float o[D];
#pragma unroll
            for (int i = 0; i < D; i++) o[i] = 0.0f;
            auto fold = [&]() {
#pragma unroll
                for (int b = 0; b < D; b += 16) {
                    uint32_t r[16];
                    ptx::tmem_ld16(o_at + b, r);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i += 2)
                        upk2(add2(pk2(o[b + i], o[b + i + 1]), pk2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]))), o[b + i], o[b + i + 1]);
                }
            };
            const int step = split_keys ? 2 : 1, j0 = split_keys ? chain : 0;
            const bool works = T::CHAINS == 2 ? (split_keys || g.two || chain == 0) : chain == 0;
            if (works && j0 < g.tiles) {
                for (int j = j0; j < g.tiles; j += step) {
                    const int tile_no = tile_base + j, k0 = g.k0 + j * TKT;
                    wait_s();
                    if (!ok) break;
                    if (j == j0 && split_keys && chain == 1 && !T::DIRECT) c_row = reinterpret_cast<const float*>(q1)[row];
                    // What comes with V_j (its scales, the positions taken out of it) is there once
                    // V_j has landed, which its product waits for, not the scores.  (Not the ring
                    // slot's barrier, which may be two phases away here: up to two later V
                    // tiles may have landed too, hence four barriers.)
                    auto wait_v = [&]() {
                        ok = wait_warp(&bar.v_notes[tile_no & 3], (tile_no >> 2) & 1, abort_flag, p.err, ERR_P_SOFT);
                    };
                    if (any_live) {
                        const float* ks = reinterpret_cast<const float*>(smem + T::OFF_KS) + tile_no % (T::DIRECT ? 1 : T::KSD) * 128;
                        const float* vs = reinterpret_cast<const float*>(smem + T::OFF_VS) + tile_no % (T::DIRECT ? 1 : T::VSD) * 128;
                        const uint32_t* okw = bar.ok[tile_no & 7];
                        const bool whole = lo_row <= k0 && hi_row >= k0 + TKT && (okw[0] & okw[1] & okw[2] & okw[3]) == 0xffffffffu;
                        const bool masked = __any_sync(0xffffffffu, live && !whole);
                        // the largest score
                        float top = -INFINITY;
#pragma unroll
                        for (int b = 0; b < TKT; b += 16) {
                            uint32_t r[16];
                            ptx::tmem_ld16(s_at + b, r);
                            ptx::tmem_ld_wait();
                            float x[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = __uint_as_float(r[i]);
                            if constexpr (!T::DIRECT) {
#pragma unroll
                                for (int i = 0; i < 16; i += 4) {
                                    const float4 k = *reinterpret_cast<const float4*>(ks + b + i);
                                    x[i] *= k.x; x[i + 1] *= k.y; x[i + 2] *= k.z; x[i + 3] *= k.w;
                                }
                            }
                            if (masked) {
                                const uint32_t w = okw[b >> 5] >> (b & 16);
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (!((w >> i & 1) && k0 + b + i >= lo_row && k0 + b + i < hi_row)) x[i] = -INFINITY;
                            }
#pragma unroll
                            for (int i = 0; i < 16; i += 2) top = max3f(top, x[i], x[i + 1]);
                        }
                        top *= c_row;
                        if (j > j0) fold();
                        if (!T::DIRECT || masked) {
                            wait_v();
                            if (!ok) break;
                        }
                        // the reference
                        float tile_v = 1.0f;
                        if constexpr (!T::DIRECT) {
                            const float* vm = bar.vmax[tile_no & 3];
                            tile_v = fmaxf(fmaxf(vm[0], vm[1]), fmaxf(vm[2], vm[3]));
                        }
                        const bool raise = top > m + RAISE, wider = !T::DIRECT && tile_v > v_top;
                        if (raise) m = top;
                        if (wider) v_top = 4.0f * tile_v;
                        if (__any_sync(0xffffffffu, raise || wider)) {
                            const float to = (m == -INFINITY ? 0.0f : m) + (T::DIRECT ? 0.0f : fmaxf(log2f(v_top), -100.0f) - W_LOG2);
                            const float f = l == 0.0f ? 0.0f : exp2_fast(ref - to);   // (nothing summed yet: o = 0)
                            ref = to;
                            l *= f;
                            const unsigned long long ff = pk2(f, f);
#pragma unroll
                            for (int i = 0; i < D; i += 2) upk2(mul2(pk2(o[i], o[i + 1]), ff), o[i], o[i + 1]);
                        }
                        // weights
                        unsigned long long sum = pk2(0.0f, 0.0f);
                        const unsigned long long cc = pk2(c_row, c_row), nr = pk2(-ref, -ref);
#pragma unroll
                        for (int b = 0; b < TKT; b += 16) {
                            uint32_t r[16];
                            ptx::tmem_ld16(s_at + b, r);
                            ptx::tmem_ld_wait();
                            float x[16];
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                unsigned long long y = pk2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                                if constexpr (!T::DIRECT) y = mul2(y, *reinterpret_cast<const unsigned long long*>(ks + b + i));
                                upk2(fma2(y, cc, nr), x[i], x[i + 1]);
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = exp2_fast(x[i]);
                            if (masked) {
                                const uint32_t w = okw[b >> 5] >> (b & 16);
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (!((w >> i & 1) && k0 + b + i >= lo_row && k0 + b + i < hi_row)) x[i] = 0.0f;
                            }
#pragma unroll
                            for (int i = 0; i < 16; i += 2) sum = add2(sum, pk2(x[i], x[i + 1]));
                            if constexpr (!T::DIRECT) {
#pragma unroll
                                for (int i = 0; i < 16; i += 2) {
                                    const bool z0 = masked && x[i] == 0.0f, z1 = masked && x[i + 1] == 0.0f;
                                    upk2(mul2(pk2(x[i], x[i + 1]), *reinterpret_cast<const unsigned long long*>(vs + b + i)), x[i], x[i + 1]);
                                    if (z0) x[i] = 0.0f;   // a position that is not seen may have any scale
                                    if (z1) x[i + 1] = 0.0f;
                                }
                            }
                            uint32_t hi[8];
                            if constexpr (T::DIRECT) {
#pragma unroll
                                for (int i = 0; i < 8; i++) hi[i] = bf16_pair_rn(x[2 * i], x[2 * i + 1]);
                            } else if constexpr (T::QP == 1) {
#pragma unroll
                                for (int i = 0; i < 8; i++) hi[i] = f16x2_rn(x[2 * i], x[2 * i + 1]);
                            } else {
                                uint32_t lo[8];
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    const float a = __uint_as_float(__float_as_uint(x[2 * i]) & 0xffffe000u);
                                    const float d = __uint_as_float(__float_as_uint(x[2 * i + 1]) & 0xffffe000u);
                                    hi[i] = f16x2_rn(a, d);
                                    lo[i] = f16x2_rn(x[2 * i] - a, x[2 * i + 1] - d);
                                }
                                ptx::tmem_st8(s_at + b + 8, lo);
                            }
                            ptx::tmem_st8(s_at + b, hi);
                        }
                        float s0, s1;
                        upk2(sum, s0, s1);
                        l += s0 + s1;
                        if constexpr (T::DIRECT) {
                            if (masked) {   // values that are not finite were taken out: rows that see one get NaN
                                const uint32_t* sw = bar.strange[tile_no & 7];
                                if (sw[0] | sw[1] | sw[2] | sw[3])
                                    for (int i = 0; i < TKT; i++)
                                        if ((sw[i >> 5] >> (i & 31) & 1) && k0 + i >= lo_row && k0 + i < hi_row) l = __uint_as_float(0x7fc00000u);
                            }
                        }
                        ptx::tmem_st_wait();
                    }
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(&bar.p_full[chain]);
                }
                if (ok) wait_s();
                if (!ok) break;
                if (any_live) fold();
                ptx::tc_fence_before();
            }
            // ---- the other chain's share of the keys ----
            if (split_keys) {
                float* x = reinterpret_cast<float*>(q1);
                if (chain == 1) {
                    x[row] = l == 0.0f ? -INFINITY : ref;
                    x[128 + row] = l;
                }
                meet();
                if (!ok) break;
                float f0 = 1.0f, f1 = 0.0f;
                if (chain == 0) {
                    const float r1 = x[row], l1 = x[128 + row];
                    const float r0 = l == 0.0f ? -INFINITY : ref, to = fmaxf(r0, r1);
                    if (to != -INFINITY) {
                        f0 = l == 0.0f ? 0.0f : exp2_fast(r0 - to);
                        f1 = l1 == 0.0f ? 0.0f : exp2_fast(r1 - to);
                        l = l * f0 + l1 * f1;
                        ref = to;
                    }
                }
                meet();
                if (!ok) break;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    if (chain == 1) {
#pragma unroll
                        for (int i = 0; i < D / 2; i++) x[i * 128 + row] = o[half * (D / 2) + i];
                    }
                    meet();
                    if (!ok) break;
                    if (chain == 0) {
#pragma unroll
                        for (int i = 0; i < D / 2; i++) o[half * (D / 2) + i] = o[half * (D / 2) + i] * f0 + x[i * 128 + row] * f1;
                    }
                    meet();
                    if (!ok) break;
                }
                if (!ok) break;
            }
            // ---- out ----
            if (live && (chain == 0 || g.two)) {
                if (cur.i == 0 && g.tiles == cur.t.count) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int64_t at = paged_out_at(p, s, cur.h, my_row);
                    if (!vec_out) {
#pragma unroll
                        for (int i = 0; i < D; i++) {
                            if (p.a.dtype == RT_BF16) static_cast<__nv_bfloat16*>(p.a.out)[at + i] = __float2bfloat16_rn(o[i] * inv);
                            else static_cast<float*>(p.a.out)[at + i] = o[i] * inv;
                        }
                    } else if (p.a.dtype == RT_BF16) {
                        uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + at);
#pragma unroll
                        for (int i = 0; i < D / 8; i++)
                            out[i] = make_uint4(bf16_pair_rn(o[8 * i] * inv, o[8 * i + 1] * inv), bf16_pair_rn(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                                bf16_pair_rn(o[8 * i + 4] * inv, o[8 * i + 5] * inv), bf16_pair_rn(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                    } else {
                        float4* out = reinterpret_cast<float4*>(static_cast<float*>(p.a.out) + at);
#pragma unroll
                        for (int i = 0; i < D / 4; i++)
                            out[i] = make_float4(o[4 * i] * inv, o[4 * i + 1] * inv, o[4 * i + 2] * inv, o[4 * i + 3] * inv);
                    }
                    paged_store_lse(p, s, cur.h, my_row, ref, l);
                } else {
                    float* part = p.part + (int64_t)(2 * blockIdx.x + (cur.i == 0)) * T::OUT;
                    const int r = my_row - g.row0;
                    float4* out = reinterpret_cast<float4*>(part + r * D);
#pragma unroll
                    for (int i = 0; i < D / 4; i++) out[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    part[T::R * D + r] = l == 0.0f ? -INFINITY : ref;
                    part[T::R * D + T::R + r] = l;
                }
            }
            tile_base += g.tiles;
            u += g.tiles;
            cur.next_item<T::R, TKT>(p);
        }
    }
    __syncthreads();
    if (warp == 4) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

constexpr int MIN_UNITS = 4;

// Blocks of a call: one per SM, no more than it has work for.
int tiles_blocks(const RtPagedAttention& p) {
    const int R = p.cache.dtype == RT_F32 ? 128 : 256;
    const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(p.max_new, p.total_new)) * (p.n_q_heads / p.cache.n_heads);
    const int64_t units = (int64_t)p.n_seqs * p.cache.n_heads * ((rows + R - 1) / R) * std::max(1, (p.max_kv + TKT - 1) / TKT);
    return (int)std::max<int64_t>(1, std::min<int64_t>(g_num_sms, (units + MIN_UNITS - 1) / MIN_UNITS));
}

bool rows16(const void* p, const int64_t st[2], int dtype) {
    return aligned16(p) && (st[0] * dtype_bytes(dtype)) % 16 == 0 && (st[1] * dtype_bytes(dtype)) % 16 == 0;
}

template <int CT, bool F32ACT, int D>
Status tiles_as(PagedArgs& p, void* ws, cudaStream_t st) {
    using T = Tile<CT, F32ACT, D>;
    static const cudaError_t set = cudaFuncSetAttribute(paged_tiles_kernel<CT, F32ACT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    RT_CUDA_CHECK(set);
    const int blocks = tiles_blocks(p.a);
    p.part = static_cast<float*>(ws);
    p.whole = 0;
    p.min_units = MIN_UNITS;
    paged_tiles_kernel<CT, F32ACT, D><<<blocks, TT, T::SMEM, st>>>(p, rows16(p.a.q, p.a.q_stride, p.a.dtype), rows16(p.a.out, p.a.out_stride, p.a.dtype));
    RT_LAUNCH_CHECK();
    return blocks == 1 ? Status::ok() : launch_paged_join<D, T::R, TKT>(p, blocks, st);
}
template <int CT, bool F32ACT>
Status tiles_dim(PagedArgs& p, void* ws, cudaStream_t st) {
    return p.a.cache.head_dim == 128 ? tiles_as<CT, F32ACT, 128>(p, ws, st) : tiles_as<CT, F32ACT, 64>(p, ws, st);
}

}  // namespace

bool paged_tiles_takes(const RtPagedAttention& p) { return p.cache.head_dim == 64 || p.cache.head_dim == 128; }

size_t paged_tiles_workspace(const RtPagedAttention& p) {
    const int R = p.cache.dtype == RT_F32 ? 128 : 256;
    return (size_t)tiles_blocks(p) * 2 * (R * p.cache.head_dim + 2 * R) * sizeof(float);
}

Status launch_paged_tiles(PagedArgs& p, void* ws, cudaStream_t st) {
    const bool f32 = p.a.dtype == RT_F32;
    switch (p.a.cache.dtype) {
        case RT_F32: return tiles_dim<RT_F32, true>(p, ws, st);   // (bf16 activations need the same products)
        case RT_BF16: return f32 ? tiles_dim<RT_BF16, true>(p, ws, st) : tiles_dim<RT_BF16, false>(p, ws, st);
        case RT_F8E4M3: return f32 ? tiles_dim<RT_F8E4M3, true>(p, ws, st) : tiles_dim<RT_F8E4M3, false>(p, ws, st);
        default: return f32 ? tiles_dim<RT_I8, true>(p, ws, st) : tiles_dim<RT_I8, false>(p, ws, st);
    }
}

}  // namespace rt
