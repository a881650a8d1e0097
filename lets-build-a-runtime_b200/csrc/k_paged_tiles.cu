// k_paged_tiles.cu -- paged attention for chunks of new tokens, on the 5th
// generation tensor cores.
//
// Tiles of 128 rows (new token x query head of one cache head) x 128 cached
// positions: S = Q.K^T into TMEM, weights P = 2^(S c - m) back into TMEM over
// S, O = P.V with A from TMEM.  S, P and O exist twice, so that softmax works on
// one while the tensor cores run the other's products:
//   bf16 activations, more than 128 rows: two row tiles over the same key tiles,
//     a warpgroup each;
//   bf16 activations, up to 128 rows: one row tile, a warpgroup takes every other
//     key tile with a maximum of its own; the two are added at the end of the item;
//   fp32 activations: one row tile, both warpgroups on every key tile, each half
//     of its positions (a row's sums need the registers of two threads).
// 512 threads: warps 0-3 fetch K and V from the pages into a ring of shared
// memory tiles (128-byte swizzle; K as [position][64 features], which is
// K-major for Q.K^T, V the same, which is MN-major for P.V -- nothing is
// transposed), warp 4 issues the MMAs, warps 8-15 are the softmax.
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
// The tensor core's own sum truncates (2^-24 of the sum per step, always down):
// with bf16 outputs that is nothing even over long caches and O stays in TMEM,
// with fp32 outputs every key tile's O is folded into fp32 registers.
//
// Bound: the two products of a 128 x 128 tile take 1024 cycles at D = 128, its
// 16384 exponentials 1024 as well.  Measured it is neither, but the chain of a
// tile: 4096 tokens over 16384 positions, 16 heads of 128, bf16, 537 us = 897
// TF/s (2550 cycles a tile).  P lies over S, so the next scores of a chain wait
// for all of its weights and then for all of P.V; of 4 warps a scheduler 0.5
// could issue on average (2048 tokens over 8192: tensor pipe busy 43 %, issue
// slots 36 %, exponential unit 38 %).  With a quarter of the exponentials on the
// FMA pipe instead it was slower (566 -> 628 us when measured), and with waits
// that poll harder (574 - 628).  fp32 activations have two products for one, two
// threads a row that exchange their maximum, and weights in two parts: 12 heads
// of 64 over int8, chunks of up to 1400 tokens, 490 us = 155 TF/s of plain
// products (chunks of 700: tensor pipe 25 %, issue slots 41 %).  128 registers a
// thread at launch cost every instance 400 - 730 bytes of spills.
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
constexpr int W_LOG2 = 6;          // fp16 weights reach 2^8 * 2^6 (* 2: value scales count by their exponent)

template <int CT, bool F32ACT, int D>
struct Tile {
    static constexpr int ES = CT == RT_F32 ? 4 : CT == RT_BF16 ? 2 : 1;
    static constexpr bool Q8 = ES == 1;
    static constexpr bool DIRECT = CT == RT_BF16 && !F32ACT;     // bf16 all the way
    static constexpr int R = F32ACT ? 128 : 256;                 // rows of an item
    static constexpr int QP = F32ACT ? 2 : 1;                    // parts of Q and of P
    static constexpr int VP = CT == RT_F32 ? 2 : 1;              // parts of K and of V
    static constexpr int PLANE = 128 * D * 2;                    // one part of a 128-row tile
    static constexpr int SLOT = VP * PLANE;                      // ring slot
    static constexpr int SLOTS = DIRECT ? 5 : VP == 2 ? 2 : 3;
    static constexpr int RB = 4, RAW_PIECE = RB * 128 * 16;      // raw ring: RB loads of 16 bytes a thread
    static constexpr int NRAW = DIRECT ? 0 : VP == 2 ? 3 : 6;
    // Scales are written with their tile and read by its softmax, which may be
    // behind the loads: V_j is still held while K_{j+2} (2 or 3 slots) and
    // V_{j+1} (3 slots) may be written.
    static constexpr int KSD = DIRECT ? 0 : 3, VSD = DIRECT ? 0 : 2;
    static constexpr int OFF_RING = R / 128 * QP * PLANE;
    static constexpr int OFF_RAW = OFF_RING + SLOTS * SLOT;
    static constexpr int OFF_RAW_SCALE = OFF_RAW + NRAW * RAW_PIECE;   // by load & 7
    static constexpr int OFF_KS = OFF_RAW_SCALE + (Q8 ? 4096 : 0);
    static constexpr int OFF_VS = OFF_KS + KSD * 512;
    static constexpr int OFF_QS = OFF_VS + VSD * 512;                  // per row: scale of a score
    static constexpr int OFF_RED = OFF_QS + (DIRECT ? 0 : R * 4);      // fp32 activations: [2][2][128] maxima of half rows
    static constexpr int OFF_BAR = OFF_RED + (F32ACT ? 2048 : 0);
    static constexpr int SMEM = OFF_BAR + 1024;
    static constexpr uint32_t COL_S = 0, COL_O = 256;            // + 128 for the second
    static constexpr int OUT = R * D + 2 * R;                    // floats of an unfinished result
    static_assert(SMEM <= 232448, "shared memory");
};

struct Bars {
    uint64_t full[5], empty[5];
    uint64_t s_full[2], p_full[2], q_full[2], v_notes[4], join, half[4], drain;
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Arrives once on `bar` (an arrival that its count includes) when the copies of
// this thread so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ptx::smem_u32(bar)) : "memory");
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
// hi pairs, then (two parts) 8 of lo pairs.
template <class T, int D, int... I>
__device__ __forceinline__ void issue_scores(uint32_t d, uint32_t q, uint32_t k, uint32_t kind, std::integer_sequence<int, I...>) {
    constexpr uint32_t part = T::PLANE >> 4;
    constexpr bool CROSS = T::QP == 2 || T::VP == 2;
    (([&] {   // the small products first: what the sum truncates is of their own size then
         constexpr uint32_t o = ((I / 4) * 16384 + (I % 4) * 32) >> 4;
         if constexpr (T::QP == 2) ptx::mma_f16_ss<o + part, o>(d, q, k, kind, I ? 1u : 0u);
         if constexpr (T::VP == 2) ptx::mma_f16_ss<o, o + part>(d, q, k, kind, I || T::QP == 2 ? 1u : 0u);
     }()),
     ...);
    (([&] {
         constexpr uint32_t o = ((I / 4) * 16384 + (I % 4) * 32) >> 4;
         ptx::mma_f16_ss<o, o>(d, q, k, kind, I || CROSS ? 1u : 0u);
     }()),
     ...);
}
template <class T, int... I>
__device__ __forceinline__ void issue_values(uint32_t d, uint32_t a, uint32_t v, uint32_t kind, uint32_t add, std::integer_sequence<int, I...>) {
    constexpr uint32_t part = T::PLANE >> 4;
    constexpr bool CROSS = T::QP == 2 || T::VP == 2;
    (([&] {
         constexpr uint32_t o = I * 2048 >> 4, col = I * 8 * T::QP;
         if constexpr (T::QP == 2) ptx::mma_f16_ts<col + 8, o>(d, a, v, kind, I ? 1u : add);
         if constexpr (T::VP == 2) ptx::mma_f16_ts<col, o + part>(d, a, v, kind, I || T::QP == 2 ? 1u : add);
     }()),
     ...);
    (([&] {
         constexpr uint32_t o = I * 2048 >> 4, col = I * 8 * T::QP;
         ptx::mma_f16_ts<col, o>(d, a, v, kind, I || CROSS ? 1u : add);
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
    int all_lo, all_hi;   // positions that every row of the item sees
    // Do rows of the item see the key tile at k differently?
    __device__ __forceinline__ bool differ(int k) const { return k < all_lo || k + TKT > all_hi; }
};
template <class T>
__device__ __forceinline__ Segment segment_of(const PagedArgs& p, const PagedCursor& c, int u, int u_end) {
    Segment g;
    g.tiles = min(c.t.count - c.i, u_end - u);
    g.k0 = (c.t.t0 + c.i) * TKT;
    g.row0 = c.qt * T::R;
    g.rows = min(T::R, c.s.n * p.group - g.row0);
    g.two = T::R == 256 && g.rows > 128;
    const int tok0 = g.row0 / p.group, tok1 = (g.row0 + g.rows - 1) / p.group, at0 = c.s.L - c.s.n;
    g.all_lo = tok1 > tok0 ? paged_lo(p, at0 + tok1) : 0;   // (a single token: all alike)
    g.all_hi = tok1 > tok0 && p.a.causal ? at0 + tok0 + 1 : 0x7fffffff;
    return g;
}

template <int CT, bool F32ACT, int D>
__global__ void __launch_bounds__(TT, 1) paged_tiles_kernel(const __grid_constant__ PagedArgs p) {
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
    bool rest;
    const bool some = paged_schedule<TT, T::R>(p, blockIdx.x, gridDim.x, reinterpret_cast<int*>(smem), cur, u, per, total, rest);
    paged_note<T::R>(p, some, cur, u, per);
    if (rest) paged_rest<TT>(p);
    if (!some) return;
    const int u_end = (int)min((int64_t)u + per, (int64_t)total);

    if (tid == 0) {
        for (int i = 0; i < T::SLOTS; i++) {
            ptx::mbar_init(&bar.full[i], T::DIRECT ? 128 + 4 : 128);   // (+ 4: the warps' notes)
            ptx::mbar_init(&bar.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            ptx::mbar_init(&bar.s_full[i], 1);
            ptx::mbar_init(&bar.p_full[i], F32ACT ? 256 : 128);
            ptx::mbar_init(&bar.q_full[i], F32ACT ? 256 : 128);
            ptx::mbar_init(&bar.v_notes[i], 128);
            ptx::mbar_init(&bar.v_notes[2 + i], 128);
        }
        ptx::mbar_init(&bar.join, 256);
        for (int i = 0; i < 4; i++) ptx::mbar_init(&bar.half[i], 64);
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
        // A lane looks up one position of the warp's 32, all lanes then copy rows with
        // cp.async: bf16 all the way straight into the ring, where the copies themselves
        // arrive on the slot's barrier; the rest, in pieces of RB loads a lane, into a raw
        // ring from which the same thread converts its own bytes, AHEAD pieces later.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_LOAD));
        bool ok = true;
        const uint32_t ring = ptx::smem_u32(smem + T::OFF_RING), raw = ptx::smem_u32(smem + T::OFF_RAW) + tid * 16;
        constexpr int LANES = D * T::ES / 16, ROWS = 32 / LANES;          // lanes of a row, rows of a warp's load
        constexpr int LOADS = 32 / ROWS;                                  // loads of a warp's 32 rows
        constexpr int PIECES = T::DIRECT ? 1 : LOADS / T::RB, PER = LOADS / PIECES;
        const int sub_row = lane / LANES, piece16 = lane % LANES;
        const uint8_t* const k_lane = static_cast<const uint8_t*>(c.k) + piece16 * 16;
        const uint8_t* const v_lane = static_cast<const uint8_t*>(c.v) + piece16 * 16;
        // Place of this lane's part of row i * ROWS + sub_row of the warp's 32 in a tile of
        // 2-byte elements: the swizzle repeats every 8 rows.
        constexpr int OUT_B = T::VP == 2 ? 8 : T::Q8 ? 32 : 16, TURN = 8 / ROWS ? 8 / ROWS : 1;   // bytes of the part; loads of 8 rows
        uint32_t place[TURN];
#pragma unroll
        for (int i = 0; i < TURN; i++) place[i] = tile_at(warp * 32 + i * ROWS + sub_row, piece16 * OUT_B);
        auto place_of = [&](int i) { return place[i % TURN] + (uint32_t)(i / TURN) * 1024u; };

        // ---- the copies ----
        Segment g = segment_of<T>(p, cur, u, u_end);
        int idx = 0, tile_base = 0, n_copy = 0;             // load of the segment, tiles before it, loads begun
        uint32_t off0 = ~0u, off1 = ~0u, off_now = ~0u;     // this lane's row of even / odd tiles, units of 16 bytes
        int sp0 = 0, sp1 = 0, sp_now = 0, page_next = 0;    // its scale; the page of the next key tile
        bool is_v = false, mixed = false;
        int tile_no = 0;
        uint32_t live = 0;                                  // positions of the warp's 32 that exist
        auto page_of = [&](int j) -> int {
            const int pos = g.k0 + j * TKT + warp * 32 + lane;
            if (pos < cur.t.lo || pos >= cur.t.hi) return -1;
            int ip, slot;
            paged_split(p, pos, ip, slot);
            const int page = p.a.page_table[cur.s.b * p.a.table_stride + ip];
            return page < 0 ? 0x7fffffff : page;
        };
        auto begin_load = [&]() {
            const int a = g.two ? 1 : 2, n = g.tiles, head = min(a, n), r = idx - head, both = max(0, n - a);
            int j;   // K0 (K1) | V0 K(a) | V1 K(a+1) | ... | the last V
            if (r < 0) is_v = false, j = idx;
            else if (r < 2 * both) is_v = !(r & 1), j = (r >> 1) + (r & 1 ? a : 0);
            else is_v = true, j = r - both;
            tile_no = tile_base + j;
            if (idx == 0) page_next = page_of(0);
            if (!is_v) {
                uint32_t off = ~0u;
                int sp = 0;
                if (page_next >= c.n_pages) {
                    atomicCAS(p.err, 0, KERR_PAGE);
                } else if (page_next >= 0) {
                    int ip, slot;
                    paged_split(p, g.k0 + j * TKT + warp * 32 + lane, ip, slot);
                    off = (uint32_t)((page_next * c.stride[0] + slot * c.stride[1] + cur.h * c.stride[2]) * T::ES >> 4);
                    if constexpr (T::Q8) sp = (int)(page_next * c.scale_stride[0] + slot * c.scale_stride[1] + cur.h * c.scale_stride[2]);
                }
                if (j + 1 < n) page_next = page_of(j + 1);
                if (j & 1) off1 = off, sp1 = sp;
                else off0 = off, sp0 = sp;
            }
            off_now = j & 1 ? off1 : off0;
            sp_now = j & 1 ? sp1 : sp0;
            live = __ballot_sync(0xffffffffu, off_now != ~0u);
            if constexpr (T::DIRECT || CT == RT_F8E4M3) mixed = is_v && g.differ(g.k0 + j * TKT);
        };
        auto end_load = [&]() {
            n_copy++;
            if (++idx == 2 * g.tiles) {
                idx = 0;
                tile_base += g.tiles;
                u += g.tiles;
                cur.next_item<T::R>(p);
                if (u < u_end) g = segment_of<T>(p, cur, u, u_end);
            }
        };
        // Rows i0 .. i0 + N - 1 (of the warp's loads) to to(i).
        auto copy_rows = [&](int i0, auto to) {
            const uint8_t* base = is_v ? v_lane : k_lane;
            if (live == 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const uint32_t o = __shfl_sync(0xffffffffu, off_now, (i0 + i) * ROWS + sub_row);
                    cp_async16(to(i), base + ((uint64_t)o << 4));
                }
            } else {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const uint32_t o = __shfl_sync(0xffffffffu, off_now, (i0 + i) * ROWS + sub_row);
                    cp_async16(to(i), o == ~0u ? base : base + ((uint64_t)o << 4), o != ~0u);
                }
            }
        };

        if constexpr (T::DIRECT) {
            while (ok && u < u_end) {
                begin_load();
                const int s = n_copy % T::SLOTS;
                const uint32_t dst = ring + (uint32_t)s * T::SLOT;
                if (n_copy >= T::SLOTS)
                    ok = wait_warp(&bar.empty[s], (n_copy / T::SLOTS - 1) & 1, abort_flag, p.err, ERR_P_LOAD);
                if (!ok) break;
                copy_rows(0, [&](int i) { return dst + place_of(i); });
                if (is_v && warp == 0 && lane < 4) bar.strange[(tile_no + 4) & 7][lane] = 0;   // four tiles ahead of its use
                if (mixed) {
                    // Rows of the item see this tile differently: values that are not finite
                    // leave it (0 times them is not 0) and their positions are noted.
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    cp_wait<0>();
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
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive(&bar.full[s]);
                } else {
                    cp_async_arrive(&bar.full[s]);       // when this thread's copies so far have landed
                }
                if (!is_v && lane == 0) bar.ok[tile_no & 7][warp] = live;
                if (lane == 0) ptx::mbar_arrive(&bar.full[s]);   // the notes
                if (is_v) ptx::mbar_arrive(&bar.v_notes[tile_no & 3]);
                end_load();
            }
            cp_wait<0>();
        } else {
            constexpr int AHEAD = T::NRAW - 1;
            volatile uint32_t* meta = bar.meta[warp];       // by load & 7: is_v | mixed << 1 | tile << 2
            volatile uint32_t* there = bar.there[warp];
            int part = 0, raw_c = 0;                        // piece of the load, raw slot
            auto copy_piece = [&]() {
                if (part == 0) {
                    begin_load();
                    if (lane == 0) {
                        meta[n_copy & 7] = (is_v ? 1u : 0u) | (mixed ? 2u : 0u) | (uint32_t)tile_no << 2;
                        there[n_copy & 7] = live;
                    }
                    if constexpr (T::Q8)
                        cp_async4(ptx::smem_u32(smem + T::OFF_RAW_SCALE) + ((n_copy & 7) * 128 + tid) * 4, (is_v ? c.v_scale : c.k_scale) + sp_now,
                                  off_now != ~0u);
                }
                const uint32_t dst = raw + (uint32_t)raw_c * T::RAW_PIECE;
                copy_rows(part * PER, [&](int i) { return dst + i * 2048; });
                asm volatile("cp.async.commit_group;" ::: "memory");
                raw_c = raw_c + 1 == T::NRAW ? 0 : raw_c + 1;
                if (++part == PIECES) {
                    part = 0;
                    end_load();
                }
            };
            // ---- handing over ----
            int n_done = 0, done_part = 0, raw_d = 0;
            uint32_t top_all = 0;   // own scales: the largest of this lane's rows (bits)
            auto hand_piece = [&]() {
                const uint32_t what = meta[n_done & 7];
                const bool v = what & 1;
                const int tile = (int)(what >> 2), s = n_done % T::SLOTS;
                const uint32_t dst = ring + (uint32_t)s * T::SLOT, src = raw + (uint32_t)raw_d * T::RAW_PIECE;
                float* scales = v ? reinterpret_cast<float*>(smem + T::OFF_VS) + tile % (T::DIRECT ? 1 : T::VSD) * 128
                                  : reinterpret_cast<float*>(smem + T::OFF_KS) + tile % (T::DIRECT ? 1 : T::KSD) * 128;
                uint32_t w[PER][4];   // all of the piece at once: the conversions of its rows overlap
#pragma unroll
                for (int i = 0; i < PER; i++) ld_shared16(src + i * 2048, w[i]);
                if (done_part == 0) {
                    if (!v && lane == 0) bar.ok[tile & 7][warp] = there[n_done & 7];
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
                if constexpr (CT == RT_F8E4M3) {
                    // Codes 0x7f and 0xff are NaN, and so is 0 times them. Where rows see the tile
                    // differently such a row of values becomes zeros with a scale of NaN.
                    if (what & 2u) {
                        __syncwarp();   // (the scales are there)
#pragma unroll
                        for (int i = 0; i < PER; i++) {
                            uint32_t top = 0;
#pragma unroll
                            for (int k = 0; k < 4; k++) top |= (w[i][k] & 0x7f7f7f7fu) + 0x01010101u;
                            if (top & 0x80808080u) {
                                w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0;
                                scales[warp * 32 + (done_part * PER + i) * ROWS + sub_row] = __uint_as_float(0x7fc00000u);
                            }
                        }
                    }
                }
                if constexpr (T::Q8) {
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        uint32_t h[8];
#pragma unroll
                        for (int k = 0; k < 4; k++) codes_f16<CT>(w[i][k], h[2 * k], h[2 * k + 1]);
                        // (the two halves of 32 bytes are neighbours up to the swizzle's lowest bit)
                        const uint32_t at = dst + place_of(done_part * PER + i);
                        st_shared16(at, h[0], h[1], h[2], h[3]);
                        st_shared16(at ^ 16u, h[4], h[5], h[6], h[7]);
                    }
                } else {
                    constexpr int N = 16 / T::ES;
                    uint32_t top[PER];   // over the bits of |x|: what is not finite comes out on top
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        top[i] = 0;
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            top[i] = CT == RT_BF16 ? max(top[i], max(w[i][k] << 16 & 0x7fffffffu, w[i][k] & 0x7fff0000u)) : max(top[i], w[i][k] & 0x7fffffffu);
                    }
#pragma unroll
                    for (int o = LANES / 2; o; o >>= 1)
#pragma unroll
                        for (int i = 0; i < PER; i++) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        const int at_row = done_part * PER + i, r = warp * 32 + at_row * ROWS + sub_row;
                        const int e = f16_scale_exp(__uint_as_float(top[i]));
                        const bool finite = top[i] < 0x7f800000u;
                        const float up = finite ? pow2i(e) : 0.0f;
                        const float down = finite ? pow2i(-e) : __uint_as_float(0x7fc00000u);
                        float x[N];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if constexpr (CT == RT_BF16) {
                                x[2 * k] = __uint_as_float(w[i][k] << 16) * up;
                                x[2 * k + 1] = __uint_as_float(w[i][k] & 0xffff0000u) * up;
                            } else {
                                x[k] = __uint_as_float(w[i][k]) * up;
                            }
                        }
                        if (!finite) {
#pragma unroll
                            for (int k = 0; k < N; k++) x[k] = 0.0f;
                        }
                        // (a row of zeros has scale 0: weights are as large as the other rows' scales are small)
                        if (piece16 == 0) scales[r] = top[i] ? down : 0.0f;
                        if (finite && top[i]) top_all = max(top_all, __float_as_uint(down));
                        const uint32_t at = dst + place_of(at_row);
                        if constexpr (T::VP == 1) {
                            st_shared16(at, f16x2_rn(x[0], x[1]), f16x2_rn(x[2], x[3]), f16x2_rn(x[4 % N], x[5 % N]), f16x2_rn(x[6 % N], x[7 % N]));
                        } else {
                            float h[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) h[k] = round11(x[k]);
                            st_shared8(at, f16x2_rn(h[0], h[1]), f16x2_rn(h[2], h[3]));
                            st_shared8(at + T::PLANE, f16x2_rn(x[0] - h[0], x[1] - h[1]), f16x2_rn(x[2] - h[2], x[3] - h[3]));
                        }
                    }
                }
                if (v && done_part == PIECES - 1) {
                    const uint32_t top = __reduce_max_sync(0xffffffffu, top_all);
                    if (lane == 0) bar.vmax[tile & 3][warp] = __uint_as_float(top);
                }
                raw_d = raw_d + 1 == T::NRAW ? 0 : raw_d + 1;
                if (++done_part == PIECES) {
                    done_part = 0;
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive(&bar.full[s]);
                    if (v) ptx::mbar_arrive(&bar.v_notes[tile & 3]);
                    n_done++;
                }
            };
            int ahead = 0;
            while (ok && u < u_end) {
                copy_piece();
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
        }
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
                if constexpr (T::DIRECT) ptx::fence_proxy_async_smem();   // the copies landed as ordinary writes
            };
            auto release = [&](int n) { ptx::mma_commit(&bar.empty[n % T::SLOTS]); };
            auto scores = [&](int chain, int q_tile, int load) {   // S = Q.K^T: all features
                issue_scores<T, D>(tmem + T::COL_S + chain * 128, q_desc + (uint32_t)(q_tile * (T::QP * T::PLANE >> 4)),
                                   k_desc + (uint32_t)(load % T::SLOTS * (T::SLOT >> 4)), kind_s, std::make_integer_sequence<int, D / 16>());
            };
            auto values = [&](int chain, int load, bool add) {   // O (+)= P.V over 128 positions
                issue_values<T>(tmem + T::COL_O + chain * 128, tmem + T::COL_S + chain * 128,
                                v_desc + (uint32_t)(load % T::SLOTS * (T::SLOT >> 4)), kind_o, add ? 1u : 0u,
                                std::make_integer_sequence<int, TKT / 16>());
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
                if (!g.two) {
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
                        values(t, n_use, !F32ACT && j >= 2);
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
                    scores(1, 1, n_use);
                    ptx::mma_commit(&bar.s_full[1]);
                    release(n_use++);
                    for (int j = 0; j < g.tiles && ok; j++) {
                        const int v = n_use, k = n_use + 1;
                        const bool more = j + 1 < g.tiles;
                        wait_load(v);
                        wait_p(0);
                        if (!ok) break;
                        values(0, v, j > 0);
                        if (more) {
                            wait_load(k);
                            if (!ok) break;
                            scores(0, 0, k);
                        }
                        ptx::mma_commit(&bar.s_full[0]);
                        wait_p(1);
                        if (!ok) break;
                        values(1, v, j > 0);
                        release(v);
                        if (more) {
                            scores(1, 1, k);
                            release(k);
                        }
                        ptx::mma_commit(&bar.s_full[1]);
                        n_use += more ? 2 : 1;
                    }
                }
                u += g.tiles;
                cur.next_item<T::R>(p);
            }
            ptx::mma_commit(&bar.drain);   // nothing in flight when TMEM is given back
            volatile int no_abort = 0;
            ptx::wait_bounded(&bar.drain, 0, &no_abort, p.err, ERR_P_MMA, WAIT_NS);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_SOFT));
        const int wg = (warp - 8) >> 2, quarter = warp & 3, row = quarter * 32 + lane;   // TMEM lane `row` is this thread's
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const float base = p.a.scale * 1.4426950408889634f;   // scores in log2 units
        float* qs = reinterpret_cast<float*>(smem + T::OFF_QS);
        int n_s[2] = {0, 0}, n_join = 0, n_half = 0, tile_base = 0;
        bool ok = true, was_two = false;
        auto wait_s = [&](int t) {
            ok = wait_warp(&bar.s_full[t], n_s[t]++ & 1, abort_flag, p.err, ERR_P_SOFT);
            ptx::tc_fence_after();
        };
        auto meet = [&]() {   // all softmax threads
            ptx::mbar_arrive(&bar.join);
            ok = wait_warp(&bar.join, n_join++ & 1, abort_flag, p.err, ERR_P_SOFT);
        };
        // What comes with a tile's V (its scales, the positions taken out of it) is there once
        // V has landed, which its product waits for, not the scores.  (Not the ring slot's
        // barrier, which may be two phases away here: up to two later V tiles may have landed
        // too, hence four barriers.)
        auto wait_v = [&](int tile_no) {
            ok = wait_warp(&bar.v_notes[tile_no & 3], (tile_no >> 2) & 1, abort_flag, p.err, ERR_P_SOFT);
        };
        while (ok && u < u_end) {
            const Segment g = segment_of<T>(p, cur, u, u_end);
            const PagedSeq& s = cur.s;
            const bool split_keys = !F32ACT && !g.two;
            if (split_keys && was_two) {   // chain 1's products have read its own Q, whose place is used below
                meet();
                if (!ok) break;
            }
            was_two = g.two;
            // ---- Q into shared memory: LQ lanes a row, 8 features each ----
            if (F32ACT || wg == 0 || g.two) {
                constexpr int LQ = D / 8, STEP = (F32ACT ? 256 : 128) / LQ;
                const int q_tile = g.two ? wg : 0, first = q_tile * 128, n = min(128, g.rows - first);
                const uint32_t dst = ptx::smem_u32(smem) + (uint32_t)q_tile * T::QP * T::PLANE;
                const int t = F32ACT ? tid - 256 : row, d = t % LQ * 8;
                const bool bf = p.a.dtype == RT_BF16;
#pragma unroll 4
                for (int r = t / LQ; r < n; r += STEP) {   // (rows past the item hold whatever was there: their results go nowhere)
                    const int rr = g.row0 + first + r;
                    const int64_t at = (int64_t)(s.first + rr / p.group) * p.a.q_stride[0] + (cur.h * p.group + rr % p.group) * p.a.q_stride[1] + d;
                    const float* qf = static_cast<const float*>(p.a.q) + at;
                    const __nv_bfloat16* qh = static_cast<const __nv_bfloat16*>(p.a.q) + at;
                    const uint32_t a = dst + tile_at(r, d * 2);
                    if constexpr (T::DIRECT) {
                        if (p.vec_q) {
                            cp_async16(a, qh, true);
                        } else {
                            const unsigned short* q16 = reinterpret_cast<const unsigned short*>(qh);
                            st_shared16(a, q16[0] | q16[1] << 16, q16[2] | q16[3] << 16, q16[4] | q16[5] << 16, q16[6] | q16[7] << 16);
                        }
                    } else {
                        float x[8], h[8], m = 0.0f;
                        if (bf && p.vec_q) {
                            const uint4 v = *reinterpret_cast<const uint4*>(qh);
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                x[2 * i] = __uint_as_float(w[i] << 16);
                                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                            }
                        } else if (p.vec_q) {
                            const float4 v = *reinterpret_cast<const float4*>(qf), w = *reinterpret_cast<const float4*>(qf + 4);
                            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
                            x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; i++) x[i] = bf ? __bfloat162float(qh[i]) : qf[i];
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
                        const uint32_t mates = (LQ == 16 ? 0xffffu : 0xffu) << (lane / LQ * LQ);
#pragma unroll
                        for (int i = LQ / 2; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(mates, m, i));
                        const int e = f16_scale_exp(m);
                        const float up = pow2i(e);
                        if (t % LQ == 0) qs[first + r] = base * pow2i(-e);
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
                if constexpr (T::DIRECT) {
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    cp_wait<0>();
                }
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(&bar.q_full[q_tile]);
            }
            // ---- this thread's row ----
            const int my_row = g.row0 + row + (g.two ? wg * 128 : 0);
            const bool live = my_row < g.row0 + g.rows, any_live = __any_sync(0xffffffffu, live);
            const int at_pos = s.L - s.n + my_row / p.group;
            const int lo_row = paged_lo(p, at_pos);
            const int hi_row = live ? (p.a.causal ? min(s.L, at_pos + 1) : s.L) : 0;
            // m, l: the row's maximum (as of the last move) and its weight sum in units of 2^m. Exponents are
            // taken against ref = m + the exponent of the value scales: weights times scales are then in
            // fp16's range, and O is in units of `unit` = 2^(ref - m), which l, with no values in it, is not.
            float c_row = base, m = -INFINITY, l = 0.0f, ref = 0.0f, v_top = 0.0f, unit = 1.0f;
            // Scores of N positions from b on: times their scales, -inf where the row does not see them; their maximum.
            auto see = [&](auto& x, int b, int tile_no, int k0, bool masked) -> float {
                constexpr int N = sizeof(x) / 4;
                if constexpr (!T::DIRECT) {
                    const float* ks = reinterpret_cast<const float*>(smem + T::OFF_KS) + tile_no % T::KSD * 128 + b;
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        const float4 k = *reinterpret_cast<const float4*>(ks + i);
                        upk2(mul2(pk2(x[i], x[i + 1]), pk2(k.x, k.y)), x[i], x[i + 1]);
                        upk2(mul2(pk2(x[i + 2], x[i + 3]), pk2(k.z, k.w)), x[i + 2], x[i + 3]);
                    }
                }
                if (masked) {
#pragma unroll
                    for (int w = 0; w < N / 32; w++) {
                        const uint32_t there = bar.ok[tile_no & 7][(b >> 5) + w];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const int k = k0 + b + w * 32 + i;
                            if (!((there >> i & 1) && k >= lo_row && k < hi_row)) x[w * 32 + i] = -INFINITY;
                        }
                    }
                }
                float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    t0 = max3f(t0, x[i], x[i + 1]);
                    t1 = max3f(t1, x[i + 2], x[i + 3]);
                }
                return fmaxf(t0, t1) * c_row;
            };
            auto sees_all = [&](int k0, int tile_no) {
                const uint32_t* w = bar.ok[tile_no & 7];
                return lo_row <= k0 && hi_row >= k0 + TKT && (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu;
            };
            // Moves the reference when a score or a value scale asks for it; the factor for what
            // has been summed, 1 where nothing moved.
            auto refer = [&](float top, int tile_no) -> float {
                float tile_v = 0.0f;
                if constexpr (!T::DIRECT) {
                    const float* vm = bar.vmax[tile_no & 3];
                    tile_v = fmaxf(fmaxf(vm[0], vm[1]), fmaxf(vm[2], vm[3]));
                }
                const bool raise = top > m + RAISE, wider = !T::DIRECT && tile_v > v_top;
                if (!raise && !wider) return 1.0f;
                const bool first = m == -INFINITY;   // (nothing summed yet: o = 0)
                if (raise) {
                    if (!first) l *= exp2_fast(m - top);
                    m = top;
                }
                if (wider) v_top = 4.0f * tile_v;
                const int shift = T::DIRECT ? 0 : max((int)(__float_as_uint(v_top) >> 23) - 127, -100) - W_LOG2;
                const float to = (m == -INFINITY ? 0.0f : m) + (float)shift;
                // (by the row's maximum: the weight sum of a thread that has half of the row's positions may
                // be 0 where the other's is not, and its share of the output has both)
                const float f = first ? 0.0f : exp2_fast(ref - to);
                ref = to;
                if constexpr (!T::DIRECT) unit = pow2i(shift);
                return f;
            };
            // Scores to weights, in place; their sum.  Then times the value scales.
            auto weigh = [&](auto& x, int b, int tile_no, bool masked) {
                constexpr int N = sizeof(x) / 4;
                const unsigned long long cc = pk2(c_row, c_row), nr = pk2(-ref, -ref);
                unsigned long long s0 = pk2(0.0f, 0.0f), s1 = s0;
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    upk2(fma2(pk2(x[i], x[i + 1]), cc, nr), x[i], x[i + 1]);
                    upk2(fma2(pk2(x[i + 2], x[i + 3]), cc, nr), x[i + 2], x[i + 3]);
#pragma unroll
                    for (int k = 0; k < 4; k++) x[i + k] = exp2_fast(x[i + k]);
                    s0 = add2(s0, pk2(x[i], x[i + 1]));
                    s1 = add2(s1, pk2(x[i + 2], x[i + 3]));
                }
                float a, c2;
                upk2(add2(s0, s1), a, c2);
                l += T::DIRECT ? a + c2 : (a + c2) * unit;
                if constexpr (!T::DIRECT) {
                    const float* vs = reinterpret_cast<const float*>(smem + T::OFF_VS) + tile_no % T::VSD * 128 + b;
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        const float4 v = *reinterpret_cast<const float4*>(vs + i);
                        const float w[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
                        upk2(mul2(pk2(x[i], x[i + 1]), pk2(v.x, v.y)), x[i], x[i + 1]);
                        upk2(mul2(pk2(x[i + 2], x[i + 3]), pk2(v.z, v.w)), x[i + 2], x[i + 3]);
                        if (masked) {   // a position that is not seen may have any scale
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                if (w[k] == 0.0f) x[i + k] = 0.0f;
                        }
                    }
                }
            };
            constexpr int NO = F32ACT ? D / 2 : D;   // this thread's output columns
            const int col0 = F32ACT ? wg * (D / 2) : 0;
            float o[NO];
            if constexpr (F32ACT) {
                // Two threads a row, 64 positions and D / 2 output columns each; S, P and O of even
                // and odd tiles in places of their own.  A tile's O is folded into registers two
                // tiles later, when its scores' successors are ready.
                float* red = reinterpret_cast<float*>(smem + T::OFF_RED);
                float ref_of[2] = {0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < NO; i++) o[i] = 0.0f;
                auto fold = [&](int t) {
                    const float f = ref_of[t] == ref ? 1.0f : exp2_fast(ref_of[t] - ref);
                    const unsigned long long ff = pk2(f, f);
#pragma unroll
                    for (int b = 0; b < NO; b += 32) {
                        uint32_t r[32];
                        ptx::tmem_ld32(tmem + lanes + T::COL_O + t * 128 + col0 + b, r);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            upk2(fma2(pk2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), ff, pk2(o[b + i], o[b + i + 1])), o[b + i], o[b + i + 1]);
                    }
                };
                for (int j = 0; j < g.tiles; j++) {
                    const int t = j & 1, tile_no = tile_base + j, k0 = g.k0 + j * TKT;
                    wait_s(t);
                    if (!ok) break;
                    if (j == 0) c_row = qs[row];
                    if (any_live) {
                        const uint32_t s_at = tmem + lanes + T::COL_S + t * 128 + wg * 64;
                        const bool masked = __any_sync(0xffffffffu, live && !sees_all(k0, tile_no));
                        float x[64];
                        {
                            uint32_t(&r)[64] = reinterpret_cast<uint32_t(&)[64]>(x);
                            ptx::tmem_ld32(s_at, reinterpret_cast<uint32_t(&)[32]>(r[0]));
                            ptx::tmem_ld32(s_at + 32, reinterpret_cast<uint32_t(&)[32]>(r[32]));
                            ptx::tmem_ld_wait();
                        }
                        float top = see(x, wg * 64, tile_no, k0, masked);
                        // the row's other half: read for tile j - 2 before anyone got here
                        red[(t * 2 + wg) * 128 + row] = top;
                        ptx::mbar_arrive(&bar.half[quarter]);
                        ok = wait_warp(&bar.half[quarter], n_half++ & 1, abort_flag, p.err, ERR_P_SOFT);
                        if (!ok) break;
                        top = fmaxf(top, red[(t * 2 + (wg ^ 1)) * 128 + row]);
                        wait_v(tile_no);
                        if (!ok) break;
                        const float f = refer(top, tile_no);
                        if (__any_sync(0xffffffffu, f != 1.0f)) {
                            const unsigned long long ff = pk2(f, f);
#pragma unroll
                            for (int i = 0; i < NO; i += 2) upk2(mul2(pk2(o[i], o[i + 1]), ff), o[i], o[i + 1]);
                        }
                        if (j >= 2) fold(t);
                        ref_of[t] = m == -INFINITY ? -INFINITY : ref;   // (nothing seen so far: O is 0, and the reference may come down)
                        weigh(x, wg * 64, tile_no, masked);
#pragma unroll
                        for (int b = 0; b < 64; b += 16) {   // per 16 positions: 8 columns of hi pairs, 8 of lo pairs
                            uint32_t w[16];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float ha = __uint_as_float(__float_as_uint(x[b + 2 * i]) & 0xffffe000u);
                                const float hb = __uint_as_float(__float_as_uint(x[b + 2 * i + 1]) & 0xffffe000u);
                                w[i] = f16x2_rn(ha, hb);
                                w[8 + i] = f16x2_rn(x[b + 2 * i] - ha, x[b + 2 * i + 1] - hb);
                            }
                            ptx::tmem_st16(s_at + b, w);
                        }
                        ptx::tmem_st_wait();
                    }
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(&bar.p_full[t]);
                }
                for (int j = max(0, g.tiles - 2); ok && j < g.tiles; j++) {
                    wait_s(j & 1);
                    if (ok && any_live) fold(j & 1);
                }
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < NO; i++) o[i] *= unit;
                ptx::tc_fence_before();
                if (any_live) {   // the weight sum of both halves
                    const int t = g.tiles & 1;
                    red[(t * 2 + wg) * 128 + row] = l;
                    ptx::mbar_arrive(&bar.half[quarter]);
                    ok = wait_warp(&bar.half[quarter], n_half++ & 1, abort_flag, p.err, ERR_P_SOFT);
                    if (!ok) break;
                    l = wg ? red[t * 2 * 128 + row] + l : l + red[(t * 2 + 1) * 128 + row];
                }
            } else {
                // A thread per row; O stays in TMEM and is rescaled there when the reference moves.
                const int chain = wg, step = split_keys ? 2 : 1;
                const uint32_t s_at = tmem + lanes + T::COL_S + chain * 128, o_at = tmem + lanes + T::COL_O + chain * 128;
                const int j0 = split_keys ? chain : 0;
                bool spoiled = false;   // bf16 all the way: the row sees a value that is not finite
                for (int j = j0; j < g.tiles; j += step) {
                    const int tile_no = tile_base + j, k0 = g.k0 + j * TKT;
                    wait_s(chain);
                    if (!ok) break;
                    if (!T::DIRECT && j == j0) c_row = qs[row + (g.two ? chain * 128 : 0)];
                    if (any_live) {
                        const bool masked = __any_sync(0xffffffffu, live && !sees_all(k0, tile_no));
                        float x[128];
                        {
                            uint32_t(&r)[128] = reinterpret_cast<uint32_t(&)[128]>(x);
#pragma unroll
                            for (int b = 0; b < 128; b += 32) ptx::tmem_ld32(s_at + b, reinterpret_cast<uint32_t(&)[32]>(r[b]));
                            ptx::tmem_ld_wait();
                        }
                        const float top = see(x, 0, tile_no, k0, masked);
                        // values that are not finite were taken out of a tile that rows of the item see
                        // differently, for the rows that see all of it too
                        const bool noted = T::DIRECT && g.differ(k0);
                        if (!T::DIRECT || noted) {
                            wait_v(tile_no);
                            if (!ok) break;
                        }
                        const float f = refer(top, tile_no);
                        if (j > j0 && __any_sync(0xffffffffu, f != 1.0f)) {
                            const unsigned long long ff = pk2(f, f);
#pragma unroll
                            for (int b = 0; b < D; b += 16) {
                                uint32_t r[16];
                                ptx::tmem_ld16(o_at + b, r);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 16; i += 2) {
                                    float a, c2;
                                    upk2(mul2(pk2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), ff), a, c2);
                                    r[i] = __float_as_uint(a);
                                    r[i + 1] = __float_as_uint(c2);
                                }
                                ptx::tmem_st16(o_at + b, r);
                            }
                        }
                        weigh(x, 0, tile_no, masked);
#pragma unroll
                        for (int b = 0; b < 128; b += 32) {
                            uint32_t w[16];
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                // one part, whose rounding (2^-8, 2^-11) the sum averages: below the output's own
                                w[i] = T::DIRECT ? bf16_pair_rn(x[b + 2 * i], x[b + 2 * i + 1]) : f16x2_rn(x[b + 2 * i], x[b + 2 * i + 1]);
                            ptx::tmem_st16(s_at + b / 2, w);
                        }
                        if constexpr (T::DIRECT) {
                            if (noted) {   // rows that see such a value get NaN
                                const uint32_t* sw = bar.strange[tile_no & 7];
                                if (sw[0] | sw[1] | sw[2] | sw[3])
                                    for (int i = 0; i < TKT; i++)
                                        if ((sw[i >> 5] >> (i & 31) & 1) && k0 + i >= lo_row && k0 + i < hi_row) spoiled = true;
                            }
                        }
                        ptx::tmem_st_wait();
                    }
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(&bar.p_full[chain]);
                }
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < NO; i++) o[i] = 0.0f;
                if (j0 < g.tiles) {
                    wait_s(chain);
                    if (!ok) break;
                    if (any_live) {
                        uint32_t(&r)[NO] = reinterpret_cast<uint32_t(&)[NO]>(o);
#pragma unroll
                        for (int b = 0; b < D; b += 32) ptx::tmem_ld32(o_at + b, reinterpret_cast<uint32_t(&)[32]>(r[b]));
                        ptx::tmem_ld_wait();
                    }
                    if constexpr (!T::DIRECT) {
#pragma unroll
                        for (int i = 0; i < NO; i++) o[i] *= unit;
                    }
                    if (T::DIRECT && spoiled) {
#pragma unroll
                        for (int i = 0; i < NO; i++) o[i] = __uint_as_float(0x7fc00000u);
                    }
                    ptx::tc_fence_before();
                }
                if (split_keys) {   // the other chain's share of the keys
                    float* x = reinterpret_cast<float*>(smem + T::QP * T::PLANE);   // the second Q tile's place
                    if (chain == 1) {
                        x[row] = m;
                        x[128 + row] = l;
                    }
                    meet();
                    if (!ok) break;
                    float f0 = 1.0f, f1 = 0.0f;
                    if (chain == 0) {   // (a sum of NaN has no maximum to go by, and goes into the result)
                        const float m1 = x[row], l1 = x[128 + row], to = fmaxf(m, m1);
                        f0 = l == 0.0f ? 0.0f : l == l ? exp2_fast(m - to) : l;
                        f1 = l1 == 0.0f ? 0.0f : l1 == l1 ? exp2_fast(m1 - to) : l1;
                        l = l * f0 + l1 * f1;
                        m = to;
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
            }
            // ---- out ----
            if (live && (F32ACT || wg == 0 || g.two)) {
                if (cur.i == 0 && g.tiles == cur.t.count) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int64_t at = paged_out_at(p, s, cur.h, my_row) + col0;
                    if (!p.vec_out) {
#pragma unroll
                        for (int i = 0; i < NO; i++) {
                            if (p.a.dtype == RT_BF16) static_cast<__nv_bfloat16*>(p.a.out)[at + i] = __float2bfloat16_rn(o[i] * inv);
                            else static_cast<float*>(p.a.out)[at + i] = o[i] * inv;
                        }
                    } else if (p.a.dtype == RT_BF16) {
                        uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + at);
#pragma unroll
                        for (int i = 0; i < NO / 8; i++)
                            out[i] = make_uint4(bf16_pair_rn(o[8 * i] * inv, o[8 * i + 1] * inv), bf16_pair_rn(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                                bf16_pair_rn(o[8 * i + 4] * inv, o[8 * i + 5] * inv), bf16_pair_rn(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                    } else {
                        float4* out = reinterpret_cast<float4*>(static_cast<float*>(p.a.out) + at);
#pragma unroll
                        for (int i = 0; i < NO / 4; i++)
                            out[i] = make_float4(o[4 * i] * inv, o[4 * i + 1] * inv, o[4 * i + 2] * inv, o[4 * i + 3] * inv);
                    }
                    if (col0 == 0) paged_store_lse(p, s, cur.h, my_row, m, l);
                } else {
                    float* part = p.part + (int64_t)(2 * blockIdx.x + (cur.i == 0)) * T::OUT;
                    const int r = my_row - g.row0;
                    float4* out = reinterpret_cast<float4*>(part + r * D + col0);
#pragma unroll
                    for (int i = 0; i < NO / 4; i++) out[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    if (col0 == 0) {
                        part[T::R * D + r] = m;
                        part[T::R * D + T::R + r] = l;
                    }
                }
            }
            tile_base += g.tiles;
            u += g.tiles;
            cur.next_item<T::R>(p);
        }
    }
    __syncthreads();
    if (warp == 4) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}


int tile_rows(const RtPagedAttention& p) { return p.cache.dtype == RT_F32 || p.dtype == RT_F32 ? 128 : 256; }

// Blocks of a call: one per SM, no more than there are key tiles (2 prompts of 200
// tokens, 12 heads of 64, fp32 over int8: 45 us with four tiles a block at least, 22 with one).
int tiles_blocks(const RtPagedAttention& p) {
    const int R = tile_rows(p);
    const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(p.max_new, p.total_new)) * (p.n_q_heads / p.cache.n_heads);
    const int64_t units = (int64_t)p.n_seqs * p.cache.n_heads * ((rows + R - 1) / R) * std::max(1, (p.max_kv + TKT - 1) / TKT);
    return (int)std::max<int64_t>(1, std::min<int64_t>(g_num_sms, units));
}

template <int CT, bool F32ACT, int D>
Status tiles_as(PagedArgs& p, void* ws, cudaStream_t st) {
    using T = Tile<CT, F32ACT, D>;
    static const cudaError_t set = cudaFuncSetAttribute(paged_tiles_kernel<CT, F32ACT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    RT_CUDA_CHECK(set);
    const int blocks = tiles_blocks(p.a);
    paged_set_workspace(p, ws, blocks);
    p.whole = 0;
    p.key_shift = 7;
    p.head_group = 1;
    p.head_groups = p.a.cache.n_heads;
    p.min_units = 1;
    paged_tiles_kernel<CT, F32ACT, D><<<blocks, TT, T::SMEM, st>>>(p);
    RT_LAUNCH_CHECK();
    return blocks == 1 ? Status::ok() : launch_paged_join<D, T::R>(p, blocks, st);
}
template <int CT, bool F32ACT>
Status tiles_dim(PagedArgs& p, void* ws, cudaStream_t st) {
    return p.a.cache.head_dim == 128 ? tiles_as<CT, F32ACT, 128>(p, ws, st) : tiles_as<CT, F32ACT, 64>(p, ws, st);
}

}  // namespace

bool paged_tiles_takes(const RtPagedAttention& p) { return p.cache.head_dim == 64 || p.cache.head_dim == 128; }

size_t paged_tiles_workspace(const RtPagedAttention& p) {
    const int R = tile_rows(p);
    return paged_workspace(tiles_blocks(p), 1, R * p.cache.head_dim + 2 * R);
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
