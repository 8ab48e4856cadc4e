// The tiled product of block_fp8.h: codes of x and of the weight meet in LDS, 128 values of K at a time.
//
// A workgroup of WM x WN waves owns WM * TM * 16 rows of x by WN * TN * 16 weight rows.  A step's codes of both operands come by
// LDS-DMA into two buffers, asked for a step and a half ahead, or three, two steps ahead; a step is one block of K, so a wave multiplies
// TM x TN results by one instruction each, from zero, and adds them to the sums in float32 times the two scales.
//
// LDS holds rows of 128 bytes, the 16-byte chunk c of row r at slot c ^ swizzle(r): the DMA writes 8 rows of 8 slots at a time (lane
// = 8 * row + slot, so the swizzle is in the lane's source address), and 16 lanes of a read, which take one chunk of 16
// consecutive rows, cover all 64 banks: two rows are 256 bytes, and the eight rows of one parity have different slots.  (With slots that
// repeat after four rows half of LDS' busy cycles were conflicts.)
//
// Bound by the matrix pipes and the clock that the power limit leaves them (1.6 GHz at the largest sizes): 8192^3 448 us, 2.45 PFLOP/s, where
// the library's product with a single scale takes 386; [28672 x 8192] by 8192 rows 1550 us, MFMAs on 66 % of the cycles, no LDS conflict.
// A few hundred rows are bound by the latency of a step: two groups of waves that take half of a tile's blocks each, 333 x 3211 x 2112 in
// float32 15 us against 17, 300 x 4096 x 4096 14.2 / 17.6, 40 x 11008 x 4096 11.7 against 13.3 in two splits and their sum (without the
// launch of 2.5 us that quantizes the rows).
//
// EXACT, for sums that keep float32's 24 bits (block_fp8.h): the bfloat16 MFMA, four instructions of 32 values in place of one.  x comes as
// bfloat16 numbers, rows of 256 bytes a block, and only the weight's codes are widened on the way from LDS, part by part.
#pragma once
#include "block_fp8.h"
#include "lowbit_gemm.h"

namespace lowbit {

struct TiledArgs {
    const uint8_t *x;                                        // codes (EXACT: their numbers in bfloat16), rows of ldx bytes, zeros past K
    const float *xs;                                         // [KB][ldxs], by row of x
    const uint8_t *w;
    const float *ws;
    const void *bias;
    void *y;
    float *part;                                             // sums of a split: [split][M][pitch]
    const int32_t *offsets, *order;                          // by expert: rows offsets[e] .. of the result; x row order[row] / top_k, or row
    int64_t ldx;
    int ldxs, M, N, K, KB, pitch;
    int tiles_m, tiles_n, splits, split_blocks;
    int n_exp, top_k, I, act;                                // UP: I columns of h
    int expert_rows;                                         // by expert: weight rows from one expert's to the next's, N of which the launch takes
    float *hs;                                               // UP: scales of h, [I / 128][ldhs]; its codes go to y
    int ldhs;
};

enum TiledMode { TILED_PLAIN, TILED_PART, TILED_UP };

__device__ inline int swizzle(int row) { return (row >> 1) & 7; }

// 16 bytes per lane from base + off (or from the lanes' own addresses) to LDS at lds_at + 16 * lane.  Inline assembly, because the compiler
// takes an LDS-DMA to alias every later LDS access and waits for it at once; here the wait is the one ahead of the step's barrier.
__device__ inline void dma16(uint32_t off, uint64_t base, uint32_t lds_at) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds_at) : "memory", "m0");
}
__device__ inline void dma4(uint32_t off, uint64_t base, uint32_t lds_at) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" :: "v"(off), "s"(base), "s"(lds_at) : "memory", "m0");
}
__device__ inline void dma16_at(uint64_t address, uint32_t lds_at) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(address), "s"(lds_at) : "memory", "m0");
}

// (the other two counters untouched: 4 bits of lgkmcnt at 8)
__device__ inline void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// The part of a lane's 32 codes that the p-th of four bfloat16 MFMAs takes
__device__ inline bf16x8 widen_part(const Codes &c, int p) {
    const u32x4 &h = p < 2 ? c.lo : c.hi;
    return widen8(h[2 * (p & 1)], h[2 * (p & 1) + 1]);
}
// A lane's values of x: codes, or (EXACT) the same numbers in bfloat16, part by part
template <bool EXACT> struct XOperand;
template <> struct XOperand<false> {
    Codes v;
};
template <> struct XOperand<true> {
    bf16x8 v[4];
};

template <typename OT> struct Stored;
template <> struct Stored<float> {
    static __device__ float of(float v) { return v; }
};
template <> struct Stored<_Float16> {
    static __device__ _Float16 of(float v) { return (_Float16)v; }
};
template <> struct Stored<__bf16> {
    static __device__ __bf16 of(float v) { return (__bf16)v; }
};

// BY_EXPERT: row tiles of one expert each.  GATHER: x rows by order[].  S: buffers in LDS.  KG: groups of WM x WN waves, each with buffers of
// its own, that share a tile's blocks out among them and add their sums at the end.
template <typename OT, bool EXACT, TiledMode MODE, bool BY_EXPERT, bool GATHER, int TM, int TN, int WM, int WN, int S, int MIN_WAVES, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, MIN_WAVES) void block_fp8_tiled_kernel(const TiledArgs p) {
    constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
    constexpr int XB = EXACT ? 256 : 128, XR = 1024 / XB, XP = BM / XR, WP = BN / 8;   // bytes of a row of x, rows of a piece, pieces
    constexpr int PX = XP / WAVES, PW = WP / WAVES;
    constexpr bool UP = MODE == TILED_UP;
    constexpr int TH = TN / 2;                               // UP: a wave's tiles of the gate, and as many of u
    // Two buffers: a step in two halves, each with a barrier (see the loop)
    constexpr int HALVES = S == 2 ? 2 : 1, PH = PW / HALVES;
    static_assert(KG == 1 || (KG == 2 && MODE != TILED_UP && !BY_EXPERT && (int)(S * (BM * XB + BN * FP8_BLOCK)) >= TM * TN * WAVES * 1024), "room for a group's sums");
    static_assert(WP % (WAVES * HALVES) == 0 && XP % WAVES == 0 && PX > 0 && BM / WAVES <= 64 && TN % 2 == 0 && (S > 2 || TN % 4 == 0 || TN == 2) &&
                  (!UP || BN == 256), "whole pieces per wave");
    constexpr uint32_t BUFFER = BM * XB + BN * FP8_BLOCK, SCALES = BM * 4;
    constexpr uint32_t OWN = S * (BUFFER + SCALES);          // a group's
    __shared__ __attribute__((aligned(16))) uint8_t shared[KG * OWN];
    const int lane = threadIdx.x & 63, in_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int group = KG == 1 ? 0 : in_all / WAVES, wave = in_all - group * WAVES, wm = wave / WN, wn = wave % WN;
    uint8_t *const lds = shared + group * OWN;

    // Workgroups go to the XCDs in turn: each takes a run of the tiles, eight row tiles by as many columns as its CUs hold, so that
    // its L2 serves every operand several times.  By expert: all row tiles of a column side by side, those that there are (the launch
    // counts what there may be at most; runs of tiles of which some do not exist would leave XCDs idle).
    const int tiles_m = BY_EXPERT ? count_expert_tiles<BM>(p.offsets, p.n_exp) : p.tiles_m, tall = BY_EXPERT ? tiles_m : 8;
    const uint32_t units = (uint32_t)(tiles_m * p.tiles_n * p.splits), xcd = blockIdx.x & 7;
    const uint32_t unit = (uint32_t)((uint64_t)units * xcd >> 3) + (blockIdx.x >> 3);
    if (unit >= (uint32_t)((uint64_t)units * (xcd + 1) >> 3)) return;
    const int tile = (int)(unit / p.splits), split = (int)(unit - (uint32_t)tile * p.splits);
    int tm, tn;
    {
        const int per = tall * p.tiles_n, band = tile / per, at = tile - band * per, rows = tiles_m - band * tall < tall ? tiles_m - band * tall : tall;
        tn = at / rows;
        tm = band * tall + at - tn * rows;
    }
    int m0 = tm * BM, end = p.M, expert = 0;
    if constexpr (BY_EXPERT) {
        ExpertTile t;
        if (!find_expert_tile<BM>(p.offsets, p.n_exp, tm, t)) return;
        expert = __builtin_amdgcn_readfirstlane(t.expert);
        m0 = __builtin_amdgcn_readfirstlane(t.first);
        end = __builtin_amdgcn_readfirstlane(t.end);
    }
    const int n0 = tn * (UP ? FP8_BLOCK : BN), KB = p.KB;
    // blocks of K: of this split, and of this group (an odd one out is the first group's; the other walks as far, and adds nothing for it)
    const int from = split * p.split_blocks, to = MODE == TILED_PART && from + p.split_blocks < KB ? from + p.split_blocks : KB;
    const int walk = (to - from + KG - 1) / KG, b0 = KG == 1 || group == 0 ? from : from + walk, stop = b0 + walk, b1 = stop < to ? stop : to;

    // ---- sources of this wave's pieces of 8 rows
    uint32_t xoff[GATHER ? 1 : PX], woff[PW];
    uint64_t xaddr[GATHER ? PX : 1];
    const int piece_row = lane >> 3;
    const uint64_t xbase = (uint64_t)(uintptr_t)p.x + (GATHER ? 0 : (uint64_t)m0 * p.ldx);
#pragma unroll
    for (int j = 0; j < PX; j++) {
        const int row = (wave * PX + j) * XR + lane / (XB / 16), chunk = ((lane % (XB / 16)) ^ (EXACT ? row & 15 : swizzle(row))) * 16;
        const int at = m0 + row < end ? m0 + row : end - 1;
        if constexpr (GATHER) xaddr[j] = xbase + (uint64_t)(p.order[at] / p.top_k) * p.ldx + chunk;
        else xoff[j] = (uint32_t)((at - m0) * p.ldx) + chunk;
    }
    const uint64_t wexpert = (uint64_t)(uintptr_t)p.w + (BY_EXPERT ? (uint64_t)expert * p.expert_rows * p.K : 0);
    // Which weight row lies in row `at` of LDS: a wave column's tiles of 16, each lane quarter's four rows of them neighbours of its
    // four in the next tile, so that a lane's results are neighbours in a row of y.  UP: tiles of the gate, then as many of u.
    auto weight_row = [&](int at) -> int64_t {
        const int col = at / (TN * 16), i = at / 16 % TN, q = at / 4 % 4, t = at % 4;
        if constexpr (UP) return (int64_t)(i / TH) * p.I + n0 + col * (TH * 16) + q * (TH * 4) + i % TH * 4 + t;
        const int n = n0 + col * (TN * 16) + i / 2 * 32 + q * 8 + i % 2 * 4 + t;
        return n < p.N ? n : p.N - 1;
    };
    // Row of LDS where the wave's piece j starts: with two halves the first PH pieces are of the first half of every wave column's tiles
    auto piece_at = [&](int j) {
        const int id = wave * PH + j % PH;
        return HALVES == 1 ? id * 8 : (id / TN) * (TN * 16) + j / PH * (TN * 8) + id % TN * 8;
    };
    uint32_t wchunk[2];                                      // of even and odd rows of eight: 8 rows more turn one bit of the swizzle
#pragma unroll
    for (int j = 0; j < 2; j++) wchunk[j] = ((lane & 7) ^ swizzle(j * 8 + piece_row)) * 16;
    uint64_t wbase[UP ? PW : 1];
    if constexpr (!UP) wbase[0] = wexpert + (uint64_t)n0 * p.K;
#pragma unroll
    for (int j = 0; j < PW; j++) {
        const int first = piece_at(j);
        const int64_t from = UP ? weight_row(first) : n0;    // (a piece is of one tile: the first of its rows is the lowest)
        if constexpr (UP) wbase[j] = wexpert + (uint64_t)from * p.K;
        woff[j] = (uint32_t)(weight_row(first + piece_row) - from) * p.K + wchunk[first / 8 & 1];
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const uint32_t lds_x = lds0 + wave * PX * 1024, lds_w = lds0 + BM * XB;
    // x's scales of a block come the same way, BM / WAVES rows per wave (rows past the end: the last one's)
    constexpr int RS = BM / WAVES;
    const int sat = m0 + wave * RS + (lane < RS ? lane : 0), srow = sat < end ? sat : end - 1;
    const uint32_t soff = (uint32_t)(GATHER ? p.order[srow] / p.top_k : srow) * 4, lds_s = lds0 + S * BUFFER + wave * RS * 4;
    // Pieces of a block in the order in which a wave asks for them: x, its scales, weights.  They are asked for one at a time between the
    // products: all at once, from all waves, they queue at the CU's address unit and the waves stand still (8192^3: 553 us against 489).
    constexpr int PIECES = PX + 1 + PW;
    auto fetch = [&](int kb, int which, int q) __attribute__((always_inline)) {
        const uint32_t buffer = which * BUFFER;
        if (q < PX) {
            if constexpr (GATHER) dma16_at(xaddr[q] + (uint64_t)kb * XB, lds_x + buffer + q * 1024);
            else dma16(xoff[q], xbase + (uint64_t)kb * XB, lds_x + buffer + q * 1024);
        } else if (q == PX) {
            if (lane < RS) dma4(soff, (uint64_t)(uintptr_t)(p.xs + (int64_t)kb * p.ldxs), lds_s + which * SCALES);
        } else {
            // A row that ends inside the block: in place of the chunks past its end the block's first one.  x has zeros there, so it
            // counts nothing (a NaN among it is one of the row's own).
            const int j = q - PX - 1, left = p.K - kb * FP8_BLOCK;
            uint32_t off = woff[j];
            if (left < FP8_BLOCK) {
                const uint32_t chunk = wchunk[piece_at(j) / 8 & 1];
                off -= chunk < (uint32_t)left ? 0u : chunk;
            }
            dma16(off, wbase[UP ? j : 0] + (uint64_t)kb * FP8_BLOCK, lds_w + buffer + piece_at(j) * FP8_BLOCK);
        }
    };

    // ---- scales.  A weight's of up to 64 blocks lie in the lanes of one register
    const int nb0 = UP ? n0 / FP8_BLOCK : (n0 + wn * TN * 16) / FP8_BLOCK, NB = fp8_blocks(p.N);
    const float *const wscale = p.ws + ((BY_EXPERT ? (int64_t)expert * fp8_blocks(p.expert_rows) : 0) + (nb0 < NB ? nb0 : NB - 1)) * KB;
    const int64_t u_scale = UP ? (int64_t)(p.I / FP8_BLOCK) * KB : 0;
    float wheld[UP ? 2 : 1];
    auto hold = [&](int kb) __attribute__((always_inline)) {
        const int b = kb + lane < KB ? kb + lane : KB - 1;
        wheld[0] = wscale[b];
        if constexpr (UP) wheld[1] = wscale[u_scale + b];
        // (waited for here: a load that may be under way at the loop's head makes the compiler wait there for all, in every step)
        asm volatile("" : "+v"(wheld[0]));
        if constexpr (UP) asm volatile("" : "+v"(wheld[1]));
    };
    // ---- operands: lane (r, g) reads the chunks g and 4 + g of row r of a tile (EXACT: of x those of the same numbers, 2 g and 2 g + 1 and
    // eight on; its sixteen slots are turned by the row)
    const int wlo = BM * XB + (wn * TN * 16 + r) * FP8_BLOCK + (g ^ swizzle(r)) * 16;
    const int xlo = (wm * TM * 16 + r) * XB + ((EXACT ? 2 * g : g) ^ (EXACT ? r : swizzle(r))) * 16;
    auto read_x = [&](int buffer, int i, XOperand<EXACT> &o) __attribute__((always_inline)) {
        const uint8_t *const at = lds + buffer + i * 16 * XB;
        if constexpr (EXACT) {
#pragma unroll
            for (int c = 0; c < 4; c++) o.v[c] = *(const bf16x8 *)(at + (xlo ^ ((c & 1) * 16 + (c >> 1) * 128)));
        } else o.v = Codes{*(const u32x4 *)(at + xlo), *(const u32x4 *)(at + (xlo ^ 64))};
    };
    auto read_w = [&](int buffer, int i, Codes &o) __attribute__((always_inline)) {
        const uint8_t *const at = lds + buffer + i * 16 * FP8_BLOCK;
        o = Codes{*(const u32x4 *)(at + wlo), *(const u32x4 *)(at + (wlo ^ 64))};
    };

    // A step: TN tiles of TM products each.  A product is added while the next ones run, LAG instructions later; a tile's operands are read
    // one tile ahead.  The barrier that publishes the next block stands ahead of the last tile, whose operands are in registers: its
    // products cover the first reads of the next block (of x into the registers that they free), and the buffer that has been read is filled
    // again from there on.  The order is fixed: left alone the compiler issues all products first and spills them.
    //
    // A load takes about as long as a step of the largest tile, so it is asked for more than a step ahead.  Where there is room for two
    // buffers only, a second barrier stands in the middle: it frees x, which is in registers, and the first half of the weights, whose
    // next block but one is asked for there; the second half's at the other barrier.  Each has a step and a half to arrive.
    constexpr int COUNT = TN * TM, LAG = EXACT ? TM : COUNT - TM < 3 ? COUNT - TM : 3, PARTS = EXACT ? 4 : 1, EARLY = PIECES - (HALVES - 1) * PH, TURN = HALVES == 2 ? (TN / 2 - 1) * TM : -1;
    constexpr int IN_FLIGHT = HALVES == 2 ? PIECES : (S - 2) * PIECES;       // loads of this wave that a barrier leaves under way
    constexpr int SLOTS = COUNT / HALVES, PER = ((HALVES == 2 ? EARLY : PIECES) + SLOTS - 1) / SLOTS;       // pieces asked for per product
    static_assert(IN_FLIGHT < 64, "vmcnt has 6 bits");
    f32x4 acc[TN][TM] = {};
    XOperand<EXACT> b[TM];
    Codes a[2];
    bf16x8 wide[2];                                          // EXACT: the part in use and the next one
    constexpr int RING = EXACT ? 2 * TM : LAG + 1;
    f32x4 d[RING];
    float s[UP ? 2 : 1][TM], xs[TM];
    auto read_xs = [&](int which) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TM; i++) xs[i] = *(const float *)(lds + S * BUFFER + which * SCALES + ((wm * TM + i) * 16 + r) * 4);
    };
    auto scales = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < (UP ? 2 : 1); h++) {
            const float sw = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wheld[h]), (kb - b0) & 63));
#pragma unroll
            for (int i = 0; i < TM; i++) s[h][i] = KG == 1 || kb < b1 ? xs[i] * sw : 0.0f;
        }
    };
    auto add = [&](int o) __attribute__((always_inline)) {
        f32x4 &sum = acc[o / TM][o % TM];
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] = fmaf(s[UP ? o / TM / TH : 0][o % TM], d[o % RING][j], sum[j]);
        asm volatile("" : "+v"(sum));                        // (here, and not behind the barrier, where nothing covers them)
    };
    // pieces first .. last - 1 of a block, PER of them in slot 0, 1, ..
    auto fetch_slot = [&](int kb, int which, int first, int last, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int q = first + slot * PER; q < first + (slot + 1) * PER && q < last; q++) fetch(kb, which, q);
    };
    // part c of product (t, i); EXACT: the parts of a tile's products one after the other, the next part widened among the first of them
    auto product = [&](int t, int i, int c, const Codes &w, const Codes &then) __attribute__((always_inline)) {
        f32x4 &to = d[(t * TM + i) % RING];
        if constexpr (EXACT) {
            to = mfma16(wide[c & 1], b[i].v[c], c ? to : f32x4{});
            if (i == 0) wide[(c + 1) & 1] = c < 3 ? widen_part(w, c + 1) : widen_part(then, 0);
        } else to = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(joined(w), joined(b[i].v), f32x4{}, 0, 0, 0, 0, 0, 0);
    };
    auto meet = [&]() __attribute__((always_inline)) {       // what was asked for IN_FLIGHT pieces ago is there, and every wave's reads are done
        wait_loads_but<IN_FLIGHT>();
        wait_lds();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const int last = b1 - 1;                                 // (past it: this block again, whose products nobody adds)

    hold(b0);
    constexpr int AHEAD = S - 1;                             // whole blocks asked for ahead of the loop but for what slot 0 .. ask for
#pragma unroll
    for (int v = 0; v < AHEAD; v++)
#pragma unroll
        for (int q = 0; q < PIECES; q++) fetch(b0 + v < last ? b0 + v : last, v, q);
    if constexpr (HALVES == 2) {
#pragma unroll
        for (int q = 0; q < EARLY; q++) fetch(b0 + 1 < last ? b0 + 1 : last, 1, q);
        wait_loads_but<EARLY>();
    } else wait_loads_but<(S - 2) * PIECES>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int which = 0;
#pragma unroll
    for (int i = 0; i < TM; i++) read_x(0, i, b[i]);
    read_w(0, 0, a[0]);
    if constexpr (EXACT) wide[0] = widen_part(a[0], 0);
    read_xs(0);
#pragma unroll
    for (int i = 0; i < TM; i++) {                           // what the last tile of a step before this one would have asked for
        if constexpr (HALVES == 2) fetch_slot(b0 + 1 < last ? b0 + 1 : last, 1, EARLY, PIECES, i);
        else fetch_slot(b0 + S - 1 < last ? b0 + S - 1 : last, S - 1, 0, PIECES, i);
    }
    // A wave whose rows are all past the end loads its share and keeps the barriers: a tile of up to half its rows takes little more than half
    // the time, where an expert's last one would otherwise cost as much as a whole one.
    if (m0 + wm * TM * 16 >= end) {
        for (int kb = b0; kb < stop; kb++) {
            const int late = kb + S - 1 < last ? kb + S - 1 : last, next = kb + S < last ? kb + S : last, behind = which > 0 ? which - 1 : S - 1;
#pragma unroll
            for (int o = 0; o < COUNT - TM; o++) {
                if (o == TURN) meet();
                if constexpr (HALVES == 2) {
                    if (o < TURN) fetch_slot(late, behind, EARLY, PIECES, TM + o);
                    else fetch_slot(next, which, 0, EARLY, o - TURN);
                } else fetch_slot(late, behind, 0, PIECES, TM + o);
            }
            meet();
#pragma unroll
            for (int i = 0; i < TM; i++) {
                if constexpr (HALVES == 2) fetch_slot(next, which, EARLY, PIECES, i);
                else fetch_slot(next, which, 0, PIECES, i);
            }
            which = which + 1 < S ? which + 1 : 0;
        }
    } else
    for (int kb = b0;;) {
        const int buffer = which * BUFFER, then = which + 1 < S ? which + 1 : 0, other = then * BUFFER;
        const int late = kb + S - 1 < last ? kb + S - 1 : last, next = kb + S < last ? kb + S : last;
        const int behind = which > 0 ? which - 1 : S - 1;    // the buffer that the step before this one freed
        scales(kb);
#pragma unroll
        for (int t = 0; t < TN - 1; t++) {
            if (t * TM == TURN) meet();
            read_w(buffer, t + 1, a[(t + 1) & 1]);
#pragma unroll
            for (int c = 0; c < PARTS; c++)
#pragma unroll
                for (int i = 0; i < TM; i++) {
                    const int o = t * TM + i;
                    product(t, i, c, a[t & 1], a[(t + 1) & 1]);
                    if (c == PARTS / 4 && o >= LAG) add(o - LAG);
                    if (c == 0) {
                        if constexpr (HALVES == 2) {
                            if (o < TURN) fetch_slot(late, behind, EARLY, PIECES, TM + o);
                            else fetch_slot(next, which, 0, EARLY, o - TURN);
                        } else fetch_slot(late, behind, 0, PIECES, TM + o);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
        meet();
        read_w(other, 0, a[TN & 1]);
#pragma unroll
        for (int c = 0; c < PARTS; c++)
#pragma unroll
            for (int i = 0; i < TM; i++) {
                product(TN - 1, i, c, a[(TN - 1) & 1], a[TN & 1]);
                if (c == PARTS - 1) read_x(other, i, b[i]);
                if (c == PARTS / 4) add(COUNT - TM + i - LAG);
                if (c == 0) {
                    if constexpr (HALVES == 2) fetch_slot(next, which, EARLY, PIECES, i);
                    else fetch_slot(next, which, 0, PIECES, i);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        read_xs(then);
#pragma unroll
        for (int o = COUNT - LAG; o < COUNT; o++) add(o);
        if (++kb >= stop) break;
        if (((kb - b0) & 63) == 0) hold(kb);
        which = then;
    }
    wait_all_loads();
    __syncthreads();
    if constexpr (KG == 2) {
        f32x4 *const sums = (f32x4 *)(shared + OWN) + wave * TN * TM * 64 + lane;
        if (group == 1)
#pragma unroll
            for (int o = 0; o < COUNT; o++) sums[o * 64] = acc[o / TM][o % TM];
        __syncthreads();
        if (group == 1) return;
#pragma unroll
        for (int o = 0; o < COUNT; o++) acc[o / TM][o % TM] += sums[o * 64];
    }

    // ---- results: lane = row r of tile i, columns 4 g .. 4 g + 3 of tile t's sixteen
    if constexpr (UP) {
        float *const most = (float *)lds;                    // [WN][BM] largest magnitudes, as bits
        float h[TM][TH][4];
#pragma unroll
        for (int i = 0; i < TM; i++) {
            uint32_t m = 0;
#pragma unroll
            for (int t = 0; t < TH; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    h[i][t][j] = gate_act(acc[t][i][j], p.act) * acc[TH + t][i][j];
                    m = max_u32(m, magnitude(h[i][t][j]));
                }
            m = max_u32(m, (uint32_t)__shfl_xor((int)m, 16));
            m = max_u32(m, (uint32_t)__shfl_xor((int)m, 32));
            if (g == 0) most[wn * BM + (wm * TM + i) * 16 + r] = __builtin_bit_cast(float, m);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int row = (wm * TM + i) * 16 + r, m = m0 + row;
            uint32_t top = 0;
#pragma unroll
            for (int v = 0; v < WN; v++) top = max_u32(top, __builtin_bit_cast(uint32_t, most[v * BM + row]));
            const float s = block_scale(top), inv = __builtin_amdgcn_rcpf(s);
            uint32_t c[TH];
#pragma unroll
            for (int t = 0; t < TH; t++) c[t] = encode4(h[i][t][0] * inv, h[i][t][1] * inv, h[i][t][2] * inv, h[i][t][3] * inv);
            if (m >= end) continue;
            uint8_t *const to = (uint8_t *)p.y + (int64_t)m * p.I + n0 + wn * (TH * 16) + g * (TH * 4);
            if constexpr (TH == 4) *(u32x4 *)to = u32x4{c[0], c[1], c[2], c[3]};
            else if constexpr (TH == 2) *(u32x2 *)to = u32x2{c[0], c[1]};
            else *(uint32_t *)to = c[0];
            if (wn == 0 && g == 0) p.hs[(int64_t)(n0 / FP8_BLOCK) * p.ldhs + m] = s;
        }
    } else {
        const bool aligned = p.N % 8 == 0;
#pragma unroll
        for (int t = 0; t < TN; t += 2) {
            const int n = n0 + wn * TN * 16 + (t >> 1) * 32 + g * 8;
            float add[8] = {};
            if (MODE == TILED_PLAIN && p.bias) {
#pragma unroll
                for (int j = 0; j < 8; j++) add[j] = n + j < p.N ? (float)((const OT *)p.bias)[n + j] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const int m = m0 + (wm * TM + i) * 16 + r;
                if (m >= end) continue;
                if constexpr (MODE == TILED_PART) {
                    float *const to = p.part + ((int64_t)split * p.M + m) * p.pitch + n;
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (n + 4 * h < p.pitch) *(f32x4 *)(to + 4 * h) = acc[t + h][i];
                } else {
                    OT *const to = (OT *)p.y + (int64_t)m * p.N + n;
                    typedef OT out_v __attribute__((ext_vector_type(8)));
                    out_v o;
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = Stored<OT>::of(acc[t + j / 4][i][j & 3] + add[j]);
                    // (one store of 8 results also where rows of y start at odd places: value by value 5753 x 12291 x 3328 took 347 us)
                    if (aligned) {
                        if (n < p.N) *(out_v *)to = o;
                    } else if (n + 8 <= p.N) __builtin_memcpy(to, &o, sizeof(o));
                    else {
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (n + j < p.N) to[j] = o[j];
                    }
                }
            }
        }
    }
}

template <typename OT, bool EXACT, TiledMode MODE, bool BY_EXPERT, bool GATHER, int TM, int TN, int WM, int WN, int S, int MIN_WAVES, int KG = 1>
void launch_tiled(TiledArgs p, hipStream_t st) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
    if (!BY_EXPERT) p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = MODE == TILED_UP ? p.I / FP8_BLOCK : (p.N + BN - 1) / BN;
    if (MODE != TILED_PART) {
        p.splits = 1;
        p.split_blocks = p.KB;
    }
    const uint32_t units = (uint32_t)(p.tiles_m * p.tiles_n * p.splits);
    hipLaunchKernelGGL((block_fp8_tiled_kernel<OT, EXACT, MODE, BY_EXPERT, GATHER, TM, TN, WM, WN, S, MIN_WAVES, KG>), dim3((units + 7) / 8 * 8),
                       dim3(64 * WM * WN * KG), 0, st, p);
}

}  // namespace lowbit
