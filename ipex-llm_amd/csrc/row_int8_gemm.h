// The tiled product of row_int8.h: codes of x and of the weight meet in LDS, 128 values of K at a time.
//
// A workgroup of WM x WN waves owns WM * TM * 16 rows of x by WN * TN * 16 weight rows.  A step's codes of both operands come by LDS-DMA
// into S buffers, asked for a step and a half ahead (two buffers) or S - 1 steps; a wave multiplies TM x TN results by two instructions
// each, on into the same 32-bit sums, and the two scales meet them once, at the end.
//
// LDS holds rows of 128 bytes, the 16-byte chunk c of row r at slot c ^ swizzle(r) (block_fp8_gemm.h).
//
// Large products are bound by the clock that their data's power leaves: 8192^3 395 us, 2780 TOP/s, at 2.0 GHz with MFMAs on 63 % of the cycles and no
// LDS conflict, the same launch on codes of zero 311, 3530 TOP/s.  Four waves of 128 x 128 results in instructions of 32 x 32 x 32, which read a third
// less from LDS, take 471 at 1.87 GHz.  [28672 x 8192] by 8192 rows 1400 to 1430 us, where the library's largest product reaches 2150 TOP/s.  Products of a few hundred
// rows are bound by the latency of a step and by how many CUs have a tile (row_int8_tiled.h).
#pragma once
#include "row_int8.h"
#include "lowbit_gemm.h"

namespace lowbit {

struct Int8Args {
    const uint8_t *x;                                        // codes, rows of ldx bytes: whole blocks, zeros past K
    const float *xs;
    const uint8_t *w;
    const float *ws;
    const void *bias;
    void *y;
    int32_t *part;                                           // sums of a split: [split][M][pitch]
    const int32_t *offsets, *order;                          // by expert: rows offsets[e] .. of the result; x row order[row] / top_k, or row
    int64_t ldx;
    int M, N, K, KB, pitch;
    int tiles_m, tiles_n, splits, split_blocks;
    int n_exp, top_k, I, act;                                // UP: I columns of h, float32 to y
    int expert_rows;                                         // by expert: weight rows from one expert's to the next's, N of which the launch takes
};

enum Int8Mode { INT8_PLAIN, INT8_PART, INT8_UP };

// Which tile a workgroup of a product grouped by expert works on: expert after expert, of each its columns in turn, of each column its row tiles of
// ROWS rows side by side: they share its weights, and all of an expert's tiles its rows, mostly in one XCD's L2.  Called by whole waves; false past the last.
struct ExpertUnit {
    int expert, first, end, column;                          // rows first .. end - 1 (end: the expert's, not the tile's)
};
template <int ROWS> __device__ inline bool find_expert_unit(const int32_t *__restrict__ offsets, int n_exp, int unit, int tiles_n, ExpertUnit &u) {
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < n_exp; e0 += 64) {
        const int e = e0 + lane, from = e < n_exp ? offsets[e] : 0, to = e < n_exp ? offsets[e + 1] : 0, own = (to - from + ROWS - 1) / ROWS;
        int upto = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(upto, d);
            if (lane >= d) upto += up;
        }
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (unit < all * tiles_n) {
            const int l = __builtin_ctzll(__ballot(upto * tiles_n > unit)), tiles = __builtin_amdgcn_readlane(own, l);
            const int at = unit - (__builtin_amdgcn_readlane(upto, l) - tiles) * tiles_n;
            u.expert = e0 + l;
            u.column = at / tiles;
            u.first = __builtin_amdgcn_readlane(from, l) + (at - u.column * tiles) * ROWS;
            u.end = __builtin_amdgcn_readlane(to, l);
            return true;
        }
        unit -= all * tiles_n;
    }
    return false;
}

// BY_EXPERT: row tiles of one expert each.  GATHER: x rows by order[].  S: buffers in LDS.  KG: groups of WM x WN waves, each with buffers of
// its own, that share a tile's blocks out among them and add their sums at the end.
template <typename OT, Int8Mode MODE, bool BY_EXPERT, bool GATHER, int TM, int TN, int WM, int WN, int S, int MIN_WAVES, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, MIN_WAVES) void row_int8_tiled_kernel(const Int8Args p) {
    constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
    constexpr int XP = BM / 8, WP = BN / 8, PX = XP / WAVES, PW = WP / WAVES;        // pieces of 8 rows
    constexpr bool UP = MODE == INT8_UP;
    constexpr int TH = TN / 2;                               // UP: a wave's tiles of the gate, and as many of u
    constexpr int UP_COLUMNS = BN / 2;
    // Two buffers: a step in two halves, each with a barrier (see the loop)
    constexpr int HALVES = S == 2 ? 2 : 1, PH = PW / HALVES;
    static_assert(KG == 1 || (MODE != INT8_UP && !BY_EXPERT && S * (BM + BN) * INT8_BLOCK >= TM * TN * WAVES * 1024), "room for a group's sums");
    static_assert(WP % (WAVES * HALVES) == 0 && XP % WAVES == 0 && PX > 0 && TN % 2 == 0 && (S > 2 || TN % 4 == 0 || TN == 2), "whole pieces per wave");
    constexpr uint32_t BUFFER = (BM + BN) * INT8_BLOCK, OWN = S * BUFFER;            // a group's
    __shared__ __attribute__((aligned(16))) uint8_t shared[KG * OWN];
    const int lane = threadIdx.x & 63, in_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int group = KG == 1 ? 0 : in_all / WAVES, wave = in_all - group * WAVES, wm = wave / WN, wn = wave % WN;
    uint8_t *const lds = shared + group * OWN;

    // Runs of tiles to the XCDs in turn, so that an L2 serves every operand several times (block_fp8_gemm.h).
    const int tiles_m = BY_EXPERT ? count_expert_tiles<BM>(p.offsets, p.n_exp) : p.tiles_m;
    const uint32_t units = (uint32_t)(tiles_m * p.tiles_n * p.splits), xcd = blockIdx.x & 7;
    const uint32_t unit = (uint32_t)((uint64_t)units * xcd >> 3) + (blockIdx.x >> 3);
    if (unit >= (uint32_t)((uint64_t)units * (xcd + 1) >> 3)) return;
    int m0, tn, end = p.M, expert = 0, split = 0;
    if constexpr (BY_EXPERT) {
        ExpertUnit u;
        if (!find_expert_unit<BM>(p.offsets, p.n_exp, (int)unit, p.tiles_n, u)) return;
        expert = __builtin_amdgcn_readfirstlane(u.expert);
        m0 = __builtin_amdgcn_readfirstlane(u.first);
        end = __builtin_amdgcn_readfirstlane(u.end);
        tn = __builtin_amdgcn_readfirstlane(u.column);
    } else {
        const int tile = (int)(unit / p.splits), per = 8 * p.tiles_n, band = tile / per, at = tile - band * per;
        const int rows = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
        split = (int)(unit - (uint32_t)tile * p.splits);
        tn = at / rows;
        m0 = (band * 8 + at - tn * rows) * BM;
    }
    const int n0 = tn * (UP ? UP_COLUMNS : BN), KB = p.KB;
    // blocks of K: of this split, and of this group (the first ones have them all; the last walks as far, over zeros of x)
    const int from = split * p.split_blocks, to = MODE == INT8_PART && from + p.split_blocks < KB ? from + p.split_blocks : KB;
    const int walk = (to - from + KG - 1) / KG, b0 = from + group * walk, stop = b0 + walk, b1 = stop < to ? stop : to;

    // ---- sources of this wave's pieces of 8 rows
    uint32_t xoff[GATHER ? 1 : PX], woff[PW];
    uint64_t xaddr[GATHER ? PX : 1];
    const int piece_row = lane >> 3;
    const uint64_t xbase = (uint64_t)(uintptr_t)p.x + (GATHER ? 0 : (uint64_t)m0 * p.ldx);
#pragma unroll
    for (int j = 0; j < PX; j++) {
        const int row = (wave * PX + j) * 8 + piece_row, chunk = ((lane & 7) ^ swizzle(row)) * 16;
        const int at = m0 + row < end ? m0 + row : end - 1;
        if constexpr (GATHER) xaddr[j] = xbase + (uint64_t)(p.order[at] / p.top_k) * p.ldx + chunk;
        else xoff[j] = (uint32_t)((at - m0) * p.ldx) + chunk;
    }
    const uint64_t wexpert = (uint64_t)(uintptr_t)p.w + (BY_EXPERT ? (uint64_t)expert * p.expert_rows * p.K : 0);
    // Which weight row lies in row `at` of LDS: a wave column's tiles of 16, each lane quarter's four rows of them neighbours of its
    // four in the next tile, so that a lane's results are neighbours in a row of y.  UP: tiles of the gate, then as many of u.
    auto weight_row = [&](int at) -> int64_t {
        const int col = at / (TN * 16), i = at / 16 % TN, q = at / 4 % 4, t = at % 4;
        if constexpr (UP) {
            const int c = n0 + col * (TH * 16) + q * (TH * 4) + i % TH * 4 + t;
            return (int64_t)(i / TH) * p.I + (c < p.I ? c : p.I - 1);
        }
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
        const int64_t at = UP ? weight_row(first) : n0;      // (a piece is of one tile: the first of its rows is the lowest)
        if constexpr (UP) wbase[j] = wexpert + (uint64_t)at * p.K;
        woff[j] = (uint32_t)(weight_row(first + piece_row) - at) * p.K + wchunk[first / 8 & 1];
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const uint32_t lds_x = lds0 + wave * PX * 1024, lds_w = lds0 + BM * INT8_BLOCK;
    // Pieces of a block in the order in which a wave asks for them, x first; one at a time between the products, since all at once, from
    // all waves, they queue at the CU's address unit.
    constexpr int PIECES = PX + PW;
    auto fetch = [&](int kb, int which, int q) __attribute__((always_inline)) {
        const uint32_t buffer = which * BUFFER;
        if (q < PX) {
            if constexpr (GATHER) dma16_at(xaddr[q] + (uint64_t)kb * INT8_BLOCK, lds_x + buffer + q * 1024);
            else dma16(xoff[q], xbase + (uint64_t)kb * INT8_BLOCK, lds_x + buffer + q * 1024);
        } else {
            // A row that ends inside the block: in place of the chunks past its end the block's first one.  x has zeros there.
            const int j = q - PX, left = p.K - kb * INT8_BLOCK;
            uint32_t off = woff[j];
            if (left < INT8_BLOCK) {
                const uint32_t chunk = wchunk[piece_at(j) / 8 & 1];
                off -= chunk < (uint32_t)left ? 0u : chunk;
            }
            dma16(off, wbase[UP ? j : 0] + (uint64_t)kb * INT8_BLOCK, lds_w + buffer + piece_at(j) * INT8_BLOCK);
        }
    };

    // ---- operands: lane (r, g) reads the chunks g and 4 + g of row r of a tile
    const int wlo = BM * INT8_BLOCK + (wn * TN * 16 + r) * INT8_BLOCK + (g ^ swizzle(r)) * 16;
    const int xlo = (wm * TM * 16 + r) * INT8_BLOCK + (g ^ swizzle(r)) * 16;
    // (dead: a block past this group's, whose products count nothing)
    auto read_x = [&](int buffer, int i, Codes &o, bool dead) __attribute__((always_inline)) {
        const uint8_t *const at = lds + buffer + i * 16 * INT8_BLOCK;
        o = Codes{*(const u32x4 *)(at + xlo), *(const u32x4 *)(at + (xlo ^ 64))};
        if (KG > 1 && dead) o = Codes{};
    };
    auto read_w = [&](int buffer, int i, Codes &o) __attribute__((always_inline)) {
        const uint8_t *const at = lds + buffer + i * 16 * INT8_BLOCK;
        o = Codes{*(const u32x4 *)(at + wlo), *(const u32x4 *)(at + (wlo ^ 64))};
    };

    // A step: TN tiles of TM products each, every product in two instructions TM apart, so that none waits for its own sum.  A tile's operands
    // are read one tile ahead.  The barrier that publishes the next block stands ahead of the last tile, whose operands are in registers: its
    // products cover the first reads of the next block (of x into the registers that they free), and the buffer that has been read is filled
    // again from there on.  The order is fixed: left alone the compiler issues all products first and spills them.
    //
    // A load takes about as long as a step of the largest tile, so it is asked for more than a step ahead.  Where there is room for two
    // buffers only, a second barrier stands in the middle: it frees x, which is in registers, and the first half of the weights, whose
    // next block but one is asked for there; the second half's at the other barrier.  Each has a step and a half to arrive.
    constexpr int COUNT = TN * TM, EARLY = PIECES - (HALVES - 1) * PH, TURN = HALVES == 2 ? (TN / 2 - 1) * TM : -1;
    constexpr int IN_FLIGHT = HALVES == 2 ? PIECES : (S - 2) * PIECES;       // loads of this wave that a barrier leaves under way
    constexpr int SLOTS = COUNT / HALVES, PER = ((HALVES == 2 ? EARLY : PIECES) + SLOTS - 1) / SLOTS;       // pieces asked for per product
    static_assert(IN_FLIGHT < 64, "vmcnt has 6 bits");
    i32x4 acc[TN][TM] = {};
    Codes b[TM], a[2];
    // pieces first .. last - 1 of a block, PER of them in slot 0, 1, ..
    auto fetch_slot = [&](int kb, int which, int first, int last, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int q = first + slot * PER; q < first + (slot + 1) * PER && q < last; q++) fetch(kb, which, q);
    };
    auto product = [&](int t, int i, int c) __attribute__((always_inline)) {
        const u32x4 &u = c ? a[t & 1].hi : a[t & 1].lo, &v = c ? b[i].hi : b[i].lo;
        acc[t][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, u), __builtin_bit_cast(i32x4, v), acc[t][i], 0, 0, 0);
    };
    auto meet = [&]() __attribute__((always_inline)) {       // what was asked for IN_FLIGHT pieces ago is there, and every wave's reads are done
        wait_loads_but<IN_FLIGHT>();
        wait_lds();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const int last = b1 - 1;                                 // (past it: this block again, whose products nobody adds)

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
    for (int i = 0; i < TM; i++) read_x(0, i, b[i], b0 >= b1);
    read_w(0, 0, a[0]);
#pragma unroll
    for (int i = 0; i < TM; i++) {                           // what the last tile of a step before this one would have asked for
        if constexpr (HALVES == 2) fetch_slot(b0 + 1 < last ? b0 + 1 : last, 1, EARLY, PIECES, i);
        else fetch_slot(b0 + S - 1 < last ? b0 + S - 1 : last, S - 1, 0, PIECES, i);
    }
    // A wave whose rows are all past the end loads its share and keeps the barriers.
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
    for (int kb = b0; kb < stop; kb++) {
        const int buffer = which * BUFFER, then = which + 1 < S ? which + 1 : 0, other = then * BUFFER;
        const int late = kb + S - 1 < last ? kb + S - 1 : last, next = kb + S < last ? kb + S : last;
        const int behind = which > 0 ? which - 1 : S - 1;    // the buffer that the step before this one freed
#pragma unroll
        for (int t = 0; t < TN - 1; t++) {
            if (t * TM == TURN) meet();
            read_w(buffer, t + 1, a[(t + 1) & 1]);
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int i = 0; i < TM; i++) {
                    const int o = t * TM + i;
                    product(t, i, c);
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
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int i = 0; i < TM; i++) {
                product(TN - 1, i, c);
                if (c == 1) read_x(other, i, b[i], kb + 1 >= b1);
                if (c == 0) {
                    if constexpr (HALVES == 2) fetch_slot(next, which, EARLY, PIECES, i);
                    else fetch_slot(next, which, 0, PIECES, i);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        which = then;
    }
    wait_all_loads();
    __syncthreads();
    if constexpr (KG > 1) {
        constexpr int NEXT = OWN / 16;
        i32x4 *const sums = (i32x4 *)shared + wave * TN * TM * 64 + lane;
        if (group > 0)
#pragma unroll
            for (int o = 0; o < COUNT; o++) sums[group * NEXT + o * 64] = acc[o / TM][o % TM];
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int v = 1; v < KG; v++)
#pragma unroll
            for (int o = 0; o < COUNT; o++) acc[o / TM][o % TM] += sums[v * NEXT + o * 64];
    }

    // ---- results: lane = row r of tile i, columns 4 g .. 4 g + 3 of tile t's sixteen
    float xs[TM];
    if constexpr (MODE != INT8_PART) {
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int m = m0 + (wm * TM + i) * 16 + r, at = m < end ? m : end - 1;
            xs[i] = p.xs[GATHER ? p.order[at] / p.top_k : at];
        }
    }
    if constexpr (UP) {
        const float *const ws = p.ws + (int64_t)expert * 2 * p.I;
        const int c0 = n0 + wn * (TH * 16) + g * (TH * 4);
#pragma unroll
        for (int t = 0; t < TH; t++) {
            const int c = c0 + t * 4;                        // (I is a multiple of 16: all four columns or none)
            if (c >= p.I) continue;
            const f32x4 sg = *(const f32x4 *)(ws + c), su = *(const f32x4 *)(ws + p.I + c);
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const int m = m0 + (wm * TM + i) * 16 + r;
                if (m >= end) continue;
                f32x4 h;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    h[j] = gate_act((float)acc[t][i][j] * xs[i] * sg[j], p.act) * ((float)acc[TH + t][i][j] * xs[i] * su[j]);
                *(f32x4 *)((float *)p.y + (int64_t)m * p.I + c) = h;
            }
        }
    } else {
        const bool aligned = p.N % 8 == 0;
        // the columns' scales and bias, all on their way together
        float by[TN / 2][8], add[TN / 2][8] = {};
        if constexpr (MODE == INT8_PLAIN) {
            const float *const ws = p.ws + (BY_EXPERT ? (int64_t)expert * p.expert_rows : 0);
            const int first = n0 + wn * TN * 16 + g * 8;
            if (n0 + BN <= p.N) {
#pragma unroll
                for (int t = 0; t < TN / 2; t++) __builtin_memcpy(by[t], ws + first + t * 32, sizeof(by[t]));
                if (p.bias) {
                    typedef OT v8 __attribute__((ext_vector_type(8)));
                    v8 given[TN / 2];
#pragma unroll
                    for (int t = 0; t < TN / 2; t++) __builtin_memcpy(&given[t], (const OT *)p.bias + first + t * 32, sizeof(v8));
#pragma unroll
                    for (int t = 0; t < TN / 2; t++)
#pragma unroll
                        for (int j = 0; j < 8; j++) add[t][j] = (float)given[t][j];
                }
            } else {
#pragma unroll
                for (int t = 0; t < TN / 2; t++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int n = first + t * 32 + j < p.N ? first + t * 32 + j : p.N - 1;
                        by[t][j] = ws[n];
                        if (p.bias) add[t][j] = (float)((const OT *)p.bias)[n];
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < TN; t += 2) {
            const int n = n0 + wn * TN * 16 + (t >> 1) * 32 + g * 8;
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const int m = m0 + (wm * TM + i) * 16 + r;
                if (m >= end) continue;
                if constexpr (MODE == INT8_PART) {
                    int32_t *const to = p.part + ((int64_t)split * p.M + m) * p.pitch + n;
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (n + 4 * h < p.pitch) *(i32x4 *)(to + 4 * h) = acc[t + h][i];
                } else {
                    OT *const to = (OT *)p.y + (int64_t)m * p.N + n;
                    typedef OT out_v __attribute__((ext_vector_type(8)));
                    out_v o;
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = Stored<OT>::of((float)acc[t + j / 4][i][j & 3] * xs[i] * by[t / 2][j] + add[t / 2][j]);
                    // (one store of 8 results also where rows of y start at odd places)
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

template <typename OT, Int8Mode MODE, bool BY_EXPERT, bool GATHER, int TM, int TN, int WM, int WN, int S, int MIN_WAVES, int KG = 1>
void launch_int8_tile(Int8Args p, hipStream_t st) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
    if (!BY_EXPERT) p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = MODE == INT8_UP ? (p.I + BN / 2 - 1) / (BN / 2) : (p.N + BN - 1) / BN;
    if (MODE != INT8_PART) {
        p.splits = 1;
        p.split_blocks = p.KB;
    }
    const uint32_t units = (uint32_t)(p.tiles_m * p.tiles_n * p.splits);
    hipLaunchKernelGGL((row_int8_tiled_kernel<OT, MODE, BY_EXPERT, GATHER, TM, TN, WM, WN, S, MIN_WAVES, KG>), dim3((units + 7) / 8 * 8),
                       dim3(64 * WM * WN * KG), 0, st, p);
}

}  // namespace lowbit
