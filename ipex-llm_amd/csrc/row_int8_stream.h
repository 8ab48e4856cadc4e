// Some dozens of rows of codes times a weight with a scale for each row (row_int8.h), the weight streamed past once.
//
// A workgroup owns 16 weight rows and all rows of x, MT * 16 at most.  Its waves take the blocks of K in turn, both operands from memory
// straight to registers, DEPTH blocks in flight, and their whole sums meet in LDS: no barrier stands between a load and its use, which tiles pay for
// in every step.  Each workgroup reads all of x from L2, so that tiles overtake it as rows and weight rows grow: 16 rows on [4096 x 4096] 7.4 us
// against 8.9 in tiles, 4 on [512 x 4096] 5.6 / 7.4; 16 on [11008 x 4096] 15.4 / 12.5, 64 on [4096 x 4096] 12.7 / 10.2.
#pragma once
#include "row_int8_tiled.h"

namespace lowbit {

constexpr int STREAM_ROWS = 32;

// PART: the sums of split blockIdx.y's blocks of K.
template <typename OT, bool PART, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void row_int8_stream_kernel(const Int8Args p) {
    constexpr int DEPTH = 4;
    __shared__ int32_t sums[WAVES][MT][64 * 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, K = p.K, b0 = PART ? blockIdx.y * p.split_blocks : 0, KB = PART && b0 + p.split_blocks < p.KB ? b0 + p.split_blocks : p.KB;
    const uint8_t *const wrow = p.w + (int64_t)(n0 + r < p.N ? n0 + r : p.N - 1) * K;
    const uint8_t *xrow[MT];
    // (rows past M: the last one, whose results are not stored)
#pragma unroll
    for (int i = 0; i < MT; i++) xrow[i] = (const uint8_t *)p.x + (int64_t)(i * 16 + r < p.M ? i * 16 + r : p.M - 1) * p.ldx + g * 16;
    Codes w[DEPTH], x[DEPTH][MT];
    auto load = [&](int kb, Codes &wc, Codes (&xc)[MT]) __attribute__((always_inline)) {
        const int left = K - kb * INT8_BLOCK;
        // (chunks past the row's end: the block's first one, which meets zeros of x)
        const uint8_t *const at = wrow + kb * INT8_BLOCK;
        wc = Codes{ld<u32x4, true>(at + (g * 16 < left ? g * 16 : 0)), ld<u32x4, true>(at + (64 + g * 16 < left ? 64 + g * 16 : 0))};
#pragma unroll
        for (int i = 0; i < MT; i++) xc[i] = Codes{*(const u32x4 *)(xrow[i] + kb * INT8_BLOCK), *(const u32x4 *)(xrow[i] + kb * INT8_BLOCK + 64)};
    };
    i32x4 acc[MT] = {};
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (b0 + wave + d * WAVES < KB) load(b0 + wave + d * WAVES, w[d], x[d]);
    for (int i0 = 0; b0 + wave + i0 * WAVES < KB; i0 += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int kb = b0 + wave + (i0 + d) * WAVES, next = kb + DEPTH * WAVES;
            if (kb >= KB) break;                             // (the same for the whole wave)
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i] = int8_dot(w[d], x[d][i], acc[i]);
            if (next < KB) load(next, w[d], x[d]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) *(i32x4 *)&sums[wave][i][lane * 4] = acc[i];
    __syncthreads();
    // thread: row m of x, four columns
    for (int q = threadIdx.x; q < MT * 64; q += 64 * WAVES) {
        const int tile = q >> 6, l = q & 63, m = tile * 16 + (l & 15), n = n0 + (l >> 4) * 4;
        if (m >= p.M) continue;
        i32x4 sum = {};
#pragma unroll
        for (int v = 0; v < WAVES; v++) sum += *(const i32x4 *)&sums[v][tile][l * 4];
        if constexpr (PART) {
            if (n < p.pitch) *(i32x4 *)(p.part + ((int64_t)blockIdx.y * p.M + m) * p.pitch + n) = sum;
            continue;
        }
        const float xs = p.xs[m];
        OT *const y = (OT *)p.y + (int64_t)m * p.N + n;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n + j < p.N) y[j] = Stored<OT>::of((float)sum[j] * xs * p.ws[n + j] + (p.bias ? (float)((const OT *)p.bias)[n + j] : 0.0f));
    }
}

}  // namespace lowbit
