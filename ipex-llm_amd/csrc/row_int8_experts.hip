// The experts of a mixture-of-experts block with weights and activations in int8, a scale for each row (row_int8.h):
//     out_t = sum_j p_tj * (Q(act(g) u) down_e^T),  (g | u) = Q(x_t) gate_up_e^T,  e = ids_tj
//
// Few pairs: each pair streams its expert's weights, two launches, h = act(g) u between them in float32.  More: the pairs sorted by expert, and tiles
// of rows of one expert (row_int8_gemm.h).  A row of h has one scale, which its last column may set, so h leaves the first product in float32 and
// a launch of its own makes codes of it.  h is never a 16-bit number, and neither is a pair's result.
#include "expert_sort.h"
#include "row_int8_tiled.h"

#include <math.h>

namespace lowbit {

void launch_moe_combine_f32(const float *y, const int32_t *pos, const void *weight, int w_dtype, void *out, int act_dtype, int tokens, int top_k,
                            int N, int pitch, hipStream_t st);

struct Int8Experts {
    const void *x;                                           // [tokens, H]
    const int64_t *ids;
    const uint8_t *gate_up, *down;
    const float *gate_up_scale, *down_scale;
    float *h;                                                // [pairs, I]: few pairs: by pair; else by sorted position
    uint32_t *most;                                          // few pairs: [pairs, I / 16] largest magnitudes of 16 columns of h each
    int n_exp, top_k, H, I, act;
};

// Both chunks of a lane (row_int8.h) of one block of a row; past the row's end the block's first chunk, which meets zeros of x
__device__ inline Codes load_block(const uint8_t *row, int kb, int g, int K) {
    const uint8_t *const at = row + kb * INT8_BLOCK;
    const int left = K - kb * INT8_BLOCK;
    return Codes{ld<u32x4, true>(at + (g * 16 < left ? g * 16 : 0)), ld<u32x4, true>(at + (64 + g * 16 < left ? 64 + g * 16 : 0))};
}

constexpr size_t TOKEN_LDS = 65536 - 4096;                   // codes of a row of x, or of h of all pairs of a token

// One pair's 16 columns of h per workgroup: 16 rows of the gate and 16 of u.  The blocks of K are dealt to the waves, STEPS of them in flight
// per wave, whose sums meet in LDS.  x is quantized by each workgroup.  Bound by memory: two experts of [14336 x 4096] 46.8 us, 5.0 TB/s (two steps in
// flight 51.5); rows of up to 2048 in four waves of two steps, one of [7168 x 512] 10.4 us against 16.2 in eight.
template <typename AT, int WAVES, int STEPS>
__global__ __launch_bounds__(64 * WAVES, 2) void row_int8_expert_token_up_kernel(const Int8Experts p) {
    constexpr int THREADS = 64 * WAVES, HELD = 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ int32_t sums[WAVES][2][16];
    __shared__ uint32_t part[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.x * 16, pair = blockIdx.y, H = p.H, KB = int8_blocks(H);
    const int64_t e = p.ids[pair];
    if (e < 0 || e >= p.n_exp) return;                       // (the second product skips the pair)

    // x is asked for ahead of the weights: loads return in order
    typedef AT V8 __attribute__((ext_vector_type(8)));
    const V8 *const x = (const V8 *)((const AT *)p.x + (int64_t)(pair / p.top_k) * H);
    const int pieces = KB * 16;
    V8 first[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int at = threadIdx.x + i * THREADS;
        first[i] = at * 8 < H ? x[at] : V8{};
    }
    __builtin_amdgcn_sched_barrier(0);

    const uint8_t *row[2];
#pragma unroll
    for (int t = 0; t < 2; t++) row[t] = p.gate_up + (e * 2 * p.I + t * p.I + c0 + r) * H;
    Codes wc[STEPS][2];
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int t = 0; t < 2; t++) wc[s][t] = load_block(row[t], wave + s * WAVES < KB ? wave + s * WAVES : KB - 1, g, H);
    __builtin_amdgcn_sched_barrier(0);

    uint32_t most = 0;
    auto look = [&](const V8 &v) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i++) most = max_u32(most, magnitude((float)v[i]));
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) look(first[i]);
    for (int at = threadIdx.x + HELD * THREADS; at * 8 < H; at += THREADS) look(x[at]);
    most = max_of_wave(most);
    if (lane == 0) part[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) most = max_u32(most, part[w]);
    const RowCoder code(most);
    auto put = [&](int at, const V8 &v) __attribute__((always_inline)) {
        float f[8];
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = (float)v[i];
        code(f, c);
        *(u32x2 *)(lds + at * 8) = u32x2{c[0], c[1]};
    };
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if ((int)threadIdx.x + i * THREADS < pieces) put(threadIdx.x + i * THREADS, first[i]);
    for (int at = threadIdx.x + HELD * THREADS; at < pieces; at += THREADS) put(at, at * 8 < H ? x[at] : V8{});
    __syncthreads();

    i32x4 acc[2] = {};
    for (int i0 = 0; wave + i0 * WAVES < KB; i0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = wave + (i0 + s) * WAVES, in = kb < KB ? kb : KB - 1, next = kb + STEPS * WAVES;
            const uint8_t *const xr = lds + in * INT8_BLOCK + g * 16;    // (all 16 rows of the operand are the one)
            Codes xc = {*(const u32x4 *)xr, *(const u32x4 *)(xr + 64)};
            if (kb >= KB) xc = Codes{};
#pragma unroll
            for (int t = 0; t < 2; t++) {
                acc[t] = int8_dot(wc[s][t], xc, acc[t]);
                if (next < KB) wc[s][t] = load_block(row[t], next, g, H);
            }
        }
    }
    if (r == 0)
#pragma unroll
        for (int t = 0; t < 2; t++) *(i32x4 *)&sums[wave][t][g * 4] = acc[t];
    __syncthreads();
    if (threadIdx.x >= 16) return;
    int32_t v[2] = {};
#pragma unroll
    for (int w = 0; w < WAVES; w++)
#pragma unroll
        for (int t = 0; t < 2; t++) v[t] += sums[w][t][threadIdx.x];
    const float xs = row_scale(most);
    const float *const ws = p.gate_up_scale + e * 2 * p.I + c0 + threadIdx.x;
    const float h = gate_act((float)v[0] * xs * ws[0], p.act) * ((float)v[1] * xs * ws[p.I]);
    p.h[(int64_t)pair * p.I + c0 + threadIdx.x] = h;
    const uint32_t top = max_of_16(magnitude(h));
    if (threadIdx.x == 0) p.most[(int64_t)pair * (p.I / 16) + blockIdx.x] = top;
}

// One token's 16 columns per workgroup, which quantizes h of all its pairs; their blocks are dealt to the waves, STEPS of them in flight per
// wave.  A wave's blocks of one pair are summed in whole numbers, then scaled into the sum over the pairs.  Two experts of [4096 x 14336] 28 us, 4.2
// TB/s: ahead of the first product 115 KB of h come from L2 and become codes; six or eight steps in flight make no difference.
template <typename AT, typename PT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void row_int8_expert_down_token_kernel(const Int8Experts p, const PT *__restrict__ weight, AT *__restrict__ out) {
    constexpr int STEPS = 4, HELD = 4, THREADS = 64 * WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float sums[WAVES][16];
    __shared__ uint32_t top[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, token = blockIdx.y, I = p.I, IB = int8_blocks(I), top_k = p.top_k;
    // the pairs' experts (-1: none) and weights in the lanes of registers: top_k is 64 at most
    const int pair0 = token * top_k;
    int expert = -1;
    float route = 0.0f;
    if (lane < top_k) {
        const int64_t e = p.ids[pair0 + lane];
        expert = e >= 0 && e < p.n_exp ? (int)e : -1;
        route = (float)weight[pair0 + lane];
    }
    // h of the pairs, rows of whole blocks in LDS (what a pair of no expert left there is not used)
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    const float *const h = p.h + (int64_t)pair0 * I;
    const int units = top_k * IB, pieces = units * 16;
    auto load_h = [&](int at) __attribute__((always_inline)) {
        const int j = at / (IB * 16), k = (at - j * IB * 16) * 8;
        return k < I ? *(const f32x8 *)(h + (int64_t)j * I + k) : f32x8{};
    };
    f32x8 first[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int at = threadIdx.x + i * THREADS;
        first[i] = at < pieces ? load_h(at) : f32x8{};
    }
    // the rows' largest magnitudes, a pair per wave
    for (int j = wave; j < top_k; j += WAVES) {
        uint32_t m = 0;
        const uint32_t *const most = p.most + (int64_t)(pair0 + j) * (I / 16);
        for (int i = lane; i < I / 16; i += 64) m = max_u32(m, most[i]);
        m = max_of_wave(m);
        if (lane == 0) top[j] = m;
    }
    __builtin_amdgcn_sched_barrier(0);

    const uint64_t valid = __ballot(expert >= 0);
    // unit u: block u % IB of pair u / IB; a wave's are a run of them, so that it changes the pair seldom
    const int per = (units + WAVES - 1) / WAVES, u0 = wave * per, u1 = u0 + per < units ? u0 + per : units;
    auto load = [&](int u, Codes &w) __attribute__((always_inline)) {
        const int j = u / IB, kb = u - j * IB;
        if (u < u1 && (valid >> j & 1))                      // (the same for the whole wave)
            w = load_block(p.down + ((int64_t)__builtin_amdgcn_readlane(expert, j) * p.H + n0 + r) * I, kb, g, I);
    };
    Codes wc[STEPS] = {};
#pragma unroll
    for (int s = 0; s < STEPS; s++) load(u0 + s, wc[s]);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();

    auto put = [&](int at, const f32x8 &v) __attribute__((always_inline)) {
        float f[8];
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = v[i];
        RowCoder{top[at / (IB * 16)]}(f, c);
        *(u32x2 *)(lds + at * 8) = u32x2{c[0], c[1]};
    };
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if ((int)threadIdx.x + i * THREADS < pieces) put(threadIdx.x + i * THREADS, first[i]);
    for (int at = threadIdx.x + HELD * THREADS; at < pieces; at += THREADS) put(at, load_h(at));
    __syncthreads();

    f32x4 acc = {};
    i32x4 sum = {};
    int pair = u0 / IB;
    auto close = [&](int j) __attribute__((always_inline)) {  // the whole sum of the wave's blocks of pair j
        if (valid >> j & 1) {
            const int e = __builtin_amdgcn_readlane(expert, j);
            const float by = row_scale(top[j]) * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, route), j));
            const f32x4 ws = *(const f32x4 *)(p.down_scale + (int64_t)e * p.H + n0 + g * 4);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf((float)sum[i] * ws[i], by, acc[i]);
        }
        sum = i32x4{};
    };
    for (int v0 = u0; v0 < u1; v0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int u = v0 + s;
            if (u >= u1) break;
            const int j = u / IB;
            if (j != pair) {
                close(pair);
                pair = j;
            }
            const uint8_t *const xr = lds + u * INT8_BLOCK + g * 16;
            if (valid >> j & 1) sum = int8_dot(wc[s], Codes{*(const u32x4 *)xr, *(const u32x4 *)(xr + 64)}, sum);
            load(u + STEPS, wc[s]);
        }
    }
    if (u0 < u1) close(pair);
    if (r == 0) *(f32x4 *)&sums[wave][g * 4] = acc;
    __syncthreads();
    if (threadIdx.x >= 16) return;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) v += sums[w][threadIdx.x];
    out[(int64_t)token * p.H + n0 + threadIdx.x] = Stored<AT>::of(v);
}

// The rows of x in codes and scales, a row per workgroup, and the pairs' sort by expert or its first half, in one launch (expert_sort.h).  The sort
// goes first: it takes the longest.
template <typename AT, bool PLACES>
__global__ __launch_bounds__(256) void row_int8_expert_rows_kernel(const AT *__restrict__ x, const int64_t *__restrict__ ids, uint8_t *__restrict__ codes,
                                                                   float *__restrict__ scale, int32_t *__restrict__ offsets, int32_t *__restrict__ order,
                                                                   int32_t *__restrict__ pos, int32_t *__restrict__ counts, int tokens, int pairs,
                                                                   int n_exp, int H, int ldc, int chunk, int sorting) {
    const int row = (int)blockIdx.x - sorting;
    if (row < 0) {
        if constexpr (PLACES) sort_pairs(ids, offsets, order, pos, pairs, n_exp);
        else count_pairs(ids, counts, pairs, n_exp, chunk, blockIdx.x);
        return;
    }
    const float s = quantize_row<AT, 4, 1>(x + (int64_t)row * H, codes + (int64_t)row * ldc, H, ldc, threadIdx.x);
    if (threadIdx.x == 0) scale[row] = s;
}

// Pair by pair or sorted, by estimated time in us, fitted to 110 sizes of 1 to 48 tokens; the pick is 0.3 % above the shorter way on average, 12 % at
// worst.  Pair by pair: the reads, as many as there are pairs; workgroups of the first launch; of the second, and the codes of h that each of its
// rounds makes.  Sorted: a weight is read once, of the experts that tokens routed evenly would meet.  The codes of a row of x and those of a
// token's rows of h have to fit LDS.  2 tokens through 2 of 8 of [14336 x 4096] 150 us pair by pair, 110 sorted, 4 through 6 of 64 of [1408 x 2048]
// 43 / 53, 8 81 / 79, 12 through 2 of 4 of [512 x 1024] 16 / 21.
static size_t token_up_lds(int H) { return (size_t)int8_blocks(H) * INT8_BLOCK; }
static size_t token_down_lds(int top_k, int I) { return (size_t)top_k * int8_blocks(I) * INT8_BLOCK; }
static bool direct(int tokens, int top_k, int n_exp, int H, int I) {
    if (token_up_lds(H) > TOKEN_LDS || token_down_lds(top_k, I) > TOKEN_LDS || (int64_t)tokens * top_k > 4096) return false;
    const double pairs = (double)tokens * top_k, expert = 3.0e-6 * H * I, met = n_exp * (1.0 - pow(1.0 - (double)top_k / n_exp, tokens));
    const double rounds = tokens * (double)H / (16 * 256);
    const double each = 6.6 + 0.08 * pairs * expert + 2.5 * pairs * I / (16 * 512) + 0.114 * rounds + 0.117 * top_k * int8_blocks(I) * fmax(1.0, rounds);
    return each <= 20.1 + 0.1815 * met * expert + 0.0006 * pairs;
}

// The forms of the two products, by estimated time, with the row tiles that tokens routed evenly would make: of m rows for an expert, with a deviation
// of sqrt(m), the sum of the chances that there are more than 0, R, 2 R .. of them.
static double expert_tiles(int pairs, int n_exp, int rows) {
    const double mean = (double)pairs / n_exp;
    const double spread = sqrt(2.0 * mean);
    const int sure = (int)fmax(0.0, (mean - 4.0 * spread) / rows);
    double tiles = 1.0 + sure;
    for (int k = sure + 1; k * (double)rows < mean + 4.0 * spread; k++) tiles += 0.5 * erfc((k * (double)rows - mean) / spread);
    return tiles * (pairs < n_exp ? pairs : n_exp);
}
//
// Both launches' times are fitted to 37 sizes, 4 to 4096 tokens through 1 to 8 of 4 to 160 experts, [256 to 14336 x 512 to 8192]: for each round of
// workgroups over the GPU what goes by the tile, and by its steps for each whole one.  The picks are 2.6 % and 2.7 % above the fastest of fourteen
// forms on average, 18 and 22 % at worst.  First product, us at 32 / 64 / 128 / 192 rows: 64 experts of [1408 x 2048], 47 rows each in the mean, 92 / 81 / 88 / 88, 8
// of [14336 x 4096], 8 rows 162 / 162 / 163 / 174, 128 rows 327 / 277 / 260 / 220, 500 rows 1011 / 782 / 634 / 514.
struct ExpertForm {
    int rows, cols, per_cu;                                  // cols: of weight rows, half of which are u's in the first product
    float tile_us, step_us;
};
enum { UP_32, UP_64, UP_128, UP_192 };
static const ExpertForm UP_FORMS[4] = {{32, 128, 2, 3.83f, 0.635f}, {64, 128, 3, 2.68f, 1.05f}, {128, 128, 2, 4.35f, 0.995f}, {192, 256, 1, 5.42f, 1.15f}};
enum { DOWN_64_64, DOWN_64, DOWN_128, DOWN_256 };
static const ExpertForm DOWN_FORMS[4] = {{64, 64, 2, 3.53f, 0.565f}, {64, 128, 3, 4.62f, 0.85f}, {128, 256, 1, 5.97f, 0.98f}, {256, 256, 1, 7.6f, 1.105f}};

static int expert_form(const ExpertForm (&forms)[4], int pairs, int n_exp, int N, int K) {
    int best = 0;
    float least = 0.0f;
    for (int i = 0; i < 4; i++) {
        const ExpertForm &f = forms[i];
        const float rounds = (float)expert_tiles(pairs, n_exp, f.rows) * ((N + f.cols - 1) / f.cols) / (256 * f.per_cu);
        const float us = (rounds > 1.0f ? rounds : 1.0f) * f.tile_us + ceilf(rounds) * f.step_us * int8_blocks(K);
        if (i == 0 || us < least) {
            least = us;
            best = i;
        }
    }
    return best;
}
static int up_form(int pairs, int n_exp, int H, int I) { return expert_form(UP_FORMS, pairs, n_exp, 2 * I, H); }
static int down_form(int pairs, int n_exp, int H, int I) { return expert_form(DOWN_FORMS, pairs, n_exp, H, I); }

// Tokens that go through the sorted launches together: as many as keep h, its codes and the pairs' results within 2 GiB.
constexpr int64_t EXPERTS_HELD = (int64_t)1 << 31;
static int tokens_at_once(int tokens, int top_k, int H, int I) {
    const int64_t fit = EXPERTS_HELD / ((int64_t)top_k * (5 * (int64_t)I + 4 * (int64_t)H));
    return (int)(fit >= tokens ? tokens : fit < 1 ? 1 : fit);
}

void row_int8_experts_plan(int tokens, int top_k, int n_exp, int H, int I, int *plan4) {
    plan4[0] = plan4[1] = plan4[2] = plan4[3] = 0;
    if (direct(tokens, top_k, n_exp, H, I)) return;
    const int pairs = tokens_at_once(tokens, top_k, H, I) * top_k;
    const ExpertForm &down = DOWN_FORMS[down_form(pairs, n_exp, H, I)];
    plan4[0] = UP_FORMS[up_form(pairs, n_exp, H, I)].rows;
    plan4[1] = down.rows;
    plan4[2] = down.cols;
    plan4[3] = !one_sorts(pairs, n_exp);
}

struct ExpertsSpace {
    size_t h, most, codes, hs, x, xs, offsets, order, pos, counts, y, bytes;
};
static ExpertsSpace experts_space(int tokens, int top_k, int n_exp, int H, int I) {
    const bool one_each = direct(tokens, top_k, n_exp, H, I);
    const int at_once = one_each ? tokens : tokens_at_once(tokens, top_k, H, I);
    const int64_t pairs = (int64_t)at_once * top_k;
    ExpertsSpace w{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    w.h = take((size_t)pairs * I * sizeof(float));
    if (one_each) w.most = take((size_t)pairs * (I / 16) * sizeof(uint32_t));
    else {
        w.codes = take((size_t)pairs * int8_blocks(I) * INT8_BLOCK);
        w.hs = take((size_t)pairs * 4);
        w.x = take((size_t)at_once * int8_blocks(H) * INT8_BLOCK);
        w.xs = take((size_t)at_once * 4);
        w.offsets = take((size_t)(n_exp + 1) * 4);
        w.order = take((size_t)pairs * 4);
        w.pos = take((size_t)pairs * 4);
        if (!one_sorts(pairs, n_exp)) w.counts = take((size_t)EXPERTS_CHUNKS * n_exp * 4);
        w.y = take((size_t)pairs * H * sizeof(float));       // (rounded once, when a token's are summed)
    }
    w.bytes = at;
    return w;
}
size_t row_int8_experts_workspace_bytes(int tokens, int top_k, int n_exp, int H, int I) { return experts_space(tokens, top_k, n_exp, H, I).bytes; }

// 16 waves where there are no more workgroups than CUs
static int down_token_waves(int tokens, int H) { return (int64_t)(H / 16) * tokens <= 256 ? 16 : 8; }

// waves of a workgroup of the second launch where each pair streams its weights; 0 where the pairs are sorted
int row_int8_experts_waves(int tokens, int top_k, int n_exp, int H, int I) {
    return direct(tokens, top_k, n_exp, H, I) ? down_token_waves(tokens, H) : 0;
}

template <typename AT, typename PT> static void launch_down_token(const Int8Experts &p, const PT *weight, AT *out, int tokens, hipStream_t st) {
    const dim3 grid(p.H / 16, tokens);
    const size_t lds = token_down_lds(p.top_k, p.I);
    if (down_token_waves(tokens, p.H) == 16)
        hipLaunchKernelGGL((row_int8_expert_down_token_kernel<AT, PT, 16>), grid, dim3(1024), lds, st, p, weight, out);
    else hipLaunchKernelGGL((row_int8_expert_down_token_kernel<AT, PT, 8>), grid, dim3(512), lds, st, p, weight, out);
}

// the sorted launches, for tokens that fit the workspace together
template <typename AT> static int launch_sorted(Int8Experts p, const ExpertsSpace &at, uint8_t *ws, const void *weight, int w_dtype, AT *out, int act_dtype,
                                                int tokens, hipStream_t st) {
    const int pairs = tokens * p.top_k, ldx = int8_blocks(p.H) * INT8_BLOCK, ldh = int8_blocks(p.I) * INT8_BLOCK;
    int32_t *const offsets = (int32_t *)(ws + at.offsets), *const order = (int32_t *)(ws + at.order), *const pos = (int32_t *)(ws + at.pos);
    int32_t *const counts = (int32_t *)(ws + at.counts);
    if ((int64_t)tokens + pairs + p.n_exp > most_groups(256)) return -3;
    const AT *const x = (const AT *)p.x;
    float *const xs = (float *)(ws + at.xs), *const hs = (float *)(ws + at.hs);
    if (one_sorts(pairs, p.n_exp))
        hipLaunchKernelGGL((row_int8_expert_rows_kernel<AT, true>), dim3(1 + tokens), dim3(256), sort_lds(p.n_exp), st, x, p.ids, ws + at.x, xs, offsets, order,
                           pos, nullptr, tokens, pairs, p.n_exp, p.H, ldx, 0, 1);
    else {
        const int chunk = sort_chunk(pairs), chunks = (pairs + chunk - 1) / chunk;
        hipLaunchKernelGGL((row_int8_expert_rows_kernel<AT, false>), dim3(chunks + tokens), dim3(256), (size_t)p.n_exp * 4, st, x, p.ids, ws + at.x, xs,
                           offsets, order, pos, counts, tokens, pairs, p.n_exp, p.H, ldx, chunk, chunks);
        launch_expert_place(p.ids, counts, offsets, order, pos, pairs, p.n_exp, st);
    }

    Int8Args t{};
    t.offsets = offsets; t.order = order; t.n_exp = p.n_exp; t.top_k = p.top_k; t.M = pairs; t.I = p.I; t.act = p.act;
    Int8Args u = t;
    u.x = ws + at.x; u.xs = xs; u.ldx = ldx;
    u.w = p.gate_up; u.ws = p.gate_up_scale; u.N = 2 * p.I; u.K = p.H; u.KB = int8_blocks(p.H);
    u.expert_rows = u.N;
    u.y = p.h;
    Int8Args d = t;
    d.x = ws + at.codes; d.xs = hs; d.ldx = ldh;
    d.w = p.down; d.ws = p.down_scale; d.N = p.H; d.K = p.I; d.KB = int8_blocks(p.I);
    d.expert_rows = p.H;
    d.y = ws + at.y;
    const int up = up_form(pairs, p.n_exp, p.H, p.I), down = down_form(pairs, p.n_exp, p.H, p.I), used = pairs < p.n_exp ? pairs : p.n_exp;
    u.tiles_m = pairs / UP_FORMS[up].rows + used;            // at most
    d.tiles_m = pairs / DOWN_FORMS[down].rows + used;
    if ((int64_t)u.tiles_m * ((p.I + 63) / 64) > most_groups(512) || (int64_t)d.tiles_m * ((p.H + 63) / 64) > most_groups(512)) return -3;
    if (up == UP_32) launch_int8_tile<float, INT8_UP, true, true, 2, 2, 1, 4, 4, 2>(u, st);
    else if (up == UP_64) launch_int8_tile<float, INT8_UP, true, true, 2, 4, 2, 2, 2, 2>(u, st);
    else if (up == UP_128) launch_int8_tile<float, INT8_UP, true, true, 4, 4, 2, 2, 2, 2>(u, st);
    else launch_int8_tile<float, INT8_UP, true, true, 6, 4, 2, 4, 2, 2>(u, st);
    if (int rc = launch_row_int8_quantize(p.h, DT_F32, pairs, p.I, ws + at.codes, ldh, hs, offsets + p.n_exp, st)) return rc;
    if (down == DOWN_64_64) launch_int8_tile<float, INT8_PLAIN, true, false, 2, 2, 2, 2, 4, 2>(d, st);
    else if (down == DOWN_64) launch_int8_tile<float, INT8_PLAIN, true, false, 2, 4, 2, 2, 2, 2>(d, st);
    else if (down == DOWN_128) launch_int8_tile<float, INT8_PLAIN, true, false, 4, 4, 2, 4, 3, 2>(d, st);
    else launch_int8_tile<float, INT8_PLAIN, true, false, 4, 8, 4, 2, 2, 2>(d, st);
    launch_moe_combine_f32((const float *)(ws + at.y), pos, weight, w_dtype, out, act_dtype, tokens, p.top_k, p.H, p.H, st);
    return 0;
}

template <typename AT> static int launch_experts_t(Int8Experts p, const ExpertsSpace &at, uint8_t *ws, const void *weight, int w_dtype, void *out,
                                                   int act_dtype, int tokens, hipStream_t st) {
    if (direct(tokens, p.top_k, p.n_exp, p.H, p.I)) {
        const dim3 grid(p.I / 16, tokens * p.top_k);
        if (int8_blocks(p.H) <= 16) hipLaunchKernelGGL((row_int8_expert_token_up_kernel<AT, 4, 2>), grid, dim3(256), token_up_lds(p.H), st, p);
        else hipLaunchKernelGGL((row_int8_expert_token_up_kernel<AT, 8, 4>), grid, dim3(512), token_up_lds(p.H), st, p);
        if (w_dtype == DT_F32) launch_down_token(p, (const float *)weight, (AT *)out, tokens, st);
        else if (w_dtype == DT_F16) launch_down_token(p, (const _Float16 *)weight, (AT *)out, tokens, st);
        else launch_down_token(p, (const __bf16 *)weight, (AT *)out, tokens, st);
        return 0;
    }
    const int step = tokens_at_once(tokens, p.top_k, p.H, p.I);
    for (int t = 0; t < tokens; t += step) {
        Int8Experts q = p;
        q.x = (const AT *)p.x + (int64_t)t * p.H;
        q.ids = p.ids + (int64_t)t * p.top_k;
        const void *const w = (const uint8_t *)weight + (int64_t)t * p.top_k * (w_dtype == DT_F32 ? 4 : 2);
        if (int rc = launch_sorted(q, at, ws, w, w_dtype, (AT *)out + (int64_t)t * p.H, act_dtype, tokens - t < step ? tokens - t : step, st)) return rc;
    }
    return 0;
}

int launch_row_int8_experts(const void *x, const int64_t *ids, const void *weight, int w_dtype, int tokens, int top_k, int n_exp,
                            const uint8_t *gate_up, const float *gate_up_scale, const uint8_t *down, const float *down_scale, void *workspace,
                            void *out, int act_dtype, int H, int I, int act, hipStream_t st) {
    const ExpertsSpace at = experts_space(tokens, top_k, n_exp, H, I);
    uint8_t *const ws = (uint8_t *)workspace;
    Int8Experts p{};
    p.x = x; p.ids = ids;
    p.gate_up = gate_up; p.down = down; p.gate_up_scale = gate_up_scale; p.down_scale = down_scale;
    p.h = (float *)(ws + at.h); p.most = (uint32_t *)(ws + at.most);
    p.n_exp = n_exp; p.top_k = top_k; p.H = H; p.I = I; p.act = act;
    if (act_dtype == DT_F16) return launch_experts_t<_Float16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st);
    if (act_dtype == DT_F32) return launch_experts_t<float>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st);
    return launch_experts_t<__bf16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st);
}

}  // namespace lowbit
