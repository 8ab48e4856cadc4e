// The experts of a mixture-of-experts block with weights and activations in e4m3, a scale for each block of 128 (block_fp8.h):
//     out_t = sum_j p_tj * (Q(act(g) u) down_e^T),  (g | u) = Q(x_t) gate_up_e^T,  e = ids_tj
//
// The first product's sums go through the bfloat16 MFMA, which is exact (block_fp8.h): what the fp8 instruction drops, 1e-5 and more of a sum, would put one
// of 3000 values of h on the other side of the border between two codes, 1.5e-3 of the result, more than its rounding to bfloat16 costs.
// While the experts' weights are what takes the time, that costs nothing.
//
// Few pairs: each pair streams its expert's weights, two launches, h between them in float32.  More: the pairs sorted by expert, and tiles of
// rows of one expert (block_fp8_gemm.h).  A tile of the first product owns 128 columns of h = act(g) u, which are one block of h's rows: it
// has every value that the block's scale depends on, so h leaves as codes.  h is never a 16-bit number, and neither is a pair's result.
// Bound by memory up to some 30 rows per expert (64 experts of [1408 x 2048], 300 tokens, six each: 554 MB in 137 us), by the first product's
// bfloat16 MFMAs beyond.
#include "block_fp8_tiled.h"
#include "expert_sort.h"

#include <math.h>

namespace lowbit {

void launch_moe_combine_f32(const float *y, const int32_t *pos, const void *weight, int w_dtype, void *out, int act_dtype, int tokens, int top_k,
                            int N, int pitch, hipStream_t st);
struct ExpertsArgs {
    const void *x;                                           // [tokens, H]
    const int64_t *ids;
    const uint8_t *gate_up, *down;
    const float *gate_up_scale, *down_scale;
    uint8_t *h;                                              // few pairs: float32 [pairs, I]; else codes [pairs, I], by sorted position
    int n_exp, top_k, H, I, act;
};

// Both chunks of a lane (block_fp8.h) of one block of a row; past the row's end the block's first chunk, which meets zeros of x
__device__ inline Codes load_chunks(const uint8_t *row, int kb, int g, int K) {
    const int left = K - kb * FP8_BLOCK;
    const uint8_t *const at = row + kb * FP8_BLOCK;
    return Codes{ld<u32x4, true>(at + (g * 16 < left ? g * 16 : 0)), ld<u32x4, true>(at + (64 + g * 16 < left ? 64 + g * 16 : 0))};
}

__device__ inline float lane_value(float held, int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), l));
}

// Codes and scales of a row that the two kernels below keep in LDS, and the blocks that fit: at most 64 for each of 8 waves
constexpr size_t ROW_LDS = 65536 - 4096, BLOCK_LDS = FP8_BLOCK + sizeof(float);
constexpr int MOST_BLOCKS = (int)(ROW_LDS / BLOCK_LDS);
static_assert(MOST_BLOCKS <= 8 * 64, "a wave's scales lie in the 64 lanes of a register");

// One pair's 16 columns of h per workgroup: 16 rows of the gate and 16 of u.  The blocks of K are dealt to the waves, STEPS of them in flight
// per wave, whose sums meet in LDS.  x is quantized by each workgroup; h leaves in float32, since its blocks are of 128 columns: with 128
// columns per workgroup six experts of [1408 x 2048] would keep 66 CUs busy.  Bound by memory: two experts of [14336 x 4096], 235 MB, in 45 us.
template <typename AT>
__global__ __launch_bounds__(512) void block_fp8_expert_token_up_kernel(const ExpertsArgs p) {
    constexpr int STEPS = 2, WAVES = 8, THREADS = 64 * WAVES, HELD = 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float sums[WAVES][2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.x * 16, pair = blockIdx.y, H = p.H, KB = fp8_blocks(H);
    const int64_t e = p.ids[pair];
    if (e < 0 || e >= p.n_exp) return;                       // (the second product skips the pair)

    // x is asked for ahead of the weights: loads return in order
    using V8 = typename Vec8<AT>::type;
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
    float held[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        row[t] = p.gate_up + (e * 2 * p.I + t * p.I + c0 + r) * H;
        // the scales of this wave's blocks in the lanes of a register (MOST_BLOCKS)
        const float *const ws = p.gate_up_scale + ((e * 2 + t) * (p.I / FP8_BLOCK) + c0 / FP8_BLOCK) * KB;
        held[t] = ws[wave + lane * WAVES < KB ? wave + lane * WAVES : KB - 1];
    }
    Codes wc[STEPS][2];
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int t = 0; t < 2; t++) wc[s][t] = load_chunks(row[t], wave + s * WAVES < KB ? wave + s * WAVES : KB - 1, g, H);
    __builtin_amdgcn_sched_barrier(0);

    float *const xs = (float *)(lds + KB * FP8_BLOCK);
    auto put = [&](int at, const V8 &v) __attribute__((always_inline)) { put8<AT>(v, lds + at * 8, xs + (at >> 4), (at & 15) == 0); };
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if ((int)threadIdx.x + i * THREADS < pieces) put(threadIdx.x + i * THREADS, first[i]);    // (the 16 lanes of a block are in or out together)
    for (int at = threadIdx.x + HELD * THREADS; at < pieces; at += THREADS) put(at, at * 8 < H ? x[at] : V8{});
    __syncthreads();

    f32x4 acc[2] = {};
    for (int i0 = 0; wave + i0 * WAVES < KB; i0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = wave + (i0 + s) * WAVES, in = kb < KB ? kb : KB - 1, next = kb + STEPS * WAVES;
            const uint8_t *const xr = lds + in * FP8_BLOCK + g * 16;     // (all 16 rows of the operand are the one)
            const Codes xc = {*(const u32x4 *)xr, *(const u32x4 *)(xr + 64)};
            const float sx = xs[in];                         // (past the last block: it again, not added)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f32x4 d = block_dot<true>(wc[s][t], xc);
                const float sc = sx * lane_value(held[t], i0 + s);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[t][j] = kb < KB ? fmaf(sc, d[j], acc[t][j]) : acc[t][j];
                if (next < KB) wc[s][t] = load_chunks(row[t], next, g, H);
            }
        }
    }
    if (r == 0)
#pragma unroll
        for (int t = 0; t < 2; t++) *(f32x4 *)&sums[wave][t][g * 4] = acc[t];
    __syncthreads();
    if (threadIdx.x >= 16) return;
    float v[2] = {};
#pragma unroll
    for (int w = 0; w < WAVES; w++)
#pragma unroll
        for (int t = 0; t < 2; t++) v[t] += sums[w][t][threadIdx.x];
    ((float *)p.h)[(int64_t)pair * p.I + c0 + threadIdx.x] = gate_act(v[0], p.act) * v[1];
}

// One token's 16 columns per workgroup, which quantizes h of all its pairs; their blocks are dealt to the waves, STEPS of them in flight per
// wave.  Bound by memory: two experts of [4096 x 14336], 117 MB, in 25 us.
template <typename AT, typename PT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void block_fp8_expert_down_token_kernel(const ExpertsArgs p, const PT *__restrict__ weight, AT *__restrict__ out) {
    constexpr int STEPS = 4, HELD = 4, THREADS = 64 * WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float sums[WAVES][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, token = blockIdx.y, I = p.I, IB = I / FP8_BLOCK, HB = fp8_blocks(p.H), top_k = p.top_k;
    // the pairs' experts (-1: none) and weights in the lanes of registers: top_k is 64 at most
    const int pair0 = token * top_k;
    int expert = -1;
    float route = 0.0f;
    if (lane < top_k) {
        const int64_t e = p.ids[pair0 + lane];
        expert = e >= 0 && e < p.n_exp ? (int)e : -1;
        route = (float)weight[pair0 + lane];
    }
    // h of the pairs, one row after the other (what a pair of no expert left there is not used)
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    const f32x8 *const h = (const f32x8 *)((const float *)p.h + (int64_t)pair0 * I);
    const int units = top_k * IB, pieces = units * 16;
    f32x8 first[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int at = threadIdx.x + i * THREADS;
        first[i] = at < pieces ? h[at] : f32x8{};
    }
    __builtin_amdgcn_sched_barrier(0);

    const uint64_t valid = __ballot(expert >= 0);
    // unit u: block u % IB of pair u / IB; a wave's are wave, wave + WAVES, ..
    float held;                                              // what their sums count, but for h's scale, in the lanes of a register (MOST_BLOCKS)
    {
        const int u = wave + lane * WAVES, j = u < units ? u / IB : 0, kb = u < units ? u - j * IB : 0;
        const int e = __shfl(expert, j);
        const float by = __shfl(route, j);
        held = u < units && e >= 0 ? p.down_scale[((int64_t)e * HB + n0 / FP8_BLOCK) * IB + kb] * by : 0.0f;
    }
    auto load = [&](int u, Codes &w) __attribute__((always_inline)) {
        const int j = u / IB, kb = u - j * IB;
        if (u < units && (valid >> j & 1))                   // (the same for the whole wave)
            w = load_chunks(p.down + ((int64_t)__builtin_amdgcn_readlane(expert, j) * p.H + n0 + r) * I, kb, g, I);
    };
    Codes wc[STEPS] = {};
#pragma unroll
    for (int s = 0; s < STEPS; s++) load(wave + s * WAVES, wc[s]);
    __builtin_amdgcn_sched_barrier(0);

    float *const hs = (float *)(lds + pieces * 8);
    auto put = [&](int at, const f32x8 &v) __attribute__((always_inline)) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) m = max_u32(m, magnitude(v[i]));
        const float s = block_scale(max_of_16(m)), inv = __builtin_amdgcn_rcpf(s);
        *(u32x2 *)(lds + at * 8) = u32x2{encode4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), encode4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
        if ((at & 15) == 0) hs[at >> 4] = s;
    };
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if ((int)threadIdx.x + i * THREADS < pieces) put(threadIdx.x + i * THREADS, first[i]);
    for (int at = threadIdx.x + HELD * THREADS; at < pieces; at += THREADS) put(at, h[at]);
    __syncthreads();

    f32x4 acc = {};
    for (int i0 = 0; wave + i0 * WAVES < units; i0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int u = wave + (i0 + s) * WAVES, in = u < units ? u : units - 1;
            const uint8_t *const xr = lds + in * FP8_BLOCK + g * 16;
            const f32x4 d = block_dot<false>(wc[s], Codes{*(const u32x4 *)xr, *(const u32x4 *)(xr + 64)});
            const float sc = hs[in] * lane_value(held, i0 + s);
            const bool counts = u < units && (valid >> (in / IB) & 1);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = counts ? fmaf(sc, d[j], acc[j]) : acc[j];
            load(u + STEPS * WAVES, wc[s]);
        }
    }
    if (r == 0) *(f32x4 *)&sums[wave][g * 4] = acc;
    __syncthreads();
    if (threadIdx.x >= 16) return;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) v += sums[w][threadIdx.x];
    out[(int64_t)token * p.H + n0 + threadIdx.x] = to_at<AT>(v);
}

// The rows of x in codes (as bfloat16 numbers, see EXACT) and scales, and the pairs' sort by expert or its first half, in one launch: the
// first workgroups quantize (32 blocks each); the rest place a pair for each wave, or one sorts them all, or as many as there are chunks count them for the launch
// that places them (expert_sort.h).
enum ExpertSort { SORT_EACH, SORT_ONE, SORT_CHUNKS };
static ExpertSort expert_sort(int64_t pairs, int n_exp) { return counted_by_each(pairs, n_exp) ? SORT_EACH : one_sorts(pairs, n_exp) ? SORT_ONE : SORT_CHUNKS; }

template <typename AT, ExpertSort SORT>
__global__ __launch_bounds__(256) void block_fp8_expert_rows_kernel(const AT *__restrict__ x, const int64_t *__restrict__ ids, uint8_t *__restrict__ codes,
                                                                    float *__restrict__ scale, int32_t *__restrict__ offsets, int32_t *__restrict__ order,
                                                                    int32_t *__restrict__ pos, int32_t *__restrict__ counts, int tokens, int pairs,
                                                                    int n_exp, int K, int KB, int quantizing, int chunk) {
    if ((int)blockIdx.x < quantizing) {
        const int64_t unit = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
        if (unit >= (int64_t)tokens * KB) return;
        const int row = (int)(unit / KB), kb = (int)(unit - (int64_t)row * KB), k = kb * FP8_BLOCK + (threadIdx.x & 7) * 16;
        float v[16] = {}, s;
        if (k < K) load16(x + (int64_t)row * K + k, v);
        store16<true>(codes + (int64_t)row * KB * (2 * FP8_BLOCK), k, quantize16<AT>(v, s));
        if ((threadIdx.x & 7) == 0) scale[(int64_t)kb * tokens + row] = s;
        return;
    }
    if constexpr (SORT == SORT_EACH) count_for_each(ids, offsets, order, pos, pairs, n_exp, blockIdx.x - quantizing);
    else if constexpr (SORT == SORT_ONE) sort_pairs(ids, offsets, order, pos, pairs, n_exp);
    else count_pairs(ids, counts, pairs, n_exp, chunk, blockIdx.x - quantizing);
}

// Few pairs: each streams its expert's weights, which costs as many reads as there are pairs; the codes of a row of x and those of a token's
// rows of h have to fit LDS.  Sorted by expert a weight is read once, by launches that take some 10 us more and leave a quarter of a round
// of the first product's tiles idle.  The estimate counts the experts that tokens routed evenly would meet, at 5.5 TB/s.  Pair by pair /
// sorted, us: 3 tokens through 2 of 8 of [14336 x 4096] 197 / 167, two tokens 134 / 148; 4 through 6 of 64 of [1408 x 2048] 44 / 45, 8 81 / 72;
// 8 through 8 of 128 of [768 x 2048] 61 / 66, 12 89 / 79; 4 through 8 of 256 of [2048 x 7168] 260 / 251, 16 1028 / 784.
static size_t token_up_lds(int H) { return fp8_blocks(H) * BLOCK_LDS; }
static size_t token_down_lds(int top_k, int I) { return (size_t)top_k * (I / FP8_BLOCK) * BLOCK_LDS; }
static bool direct(int tokens, int top_k, int n_exp, int H, int I) {
    if (fp8_blocks(H) > MOST_BLOCKS || (int64_t)top_k * (I / FP8_BLOCK) > MOST_BLOCKS) return false;
    if (tokens == 1) return true;
    if ((int64_t)tokens * top_k > n_exp) return false;
    const double expert_us = 3.0 * H * I / 5.5e6, met = n_exp * (1.0 - pow(1.0 - (double)top_k / n_exp, tokens));
    return (tokens * top_k - met) * expert_us <= 10.0 + 64.0 * 2 * FP8_BLOCK * H / 5.5e6;
}

// The forms of the two products.
//
// Both by estimated time, with the row tiles that tokens routed evenly would make: of m rows for an expert, with a deviation of sqrt(m), the
// sum of the chances that there are more than 0, R, 2 R .. of them.
//
// First: tiles of 64, 96 or 128 rows (waves of 32, 48 and 64 x 64), one to a CU.  Whole blocks at 64 / 96 / 128 rows, us: 8 experts of [14336 x
// 4096], 64 rows each in the mean 349 / 312 / 333, 96 rows 438 / 434 / 389, 150 551 / 503 / 545, 512 1611 / 1451 / 1392; 64 of [1408 x
// 2048], 28 rows 138 / 139 / 144, 84 246 / 206 / 220; 4 of [2304 x 640], 94 rows 28 / 31 / 32, 300 43 / 47 / 38.  Whole calls at 70 other
// sizes, 4 to 256 experts of [256 to 14336 x 512 to 8192], 16 to 8192 tokens: the pick is 0.3 % above the fastest of the three on average, 6 %
// at worst (96 rows for all 4 %, 16 %; 64 4 %, 25 %; 128 9 %, 29 %).
//
// Second: the dense forms (tiled_walk_us).  16 rows for each of 8 experts of [4096 x 14336] 323 us in tiles of 32 rows against 358 of 256,
// 512 rows 1582 / 1328; counting tiles this way and not as pairs / rows + experts / 2 took 80 rows from 342 to 320, 96 from 392 to 368.
static double expert_tiles(int pairs, int n_exp, int rows) {
    const double mean = (double)pairs / n_exp;
    const double spread = sqrt(2.0 * mean);
    const int sure = (int)fmax(0.0, (mean - 4.0 * spread) / rows);
    double tiles = 1.0 + sure;
    for (int k = sure + 1; k * (double)rows < mean + 4.0 * spread; k++) tiles += 0.5 * erfc((k * (double)rows - mean) / spread);
    return tiles * (pairs < n_exp ? pairs : n_exp);
}
static int up_rows(int pairs, int n_exp, int I) {
    static const struct {
        int rows;
        float step_us, alone_us;
    } forms[] = {{64, 1.23f, 1.05f}, {96, 1.6f, 1.3f}, {128, 2.0f, 1.6f}};
    int best = 0;
    double least = 0.0;
    for (const auto &f : forms) {
        const double rounds = expert_tiles(pairs, n_exp, f.rows) * (I / FP8_BLOCK) / 256.0, us = rounds <= 1.0 ? f.alone_us : rounds * f.step_us;
        if (!best || us < least) {
            least = us;
            best = f.rows;
        }
    }
    return best;
}
static int down_form(int pairs, int n_exp, int H, int I) {
    int best = TILED_32;
    float least = 0.0f;
    for (int form = 0; form < TILED_COUNT; form++) {
        const TiledForm &f = TILED_FORMS[form];
        if (f.groups > 1) continue;                          // (an expert's last tile, of few rows, would hold a CU for twice as many waves)
        const float us = tiled_walk_us(f.step_us, f.alone_us, f.per_cu, (int64_t)(expert_tiles(pairs, n_exp, f.rows) * ((H + f.cols - 1) / f.cols) + 0.5), I / FP8_BLOCK);
        if (form == 0 || us < least) {
            least = us;
            best = form;
        }
    }
    return best;
}

// Columns of the result that one launch of the second product and its sum over pairs take, with the pairs' results between them in float32: all
// of them up to a GiB, beyond that as many whole tiles as fit it.  A launch of a GiB has thousands of tiles, so that one more costs little:
// what is read again is h, pairs * I bytes.  16384 tokens through 8 of 128 of [1024 x 7168], four parts, 6.71 ms with 1.6 GB of workspace, 6.60
// with 4.2 in one.
constexpr int64_t EXPERTS_SUMS = (int64_t)1 << 30;
static int down_columns(int64_t pairs, int H) {
    const int64_t fit = EXPERTS_SUMS / ((int64_t)sizeof(float) * pairs) / 256 * 256;
    return (int)(fit >= H ? H : fit < 256 ? (H < 256 ? H : 256) : fit);
}

void block_fp8_experts_plan(int tokens, int top_k, int n_exp, int H, int I, int *plan4) {
    const int pairs = tokens * top_k;
    plan4[0] = plan4[1] = plan4[2] = plan4[3] = 0;
    if (direct(tokens, top_k, n_exp, H, I)) return;
    const TiledForm &down = TILED_FORMS[down_form(pairs, n_exp, down_columns(pairs, H), I)];
    plan4[0] = up_rows(pairs, n_exp, I);
    plan4[1] = down.rows;
    plan4[2] = down.cols;
    plan4[3] = expert_sort(pairs, n_exp) == SORT_CHUNKS;
}

struct ExpertsSpace {
    size_t h, hs, x, xs, offsets, order, pos, counts, y, bytes;
    int ldx, ldxs;
};
static ExpertsSpace experts_space(int tokens, int top_k, int n_exp, int H, int I) {
    const int64_t pairs = (int64_t)tokens * top_k;
    ExpertsSpace w{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    w.ldx = fp8_blocks(H) * FP8_BLOCK * 2;
    w.ldxs = tokens;
    const bool one_each = direct(tokens, top_k, n_exp, H, I);
    w.h = take((size_t)pairs * I * (one_each ? sizeof(float) : 1));
    if (!one_each) {
        w.hs = take((size_t)pairs * (I / FP8_BLOCK) * 4);
        w.x = take((size_t)tokens * w.ldx);
        w.xs = take((size_t)tokens * fp8_blocks(H) * 4);
        w.offsets = take((size_t)(n_exp + 1) * 4);
        w.order = take((size_t)pairs * 4);
        w.pos = take((size_t)pairs * 4);
        if (expert_sort(pairs, n_exp) == SORT_CHUNKS) w.counts = take((size_t)EXPERTS_CHUNKS * n_exp * 4);
        w.y = take((size_t)pairs * down_columns(pairs, H) * sizeof(float));        // (rounded once, when a token's are summed: 16 bits would cost its precision twice)
    }
    w.bytes = at;
    return w;
}
size_t block_fp8_experts_workspace_bytes(int tokens, int top_k, int n_exp, int H, int I) {
    return experts_space(tokens, top_k, n_exp, H, I).bytes;
}

// 16 waves where there are no more workgroups than CUs: two experts of [4096 x 14336] 26 us
static int down_token_waves(int tokens, int H) { return (int64_t)(H / 16) * tokens <= 256 ? 16 : 8; }

// waves of a workgroup of the second launch where each pair streams its weights; 0 where the pairs are sorted
int block_fp8_experts_waves(int tokens, int top_k, int n_exp, int H, int I) {
    return direct(tokens, top_k, n_exp, H, I) ? down_token_waves(tokens, H) : 0;
}

template <typename AT, typename PT> static void launch_down_token(const ExpertsArgs &p, const PT *weight, AT *out, int tokens, hipStream_t st) {
    const dim3 grid(p.H / 16, tokens);
    const size_t lds = token_down_lds(p.top_k, p.I);
    if (down_token_waves(tokens, p.H) == 16)
        hipLaunchKernelGGL((block_fp8_expert_down_token_kernel<AT, PT, 16>), grid, dim3(1024), lds, st, p, weight, out);
    else hipLaunchKernelGGL((block_fp8_expert_down_token_kernel<AT, PT, 8>), grid, dim3(512), lds, st, p, weight, out);
}

template <typename AT> static int launch_experts_t(ExpertsArgs p, const ExpertsSpace &at, uint8_t *ws, const void *weight, int w_dtype, void *out,
                                                   int act_dtype, int tokens, hipStream_t st) {
    const int pairs = tokens * p.top_k;
    const bool one_each = direct(tokens, p.top_k, p.n_exp, p.H, p.I);
    if (one_each) {
        hipLaunchKernelGGL((block_fp8_expert_token_up_kernel<AT>), dim3(p.I / 16, pairs), dim3(512), token_up_lds(p.H), st, p);
        if (w_dtype == DT_F32) launch_down_token(p, (const float *)weight, (AT *)out, tokens, st);
        else if (w_dtype == DT_F16) launch_down_token(p, (const _Float16 *)weight, (AT *)out, tokens, st);
        else launch_down_token(p, (const __bf16 *)weight, (AT *)out, tokens, st);
        return 0;
    }
    int32_t *const offsets = (int32_t *)(ws + at.offsets), *const order = (int32_t *)(ws + at.order), *const pos = (int32_t *)(ws + at.pos);
    const int KB = fp8_blocks(p.H);
    if (((int64_t)tokens * KB + 31) / 32 + pairs + p.n_exp > most_groups(256)) return -3;
    const int quantizing = (int)(((int64_t)tokens * KB + 31) / 32);
    int32_t *const counts = (int32_t *)(ws + at.counts);
    const AT *const x = (const AT *)p.x;
    float *const xs = (float *)(ws + at.xs);
    const ExpertSort sort = expert_sort(pairs, p.n_exp);
    if (sort == SORT_EACH)
        hipLaunchKernelGGL((block_fp8_expert_rows_kernel<AT, SORT_EACH>), dim3(quantizing + (pairs + p.n_exp + 4) / 4), dim3(256), 0, st, x, p.ids, ws + at.x,
                           xs, offsets, order, pos, nullptr, tokens, pairs, p.n_exp, p.H, KB, quantizing, 0);
    else if (sort == SORT_ONE)
        hipLaunchKernelGGL((block_fp8_expert_rows_kernel<AT, SORT_ONE>), dim3(quantizing + 1), dim3(256), sort_lds(p.n_exp), st, x, p.ids, ws + at.x,
                           xs, offsets, order, pos, nullptr, tokens, pairs, p.n_exp, p.H, KB, quantizing, 0);
    else {
        const int chunk = sort_chunk(pairs), chunks = (pairs + chunk - 1) / chunk;
        hipLaunchKernelGGL((block_fp8_expert_rows_kernel<AT, SORT_CHUNKS>), dim3(quantizing + chunks), dim3(256), (size_t)p.n_exp * 4, st, x, p.ids, ws + at.x,
                           xs, offsets, order, pos, counts, tokens, pairs, p.n_exp, p.H, KB, quantizing, chunk);
        launch_expert_place(p.ids, counts, offsets, order, pos, pairs, p.n_exp, st);
    }

    TiledArgs t{};
    t.offsets = offsets; t.order = order; t.n_exp = p.n_exp; t.top_k = p.top_k; t.M = pairs; t.I = p.I; t.act = p.act;
    TiledArgs u = t;
    u.x = ws + at.x; u.xs = (float *)(ws + at.xs); u.ldx = at.ldx; u.ldxs = at.ldxs;
    u.w = p.gate_up; u.ws = p.gate_up_scale; u.N = 2 * p.I; u.K = p.H; u.KB = KB;
    u.expert_rows = u.N;
    u.y = p.h; u.hs = (float *)(ws + at.hs); u.ldhs = pairs;
    TiledArgs d = t;
    d.x = p.h; d.xs = u.hs; d.ldx = p.I; d.ldxs = pairs;
    d.expert_rows = p.H; d.K = p.I; d.KB = p.I / FP8_BLOCK;
    d.y = ws + at.y;
    const int columns = down_columns(pairs, p.H);
    const int rows = up_rows(pairs, p.n_exp, p.I), form = down_form(pairs, p.n_exp, columns, p.I), used = pairs < p.n_exp ? pairs : p.n_exp;
    u.tiles_m = pairs / rows + used;           // at most
    d.tiles_m = pairs / TILED_FORMS[form].rows + used;
    if ((int64_t)u.tiles_m * (p.I / FP8_BLOCK) > most_groups(512) || (int64_t)d.tiles_m * ((p.H + 127) / 128) > most_groups(512)) return -3;
    if (rows == 64) launch_tiled<AT, true, TILED_UP, true, true, 2, 4, 2, 4, 3, 2>(u, st);
    else if (rows == 96) launch_tiled<AT, true, TILED_UP, true, true, 3, 4, 2, 4, 2, 2>(u, st);
    else launch_tiled<AT, true, TILED_UP, true, true, 4, 4, 2, 4, 2, 2>(u, st);
    for (int n = 0; n < p.H; n += columns) {                 // (n: a multiple of a block)
        d.N = p.H - n < columns ? p.H - n : columns;
        d.w = p.down + (int64_t)n * p.I;
        d.ws = p.down_scale + (int64_t)(n / FP8_BLOCK) * d.KB;
        launch_tiled_form<float, false, TILED_PLAIN, true>(d, form, st);
        launch_moe_combine_f32((const float *)(ws + at.y), pos, weight, w_dtype, (AT *)out + n, act_dtype, tokens, p.top_k, d.N, p.H, st);
    }
    return 0;
}

int launch_block_fp8_experts(const void *x, const int64_t *ids, const void *weight, int w_dtype, int tokens, int top_k, int n_exp,
                             const uint8_t *gate_up, const float *gate_up_scale, const uint8_t *down, const float *down_scale, void *workspace,
                             void *out, int act_dtype, int H, int I, int act, hipStream_t st) {
    const ExpertsSpace at = experts_space(tokens, top_k, n_exp, H, I);
    uint8_t *const ws = (uint8_t *)workspace;
    ExpertsArgs p{};
    p.x = x; p.ids = ids;
    p.gate_up = gate_up; p.down = down; p.gate_up_scale = gate_up_scale; p.down_scale = down_scale;
    p.h = ws + at.h;
    p.n_exp = n_exp; p.top_k = top_k; p.H = H; p.I = I; p.act = act;
    return act_dtype == DT_F16 ? launch_experts_t<_Float16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st)
                               : launch_experts_t<__bf16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st);
}

}  // namespace lowbit
