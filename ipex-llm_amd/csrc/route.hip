// Which experts a token is sent to, with which weights, and the gradients of both operands:
//     z[t, e] = sum_h x[t, h] R[e, h],  s = softmax(z[t, :]) or sigmoid(z[t, :])
//     ids[t, :]: the top_k largest z (s + bias where a bias is given), in descending order, ties to the lowest index, a NaN above all numbers
//     w[t, j] = factor * s[ids_j] (/ sum of the chosen s where renormalized)
//
// z, s and the sums are float64.  Operands are float16, bfloat16 or float32, whose products are exact in float64; v_mfma_f64_16x16x4 adds them.  A sum of H
// products is off by H * 2^-53 of the sum of their magnitudes at most: of experts whose logits (biased scores) are farther apart than that, of both, every call takes the same,
// whatever the order of its sums, which goes by how many tokens it holds.  An operand of it is one value a
// lane (row l & 15, k = l >> 4): a lane loads eight neighbours of its row, k = 8 (l >> 4) .. + 7 of 32, and eight instructions take one of
// them each, since the order of the terms is free as long as both operands agree.
//
// (Two waves per SIMD are asked for so that the sums stay in vector registers: left alone the compiler keeps them in accumulation registers and copies
// them back and forth in every turn of the loops below.)
//
// The first launch sums a part of H for 16 tokens by 16 TN experts per workgroup, the second one, a wave per token, adds the parts and chooses.  Small routers
// take one launch, a token per workgroup.
#include "row_int8.h"

#include <type_traits>

namespace lowbit {

typedef double f64x4 __attribute__((ext_vector_type(4)));

struct RouteArgs {
    const void *x, *r;                                       // [T, H], [E, H]
    double *part;                                            // [splits][T][E]
    int T, E, H, splits, chunks;                             // chunks of 32 of H per split
};

// Eight values of AT from memory as they are; zeros past the row's end
template <typename AT> struct Octet {
    typedef AT type __attribute__((ext_vector_type(8)));
};

template <typename AT, typename RT, int TN, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void route_logits_kernel(const RouteArgs p) {
    using X8 = typename Octet<AT>::type;
    using R8 = typename Octet<RT>::type;
    __shared__ double sums[WAVES - 1][64][TN * 4 + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int t0 = blockIdx.x * 16, e0 = blockIdx.y * 16 * TN, split = blockIdx.z;
    const int first = split * p.chunks, all = (p.H + 31) / 32, last = first + p.chunks < all ? first + p.chunks : all;
    const AT *const x = (const AT *)p.x + (int64_t)(t0 + r < p.T ? t0 + r : p.T - 1) * p.H;
    const RT *w[TN];
#pragma unroll
    for (int i = 0; i < TN; i++) w[i] = (const RT *)p.r + (int64_t)(e0 + i * 16 + r < p.E ? e0 + i * 16 + r : p.E - 1) * p.H;
    f64x4 acc[TN] = {};
    X8 xv;
    R8 wv[TN];
    auto load = [&](int c) __attribute__((always_inline)) {
        const int k = c * 32 + g * 8;
        const bool in = c < last && k < p.H;
        xv = in ? *(const X8 *)(x + k) : X8{};
#pragma unroll
        for (int i = 0; i < TN; i++) wv[i] = in ? *(const R8 *)(w[i] + k) : R8{};
    };
    load(first + wave);
    for (int c = first + wave; c < last; c += WAVES) {
        const X8 xc = xv;
        R8 wc[TN];
#pragma unroll
        for (int i = 0; i < TN; i++) wc[i] = wv[i];
        load(c + WAVES);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const double b = (double)(float)xc[j];
#pragma unroll
            for (int i = 0; i < TN; i++) acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)wc[i][j], b, acc[i], 0, 0, 0);
        }
    }
    if (wave > 0)
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) sums[wave - 1][lane][i * 4 + j] = acc[i][j];
    __syncthreads();
    if (wave > 0) return;
    for (int v = 0; v < WAVES - 1; v++)
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] += sums[v][lane][i * 4 + j];
    // lane (r, g): token r, experts g + 4 j of each sixteen
    if (t0 + r >= p.T) return;
    double *const to = p.part + ((int64_t)split * p.T + t0 + r) * p.E;
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int e = e0 + i * 16 + g + 4 * j;
            if (e < p.E) to[e] = acc[i][j];
        }
}

// ---- a wave's doubles
//
// (Maxima and sums over a wave by moves between lanes: by way of LDS the selection of 6 of 64 took 4.0 us for 500 tokens, so 3.4.)

template <int CTRL, int ROWS> __device__ inline double add_dpp(double v) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    return v + __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[0], CTRL, ROWS, 0xf, false),
                                                (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[1], CTRL, ROWS, 0xf, false)});
}
__device__ inline double from_lane(double v, int l) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)b[0], l), (uint32_t)__builtin_amdgcn_readlane((int)b[1], l)});
}
// the same in every lane: rows of 16, then the rows (max_of_wave)
__device__ inline double wave_sum(double v) {
    v = add_dpp<0x140, 0xf>(add_dpp<0x141, 0xf>(add_dpp<0x4E, 0xf>(add_dpp<0xB1, 0xf>(v))));
    return from_lane(add_dpp<0x143, 0xc>(add_dpp<0x142, 0xa>(v)), 63);
}
// Whole numbers in the order of the doubles: a NaN above all, the zeros alike, nothing at 0.
__device__ inline uint64_t ordered(double v) {
    if (v != v) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
// the largest over the wave, the same in every lane
__device__ inline uint64_t wave_max(uint64_t v) {
    const uint32_t hi = max_of_wave((uint32_t)(v >> 32)), lo = max_of_wave((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

struct ScoreArgs {
    const double *part;
    const float *bias;                                       // or null
    const float *grad;                                       // backward: [T, top_k]
    double *z;                                               // forward: [T, E] for the backward, or null; backward: those
    float *w, *dz;                                           // [T, top_k]; backward: [T, lde]
    int64_t *ids;
    int T, E, top_k, splits, lde;
    bool sigmoid, renormalize;
    float factor;
};

// Scores of a token's experts, lane + 64 i: softmax without its division, whose sum is returned, or sigmoid (1).  Lanes past E have scores of 0.
template <int NR> __device__ inline double scores(const double (&z)[NR], double (&s)[NR], int E, bool sigmoid, int lane) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < NR; i++) s[i] = lane + 64 * i < E ? 1.0 / (1.0 + exp(-z[i])) : 0.0;
        return 1.0;
    }
    uint64_t most = 0;
#pragma unroll
    for (int i = 0; i < NR; i++)
        if (lane + 64 * i < E) {
            const uint64_t o = ordered(z[i]);
            most = o > most ? o : most;
        }
    most = wave_max(most);
    const double top = most == ~0ull ? __builtin_nan("") : __builtin_bit_cast(double, most >> 63 ? most & ~(1ull << 63) : ~most);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NR; i++) {
        s[i] = lane + 64 * i < E ? exp(z[i] - top) : 0.0;
        sum += s[i];
    }
    return wave_sum(sum);
}

// The choice for token t by one wave, of logits z, lane + 64 i; NR * 64 experts at most.
template <int NR> __device__ __forceinline__ void choose(const ScoreArgs &p, int64_t t, const double (&z)[NR], int lane) {
    double s[NR];
    // (the scores of all only where the choice or the weights go by them)
    const bool of_chosen = p.renormalize && !p.bias;
    double sum = 1.0;
    if (!of_chosen) sum = scores<NR>(z, s, p.E, p.sigmoid, lane);
    uint64_t key[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int e = lane + 64 * i;
        key[i] = e < p.E ? ordered(p.bias ? s[i] / sum + (double)p.bias[e] : z[i]) : 0;
    }
    double chosen = 0.0, total = 0.0;                        // lane j: the score of choice j (of_chosen: z)
    int index = 0;
    for (int j = 0; j < p.top_k; j++) {
        uint64_t best = 0;
        double score = 0.0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < NR; i++)
            if (key[i] > best) {
                best = key[i];
                score = of_chosen ? z[i] : s[i];
                at = i;
            }
        const uint64_t most = wave_max(best);
        // the lowest index among equals: the largest of its complement
        const uint32_t e = 0xffffu - max_of_wave(best == most ? 0xffffu - (uint32_t)(lane + 64 * at) : 0u);
        const double c = from_lane(score, e & 63);
        if (lane == j) {
            chosen = c;
            index = (int)e;
        }
        total += c;
#pragma unroll
        for (int i = 0; i < NR; i++)
            if (lane + 64 * i == (int)e) key[i] = 0;
    }
    if (of_chosen) {                                         // (z of the first choice is the largest)
        chosen = p.sigmoid ? 1.0 / (1.0 + exp(-chosen)) : exp(chosen - from_lane(chosen, 0));
        total = wave_sum(lane < p.top_k ? chosen : 0.0);
    }
    if (lane < p.top_k) {
        p.w[t * p.top_k + lane] = (float)((double)p.factor * (chosen / (p.renormalize ? total : sum)));
        p.ids[t * p.top_k + lane] = index;
    }
}

// One token per wave.
template <int NR> __global__ __launch_bounds__(256) void route_select_kernel(const ScoreArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= p.T) return;
    double z[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int e = lane + 64 * i;
        z[i] = 0.0;
        if (e < p.E) {
            const double *const from = p.part + t * p.E + e;
            const int64_t stride = (int64_t)p.T * p.E;
            for (int v = 0; v < p.splits; v += 8) {          // (the parts on their way together, added in order)
                double part[8];
#pragma unroll
                for (int u = 0; u < 8; u++) part[u] = v + u < p.splits ? from[(v + u) * stride] : 0.0;
#pragma unroll
                for (int u = 0; u < 8; u++) z[i] += part[u];
            }
            if (p.z) p.z[t * p.E + e] = z[i];
        }
    }
    choose<NR>(p, t, z, lane);
}

// A token per workgroup, logits and choice in one launch, where a router is small: a wave sums ROWS rows of it at a time, eight apart, in float64, and the first
// wave chooses.  EIGHTS: pieces of 512 values on their way together.
constexpr int SMALL_EXPERTS = 64;
template <typename AT, typename RT, int ROWS> __global__ __launch_bounds__(512, 2) void route_small_kernel(const RouteArgs a, const ScoreArgs p) {
    using X8 = typename Octet<AT>::type;
    using R8 = typename Octet<RT>::type;
    constexpr int EIGHTS = sizeof(RT) == 4 && ROWS == 4 ? 2 : 4;
    __shared__ double logits[SMALL_EXPERTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = blockIdx.x;
    const AT *const x = (const AT *)a.x + t * a.H;
    for (int e0 = wave; e0 < a.E; e0 += 8 * ROWS) {
        double sum[ROWS] = {};
        const RT *rows[ROWS];                                // (past the last: it again, whose sum is not kept)
#pragma unroll
        for (int i = 0; i < ROWS; i++) rows[i] = (const RT *)a.r + (int64_t)(e0 + 8 * i < a.E ? e0 + 8 * i : a.E - 1) * a.H;
        for (int h = 0; h < a.H; h += 512 * EIGHTS) {
            X8 xv[EIGHTS];
            R8 wv[ROWS][EIGHTS];
#pragma unroll
            for (int u = 0; u < EIGHTS; u++) {
                const int k = h + u * 512 + lane * 8;
                const bool in = k < a.H;
                const X8 v = *(const X8 *)(x + (in ? k : 0));
                xv[u] = in ? v : X8{};
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    const R8 w = *(const R8 *)(rows[i] + (in ? k : 0));
                    wv[i][u] = in ? w : R8{};
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < EIGHTS; u++) {
                if (h + u * 512 >= a.H) break;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const double b = (double)(float)xv[u][j];
#pragma unroll
                    for (int i = 0; i < ROWS; i++) sum[i] = fma((double)(float)wv[i][u][j], b, sum[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++) sum[i] = wave_sum(sum[i]);
#pragma unroll
        for (int i = 0; i < ROWS; i++)
            if (lane == 0 && e0 + 8 * i < a.E) logits[e0 + 8 * i] = sum[i];
    }
    __syncthreads();
    if (wave > 0) return;
    const double z[1] = {lane < a.E ? logits[lane] : 0.0};
    if (p.z && lane < a.E) p.z[t * a.E + lane] = z[0];
    choose<1>(p, t, z, lane);
}

// Gradients of z for gradients of the weights.  c: the chosen scores, w = factor c / C (C their sum, or 1):
//     dc_j = factor (g_j - sum_i g_i c_i / C) / C  (or factor g_j),  dz = s (ds - sum ds s)  or  ds s (1 - s)
template <int NR> __global__ __launch_bounds__(256) void route_grad_kernel(const ScoreArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= p.T) return;
    double z[NR], s[NR], ds[NR] = {};
#pragma unroll
    for (int i = 0; i < NR; i++) z[i] = lane + 64 * i < p.E ? p.z[t * p.E + lane + 64 * i] : 0.0;
    const double sum = scores<NR>(z, s, p.E, p.sigmoid, lane);
#pragma unroll
    for (int i = 0; i < NR; i++) s[i] /= sum;
    const int id = lane < p.top_k ? (int)p.ids[t * p.top_k + lane] : 0;
    const double g = lane < p.top_k ? (double)p.grad[t * p.top_k + lane] * (double)p.factor : 0.0;
    double chosen = 0.0;                                     // lane j: the score of choice j
    for (int j = 0; j < p.top_k; j++) {
        const int e = __builtin_amdgcn_readlane(id, j);
        double own = 0.0;
#pragma unroll
        for (int i = 0; i < NR; i++)
            if (i == e >> 6) own = s[i];
        const double c = from_lane(own, e & 63);
        if (lane == j) chosen = c;
    }
    // (by c / C, which is 1 where one expert is chosen, whose gradient is zero)
    const double total = p.renormalize ? wave_sum(chosen) : 1.0, less = p.renormalize ? wave_sum(lane < p.top_k ? g * (chosen / total) : 0.0) : 0.0;
    const double mine = (g - less) / total;
    for (int j = 0; j < p.top_k; j++) {
        const int e = __builtin_amdgcn_readlane(id, j);
        const double d = from_lane(mine, j);
#pragma unroll
        for (int i = 0; i < NR; i++)
            if (lane + 64 * i == e) ds[i] = d;
    }
    double all = 0.0;
    if (!p.sigmoid) {
#pragma unroll
        for (int i = 0; i < NR; i++) all += ds[i] * s[i];
        all = wave_sum(all);
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int e = lane + 64 * i;
        if (e < p.lde) p.dz[t * p.lde + e] = e < p.E ? (float)(p.sigmoid ? ds[i] * s[i] * (1.0 - s[i]) : s[i] * (ds[i] - all)) : 0.0f;
    }
}

// ---- gradients of the operands: C[m, h] = sum_k A(m, k) B[k, h] in float32, on v_mfma_f32_16x16x4.
//
// A lane of B loads eight neighbours of a row, which are its column of eight tiles, so that a wave owns 128 columns and a lane stores
// eight neighbours of a row of C.  ACROSS: A(m, k) = dz[k, m], the gradient of the router, whose waves take the rows k in turn and add their
// sums in LDS, in order; else A(m, k) = dz[m, k], the gradient of x, whose waves take 128 columns each.  1000 tokens x 60 experts of 4096: both in one
// launch 19.7 us (alone 13.8 and 10.8, which loads a step ahead make 15.3 and 13.0), the splits' sum 3.5, the gradient of the logits 5.4; 2000 x 160 of 1024 24.6
// (17.7 and 18.5).
struct OuterArgs {
    const float *dz;                                         // [T, lde]
    const void *b;                                           // [K, H]
    void *c;                                                 // [M, H]
    float *part;                                             // ACROSS, several splits: [split][M][H]
    int M, K, H, lde, splits, steps;                         // steps of 16 rows k per split
    uint32_t groups_h, groups_m, groups;                     // workgroups along H, along M, in all
};

template <typename BT, typename CT, int TM, bool ACROSS>
__device__ __forceinline__ void route_outer(const OuterArgs &p, float *sums, uint32_t at) {
    using B8 = typename Octet<BT>::type;
    const int at_h = at % p.groups_h, at_m = at / p.groups_h % p.groups_m, split = at / p.groups_h / p.groups_m;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int h = (ACROSS ? at_h : at_h * 4 + wave) * 128 + r * 8, m0 = at_m * 16 * TM;
    const int all = (p.K + 15) / 16, first = ACROSS ? split * p.steps : 0, last = ACROSS && first + p.steps < all ? first + p.steps : all;
    const BT *const b = (const BT *)p.b + (h < p.H ? h : 0);
    f32x4 acc[TM][8] = {};
    for (int s = ACROSS ? first + wave : first; s < last; s += ACROSS ? 4 : 1) {
        const int k = s * 16 + g * 4;
        B8 bv[4];
        float a[TM][4];
#pragma unroll
        for (int j = 0; j < 4; j++) bv[j] = k + j < p.K ? *(const B8 *)(b + (int64_t)(k + j) * p.H) : B8{};
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int m = m0 + i * 16 + r;
            if constexpr (ACROSS) {
#pragma unroll
                for (int j = 0; j < 4; j++) a[i][j] = k + j < p.K && m < p.lde ? p.dz[(int64_t)(k + j) * p.lde + m] : 0.0f;
            } else {
                const f32x4 v = m < p.M ? *(const f32x4 *)(p.dz + (int64_t)m * p.lde + k) : f32x4{};
#pragma unroll
                for (int j = 0; j < 4; j++) a[i][j] = v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int c = 0; c < 8; c++) {
                const float bf = (float)bv[j][c];
#pragma unroll
                for (int i = 0; i < TM; i++) acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][j], bf, acc[i][c], 0, 0, 0);
            }
    }
    if constexpr (ACROSS) {
        for (int v = 1; v < 4; v++) {
            if (wave == v)
#pragma unroll
                for (int i = 0; i < TM; i++)
#pragma unroll
                    for (int c = 0; c < 8; c++)
#pragma unroll
                        for (int q = 0; q < 4; q++) sums[lane * (TM * 32 + 1) + (i * 8 + c) * 4 + q] = acc[i][c][q];
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int i = 0; i < TM; i++)
#pragma unroll
                    for (int c = 0; c < 8; c++)
#pragma unroll
                        for (int q = 0; q < 4; q++) acc[i][c][q] += sums[lane * (TM * 32 + 1) + (i * 8 + c) * 4 + q];
            __syncthreads();
        }
        if (wave > 0) return;
    }
    if (h >= p.H) return;
    // lane (r, g): rows 4 g + q of each sixteen
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int m = m0 + i * 16 + g * 4 + q;
            if (m >= p.M) continue;
            if (ACROSS && p.splits > 1) {
                float *const to = p.part + ((int64_t)split * p.M + m) * p.H + h;
#pragma unroll
                for (int v = 0; v < 2; v++) *(f32x4 *)(to + 4 * v) = f32x4{acc[i][4 * v][q], acc[i][4 * v + 1][q], acc[i][4 * v + 2][q], acc[i][4 * v + 3][q]};
            } else {
                typedef CT out8 __attribute__((ext_vector_type(8)));
                out8 o;
#pragma unroll
                for (int c = 0; c < 8; c++) o[c] = (CT)acc[i][c][q];
                *(out8 *)((CT *)p.c + (int64_t)m * p.H + h) = o;
            }
        }
}

// Both gradients in one launch, the router's workgroups first, which take longer; either may have none.
constexpr int OUTER_TM = 4, OUTER_X_TM = 2;
template <typename XT, typename RT> __global__ __launch_bounds__(256, 2) void route_outer_kernel(const OuterArgs of_router, const OuterArgs of_x) {
    __shared__ float sums[64 * (OUTER_TM * 32 + 1)];
    if (blockIdx.x < of_router.groups) route_outer<XT, RT, OUTER_TM, true>(of_router, sums, blockIdx.x);
    else route_outer<RT, XT, OUTER_X_TM, false>(of_x, sums, blockIdx.x - of_router.groups);
}

// the splits' sums in their order, rounded once; four values per thread
template <typename CT>
__global__ __launch_bounds__(256) void route_outer_reduce_kernel(const f32x4 *__restrict__ part, CT *__restrict__ c, int64_t quads, int splits) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= quads) return;
    f32x4 v = part[id];
    for (int s = 1; s < splits; s++) v += part[s * quads + id];
    typedef CT out4 __attribute__((ext_vector_type(4)));
    out4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = (CT)v[j];
    *(out4 *)(c + id * 4) = o;
}

// ---- launches

static int cdiv(int a, int b) { return (a + b - 1) / b; }

template <typename F> static void by_type(int dtype, F &&f) {
    if (dtype == DT_F16) f((_Float16 *)nullptr);
    else if (dtype == DT_BF16) f((__bf16 *)nullptr);
    else f((float *)nullptr);
}

// Columns of 16 experts per workgroup, and parts of H so that about a thousand workgroups run, four per CU; a part has a chunk for each of the four
// waves at least.  Two columns share a token's conversions and are taken once there are tokens enough: 500 tokens x 64 experts of 2048 take 5.7 us with
// one in 8 parts and 5.8 with two, 1000 x 60 of 4096 14.0 and 13.6, 4096 x 64 of 2048 24.1 and 23.4; with four columns they take 6.6, 14.8 and 24.8,
// and with 32 tokens by two columns 6.3, 15.4 and 26.3.  300 x 256 of 7168 takes 49 us in 512 workgroups and 32 in 1024.
struct RoutePlan {
    int tn, splits, chunks;
};
static RoutePlan route_plan(int T, int E, int H) {
    RoutePlan p;
    p.tn = E > 16 && T > 500 ? 2 : 1;
    const int tiles = cdiv(T, 16) * cdiv(E, 16 * p.tn), all = cdiv(H, 32);
    int splits = tiles < 1024 ? cdiv(1024, tiles) : 1;
    splits = splits > 16 ? 16 : splits;
    if (splits > all / 4) splits = all / 4 > 0 ? all / 4 : 1;
    p.chunks = cdiv(all, splits);
    p.splits = cdiv(all, p.chunks);
    return p;
}

// One launch where a workgroup has a token's logits in 2.5 us at most: 512 values of one, two or four rows for each of its waves take 0.17, 0.28 and 0.58, of
// which four in five are conversions to float64.  One token x 8 experts of 4096 4.6 us against 8.3 in two launches, 64 of 512 5.5 / 7.9, 64 of 1024 6.1 / 8.0, 64 of
// 2048 7.7 / 7.8; 1024 tokens x 8 of 1024 5.5 / 8.8, 4096 x 8 of 512 10.3 / 9.5.
static int small_rows(int E) { return E <= 8 ? 1 : E <= 16 ? 2 : 4; }
static bool route_small(int T, int E, int H) {
    if (E > SMALL_EXPERTS || T > 2048) return false;
    const int rows = small_rows(E);
    return cdiv(T, 512) * cdiv(E, 8 * rows) * cdiv(H, 512) * (rows == 1 ? 0.17f : rows == 2 ? 0.28f : 0.58f) <= 2.5f;
}

size_t route_workspace_bytes(int T, int E, int H) { return route_small(T, E, H) ? 0 : (size_t)route_plan(T, E, H).splits * T * E * sizeof(double); }

template <int NR> static void launch_scores(const ScoreArgs &p, bool backward, hipStream_t st) {
    const dim3 grid((p.T + 3) / 4);
    if (backward) hipLaunchKernelGGL((route_grad_kernel<NR>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((route_select_kernel<NR>), grid, dim3(256), 0, st, p);
}
static void launch_scores(const ScoreArgs &p, bool backward, hipStream_t st) {
    if (p.E <= 64) launch_scores<1>(p, backward, st);
    else if (p.E <= 128) launch_scores<2>(p, backward, st);
    else if (p.E <= 256) launch_scores<4>(p, backward, st);
    else if (p.E <= 512) launch_scores<8>(p, backward, st);
    else launch_scores<16>(p, backward, st);
}

// z: [T, E] for the backward, or null
int launch_route(const void *x, int x_dtype, const void *router, int r_dtype, const float *bias, int T, int E, int H, int top_k, bool sigmoid,
                 bool renormalize, float factor, float *w, int64_t *ids, double *z, void *space, hipStream_t st) {
    const ScoreArgs s = {(const double *)space, bias, nullptr, z, w, nullptr, ids, T, E, top_k, 0, 0, sigmoid, renormalize, factor};
    if (route_small(T, E, H)) {
        const RouteArgs a = {x, router, nullptr, T, E, H, 1, 0};
        by_type(x_dtype, [&](auto *xt) {
            by_type(r_dtype, [&](auto *rt) {
                using AT = typename std::remove_pointer<decltype(xt)>::type;
                using RT = typename std::remove_pointer<decltype(rt)>::type;
                const int rows = small_rows(E);
                if (rows == 1) hipLaunchKernelGGL((route_small_kernel<AT, RT, 1>), dim3(T), dim3(512), 0, st, a, s);
                else if (rows == 2) hipLaunchKernelGGL((route_small_kernel<AT, RT, 2>), dim3(T), dim3(512), 0, st, a, s);
                else hipLaunchKernelGGL((route_small_kernel<AT, RT, 4>), dim3(T), dim3(512), 0, st, a, s);
            });
        });
        return 0;
    }
    const RoutePlan plan = route_plan(T, E, H);
    const RouteArgs a = {x, router, (double *)space, T, E, H, plan.splits, plan.chunks};
    const dim3 grid(cdiv(T, 16), cdiv(E, 16 * plan.tn), plan.splits);
    by_type(x_dtype, [&](auto *xt) {
        by_type(r_dtype, [&](auto *rt) {
            using AT = typename std::remove_pointer<decltype(xt)>::type;
            using RT = typename std::remove_pointer<decltype(rt)>::type;
            if (plan.tn == 2) hipLaunchKernelGGL((route_logits_kernel<AT, RT, 2, 4>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((route_logits_kernel<AT, RT, 1, 4>), grid, dim3(256), 0, st, a);
        });
    });
    ScoreArgs parts = s;
    parts.splits = plan.splits;
    launch_scores(parts, false, st);
    return 0;
}

// Splits of T for the gradient of the router: at most 512 rows for each of a workgroup's four waves, so that a float32 sum rounds little, and a few
// hundred workgroups.
static int outer_steps(int T, int E, int H) {
    const int tiles = cdiv(H, 128) * cdiv(E, 16 * OUTER_TM), all = cdiv(T, 16);
    int splits = tiles < 512 ? 512 / tiles : 1;
    const int least = cdiv(all, 128);
    if (splits > cdiv(all, 8)) splits = cdiv(all, 8);
    return cdiv(all, splits < least ? least : splits);
}
static int router_columns(int E) { return cdiv(E, 16) * 16; }

struct RouteBackSpace {
    size_t part, bytes;
    int splits;
};
static RouteBackSpace route_back_space(int T, int E, int H) {
    RouteBackSpace s;
    s.part = ((size_t)T * router_columns(E) * sizeof(float) + 255) & ~(size_t)255;
    s.splits = cdiv(cdiv(T, 16), outer_steps(T, E, H));
    s.bytes = s.part + (s.splits > 1 ? (size_t)s.splits * E * H * sizeof(float) : 0);
    return s;
}
size_t route_backward_workspace_bytes(int T, int E, int H) { return route_back_space(T, E, H).bytes; }

// gx, gr: either may be null
int launch_route_backward(const float *grad, const double *z, const int64_t *ids, const void *x, int x_dtype, const void *router, int r_dtype, int T, int E,
                          int H, int top_k, bool sigmoid, bool renormalize, float factor, void *gx, void *gr, uint8_t *space, hipStream_t st) {
    const RouteBackSpace at = route_back_space(T, E, H);
    const int lde = router_columns(E);
    const ScoreArgs s = {nullptr, nullptr, grad, (double *)z, nullptr, (float *)space, (int64_t *)ids, T, E, top_k, 1, lde, sigmoid, renormalize, factor};
    launch_scores(s, true, st);
    OuterArgs r = {(const float *)space, x, gr, (float *)(space + at.part), E, T, H, lde, at.splits, outer_steps(T, E, H), (uint32_t)cdiv(H, 128),
                   (uint32_t)cdiv(E, 16 * OUTER_TM), 0};
    OuterArgs o = {(const float *)space, router, gx, nullptr, T, E, H, lde, 1, 0, (uint32_t)cdiv(H, 512), (uint32_t)cdiv(T, 16 * OUTER_X_TM), 0};
    const int64_t of_router = gr ? (int64_t)r.groups_h * r.groups_m * at.splits : 0, of_x = gx ? (int64_t)o.groups_h * o.groups_m : 0;
    if (of_router + of_x > most_groups(256)) return -3;
    if (of_router + of_x == 0) return 0;
    r.groups = (uint32_t)of_router;
    o.groups = (uint32_t)of_x;
    by_type(x_dtype, [&](auto *xt) {
        by_type(r_dtype, [&](auto *rt) {
            using XT = typename std::remove_pointer<decltype(xt)>::type;
            using RT = typename std::remove_pointer<decltype(rt)>::type;
            hipLaunchKernelGGL((route_outer_kernel<XT, RT>), dim3(r.groups + o.groups), dim3(256), 0, st, r, o);
            const int64_t quads = (int64_t)E * H / 4;
            if (gr && at.splits > 1)
                hipLaunchKernelGGL((route_outer_reduce_kernel<RT>), dim3((uint32_t)((quads + 255) / 256)), dim3(256), 0, st, (const f32x4 *)r.part, (RT *)gr, quads,
                                   at.splits);
        });
    });
    return 0;
}

}  // namespace lowbit
