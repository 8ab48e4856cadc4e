// The experts of a mixture-of-experts block with weights and activations in e4m3, a scale for each block of 128 (block_fp8.h):
//     out_t = sum_j p_tj * (Q(act(g) u) down_e^T),  (g | u) = Q(x_t) gate_up_e^T,  e = ids_tj
//
// A workgroup of the first product owns 128 columns of h = act(g) u, which are one block of h's rows: it has every value that the
// block's scale depends on, so h leaves as codes and never as 16-bit numbers.
//
// The first product's sums go through the bfloat16 MFMA, which is exact (block_fp8.h): what the fp8 instruction drops, 1e-5 of a sum, would put one
// of 3000 values of h on the other side of the border between two codes, 1.5e-3 of the result, more than its rounding to bfloat16 costs.
// While the experts' weights are what takes the time, that costs nothing.
//
// Few pairs: each pair streams its expert's weights, two launches.  More: the pairs sorted by expert, and tiles of rows of one expert
// (block_fp8_gemm.h).
#include "block_fp8_tiled.h"

namespace lowbit {

void launch_moe_route(const int64_t *ids, int pairs, int n_exp, int32_t *offsets, int32_t *order, int32_t *pos, hipStream_t st);
void launch_moe_combine(const void *y, const int32_t *pos, const void *weight, int w_dtype, void *out, int act_dtype, int tokens, int top_k,
                        int N, hipStream_t st);
struct ExpertsArgs {
    const void *x;                                           // [tokens, H]
    const int64_t *ids;
    const uint8_t *gate_up, *down;
    const float *gate_up_scale, *down_scale;
    uint8_t *h;                                              // codes [pairs, I], by pair (few pairs) or by sorted position
    float *hs;                                               // [blocks of I][ldh]
    int ldh;
    int n_exp, top_k, H, I, act;
};

__device__ inline void load_chunks(const uint8_t *row, int kb, int left, Codes &c) {
    c = Codes{};
    if (left > 0) c.lo = ld<u32x4, true>(row + kb * FP8_BLOCK);
    if (left > 64) c.hi = ld<u32x4, true>(row + kb * FP8_BLOCK + 64);
}

// Wave w: 16 columns of g and the same of u, all of K.
template <typename AT>
__global__ __launch_bounds__(512) void block_fp8_expert_token_up_kernel(const ExpertsArgs p) {
    constexpr int STEPS = 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ uint32_t part[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int cb = blockIdx.x, KB = fp8_blocks(p.H);
    const int pair = blockIdx.y;
    const int64_t e = p.ids[pair];
    if (e < 0 || e >= p.n_exp) return;                       // (the second product skips the pair)
    const int expert = (int)e;
    const uint8_t *const w = p.gate_up + (int64_t)expert * 2 * p.I * p.H;
    const uint8_t *row[2];
    const float *ws[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        row[t] = w + (int64_t)(t * p.I + cb * FP8_BLOCK + wave * 16 + r) * p.H + g * 16;
        ws[t] = p.gate_up_scale + ((int64_t)expert * 2 * (p.I / FP8_BLOCK) + t * (p.I / FP8_BLOCK) + cb) * KB;
    }
    Codes wc[STEPS][2];
#pragma unroll
    for (int s = 0; s < STEPS; s++)
        if (s < KB)
#pragma unroll
            for (int t = 0; t < 2; t++) load_chunks(row[t], s, p.H - s * FP8_BLOCK - g * 16, wc[s][t]);

    float *const xs = (float *)(lds + KB * FP8_BLOCK);
    for (int kb = threadIdx.x >> 3; kb < KB; kb += 64) {
        const int k = kb * FP8_BLOCK + (threadIdx.x & 7) * 16;
        float v[16] = {}, s;
        if (k < p.H) load16((const AT *)p.x + (int64_t)(pair / p.top_k) * p.H + k, v);
        *(u32x4 *)(lds + k) = quantize16<AT>(v, s);
        if ((threadIdx.x & 7) == 0) xs[kb] = s;
    }
    __syncthreads();

    f32x4 acc[2] = {};
    for (int kb0 = 0; kb0 < KB; kb0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = kb0 + s;
            if (kb >= KB) break;
            const uint8_t *const xr = lds + kb * FP8_BLOCK + g * 16;     // (all 16 rows of the operand are the one)
            const Codes xc = {*(const u32x4 *)xr, *(const u32x4 *)(xr + 64)};
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const float sc = xs[kb] * ws[t][kb];
                const f32x4 d = block_dot<true>(wc[s][t], xc);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[t][j] = fmaf(sc, d[j], acc[t][j]);
            }
            if (kb + STEPS < KB)
#pragma unroll
                for (int t = 0; t < 2; t++) load_chunks(row[t], kb + STEPS, p.H - (kb + STEPS) * FP8_BLOCK - g * 16, wc[s][t]);
        }
    }

    float h[4];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        h[j] = gate_act(acc[0][j], p.act) * acc[1][j];
        m = max_u32(m, magnitude(h[j]));
    }
    m = max_u32(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max_u32(m, (uint32_t)__shfl_xor((int)m, 32));
    if (lane == 0) part[wave] = m;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 8; v++) m = max_u32(m, part[v]);
    const float s = block_scale(m), inv = __builtin_amdgcn_rcpf(s);
    if (r != 0) return;
    *(uint32_t *)(p.h + (int64_t)pair * p.I + cb * FP8_BLOCK + wave * 16 + g * 4) = encode4(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
    if (wave == 0 && g == 0) p.hs[(int64_t)cb * p.ldh + pair] = s;
}

// One token's 16 columns per workgroup: the blocks of all its pairs are dealt to the waves.
template <typename AT, typename PT>
__global__ __launch_bounds__(512) void block_fp8_expert_down_token_kernel(const ExpertsArgs p, const PT *__restrict__ weight, AT *__restrict__ out) {
    constexpr int STEPS = 4;
    __shared__ f32x4 sums[8][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, token = blockIdx.y, IB = p.I / FP8_BLOCK, HB = fp8_blocks(p.H), units = p.top_k * IB;
    f32x4 acc = {};
    const int n = n0 + r;
    for (int u0 = wave; u0 < units; u0 += 8 * STEPS) {
        Codes wc[STEPS], xc[STEPS];
        float sc[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int u = u0 + s * 8, j = u / IB, kb = u - j * IB, pair = token * p.top_k + j;
            const int64_t e = u < units ? p.ids[pair] : -1;
            wc[s] = Codes{};
            xc[s] = Codes{};
            sc[s] = 0.0f;
            if (e < 0 || e >= p.n_exp) continue;
            load_chunks(p.down + ((int64_t)e * p.H + n) * p.I + g * 16, kb, FP8_BLOCK, wc[s]);
            const uint8_t *const xr = p.h + (int64_t)pair * p.I + kb * FP8_BLOCK + g * 16;
            xc[s].lo = *(const u32x4 *)xr;
            xc[s].hi = *(const u32x4 *)(xr + 64);
            sc[s] = p.hs[(int64_t)kb * p.ldh + pair] * p.down_scale[((int64_t)e * HB + n0 / FP8_BLOCK) * IB + kb] * (float)weight[pair];
        }
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const f32x4 d = block_dot<false>(wc[s], xc[s]);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = fmaf(sc[s], d[j], acc[j]);
        }
    }
    if (r == 0) sums[wave][g] = acc;
    __syncthreads();
    if (threadIdx.x < 16) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; w++) v += sums[w][threadIdx.x >> 2][threadIdx.x & 3];
        out[(int64_t)token * p.H + n0 + threadIdx.x] = to_at<AT>(v);
    }
}

// The rows of x in codes (as bfloat16 numbers, see EXACT) and scales, and the pairs sorted by expert, in one launch: the first workgroups quantize (32 blocks each), the rest place
// four pairs each.  A wave counts the pairs that come before its own - those of lower experts, and the earlier ones of its expert - as
// moe_sort_gather_kernel does; waves pairs + e write offsets[e].
constexpr int EXPERTS_SORT_PAIRS = 4096;
template <typename AT>
__global__ __launch_bounds__(256) void block_fp8_expert_rows_kernel(const AT *__restrict__ x, const int64_t *__restrict__ ids, uint8_t *__restrict__ codes,
                                                                    float *__restrict__ scale, int32_t *__restrict__ offsets, int32_t *__restrict__ order,
                                                                    int32_t *__restrict__ pos, int tokens, int pairs, int n_exp, int K, int KB,
                                                                    int quantizing) {
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
    const int lane = threadIdx.x & 63, b = (blockIdx.x - quantizing) * 4 + (threadIdx.x >> 6);
    if (b > pairs + n_exp) return;
    const bool is_pair = b < pairs;
    const int64_t own = is_pair ? ids[b] : b - pairs;
    int before = 0;
    for (int j0 = lane; j0 - lane < pairs; j0 += 512) {
        int64_t e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = j0 + i * 64 < pairs ? ids[j0 + i * 64] : -1;
#pragma unroll
        for (int i = 0; i < 8; i++)
            before += __popcll(__ballot(e[i] >= 0 && e[i] < n_exp && (e[i] < own || (is_pair && e[i] == own && j0 + i * 64 < b))));
    }
    if (lane != 0) return;
    if (!is_pair) {
        offsets[own] = before;
        return;
    }
    const bool valid = own >= 0 && own < n_exp;
    pos[b] = valid ? before : -1;
    if (valid) order[before] = b;
}

// While there are no more pairs than experts few of them share one, and each streams its weights; the row of x fits LDS.
static bool direct(int tokens, int top_k, int n_exp, int H) {
    return ((int64_t)tokens * top_k <= n_exp || tokens == 1) && fp8_blocks(H) * (FP8_BLOCK + 4) <= 65536 - 4096;
}

// Rows of a tile: as many as an expert has in the mean, that no more weights are read twice than have to be, and few rows stand idle.
static int expert_tile_rows(int pairs, int n_exp) {
    const int mean = pairs / n_exp;
    return mean <= 32 ? 32 : mean <= 64 ? 64 : 128;
}

struct ExpertsSpace {
    size_t h, hs, x, xs, offsets, order, pos, y, bytes;
    int ldx, ldxs, ldh;
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
    w.ldh = (int)pairs;
    w.h = take((size_t)pairs * I);
    w.hs = take((size_t)pairs * (I / FP8_BLOCK) * 4);
    if (!direct(tokens, top_k, n_exp, H)) {
        w.x = take((size_t)tokens * w.ldx);
        w.xs = take((size_t)tokens * fp8_blocks(H) * 4);
        w.offsets = take((size_t)(n_exp + 1) * 4);
        w.order = take((size_t)pairs * 4);
        w.pos = take((size_t)pairs * 4);
        w.y = take((size_t)pairs * H * 2);
    }
    w.bytes = at;
    return w;
}
size_t block_fp8_experts_workspace_bytes(int tokens, int top_k, int n_exp, int H, int I) {
    return experts_space(tokens, top_k, n_exp, H, I).bytes;
}

template <typename AT> static void launch_down_token(const ExpertsArgs &p, const void *weight, int w_dtype, void *out, int tokens, hipStream_t st) {
    const dim3 grid(p.H / 16, tokens), block(512);
    if (w_dtype == DT_F32)
        hipLaunchKernelGGL((block_fp8_expert_down_token_kernel<AT, float>), grid, block, 0, st, p, (const float *)weight, (AT *)out);
    else if (w_dtype == DT_F16)
        hipLaunchKernelGGL((block_fp8_expert_down_token_kernel<AT, _Float16>), grid, block, 0, st, p, (const _Float16 *)weight, (AT *)out);
    else
        hipLaunchKernelGGL((block_fp8_expert_down_token_kernel<AT, __bf16>), grid, block, 0, st, p, (const __bf16 *)weight, (AT *)out);
}

template <typename AT> static int launch_experts_t(ExpertsArgs p, const ExpertsSpace &at, uint8_t *ws, const void *weight, int w_dtype, void *out,
                                                   int act_dtype, int tokens, hipStream_t st) {
    const int pairs = tokens * p.top_k;
    const bool one_each = direct(tokens, p.top_k, p.n_exp, p.H);
    if (one_each) {
        hipLaunchKernelGGL((block_fp8_expert_token_up_kernel<AT>), dim3(p.I / FP8_BLOCK, pairs), dim3(512), (size_t)fp8_blocks(p.H) * (FP8_BLOCK + 4), st, p);
        launch_down_token<AT>(p, weight, w_dtype, out, tokens, st);
        return 0;
    }
    int32_t *const offsets = (int32_t *)(ws + at.offsets), *const order = (int32_t *)(ws + at.order), *const pos = (int32_t *)(ws + at.pos);
    const int KB = fp8_blocks(p.H), quantizing = (int)(((int64_t)tokens * KB + 31) / 32);
    const bool sorts = pairs <= EXPERTS_SORT_PAIRS;
    hipLaunchKernelGGL((block_fp8_expert_rows_kernel<AT>), dim3(quantizing + (sorts ? (pairs + p.n_exp + 4) / 4 : 0)), dim3(256), 0, st, (const AT *)p.x,
                       p.ids, ws + at.x, (float *)(ws + at.xs), offsets, order, pos, tokens, pairs, p.n_exp, p.H, KB, quantizing);
    if (!sorts) launch_moe_route(p.ids, pairs, p.n_exp, offsets, order, pos, st);

    TiledArgs t{};
    t.offsets = offsets; t.order = order; t.n_exp = p.n_exp; t.top_k = p.top_k; t.M = pairs; t.I = p.I; t.act = p.act;
    TiledArgs u = t;
    u.x = ws + at.x; u.xs = (float *)(ws + at.xs); u.ldx = at.ldx; u.ldxs = at.ldxs;
    u.w = p.gate_up; u.ws = p.gate_up_scale; u.N = 2 * p.I; u.K = p.H; u.KB = KB;
    u.y = p.h; u.hs = p.hs; u.ldhs = p.ldh;
    TiledArgs d = t;
    d.x = p.h; d.xs = p.hs; d.ldx = p.I; d.ldxs = p.ldh;
    d.w = p.down; d.ws = p.down_scale; d.N = p.H; d.K = p.I; d.KB = p.I / FP8_BLOCK;
    d.y = ws + at.y;
    const int rows = expert_tile_rows(pairs, p.n_exp);
    u.tiles_m = d.tiles_m = pairs / rows + (pairs < p.n_exp ? pairs : p.n_exp);      // at most
    if ((int64_t)u.tiles_m * (p.I / FP8_BLOCK) > 0x7fffffff - 8 || (int64_t)d.tiles_m * ((p.H + 127) / 128) > 0x7fffffff - 8) return -3;
    if (rows == 128) {
        launch_tiled<AT, true, TILED_UP, true, true, 4, 4, 2, 4, 2, 2>(u, st);
        launch_tiled<AT, false, TILED_PLAIN, true, false, 4, 4, 2, 4, 3, 2>(d, st);
    } else if (rows == 64) {
        launch_tiled<AT, true, TILED_UP, true, true, 2, 4, 2, 4, 3, 2>(u, st);
        launch_tiled<AT, false, TILED_PLAIN, true, false, 2, 4, 2, 2, 3, 2>(d, st);
    } else {
        launch_tiled<AT, true, TILED_UP, true, true, 2, 4, 1, 4, 3, 1>(u, st);
        launch_tiled<AT, false, TILED_PLAIN, true, false, 2, 2, 1, 4, 3, 2>(d, st);
    }
    launch_moe_combine(ws + at.y, pos, weight, w_dtype, out, act_dtype, tokens, p.top_k, p.H, st);
    return 0;
}

int launch_block_fp8_experts(const void *x, const int64_t *ids, const void *weight, int w_dtype, int tokens, int top_k, int n_exp,
                             const uint8_t *gate_up, const float *gate_up_scale, const uint8_t *down, const float *down_scale, void *workspace,
                             void *out, int act_dtype, int H, int I, int act, hipStream_t st) {
    const ExpertsSpace at = experts_space(tokens, top_k, n_exp, H, I);
    uint8_t *const ws = (uint8_t *)workspace;
    ExpertsArgs p{};
    p.x = x; p.ids = ids; p.ldh = at.ldh;
    p.gate_up = gate_up; p.down = down; p.gate_up_scale = gate_up_scale; p.down_scale = down_scale;
    p.h = ws + at.h; p.hs = (float *)(ws + at.hs);
    p.n_exp = n_exp; p.top_k = top_k; p.H = H; p.I = I; p.act = act;
    return act_dtype == DT_F16 ? launch_experts_t<_Float16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st)
                               : launch_experts_t<__bf16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st);
}

}  // namespace lowbit
