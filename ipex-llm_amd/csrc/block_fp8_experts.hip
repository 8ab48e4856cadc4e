// The experts of a mixture-of-experts block with weights and activations in e4m3, a scale for each block of 128 (block_fp8.h):
//     out_t = sum_j p_tj * (Q(act(g) u) down_e^T),  (g | u) = Q(x_t) gate_up_e^T,  e = ids_tj
//
// A workgroup of the first product owns 128 columns of h = act(g) u, which are one block of h's rows: it has every value that the
// block's scale depends on, so h leaves as codes and never as 16-bit numbers.
//
// Few pairs (DIRECT): each pair streams its expert's weights, two launches.  More: the pairs sorted by expert, and row tiles of one
// expert (find_expert_tile).
#include "block_fp8.h"

namespace lowbit {

void launch_moe_route(const int64_t *ids, int pairs, int n_exp, int32_t *offsets, int32_t *order, int32_t *pos, hipStream_t st);
void launch_moe_combine(const void *y, const int32_t *pos, const void *weight, int w_dtype, void *out, int act_dtype, int tokens, int top_k,
                        int N, hipStream_t st);
int launch_block_fp8_rows(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, float *scale, int64_t row_step,
                          int64_t block_step, hipStream_t st);

struct ExpertsArgs {
    const void *x;                                           // DIRECT: activations [tokens, H]; else their codes, rows of ldx bytes
    const float *xs;                                         // [blocks of H][ldxs]
    int ldx, ldxs;
    const int64_t *ids;
    const int32_t *offsets, *order;
    const uint8_t *gate_up, *down;
    const float *gate_up_scale, *down_scale;
    uint8_t *h;                                              // codes [pairs, I], by pair (DIRECT) or by sorted position
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
template <typename AT, int MT, bool DIRECT>
__global__ __launch_bounds__(512) void block_fp8_expert_up_kernel(const ExpertsArgs p) {
    constexpr int STEPS = MT == 1 ? 4 : 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ uint32_t part[8][16 * MT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int cb = blockIdx.x, KB = fp8_blocks(p.H);
    int expert, first, end;
    if constexpr (DIRECT) {
        const int64_t e = p.ids[blockIdx.y];
        if (e < 0 || e >= p.n_exp) return;                   // (the second product skips the pair)
        expert = (int)e;
        first = blockIdx.y;
        end = first + 1;
    } else {
        ExpertTile t;
        if (!find_expert_tile<16 * MT>(p.offsets, p.n_exp, blockIdx.y, t)) return;
        expert = t.expert;
        first = t.first;
        end = t.end;
    }
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

    const uint8_t *xrow[MT];
    const float *xs;
    int xs_at[MT], xs_step;
    if constexpr (DIRECT) {
        float *const xs_lds = (float *)(lds + KB * FP8_BLOCK);
        for (int kb = threadIdx.x >> 3; kb < KB; kb += 64) {
            const int k = kb * FP8_BLOCK + (threadIdx.x & 7) * 16;
            float v[16] = {}, s;
            if (k < p.H) load16((const AT *)p.x + (int64_t)(first / p.top_k) * p.H + k, v);
            *(u32x4 *)(lds + k) = quantize16<AT>(v, s);
            if ((threadIdx.x & 7) == 0) xs_lds[kb] = s;
        }
        __syncthreads();
        xrow[0] = lds + g * 16;
        xs = xs_lds;
        xs_at[0] = 0;
        xs_step = 1;
    } else {
        xs = p.xs;
        xs_step = p.ldxs;
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int at = first + i * 16 + r, token = p.order[at < end ? at : end - 1] / p.top_k;
            xrow[i] = (const uint8_t *)p.x + (int64_t)token * p.ldx + g * 16;
            xs_at[i] = token;
        }
    }

    f32x4 acc[2][MT] = {};
    for (int kb0 = 0; kb0 < KB; kb0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = kb0 + s;
            if (kb >= KB) break;
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const Codes xc = {*(const u32x4 *)(xrow[i] + kb * FP8_BLOCK), *(const u32x4 *)(xrow[i] + kb * FP8_BLOCK + 64)};
                const float sx = xs[(int64_t)kb * xs_step + xs_at[i]];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const float sc = sx * ws[t][kb];
                    const f32x4 d = block_dot<false>(wc[s][t], xc);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[t][i][j] = fmaf(sc, d[j], acc[t][i][j]);
                }
            }
            if (kb + STEPS < KB)
#pragma unroll
                for (int t = 0; t < 2; t++) load_chunks(row[t], kb + STEPS, p.H - (kb + STEPS) * FP8_BLOCK - g * 16, wc[s][t]);
        }
    }

    float h[MT][4];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            h[i][j] = gate_act(acc[0][i][j], p.act) * acc[1][i][j];
            m = max_u32(m, magnitude(h[i][j]));
        }
        m = max_u32(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max_u32(m, (uint32_t)__shfl_xor((int)m, 32));
        if (g == 0) part[wave][i * 16 + r] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; i++) {
        uint32_t m = 0;
#pragma unroll
        for (int v = 0; v < 8; v++) m = max_u32(m, part[v][i * 16 + r]);
        const float s = block_scale(m), inv = __builtin_amdgcn_rcpf(s);
        const int at = first + i * 16 + r;
        if (at >= end) continue;
        *(uint32_t *)(p.h + (int64_t)at * p.I + cb * FP8_BLOCK + wave * 16 + g * 4) =
            encode4(h[i][0] * inv, h[i][1] * inv, h[i][2] * inv, h[i][3] * inv);
        if (wave == 0 && g == 0) p.hs[(int64_t)cb * p.ldh + at] = s;
    }
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

// 16 columns of up to 16 * MT rows of one expert; the waves share K.
template <typename AT, int MT>
__global__ __launch_bounds__(512) void block_fp8_expert_down_kernel(const ExpertsArgs p, AT *__restrict__ y) {
    __shared__ f32x4 sums[8][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, IB = p.I / FP8_BLOCK, HB = fp8_blocks(p.H);
    ExpertTile t;
    if (!find_expert_tile<16 * MT>(p.offsets, p.n_exp, blockIdx.y, t)) return;
    const uint8_t *const row = p.down + ((int64_t)t.expert * p.H + n0 + r) * p.I + g * 16;
    const float *const ws = p.down_scale + ((int64_t)t.expert * HB + n0 / FP8_BLOCK) * IB;
    int at[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) at[i] = t.first + i * 16 + r < t.end ? t.first + i * 16 + r : t.end - 1;
    f32x4 acc[MT] = {};
    for (int kb = wave; kb < IB; kb += 8) {
        Codes wc;
        load_chunks(row, kb, FP8_BLOCK, wc);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const uint8_t *const xr = p.h + (int64_t)at[i] * p.I + kb * FP8_BLOCK + g * 16;
            const Codes xc = {*(const u32x4 *)xr, *(const u32x4 *)(xr + 64)};
            const float sc = p.hs[(int64_t)kb * p.ldh + at[i]] * ws[kb];
            const f32x4 d = block_dot<false>(wc, xc);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sc, d[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * 64; o += 512) {
        const int i = o >> 6, l = o & 63, m = t.first + i * 16 + (l & 15);
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < 8; w++) v += sums[w][i][l];
        if (m >= t.end) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) y[(int64_t)m * p.H + n0 + (l >> 4) * 4 + j] = to_at<AT>(v[j]);
    }
}

// While there are no more pairs than experts few of them share one, and each streams its weights; the row of x fits LDS.
static bool direct(int tokens, int top_k, int n_exp, int H) {
    return ((int64_t)tokens * top_k <= n_exp || tokens == 1) && fp8_blocks(H) * (FP8_BLOCK + 4) <= 65536 - 4096;
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
    w.ldx = fp8_blocks(H) * FP8_BLOCK;
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

template <typename AT> static void launch_up(const ExpertsArgs &p, bool one_each, int pairs, hipStream_t st) {
    const int cols = p.I / FP8_BLOCK;
    if (one_each)
        hipLaunchKernelGGL((block_fp8_expert_up_kernel<AT, 1, true>), dim3(cols, pairs), dim3(512), (size_t)fp8_blocks(p.H) * (FP8_BLOCK + 4), st, p);
    else
        hipLaunchKernelGGL((block_fp8_expert_up_kernel<AT, 4, false>), dim3(cols, (pairs + 63) / 64 + p.n_exp), dim3(512), 0, st, p);
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
        launch_up<AT>(p, true, pairs, st);
        launch_down_token<AT>(p, weight, w_dtype, out, tokens, st);
        return 0;
    }
    int32_t *const offsets = (int32_t *)(ws + at.offsets), *const order = (int32_t *)(ws + at.order), *const pos = (int32_t *)(ws + at.pos);
    if (int rc = launch_block_fp8_rows(p.x, act_dtype, tokens, p.H, ws + at.x, at.ldx, (float *)(ws + at.xs), 1, at.ldxs, st)) return rc;
    launch_moe_route(p.ids, pairs, p.n_exp, offsets, order, pos, st);
    p.x = ws + at.x;
    p.xs = (float *)(ws + at.xs);
    p.offsets = offsets;
    p.order = order;
    launch_up<AT>(p, false, pairs, st);
    hipLaunchKernelGGL((block_fp8_expert_down_kernel<AT, 4>), dim3(p.H / 16, (pairs + 63) / 64 + p.n_exp), dim3(512), 0, st, p, (AT *)(ws + at.y));
    launch_moe_combine(ws + at.y, pos, weight, w_dtype, out, act_dtype, tokens, p.top_k, p.H, st);
    return 0;
}

int launch_block_fp8_experts(const void *x, const int64_t *ids, const void *weight, int w_dtype, int tokens, int top_k, int n_exp,
                             const uint8_t *gate_up, const float *gate_up_scale, const uint8_t *down, const float *down_scale, void *workspace,
                             void *out, int act_dtype, int H, int I, int act, hipStream_t st) {
    const ExpertsSpace at = experts_space(tokens, top_k, n_exp, H, I);
    uint8_t *const ws = (uint8_t *)workspace;
    ExpertsArgs p{};
    p.x = x; p.ids = ids; p.ldx = at.ldx; p.ldxs = at.ldxs; p.ldh = at.ldh;
    p.gate_up = gate_up; p.down = down; p.gate_up_scale = gate_up_scale; p.down_scale = down_scale;
    p.h = ws + at.h; p.hs = (float *)(ws + at.hs);
    p.n_exp = n_exp; p.top_k = top_k; p.H = H; p.I = I; p.act = act;
    return act_dtype == DT_F16 ? launch_experts_t<_Float16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st)
                               : launch_experts_t<__bf16>(p, at, ws, weight, w_dtype, out, act_dtype, tokens, st);
}

}  // namespace lowbit
