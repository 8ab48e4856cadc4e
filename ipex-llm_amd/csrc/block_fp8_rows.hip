// Few rows of activations times a weight with a scale for each block of 128 (block_fp8.h): the weight streams past once.
//
// A workgroup owns 16 * T weight rows and up to 16 * MT rows of x; its waves take the blocks of K in turn and their sums meet in LDS.
// A wave's loads are 16 rows x 64 contiguous bytes, STEPS blocks ahead of their use.  FUSED: x is quantized by each workgroup, into
// LDS, while the first weights are on their way, which saves a launch; otherwise codes and scales of x come from memory (L2).
#include "block_fp8_tiled.h"

namespace lowbit {

int launch_block_fp8_rows(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, bool wide, float *scale, int64_t row_step,
                          int64_t block_step, hipStream_t st);

struct RowsProduct {
    const void *x;                                           // FUSED: activations [M, K]; else codes, rows of ldx bytes
    const float *xs;                                         // scales of the codes: [KB][ldm]
    const uint8_t *w;
    const float *ws;
    const void *bias;
    void *y;
    int M, N, K, KB, ldx, ldm;
};

template <typename AT> __device__ inline AT narrow(float v) { return to_at<AT>(v); }
template <> __device__ inline float narrow<float>(float v) { return v; }

template <typename AT, int T, int MT, bool FUSED, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void block_fp8_few_rows_kernel(const RowsProduct p) {
    constexpr bool EXACT = sizeof(AT) == 4;
    constexpr int STEPS = T * MT > 4 ? 2 : 4;                // blocks in flight per wave
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * T, m0 = blockIdx.y * 16 * MT, KB = p.KB;

    const uint8_t *wrow[T];
#pragma unroll
    for (int t = 0; t < T; t++) {
        const int n = n0 + t * 16 + r;
        wrow[t] = p.w + (int64_t)(n < p.N ? n : p.N - 1) * p.K + g * 16;
    }
    const float *const ws = p.ws + (int64_t)(n0 / FP8_BLOCK) * KB;
    auto load_w = [&](int kb, Codes (&c)[T]) {
        const int left = p.K - kb * FP8_BLOCK - g * 16;      // bytes of the row from the lane's first chunk on
#pragma unroll
        for (int t = 0; t < T; t++) {
            c[t] = Codes{};
            if (left > 0) c[t].lo = ld<u32x4, true>(wrow[t] + kb * FP8_BLOCK);
            if (left > 64) c[t].hi = ld<u32x4, true>(wrow[t] + kb * FP8_BLOCK + 64);
        }
    };
    Codes wc[STEPS][T];
    float wsc[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const int kb = wave + s * WAVES;
        if (kb < KB) {
            load_w(kb, wc[s]);
            wsc[s] = ws[kb];
        }
    }

    // FUSED: codes of up to 16 rows in LDS, rows of KB * 128 + 16 bytes (16: rows start in other banks), then their scales [KB][16]
    const int pitch = KB * FP8_BLOCK + 16, rows = p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT;
    float *const xs_lds = (float *)(lds + (size_t)rows * pitch);
    if constexpr (FUSED) {
        const int units = rows * KB;
        for (int u = threadIdx.x >> 3; u < units; u += 8 * WAVES) {
            const int row = u / KB, kb = u - row * KB, k = kb * FP8_BLOCK + (threadIdx.x & 7) * 16;
            float v[16] = {}, s;
            if (k < p.K) load16((const AT *)p.x + (int64_t)(m0 + row) * p.K + k, v);
            *(u32x4 *)(lds + row * pitch + k) = quantize16<AT>(v, s);
            if ((threadIdx.x & 7) == 0) xs_lds[kb * 16 + row] = s;
        }
        __syncthreads();
    }
    // rows past M repeat the last one; their results are not stored
    const uint8_t *xrow[MT];
    int xrow_at[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int m = i * 16 + r, mm = m < rows ? m : rows - 1;
        xrow_at[i] = FUSED ? mm : m0 + mm;
        xrow[i] = FUSED ? lds + mm * pitch + g * 16 : (const uint8_t *)p.x + (int64_t)(m0 + mm) * p.ldx + g * 16;
    }

    f32x4 acc[T][MT] = {};
    for (int kb0 = wave; kb0 < KB; kb0 += WAVES * STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = kb0 + s * WAVES;
            if (kb >= KB) break;
            Codes xc[MT];
            float scale[MT];
#pragma unroll
            for (int i = 0; i < MT; i++) {
                xc[i].lo = *(const u32x4 *)(xrow[i] + kb * FP8_BLOCK);
                xc[i].hi = *(const u32x4 *)(xrow[i] + kb * FP8_BLOCK + 64);
                scale[i] = FUSED ? xs_lds[kb * 16 + xrow_at[i]] : p.xs[(int64_t)kb * p.ldm + xrow_at[i]];
            }
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const float sc = scale[i] * wsc[s];
#pragma unroll
                for (int t = 0; t < T; t++) {
                    const f32x4 d = block_dot<EXACT>(wc[s][t], xc[i]);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[t][i][j] = fmaf(sc, d[j], acc[t][i][j]);
                }
            }
            const int next = kb + WAVES * STEPS;
            if (next < KB) {
                load_w(next, wc[s]);
                wsc[s] = ws[next];
            }
        }
    }

    // the waves' sums, [wave][t * MT + i][lane]
    if constexpr (FUSED) __syncthreads();                    // (they lie where the codes were)
    f32x4 *const sums = (f32x4 *)lds;
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
        for (int i = 0; i < MT; i++) sums[(wave * T * MT + t * MT + i) * 64 + lane] = acc[t][i];
    __syncthreads();
    for (int o = threadIdx.x; o < T * MT * 64; o += 64 * WAVES) {
        f32x4 v = sums[o];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v += sums[w * T * MT * 64 + o];
        const int l = o & 63, i = (o >> 6) % MT, t = (o >> 6) / MT;
        const int m = m0 + i * 16 + (l & 15), n = n0 + t * 16 + (l >> 4) * 4;
        if (m >= p.M) continue;
        AT *const out = (AT *)p.y + (int64_t)m * p.N + n;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n + j < p.N) out[j] = narrow<AT>(v[j] + (p.bias ? (float)((const AT *)p.bias)[n + j] : 0.0f));
    }
}

template <typename AT, int T, int MT, bool FUSED, int WAVES> static void launch_few(const RowsProduct &p, hipStream_t st) {
    size_t lds = (size_t)WAVES * T * MT * 64 * sizeof(f32x4);
    const int rows = p.M < 16 * MT ? p.M : 16 * MT;
    const size_t codes = (size_t)rows * (p.KB * FP8_BLOCK + 16) + (size_t)p.KB * 16 * sizeof(float);
    if (FUSED && codes > lds) lds = codes;
    const dim3 grid((p.N + 16 * T - 1) / (16 * T), (p.M + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((block_fp8_few_rows_kernel<AT, T, MT, FUSED, WAVES>), grid, dim3(64 * WAVES), lds, st, p);
}

template <typename AT> static void launch_few_rows_t(const RowsProduct &p, bool fused, hipStream_t st) {
    if (fused) launch_few<AT, 1, 1, true, 8>(p, st);
    else if (p.M <= 16) launch_few<AT, 1, 1, false, 8>(p, st);
    else if (p.M <= 32) launch_few<AT, 1, 2, false, 8>(p, st);
    else launch_few<AT, 2, 4, false, 8>(p, st);
}

// Rows that each workgroup quantizes by itself: their codes fit 64 KiB of LDS.
static bool fuses_rows(int M, int K) {
    return M <= 4 && (size_t)M * (fp8_blocks(K) * FP8_BLOCK + 16) + (size_t)fp8_blocks(K) * 64 <= 65536;
}

static size_t codes_bytes(int M, int K, bool wide) { return ((size_t)M * fp8_blocks(K) * FP8_BLOCK * (wide ? 2 : 1) + 255) & ~(size_t)255; }

// Up to here one pass of the weights through registers; beyond, tiles in LDS.
static bool takes_few_rows(int M) { return M <= 64; }

// codes of x (float32 results of tiles: bfloat16 numbers), their scales, a split's sums
struct LinearSpace {
    size_t xs, part, bytes;
};
static LinearSpace linear_space(int M, int N, int K, bool wide, const TiledPlan &plan) {
    LinearSpace s;
    s.xs = codes_bytes(M, K, wide);
    s.part = s.xs + (((size_t)M * fp8_blocks(K) * sizeof(float) + 255) & ~(size_t)255);
    s.bytes = s.part + block_fp8_tiled_part_bytes(plan, M, N);
    return s;
}

size_t block_fp8_linear_workspace_bytes(int dtype, int M, int N, int K) {
    if (fuses_rows(M, K)) return 0;
    const TiledPlan plan = takes_few_rows(M) ? TiledPlan{0, 1, 0.0f} : block_fp8_tiled_plan(dtype == DT_F32, M, N, K);
    return linear_space(M, N, K, dtype == DT_F32 && !takes_few_rows(M), plan).bytes;
}

int launch_block_fp8_linear(const void *x, const uint8_t *w, const float *ws, const void *bias, void *y, int dtype, int M, int N, int K,
                            uint8_t *space, hipStream_t st) {
    const bool fused = fuses_rows(M, K), few = takes_few_rows(M);
    const int KB = fp8_blocks(K), ldx = KB * FP8_BLOCK;
    RowsProduct p = {x, nullptr, w, ws, bias, y, M, N, K, KB, ldx, M};
    if (!fused) {
        const TiledPlan plan = few ? TiledPlan{0, 1, 0.0f} : block_fp8_tiled_plan(dtype == DT_F32, M, N, K);
        const bool wide = dtype == DT_F32 && !few;
        const LinearSpace at = linear_space(M, N, K, wide, plan);
        float *const xs = (float *)(space + at.xs);
        if (int rc = launch_block_fp8_rows(x, dtype, M, K, space, ldx, wide, xs, 1, M, st)) return rc;
        if (!few) {
            TiledArgs t{};
            t.x = space; t.xs = xs; t.w = w; t.ws = ws; t.bias = bias; t.y = y; t.part = (float *)(space + at.part);
            t.M = M; t.N = N; t.K = K;
            return launch_block_fp8_tiled(t, dtype, plan, st);
        }
        p.x = space;
        p.xs = xs;
    }
    if (dtype == DT_F16) launch_few_rows_t<_Float16>(p, fused, st);
    else if (dtype == DT_BF16) launch_few_rows_t<__bf16>(p, fused, st);
    else if (dtype == DT_F32) launch_few_rows_t<float>(p, fused, st);
    else return -4;
    return 0;
}

}  // namespace lowbit
