// Up to sixteen rows of activations times a weight with a scale for each block of 128 (block_fp8.h): the weight streams past once, in one
// launch.
//
// A workgroup owns 16 weight rows; its waves take the blocks of K in turn and their sums meet in LDS.  A wave's loads are 16 rows x 64
// contiguous bytes, STEPS blocks ahead of their use.  x is quantized by each workgroup, into LDS, while the first weights are on their
// way.  Loads return in order, so x is asked for ahead of them.  Bound by latency at the sizes of one token: of 5.6 us at one row of [4096 x
// 4096] an empty launch is 1.6.  More rows go to the tiles of block_fp8_gemm.h,
// which take x quantized once, by a launch of its own: 40 rows on [11008 x 4096] 28 us this way, 14.2 in both.
#include "block_fp8_tiled.h"

#include <math.h>

namespace lowbit {

int launch_block_fp8_rows(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, bool wide, float *scale, int64_t row_step,
                          int64_t block_step, hipStream_t st);

constexpr int FEW_ROWS = 16;                                 // an MFMA's

struct RowsProduct {
    const void *x;                                           // [M, K]
    const uint8_t *w;
    const float *ws;
    const void *bias;
    void *y;
    int M, N, K, KB;
};

// 8 values of AT from memory (16-byte aligned)
template <typename AT> struct Eight {
    typedef AT type __attribute__((ext_vector_type(8)));
};

template <typename AT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void block_fp8_few_rows_kernel(const RowsProduct p) {
    constexpr bool EXACT = sizeof(AT) == 4;
    constexpr int STEPS = 4;                                 // blocks in flight per wave
    constexpr int HELD = EXACT ? 2 : 4;                      // pieces of x per thread that are asked for ahead of the weights
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, KB = p.KB, M = p.M, N = p.N, K = p.K;
    // (one wait for all arguments: left alone the compiler loads each where it is first used)
    asm volatile("" :: "s"(p.x), "s"(p.w), "s"(p.ws), "s"(p.bias), "s"(p.y), "s"(M), "s"(N), "s"(K), "s"(KB));

    // pieces of 8 values of x, 16 to a block: thread, thread + 64 * WAVES, ...
    using V8 = typename Eight<AT>::type;
    const int pieces = M * KB * 16;
    auto load_x = [&](int piece) __attribute__((always_inline)) {
        const int row = piece / (KB * 16), k = (piece - row * KB * 16) * 8;
        return k < K ? *(const V8 *)((const AT *)p.x + (int64_t)row * K + k) : V8{};
    };
    V8 held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int piece = threadIdx.x + i * 64 * WAVES;
        held[i] = V8{};
        if (piece < pieces) held[i] = load_x(piece);
    }
    __builtin_amdgcn_sched_barrier(0);

    const int n = n0 + r;
    const uint8_t *const wrow = p.w + (int64_t)(n < N ? n : N - 1) * K;
    // the scales of this wave's blocks in the lanes of a register (64 blocks per wave at most: see few_rows_waves); a scalar load per block
    // would be waited for one after the other
    const float wheld = p.ws[(int64_t)(n0 / FP8_BLOCK) * KB + (wave + lane * WAVES < KB ? wave + lane * WAVES : KB - 1)];
    auto load_w = [&](int kb, Codes &c) __attribute__((always_inline)) {
        // (chunks past the row's end: the block's first one, which meets zeros of x)
        const int left = K - kb * FP8_BLOCK;
        const uint8_t *const at = wrow + kb * FP8_BLOCK;
        c.lo = ld<u32x4, true>(at + (g * 16 < left ? g * 16 : 0));
        c.hi = ld<u32x4, true>(at + (64 + g * 16 < left ? 64 + g * 16 : 0));
    };
    Codes wc[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++)
        load_w(wave + s * WAVES < KB ? wave + s * WAVES : KB - 1, wc[s]);      // (past the last block: it again, not added)
    __builtin_amdgcn_sched_barrier(0);

    // codes of x in LDS, rows of KB * 128 + 16 bytes (16: rows start in other banks), then the scales [KB][FEW_ROWS]
    const int pitch = KB * FP8_BLOCK + 16;
    float *const xs = (float *)(lds + (size_t)M * pitch);
    auto put_x = [&](int piece, const V8 &v) __attribute__((always_inline)) {
        const int row = piece / (KB * 16), at = piece - row * KB * 16;
        put8<AT>(v, lds + row * pitch + at * 8, xs + (at >> 4) * FEW_ROWS + row, (at & 15) == 0);
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int piece = threadIdx.x + i * 64 * WAVES;
        if (piece < pieces) put_x(piece, held[i]);           // (the 16 lanes of a block are in or out together)
    }
    for (int piece = threadIdx.x + HELD * 64 * WAVES; piece < pieces; piece += 64 * WAVES) put_x(piece, load_x(piece));
    __syncthreads();

    // (operand rows past M repeat the last one; their results are not stored)
    const int row = r < M ? r : M - 1;
    const uint8_t *const xrow = lds + row * pitch + g * 16;
    f32x4 acc = {};
    for (int i0 = 0; wave + i0 * WAVES < KB; i0 += STEPS) {
        Codes xc[STEPS];
        float sc[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = wave + (i0 + s) * WAVES, in = kb < KB ? kb : KB - 1;
            xc[s] = Codes{*(const u32x4 *)(xrow + in * FP8_BLOCK), *(const u32x4 *)(xrow + in * FP8_BLOCK + 64)};
            sc[s] = xs[in * FEW_ROWS + row] * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wheld), i0 + s));
        }
        f32x4 d[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            d[s] = block_dot<EXACT>(wc[s], xc[s]);
            const int next = wave + (i0 + s + STEPS) * WAVES;
            if (next < KB) load_w(next, wc[s]);
        }
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const bool in = wave + (i0 + s) * WAVES < KB;
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = in ? fmaf(sc[s], d[s][j], acc[j]) : acc[j];
        }
    }

    // the waves' sums, [wave][row][16 columns]
    __syncthreads();                                         // (they lie where the codes were)
    float *const sums = (float *)lds;
    if (r < M)
        *(f32x4 *)(sums + (wave * FEW_ROWS + r) * 16 + g * 4) = acc;
    __syncthreads();
    if ((int)threadIdx.x >= M * 16) return;
    const int m = threadIdx.x >> 4, c = threadIdx.x & 15;
    if (n0 + c >= N) return;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) v += sums[(w * FEW_ROWS + m) * 16 + c];
    if (p.bias) v += (float)((const AT *)p.bias)[n0 + c];
    ((AT *)p.y)[(int64_t)m * N + n0 + c] = Stored<AT>::of(v);
}

static size_t few_rows_lds(int M, int KB) {
    const size_t codes = (size_t)M * (KB * FP8_BLOCK + 16) + (size_t)KB * FEW_ROWS * sizeof(float);
    return codes > 16384 ? codes : 16384;                    // (the sums of 16 waves)
}

// Short walks, in which half of the loads of 8 waves would be of no block: 4 waves each.  One row on [6144 x 2048] 5.2 us against 7.2.
// Long walks of few workgroups: 16 waves each.  One row on [4096 x 11008] 13.3 us against 13.9, two on [4096 x 14336] 16.3 / 17.2; but
// one on [28672 x 8192] 53.3 / 49.9, on [4096 x 4096], where half of their loads would be of no block, 7.9 / 5.6.
//
// A row's codes and scales fit 64 KiB of LDS, so that 8 waves have 64 blocks each at most, and so have 4.
constexpr size_t FEW_LDS = 65536;
static_assert(FEW_LDS / (FP8_BLOCK + FEW_ROWS * sizeof(float)) <= 8 * 64, "a wave's scales lie in the 64 lanes of a register");
static int few_rows_waves(int N, int KB) { return KB <= 16 ? 4 : KB > 64 && N <= 8192 ? 16 : 8; }

template <typename AT> static void launch_few_rows(const RowsProduct &p, hipStream_t st) {
    const dim3 grid((p.N + 15) / 16);
    const size_t lds = few_rows_lds(p.M, p.KB);
    const int waves = few_rows_waves(p.N, p.KB);
    if (waves == 4) hipLaunchKernelGGL((block_fp8_few_rows_kernel<AT, 4>), grid, dim3(256), lds, st, p);
    else if (waves == 16) hipLaunchKernelGGL((block_fp8_few_rows_kernel<AT, 16>), grid, dim3(1024), lds, st, p);
    else hipLaunchKernelGGL((block_fp8_few_rows_kernel<AT, 8>), grid, dim3(512), lds, st, p);
}

// Rows whose codes fit 64 KiB of LDS: up to four always, up to sixteen where that is estimated shorter than tiles and the launch ahead of them.
// What grows with the rows is x, which every workgroup reads and quantizes: 8 rows on [4096 x 4096] 8.3 us against 10.7 in tiles, 16 11.2 /
// 11.2; 8 on [14336 x 4096] 21.6 / 16.2, on [1536 x 2048] 5.8 / 8.3.  Fitted to 540 sizes of 5 to 16 rows, weights from memory; the pick is 1 %
// above the shorter way on average, 31 % at worst (tiles for all 19 %).
static bool takes_few_rows(bool wide, int M, int N, int K) {
    const int KB = fp8_blocks(K);
    if (M > FEW_ROWS || few_rows_lds(M, KB) > FEW_LDS) return false;
    if (M <= 4) return true;
    const float rounds = N > 4096 ? N / 4096.0f : 1.0f;      // of a workgroup per CU
    const float bytes = (float)N * K, us = 3.1f + bytes / 5.6e6f + (wide ? 0.072f : 0.038f) * M * rounds * K / (64 * few_rows_waves(N, KB));
    return us <= fmaxf(block_fp8_tiled_plan(wide, M, N, K).us, bytes / 5.4e6f + 4.0f) + 1.5f;
}

// codes of x (float32 results: bfloat16 numbers), their scales, a split's sums
struct LinearSpace {
    size_t xs, part, bytes;
};
static LinearSpace linear_space(bool wide, int M, int N, int K, const TiledPlan &plan) {
    auto whole = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    LinearSpace s;
    s.xs = whole((size_t)M * fp8_blocks(K) * FP8_BLOCK * (wide ? 2 : 1));
    s.part = s.xs + whole((size_t)M * fp8_blocks(K) * sizeof(float));
    s.bytes = s.part + block_fp8_tiled_part_bytes(plan, M, N);
    return s;
}

size_t block_fp8_linear_workspace_bytes(int dtype, int M, int N, int K) {
    if (takes_few_rows(dtype == DT_F32, M, N, K)) return 0;
    const bool wide = dtype == DT_F32;
    return linear_space(wide, M, N, K, block_fp8_tiled_plan(wide, M, N, K)).bytes;
}

void block_fp8_linear_plan(int dtype, int M, int N, int K, int *plan4) {
    plan4[0] = plan4[1] = 0;
    plan4[2] = plan4[3] = 1;
    if (takes_few_rows(dtype == DT_F32, M, N, K)) return;
    const TiledPlan plan = block_fp8_tiled_plan(dtype == DT_F32, M, N, K);
    plan4[0] = TILED_FORMS[plan.form].rows;
    plan4[1] = TILED_FORMS[plan.form].cols;
    plan4[2] = plan.splits;
    plan4[3] = TILED_FORMS[plan.form].groups;
}

// waves of a workgroup of the kernel of few rows; 0 where tiles run
int block_fp8_linear_waves(int dtype, int M, int N, int K) {
    return takes_few_rows(dtype == DT_F32, M, N, K) ? few_rows_waves(N, fp8_blocks(K)) : 0;
}

int launch_block_fp8_linear(const void *x, const uint8_t *w, const float *ws, const void *bias, void *y, int dtype, int M, int N, int K,
                            uint8_t *space, hipStream_t st) {
    if (takes_few_rows(dtype == DT_F32, M, N, K)) {
        const RowsProduct p = {x, w, ws, bias, y, M, N, K, fp8_blocks(K)};
        if (dtype == DT_F16) launch_few_rows<_Float16>(p, st);
        else if (dtype == DT_BF16) launch_few_rows<__bf16>(p, st);
        else if (dtype == DT_F32) launch_few_rows<float>(p, st);
        else return -4;
        return 0;
    }
    const bool wide = dtype == DT_F32;
    const TiledPlan plan = block_fp8_tiled_plan(wide, M, N, K);
    const LinearSpace at = linear_space(wide, M, N, K, plan);
    float *const xs = (float *)(space + at.xs);
    if (int rc = launch_block_fp8_rows(x, dtype, M, K, space, fp8_blocks(K) * FP8_BLOCK, wide, xs, 1, M, st)) return rc;
    TiledArgs t{};
    t.x = space; t.xs = xs; t.w = w; t.ws = ws; t.bias = bias; t.y = y; t.part = (float *)(space + at.part);
    t.M = M; t.N = N; t.K = K;
    return launch_block_fp8_tiled(t, dtype, plan, st);
}

}  // namespace lowbit
