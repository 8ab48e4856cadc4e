// Up to sixteen rows of activations times a weight with a scale for each row (row_int8.h): the weight streams past once, in one launch.
//
// A workgroup owns 16 weight rows; its waves take the blocks of K in turn and their sums meet in LDS.  A wave's loads are 16 rows x 64
// contiguous bytes, STEPS blocks ahead of their use.  x is quantized by each workgroup, into LDS, while the first weights are on their
// way: its largest magnitudes by row first, then its codes.  Loads return in order, so x is asked for ahead of the weights.
#include "row_int8_tiled.h"

namespace lowbit {

constexpr int FEW_ROWS = 16;

struct Int8Rows {
    const void *x;                                           // [M, K]
    const uint8_t *w;
    const float *ws;
    const void *bias;
    void *y;
    int M, N, K, KB;
};

template <typename AT> struct Eight {
    typedef AT type __attribute__((ext_vector_type(8)));
};

template <typename V8> __device__ inline void widen_to(const V8 &v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)v[i];
}

template <typename AT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void row_int8_few_rows_kernel(const Int8Rows p) {
    constexpr int STEPS = 4;                                 // blocks in flight per wave
    constexpr int HELD = sizeof(AT) == 4 ? 2 : 4;            // pieces of x per thread that are asked for ahead of the weights
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ uint32_t most[FEW_ROWS];
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
    auto load_w = [&](int kb, Codes &c) __attribute__((always_inline)) {
        // (chunks past the row's end: the block's first one, which meets zeros of x)
        const int left = K - kb * INT8_BLOCK;
        const uint8_t *const at = wrow + kb * INT8_BLOCK;
        c.lo = ld<u32x4, true>(at + (g * 16 < left ? g * 16 : 0));
        c.hi = ld<u32x4, true>(at + (64 + g * 16 < left ? 64 + g * 16 : 0));
    };
    Codes wc[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++)
        load_w(wave + s * WAVES < KB ? wave + s * WAVES : KB - 1, wc[s]);      // (past the last block: it again, times zeros)
    __builtin_amdgcn_sched_barrier(0);

    // the rows' largest magnitudes
    if (threadIdx.x < FEW_ROWS) most[threadIdx.x] = 0;
    __syncthreads();
    auto look = [&](int piece, const V8 &v) __attribute__((always_inline)) {
        float f[8];
        widen_to(v, f);
        const uint32_t m = max_of_16(largest_of(f));         // (16 neighbouring lanes have pieces of one row)
        if ((threadIdx.x & 15) == 0) atomicMax(&most[piece / (KB * 16)], m);
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int piece = threadIdx.x + i * 64 * WAVES;
        if (piece < pieces) look(piece, held[i]);            // (the 16 lanes of a block are in or out together)
    }
    for (int piece = threadIdx.x + HELD * 64 * WAVES; piece < pieces; piece += 64 * WAVES) look(piece, load_x(piece));
    __syncthreads();

    // codes of x in LDS, rows of KB * 128 + 16 bytes (16: rows start in other banks)
    const int pitch = KB * INT8_BLOCK + 16;
    auto put_x = [&](int piece, const V8 &v) __attribute__((always_inline)) {
        const int row = piece / (KB * 16), at = piece - row * KB * 16;
        float f[8];
        widen_to(v, f);
        uint32_t c[2];
        RowCoder{most[row]}(f, c);
        *(u32x2 *)(lds + row * pitch + at * 8) = u32x2{c[0], c[1]};
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int piece = threadIdx.x + i * 64 * WAVES;
        if (piece < pieces) put_x(piece, held[i]);
    }
    for (int piece = threadIdx.x + HELD * 64 * WAVES; piece < pieces; piece += 64 * WAVES) put_x(piece, load_x(piece));
    __syncthreads();

    // (operand rows past M repeat the last one; their results are not stored)
    const uint8_t *const xrow = lds + (r < M ? r : M - 1) * pitch + g * 16;
    i32x4 acc = {};
    for (int i0 = 0; wave + i0 * WAVES < KB; i0 += STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int kb = wave + (i0 + s) * WAVES, in = kb < KB ? kb : KB - 1, next = kb + STEPS * WAVES;
            Codes xc = {*(const u32x4 *)(xrow + in * INT8_BLOCK), *(const u32x4 *)(xrow + in * INT8_BLOCK + 64)};
            if (kb >= KB) xc = Codes{};
            acc = int8_dot(wc[s], xc, acc);
            if (next < KB) load_w(next, wc[s]);
        }
    }

    // the waves' sums, [wave][row of M][16 columns]
    __syncthreads();                                         // (they lie where the codes were)
    int32_t *const sums = (int32_t *)lds;
    if (r < M) *(i32x4 *)(sums + (wave * M + r) * 16 + g * 4) = acc;
    __syncthreads();
    if ((int)threadIdx.x >= M * 16) return;
    const int m = threadIdx.x >> 4, c = threadIdx.x & 15;
    if (n0 + c >= N) return;
    int32_t sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) sum += sums[(w * M + m) * 16 + c];
    float v = (float)sum * row_scale(most[m]) * p.ws[n0 + c];
    if (p.bias) v += (float)((const AT *)p.bias)[n0 + c];
    ((AT *)p.y)[(int64_t)m * N + n0 + c] = Stored<AT>::of(v);
}

static size_t few_rows_lds(int M, int KB, int waves) {
    const size_t codes = (size_t)M * (KB * INT8_BLOCK + 16), sums = (size_t)waves * M * 16 * sizeof(int32_t);
    return codes > sums ? codes : sums;
}

template <typename AT> static void launch_few_rows(const Int8Rows &p, int waves, hipStream_t st) {
    const dim3 grid((p.N + 15) / 16);
    const size_t lds = few_rows_lds(p.M, p.KB, waves);
    if (waves == 4) hipLaunchKernelGGL((row_int8_few_rows_kernel<AT, 4>), grid, dim3(256), lds, st, p);
    else hipLaunchKernelGGL((row_int8_few_rows_kernel<AT, 8>), grid, dim3(512), lds, st, p);
}

// Waves of a workgroup, by estimated time in us; 0 where codes of x, made by a launch of their own, and a product of those are estimated shorter,
// or where x's codes do not fit 64 KiB of LDS.  What grows with the rows is x, which every workgroup reads and quantizes.  With weights in turn from memory: on
// [4096 x 4096] one row 6.1 against 5.9 and the launch ahead of it, 2.6 (5.3 where the one weight stays in the caches), four 8.9 / 6.2 + 2.6; one on
// [20000 x 512] 9.0 / 5.2 + 2.6, on [4096 x 11008] 14.4 / 15.4 + 2.6; one on [28672 x 8192] goes through tiles, 58 with the launch.  With short rows sixteen of them
// are few: 11 on [64 x 128] 3.2 against 5.4 with the launch ahead, 9 on [730 x 384] 4.5 to 5 / 5.5, 5 on [2086 x 1152] 5.2 / 6.1, 16 on [1024 x 1024] 7.4 / 7.3.  Fitted to 80 sizes of 1 to 16 rows, within 11 and 17 % at rms; 16
// waves would be the shortest at one row of very long weights only, [4096 x 11008] 13.7 against 14.3.
constexpr size_t FEW_LDS = 65536 - 64;
constexpr float ROWS_LAUNCH_US = 2.6f;
static int few_rows_waves(int M, int N, int K, float codes_us) {
    static const struct {
        int waves;
        float launch, further, block, row;
    } fits[] = {{4, 3.0f, 0.09f, 0.077f, 0.136f}, {8, 4.0f, 1.9f, 0.053f, 0.183f}};
    const int KB = int8_blocks(K);
    const float units = (N + 15) / 16 / 256.0f, load = units > 1.0f ? units : 1.0f;
    float least = codes_us + ROWS_LAUNCH_US;
    int best = 0;
    for (const auto &f : fits) {
        if (M > FEW_ROWS || few_rows_lds(M, KB, f.waves) > FEW_LDS) continue;
        // (each further workgroup on a CU waits for its rows: half a microsecond where they are many)
        const float us = f.launch + (f.further + (M > 4 ? 0.6f : 0.0f)) * (load - 1.0f) + load * KB * (f.block + f.row * M / f.waves);
        if (us < least) {
            least = us;
            best = f.waves;
        }
    }
    return best;
}

// What a product of these sizes runs as.  A call asks twice, for the workspace and for the launch: the last sizes' plan, a microsecond's
// estimates, is kept.
struct LinearPlan {
    int few;                                                 // waves of the kernel of few rows, or 0
    Int8Plan plan;
};
static LinearPlan linear_plan(int M, int N, int K) {
    static thread_local int last[3] = {};
    static thread_local LinearPlan kept;
    if (M != last[0] || N != last[1] || K != last[2]) {
        kept.plan = row_int8_product_plan(M, N, K);
        kept.few = few_rows_waves(M, N, K, kept.plan.us);
        last[0] = M; last[1] = N; last[2] = K;
    }
    return kept;
}

// codes of x, their scales, a split's sums
struct Int8Space {
    size_t xs, part, bytes;
};
static Int8Space linear_space(int M, int N, int K, const Int8Plan &plan) {
    auto whole = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    Int8Space s;
    s.xs = whole((size_t)M * int8_blocks(K) * INT8_BLOCK);
    s.part = s.xs + whole((size_t)M * sizeof(float));
    s.bytes = s.part + row_int8_part_bytes(plan, M, N);
    return s;
}

size_t row_int8_linear_workspace_bytes(int M, int N, int K) {
    const LinearPlan p = linear_plan(M, N, K);
    return p.few ? 0 : linear_space(M, N, K, p.plan).bytes;
}

// rows and columns of a tile (0, 0: the kernel of few rows; columns 16: the streaming kernel), splits, groups
void row_int8_linear_plan(int M, int N, int K, int *plan4) {
    plan4[0] = plan4[1] = 0;
    plan4[2] = plan4[3] = 1;
    const LinearPlan p = linear_plan(M, N, K);
    if (p.few) return;
    const Int8Plan &plan = p.plan;
    plan4[0] = plan.waves ? (M > 16 ? 32 : 16) : INT8_FORMS[plan.form].rows;
    plan4[1] = plan.waves ? 16 : INT8_FORMS[plan.form].cols;
    plan4[2] = plan.splits;
    plan4[3] = plan.waves ? 1 : INT8_FORMS[plan.form].groups;
}

// waves of a workgroup of the kernel of few rows or of the streaming kernel; 0 where tiles run
int row_int8_linear_waves(int M, int N, int K) {
    const LinearPlan p = linear_plan(M, N, K);
    return p.few ? p.few : p.plan.waves;
}

int launch_row_int8_linear(const void *x, const uint8_t *w, const float *ws, const void *bias, void *y, int dtype, int M, int N, int K, uint8_t *space,
                           hipStream_t st) {
    const LinearPlan all = linear_plan(M, N, K);
    if (const int waves = all.few) {
        const Int8Rows p = {x, w, ws, bias, y, M, N, K, int8_blocks(K)};
        if (dtype == DT_F16) launch_few_rows<_Float16>(p, waves, st);
        else if (dtype == DT_BF16) launch_few_rows<__bf16>(p, waves, st);
        else if (dtype == DT_F32) launch_few_rows<float>(p, waves, st);
        else return -4;
        return 0;
    }
    const Int8Plan &plan = all.plan;
    const Int8Space at = linear_space(M, N, K, plan);
    float *const xs = (float *)(space + at.xs);
    Int8Args t{};
    t.ldx = (int64_t)int8_blocks(K) * INT8_BLOCK;
    if (int rc = launch_row_int8_quantize(x, dtype, M, K, space, (int)t.ldx, xs, nullptr, st)) return rc;
    t.x = space; t.xs = xs; t.w = w; t.ws = ws; t.bias = bias; t.y = y; t.part = (int32_t *)(space + at.part);
    t.M = M; t.N = N; t.K = K;
    return launch_row_int8_codes(t, dtype, plan, st);
}

// Rows of codes that do not fill whole blocks, in rows of ldx bytes with zeros past K; 16 bytes per thread.
__global__ __launch_bounds__(256) void row_int8_pad_kernel(const u32x4 *__restrict__ codes, u32x4 *__restrict__ to, int64_t units, int quads, int ldq) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= units) return;
    const int64_t row = id / ldq;
    const int q = (int)(id - row * ldq);
    to[id] = q < quads ? codes[row * quads + q] : u32x4{};
}

static bool whole_blocks(int K) { return K % INT8_BLOCK == 0; }

// The plan of a product of codes that are given.  Those may be -128 on both sides: 128 * 128 * 2^17 is one more than 32 bits hold, so that the longest row goes in
// two parts at least, whose sums row_int8_reduce_kernel adds in 64 bits.
static Int8Plan given_codes_plan(int M, int N, int K) {
    Int8Plan plan = linear_plan(M, N, K).plan;
    if (K == INT8_MOST_K && plan.splits == 1) plan.splits = 2;
    return plan;
}

size_t row_int8_product_workspace_bytes(int M, int N, int K) {
    const size_t padded = whole_blocks(K) ? 0 : (size_t)M * int8_blocks(K) * INT8_BLOCK;
    return ((padded + 255) & ~(size_t)255) + row_int8_part_bytes(given_codes_plan(M, N, K), M, N);
}

int launch_row_int8_product(const uint8_t *codes, const float *xs, const uint8_t *w, const float *ws, const void *bias, void *y, int dtype, int M, int N,
                            int K, uint8_t *space, hipStream_t st) {
    Int8Args t{};
    t.ldx = (int64_t)int8_blocks(K) * INT8_BLOCK;
    t.x = codes;
    if (!whole_blocks(K)) {
        constexpr int most = 1 << 18;                        // rows of a launch, of up to 2^13 threads each (a grid holds fewer than 2^32)
        for (int m = 0; m < M; m += most) {
            const int64_t units = (M - m < most ? M - m : most) * (t.ldx / 16);
            hipLaunchKernelGGL(row_int8_pad_kernel, dim3((uint32_t)((units + 255) / 256)), dim3(256), 0, st, (const u32x4 *)(codes + (int64_t)m * K),
                               (u32x4 *)(space + m * t.ldx), units, K / 16, (int)(t.ldx / 16));
        }
        t.x = space;
        space += (M * t.ldx + 255) & ~(int64_t)255;
    }
    t.xs = xs; t.w = w; t.ws = ws; t.bias = bias; t.y = y; t.part = (int32_t *)space;
    t.M = M; t.N = N; t.K = K;
    return launch_row_int8_codes(t, dtype, given_codes_plan(M, N, K), st);
}

}  // namespace lowbit
