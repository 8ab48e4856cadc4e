// Codes and scales for blocks of 128 (block_fp8.h): rows of activations, blocks of weights.
//
// Both are bound by memory: an element is read once and its code written once.  bfloat16 rows of [8192 x 8192] 37 us, weights [28672 x 8192]
// 129 us: 5.4 TB/s read and written, where a copy reaches 4.8.
#include "block_fp8.h"

#include <type_traits>

namespace lowbit {

// One block of a row per 8 lanes, 16 values per lane.  Codes go to rows of ldc bytes; past the row's end they are zeros up to whole
// blocks where ldc has room for them (the products' own rows; WIDE: bfloat16 numbers in rows of 2 ldc bytes).  Scale of (row, block): scale[row * row_step + block * block_step].
template <typename AT, bool WIDE>
__global__ __launch_bounds__(256) void block_fp8_rows_kernel(const AT *__restrict__ x, uint8_t *__restrict__ codes, float *__restrict__ scale,
                                                             int64_t units, int K, int KB, int ldc, int64_t row_step, int64_t block_step) {
    const int64_t unit = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    if (unit >= units) return;                               // (the 8 lanes of a block leave together)
    const int64_t row = unit / KB;
    const int kb = (int)(unit - row * KB), k = kb * FP8_BLOCK + (threadIdx.x & 7) * 16;
    float v[16] = {};
    if (k < K) load16(x + row * K + k, v);
    float s;
    const u32x4 c = quantize16<AT>(v, s);
    if (k < ldc) store16<WIDE>(codes + row * ldc * (WIDE ? 2 : 1), k, c);
    if ((threadIdx.x & 7) == 0) scale[row * row_step + kb * block_step] = s;
}

int launch_block_fp8_rows(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, bool wide, float *scale, int64_t row_step,
                          int64_t block_step, hipStream_t st) {
    const int KB = fp8_blocks(K);
    const int64_t most = most_groups(256) * 32 / KB;
    for (; rows > most; rows -= most) {
        if (int rc = launch_block_fp8_rows(x, dtype, most, K, codes, ldc, wide, scale, row_step, block_step, st)) return rc;
        x = (const uint8_t *)x + most * K * (dtype == DT_F32 ? 4 : 2);
        codes += most * ldc * (wide ? 2 : 1);
        scale += most * row_step;
    }
    const int64_t units = rows * KB;
    const dim3 grid((uint32_t)((units + 31) / 32)), block(256);
    auto go = [&](auto *typed, auto w) {
        using AT = typename std::remove_cv<typename std::remove_pointer<decltype(typed)>::type>::type;
        hipLaunchKernelGGL((block_fp8_rows_kernel<AT, decltype(w)::value>), grid, block, 0, st, typed, codes, scale, units, K, KB, ldc, row_step, block_step);
    };
    if (dtype == DT_F16) go((const _Float16 *)x, std::false_type());
    else if (dtype == DT_BF16) go((const __bf16 *)x, std::false_type());
    else if (dtype != DT_F32) return -4;
    else if (wide) go((const float *)x, std::true_type());
    else go((const float *)x, std::false_type());
    return 0;
}

// One 128 x 128 block of a weight per workgroup of 512: thread t holds 16 values of rows t / 8 and 64 + t / 8.
template <typename AT>
__global__ __launch_bounds__(512) void block_fp8_weight_kernel(const AT *__restrict__ w, uint8_t *__restrict__ codes, float *__restrict__ scale,
                                                               int N, int K, int KB, int NB) {
    __shared__ uint32_t part[8];
    const int t = threadIdx.x, kb = blockIdx.x % KB, k = kb * FP8_BLOCK + (t & 7) * 16;
    const int at = blockIdx.x / KB, nb = at % NB;
    const int64_t base = (int64_t)(at / NB) * N * K;
    float v[2][16] = {};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int n = nb * FP8_BLOCK + i * 64 + (t >> 3);
        if (n < N && k < K) load16(w + base + (int64_t)n * K + k, v[i]);
#pragma unroll
        for (int j = 0; j < 16; j++) m = max_u32(m, magnitude(v[i][j]));
    }
    m = max_of_16(m);
    m = max_u32(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max_u32(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((t & 63) == 0) part[t >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) m = max_u32(m, part[i]);
    const float s = block_scale(m);
    const Quotient<AT> q(s, m);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int n = nb * FP8_BLOCK + i * 64 + (t >> 3);
        if (n >= N || k >= K) continue;
        u32x4 c;
#pragma unroll
        for (int j = 0; j < 4; j++) c[j] = encode4(q(v[i][4 * j]), q(v[i][4 * j + 1]), q(v[i][4 * j + 2]), q(v[i][4 * j + 3]));
        *(u32x4 *)(codes + base + (int64_t)n * K + k) = c;
    }
    if (t == 0) scale[blockIdx.x] = s;
}

int launch_block_fp8_weight(const void *w, int dtype, int64_t matrices, int N, int K, uint8_t *codes, float *scale, hipStream_t st) {
    const int KB = fp8_blocks(K), NB = fp8_blocks(N);
    const int64_t most = most_groups(512) / ((int64_t)NB * KB);
    if (most == 0) return -3;
    for (; matrices > most; matrices -= most) {
        if (int rc = launch_block_fp8_weight(w, dtype, most, N, K, codes, scale, st)) return rc;
        w = (const uint8_t *)w + most * N * K * (dtype == DT_F32 ? 4 : 2);
        codes += most * N * K;
        scale += most * NB * KB;
    }
    const dim3 grid((uint32_t)(matrices * NB * KB));
    auto go = [&](auto *typed) {
        using AT = typename std::remove_cv<typename std::remove_pointer<decltype(typed)>::type>::type;
        hipLaunchKernelGGL((block_fp8_weight_kernel<AT>), grid, dim3(512), 0, st, typed, codes, scale, N, K, KB, NB);
    };
    if (dtype == DT_F16) go((const _Float16 *)w);
    else if (dtype == DT_BF16) go((const __bf16 *)w);
    else if (dtype == DT_F32) go((const float *)w);
    else return -4;
    return 0;
}

}  // namespace lowbit
