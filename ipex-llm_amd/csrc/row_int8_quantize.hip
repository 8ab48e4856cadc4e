// Codes and scales of rows (row_int8.h): activations by token, weights by output channel.
//
// Bound by memory: a row is read once, into registers, and its codes written once.
#include "row_int8.h"

#include <type_traits>

namespace lowbit {

// A row per WAVES waves, 16 values per lane and piece; what lies past the first HELD pieces is read again behind the row's maximum.  Codes go to
// rows of ldc bytes, zeros from K up to ldc.
template <typename AT, int WAVES, int HELD>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void row_int8_quantize_kernel(const AT *__restrict__ x, uint8_t *__restrict__ codes,
                                                                                          float *__restrict__ scale, int64_t rows, int K, int ldc) {
    constexpr int THREADS = 64 * WAVES, STEP = THREADS * 16;
    const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows) return;
    const AT *const from = x + row * K;
    uint8_t *const to = codes + row * ldc;
    float v[HELD][16];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int k = i * STEP + t * 16;
#pragma unroll
        for (int j = 0; j < 16; j++) v[i][j] = 0.0f;
        if (k < K) load16(from + k, v[i]);
    }
#pragma unroll
    for (int i = 0; i < HELD; i++) m = max_u32(m, largest_of(v[i]));
    for (int k = HELD * STEP + t * 16; k < K; k += STEP) {
        float more[16];
        load16(from + k, more);
        m = max_u32(m, largest_of(more));
    }
    m = max_of_wave(m);
    if constexpr (WAVES > 1) {
        __shared__ uint32_t part[WAVES];
        if ((t & 63) == 0) part[t >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; i++) m = max_u32(m, part[i]);
    }
    const RowCoder code(m);
    auto put = [&](int k, const float (&u)[16]) {
        if (k >= ldc) return;
        uint32_t c[4];
        code(u, c);
        *(u32x4 *)(to + k) = u32x4{c[0], c[1], c[2], c[3]};
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) put(i * STEP + t * 16, v[i]);
    for (int k = HELD * STEP + t * 16; k < ldc; k += STEP) {
        float more[16] = {};
        if (k < K) load16(from + k, more);
        put(k, more);
    }
    if (t == 0) scale[row] = row_scale(m);
}

int launch_row_int8_quantize(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, float *scale, hipStream_t st) {
    if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32) return -4;
    const bool one = K <= 1024;
    const int64_t most = most_groups(256) * (one ? 4 : 1);
    for (; rows > most; rows -= most) {
        if (int rc = launch_row_int8_quantize(x, dtype, most, K, codes, ldc, scale, st)) return rc;
        x = (const uint8_t *)x + most * K * (dtype == DT_F32 ? 4 : 2);
        codes += most * ldc;
        scale += most;
    }
    auto go = [&](auto *typed) {
        using AT = typename std::remove_cv<typename std::remove_pointer<decltype(typed)>::type>::type;
        if (one) hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 1, 1>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st, typed, codes, scale, rows, K, ldc);
        else if (K <= 4096) hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 4, 1>), dim3((uint32_t)rows), dim3(256), 0, st, typed, codes, scale, rows, K, ldc);
        else if (K <= 8192) hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 4, 2>), dim3((uint32_t)rows), dim3(256), 0, st, typed, codes, scale, rows, K, ldc);
        else hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 8, 2>), dim3((uint32_t)rows), dim3(512), 0, st, typed, codes, scale, rows, K, ldc);
    };
    if (dtype == DT_F16) go((const _Float16 *)x);
    else if (dtype == DT_BF16) go((const __bf16 *)x);
    else go((const float *)x);
    return 0;
}

}  // namespace lowbit
