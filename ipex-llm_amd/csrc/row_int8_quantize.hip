// Codes and scales of rows (row_int8.h): activations by token, weights by output channel.
//
// Bound by memory: a row is read once, into registers, and its codes written once.  [28672 x 8192] in bfloat16 124 us, 5.7 TB/s read and written, [8192 x
// 8192] 47, [2048 x 11008] 15.5; 48 rows of 11008 take what a launch takes.  A wave per row up to 1024 values, so that no maximum waits for a barrier; eight
// above 8192, so that a row stays in registers.
#include "row_int8.h"

#include <type_traits>

namespace lowbit {

// A row per WAVES waves.  limit: where given, rows from *limit on are left as they are.
template <typename AT, int WAVES, int HELD>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void row_int8_quantize_kernel(const AT *__restrict__ x, uint8_t *__restrict__ codes,
                                                                                          float *__restrict__ scale, int64_t rows, int K, int ldc,
                                                                                          const int32_t *__restrict__ limit) {
    const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows || (limit && row >= *limit)) return;
    const float s = quantize_row<AT, WAVES, HELD>(x + row * K, codes + row * ldc, K, ldc, t);
    if (t == 0) scale[row] = s;
}

int launch_row_int8_quantize(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, float *scale, const int32_t *limit, hipStream_t st) {
    if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32) return -4;
    const bool one = K <= 1024;
    constexpr int64_t most = 1 << 22;                        // (of 512 threads each: a grid holds fewer than 2^32)
    for (; rows > most; rows -= most) {                      // (rows that a limit counts are fewer)
        if (int rc = launch_row_int8_quantize(x, dtype, most, K, codes, ldc, scale, limit, st)) return rc;
        x = (const uint8_t *)x + most * K * (dtype == DT_F32 ? 4 : 2);
        codes += most * ldc;
        scale += most;
    }
    auto go = [&](auto *typed) {
        using AT = typename std::remove_cv<typename std::remove_pointer<decltype(typed)>::type>::type;
        if (one) hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 1, 1>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st, typed, codes, scale, rows, K, ldc, limit);
        else if (K <= 4096) hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 4, 1>), dim3((uint32_t)rows), dim3(256), 0, st, typed, codes, scale, rows, K, ldc, limit);
        else if (K <= 8192) hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 4, 2>), dim3((uint32_t)rows), dim3(256), 0, st, typed, codes, scale, rows, K, ldc, limit);
        else hipLaunchKernelGGL((row_int8_quantize_kernel<AT, 8, 2>), dim3((uint32_t)rows), dim3(512), 0, st, typed, codes, scale, rows, K, ldc, limit);
    };
    if (dtype == DT_F16) go((const _Float16 *)x);
    else if (dtype == DT_BF16) go((const __bf16 *)x);
    else go((const float *)x);
    return 0;
}

}  // namespace lowbit
