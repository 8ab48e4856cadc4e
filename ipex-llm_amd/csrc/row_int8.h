// Products of two operands in 8-bit integers with a scale for each row: what the kernels share.
//
// A weight [N, K] is row-major int8 codes with one float32 scale for each row; activations are quantized by row in the call:
//     a = max |x[m, :]| (2^-100 at least), xs[m] = a / 127, xc[m, k] = x[m, k] * 127 / a to the nearest, ties to even, decided exactly
//     y[m, n] = xs[m] * ws[n] * sum_k xc[m, k] * wc[n, k]
// A row that holds a NaN or an infinity has the scale NaN and codes of zero.  The sum runs over all of K in 32-bit integers: it is exact in any
// order up to K = 2^17 (127 * 128 * 2^17 < 2^31: a weight's code may be -128, one made here is 127 at most; where both are given, given_codes_plan in
// row_int8_rows.hip), and float32, float16 and bfloat16 rows go through the same product.
//
// v_mfma_i32_16x16x64_i8 takes 16 bytes of a lane (row l & 15, g = l >> 4).  Two of them take 128 values of a row in the 16-byte chunks g and
// 4 + g: the order of the terms is free as long as both operands agree, and a load of one chunk by 64 lanes covers 64 contiguous bytes of 16 rows.
#pragma once
#include "block_fp8_gemm.h"

namespace lowbit {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int INT8_BLOCK = 128;                              // values of K that a step of the products takes
constexpr int INT8_MOST_K = 1 << 17;
constexpr uint32_t INFINITE_BITS = 0x7f800000u;

__host__ __device__ inline int int8_blocks(int k) { return (k + INT8_BLOCK - 1) / INT8_BLOCK; }

// D[i][j] += sum over 128 of A[i][k] B[j][k]: lane l holds D[4 * (l >> 4) + 0..3][l & 15]
__device__ inline i32x4 int8_dot(const Codes &a, const Codes &b, i32x4 d) {
    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a.lo), __builtin_bit_cast(i32x4, b.lo), d, 0, 0, 0);
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a.hi), __builtin_bit_cast(i32x4, b.hi), d, 0, 0, 0);
}

// (2^-100 at least, as block_fp8.h's)
__device__ inline float least_magnitude(uint32_t largest_bits) { return __builtin_bit_cast(float, max_u32(largest_bits, FP8_LEAST_BITS)); }

// the scale of a row whose largest magnitude has these bits
__device__ inline float row_scale(uint32_t largest_bits) {
    return largest_bits >= INFINITE_BITS ? __builtin_nanf("") : least_magnitude(largest_bits) / 127.0f;
}

// Codes of a row's values.
//
// x * (127 / a) in float32 is off by less than 127 * 2^-23 = 1.6e-5, half a unit of the reciprocal and half of the product.  Adding 1.5 * 2^23
// rounds it to a whole number, to the nearest with ties to even, whose two's complement lies in the sum's low byte.  Where some value lies
// within 2^-15 of a border between two codes (one wave in 25 for 16 values a lane, or a value of half the largest) all are taken again in 64
// bits, whose quotient is nearer to the true one than that is to a border that it is not on: 254 x and (2 n + 1) a differ by the last place
// of x at least, 2^-32 of the quotient.
struct RowCoder {
    float inv, a;
    uint32_t keep;                                           // 0 where the row is not finite
    __device__ explicit RowCoder(uint32_t largest_bits)
        : inv(127.0f / least_magnitude(largest_bits)), a(least_magnitude(largest_bits)), keep(largest_bits >= INFINITE_BITS ? 0u : ~0u) {}

    static __device__ uint32_t pack(float a, float b, float c, float d) {
        auto bits = [](float v) { return __builtin_bit_cast(uint32_t, v); };
        const uint32_t ab = __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u), cd = __builtin_amdgcn_perm(bits(d), bits(c), 0x0c0c0400u);
        return __builtin_amdgcn_perm(cd, ab, 0x05040100u);
    }
    // V of them (a multiple of four), packed
    template <int V> __device__ void operator()(const float (&x)[V], uint32_t (&codes)[V / 4]) const {
        constexpr float WHOLE = 12582912.0f;
        float m[V], off = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float t = x[i] * inv;
            m[i] = t + WHOLE;
            off = __builtin_fmaxf(off, __builtin_fabsf(t - (m[i] - WHOLE)));
        }
        if (off > 0.5f - 0x1p-15f) {
#pragma unroll
            for (int i = 0; i < V; i++) m[i] = (float)__builtin_rint((double)x[i] * 127.0 / (double)a) + WHOLE;
        }
#pragma unroll
        for (int i = 0; i < V / 4; i++) codes[i] = pack(m[4 * i], m[4 * i + 1], m[4 * i + 2], m[4 * i + 3]) & keep;
    }
};

// The largest magnitude (as bits) of V values
template <int V> __device__ inline uint32_t largest_of(const float (&v)[V]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; i++) m = max_u32(m, magnitude(v[i]));
    return m;
}
// .. over the wave, the same in every lane: of rows of 16, handed on to the second and fourth, then to the last two
__device__ inline uint32_t max_of_wave(uint32_t v) {
    v = max_of_16(v);
    v = max_u32(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = max_u32(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// One row of K values by the threads t of WAVES waves, 16 values per thread and piece; what lies past the first HELD pieces is read again behind
// the row's maximum.  Codes go to ldc bytes, zeros from K up to ldc.  Returns the scale.
template <typename AT, int WAVES, int HELD> __device__ __forceinline__ float quantize_row(const AT *__restrict__ from, uint8_t *__restrict__ to, int K, int ldc, int t) {
    constexpr int STEP = 64 * WAVES * 16;
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
    auto put = [&](int k, const float (&u)[16]) __attribute__((always_inline)) {
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
    return row_scale(m);
}

}  // namespace lowbit
