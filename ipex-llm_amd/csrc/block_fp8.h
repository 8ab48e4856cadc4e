// Products of two e4m3 operands with a scale for each block of 128: what the kernels share.
//
// A weight [N, K] is row-major e4m3 codes with one float32 scale for each 128 x 128 block, scale[N / 128][K / 128] (rounded up; the last
// blocks may end short).  Activations are quantized by row, one scale for each 128 values:
//     a = max |x| over the block (2^-100 at least), scale = a / 448, code = e4m3(x * 448 / a), to the nearest, ties to even.
//     y[m, n] = sum_kb xs[m, kb] * ws[n / 128, kb] * sum_{k in kb} xc[m, k] * wc[n, k]
// The inner sum is one v_mfma_f32_16x16x128_f8f6f4 per 16 x 16 results.  Both operands take their 32 bytes of a lane (row l & 15, g =
// l >> 4) as the 16-byte chunks g and 4 + g of the row's 128: the order of the terms is free as long as both agree, and a load of one chunk
// by 64 lanes covers 64 contiguous bytes of 16 rows.
//
// The instruction aligns the products of a small group of neighbours to the largest of them and keeps 13 bits below its leading one
// (measured: beside 2^12 a product's part below 2^-1 is lost; products in other groups, and the sum over groups, keep float32's 24).
// Of the norm of products of activations and normal weights that is 1.4e-5 (1.6 at most) for N(0, 1) activations, 2e-5 to 3.4e-5 where one
// channel in 100 to 500 is 20 times as loud, 5e-5 (5.6) for lognormal ones of deviation 1.5: a hundredth to a thirtieth of what rounding to
// bfloat16 costs, a fifteenth to a quarter of float16's.  Where large terms cancel it is as much of their root of squares, 3.5e-6 of it in
// neighbours of opposite signs, and more of the result.  Results in float32 therefore go through the bfloat16 MFMA, which keeps 24 bits:
// codes are exact in bfloat16.
#pragma once
#include "lowbit_mfma.h"

namespace lowbit {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int FP8_BLOCK = 128;
constexpr float FP8_LEAST = 0x1p-100f;                       // least magnitude that a block's scale is made for
constexpr uint32_t FP8_LEAST_BITS = 27u << 23;

// A launch has fewer than 2^32 threads in a row of its grid
constexpr int64_t most_groups(int threads) { return ((int64_t)1 << 32) / threads - 8; }

__host__ __device__ inline int fp8_blocks(int k) { return (k + FP8_BLOCK - 1) / FP8_BLOCK; }

// eight codes as bfloat16, exactly: an operand of the bfloat16 MFMA
__device__ inline bf16x8 widen8(uint32_t w0, uint32_t w1) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true);
    return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// 32 bytes of one row: chunks g and 4 + g of a block of 128.
struct Codes {
    u32x4 lo, hi;
};

__device__ inline i32x8 joined(const Codes &c) {
    return {(int)c.lo[0], (int)c.lo[1], (int)c.lo[2], (int)c.lo[3], (int)c.hi[0], (int)c.hi[1], (int)c.hi[2], (int)c.hi[3]};
}

// D[i][j] = sum over 128 of A[i][k] B[j][k]: lane l holds D[4 * (l >> 4) + 0..3][l & 15]
template <bool EXACT> __device__ inline f32x4 block_dot(const Codes &a, const Codes &b) {
    const f32x4 zero = {};
    if constexpr (!EXACT) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(joined(a), joined(b), zero, 0, 0, 0, 0, 0, 0);     // formats e4m3, no block exponents
    } else {
        f32x4 d = zero;
#pragma unroll
        for (int h = 0; h < 2; h++) d = mfma16(widen8(a.lo[2 * h], a.lo[2 * h + 1]), widen8(b.lo[2 * h], b.lo[2 * h + 1]), d);
#pragma unroll
        for (int h = 0; h < 2; h++) d = mfma16(widen8(a.hi[2 * h], a.hi[2 * h + 1]), widen8(b.hi[2 * h], b.hi[2 * h + 1]), d);
        return d;
    }
}

// The larger of two magnitudes as bit patterns: unlike fmax this keeps a NaN, whose pattern is above infinity's.
__device__ inline uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ inline uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL> __device__ inline uint32_t max_dpp(uint32_t v) {
    return max_u32(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
// over the 8 (16) lanes l & ~7 (l & ~15) ..
__device__ inline uint32_t max_of_8(uint32_t v) { return max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(v))); }
__device__ inline uint32_t max_of_16(uint32_t v) { return max_dpp<0x140>(max_of_8(v)); }

__device__ inline float block_scale(uint32_t largest_bits) {
    return __builtin_bit_cast(float, max_u32(largest_bits, FP8_LEAST_BITS)) / 448.0f;       // (correctly rounded: see the build's flags)
}

// x * 448 / a, rounded once to float32.
//
// 16-bit x: with X, A < 2^11 the quotient 448 X / A is a border of two codes (an odd C / 2, C < 2^5, times a power of two) exactly or
// differs from it by 2^-16 of itself at least (7 X against C A, whole numbers below 2^14 and 2^16 up to powers of two).  The product with
// a reciprocal is off by up to 3 units of 2^-24, and dropping its last 4 bits, rounded, puts it back on the border where it belongs
// there and moves it across none: three instructions in place of a division's ten.
// float32 x: in 64 bits, since no such gap is there.
template <typename AT> struct Quotient {
    float inv;
    __device__ Quotient(float scale, uint32_t) : inv(__builtin_amdgcn_rcpf(scale)) {}
    __device__ float operator()(float x) const {
        return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x * inv) + 8u) & ~15u);
    }
};
template <> struct Quotient<float> {
    double inv;
    __device__ Quotient(float, uint32_t largest_bits)
        : inv(1.0 / (double)__builtin_bit_cast(float, max_u32(largest_bits, FP8_LEAST_BITS))) {}
    __device__ float operator()(float x) const { return (float)((double)x * 448.0 * inv); }
};

__device__ inline uint32_t encode4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// 16 values of AT from memory (16-byte aligned) as float32
template <typename AT> __device__ inline void load16(const AT *p, float (&v)[16]) {
    if constexpr (sizeof(AT) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x4 q = ((const f32x4 *)p)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) v[4 * i + j] = q[j];
        }
    } else {
        using V8 = typename Vec8<AT>::type;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const V8 q = ((const V8 *)p)[i];
#pragma unroll
            for (int j = 0; j < 8; j++) v[8 * i + j] = (float)q[j];
        }
    }
}

// Quantizes one block of a row: the 8 lanes l & ~7 .. hold 16 values each (zeros where the row has ended).  Returns the codes of the
// lane's 16 and the block's scale.
template <typename AT> __device__ inline u32x4 quantize16(const float (&v)[16], float &scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m = max_u32(m, magnitude(v[i]));
    m = max_of_8(m);
    scale = block_scale(m);
    const Quotient<AT> q(scale, m);
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = encode4(q(v[4 * i]), q(v[4 * i + 1]), q(v[4 * i + 2]), q(v[4 * i + 3]));
    return c;
}

// One block of a row from 16 neighbouring lanes of 8 values each: their codes to LDS, and the block's scale (first: the block's first lane).
template <typename AT, typename V8> __device__ inline void put8(const V8 &v, uint8_t *codes, float *scale, bool first) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max_u32(m, magnitude((float)v[i]));
    m = max_of_16(m);
    const float s = block_scale(m);
    const Quotient<AT> q(s, m);
    *(u32x2 *)codes = u32x2{encode4(q((float)v[0]), q((float)v[1]), q((float)v[2]), q((float)v[3])),
                            encode4(q((float)v[4]), q((float)v[5]), q((float)v[6]), q((float)v[7]))};
    if (first) *scale = s;
}

// 16 codes of a row to its k-th byte, or (WIDE) the same numbers in bfloat16
template <bool WIDE> __device__ inline void store16(uint8_t *row, int k, u32x4 c) {
    if constexpr (WIDE) {
        *(bf16x8 *)(row + 2 * k) = widen8(c[0], c[1]);
        *(bf16x8 *)(row + 2 * k + 16) = widen8(c[2], c[3]);
    } else *(u32x4 *)(row + k) = c;
}

// Which rows a workgroup of a product grouped by expert works on: row tiles of ROWS rows, expert after expert; called by whole waves.
// Returns false past the last.
struct ExpertTile {
    int expert, first, end;                                  // rows first .. end - 1 (end: the expert's, not the tile's)
};
template <int ROWS> __device__ inline bool find_expert_tile(const int32_t *__restrict__ offsets, int n_exp, int tile, ExpertTile &t) {
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < n_exp; e0 += 64) {
        const int e = e0 + lane;
        const int from = e < n_exp ? offsets[e] : 0, to = e < n_exp ? offsets[e + 1] : 0;
        int before = (to - from + ROWS - 1) / ROWS;
        const int own = before;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(before, d);
            if (lane >= d) before += up;
        }
        const int all = __builtin_amdgcn_readlane(before, 63);
        if (tile < all) {
            const uint64_t hit = __ballot(before > tile);
            const int l = __builtin_ctzll(hit);
            t.expert = e0 + l;
            t.first = __builtin_amdgcn_readlane(from, l) + (tile - (__builtin_amdgcn_readlane(before, l) - __builtin_amdgcn_readlane(own, l))) * ROWS;
            t.end = __builtin_amdgcn_readlane(to, l);
            return true;
        }
        tile -= all;
    }
    return false;
}

// Number of row tiles of all experts.
template <int ROWS> __device__ inline int count_expert_tiles(const int32_t *__restrict__ offsets, int n_exp) {
    int all = 0;
    for (int e = threadIdx.x & 63; e < n_exp; e += 64) all += (offsets[e + 1] - offsets[e] + ROWS - 1) / ROWS;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d);
    return __builtin_amdgcn_readfirstlane(all);
}

// act(g) in float32.  tanh-GELU as g * sigmoid(2 u), in which nothing cancels: 1 - 1 / (1 + e^2u) is zero from g of about -5 on, where the
// values of a block may all lie.  Hardware exp2 and reciprocal are within 2^-23; the exponent's own roundings, half a unit each, count as
// much as it is large: 2^-24 times 2 |g| (SiLU) and up to 18 |u| (GELU, whose exponent takes nine), ahead of a rounding to 4 bits.
__device__ inline float gate_act(float g, int act) {
    if (act == 0) return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
    const float u = 0.7978845608028654f * (g + 0.044715f * g * g * g);
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.8853900817779268f * u));           // 0.5 g (1 + tanh u)
}

}  // namespace lowbit
