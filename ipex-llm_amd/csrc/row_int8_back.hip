// The gradient that flows on below a product with a weight in int8 and a scale for each row (row_int8.h):
//     gx[m, k] = sum_n g[m, n] * ws[n] * wc[n, k]
//
// The scale lies along the sum, so it goes into g: a launch ahead makes rows of g[m, n] * ws[n] * 2^e in float16, e by row so that the largest
// lies in [2^14, 2^15).  That rounding is half a unit of 2^-11 for every term that is 2^-29 of the row's largest or more, an eighth of
// bfloat16's and as much as float16's own; for float32 g what it leaves goes into a second float16, 22 bits in all, whose sum runs on behind the
// first's.  Codes are exact in float16, the products exact, the sums float32, and the result times 2^-e is rounded once.  A row of g that
// holds a NaN or an infinity (times ws) gives NaN throughout.
//
// The sum runs along N, across the rows of the weight, and an MFMA operand needs eight values of n per lane: codes go to LDS row by row
// by LDS-DMA, and ds_read_b64_tr_b8 hands lane i of 16 lanes byte i of eight rows; a byte c + 128 beside 0x64 is 1152 + c in float16, which
// one subtraction makes c.  g's rows lie in LDS 64 values at a time, as codes of x do in the forward (row_int8_gemm.h has the layout, the order
// of loads and the barrier ahead of the last tile, which are the same here).  A step is 64 values of n.
#include "row_int8_tiled.h"

#include <type_traits>

namespace lowbit {

struct Int8Back {
    const uint8_t *g;                                        // float16 [M][terms][ldg], zeros from N up to ldg
    const int32_t *gs;                                       // [M]: -e, or NOT_FINITE
    const uint8_t *w;
    void *gx;
    float *part;                                             // sums of a split: [split][M][K]
    int64_t ldg;
    int M, N, K, steps, all_steps;                           // steps of one term, of both
    int tiles_m, tiles_k, splits, split_steps;
};

constexpr int32_t NOT_FINITE = 1 << 20;

// a sum times 2^-e, in one rounding also where the result is below the normal numbers
__device__ inline float lowered(float v, int32_t by) { return by == NOT_FINITE ? __builtin_nanf("") : __builtin_ldexpf(v, by); }

// eight codes as float16, exactly
__device__ inline f16x8 codes_f16(u32x2 c) {
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    f16x8 o;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t u = c[i] ^ 0x80808080u;
        const f16x2 p = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
        const f16x2 q = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
        o[4 * i] = p[0]; o[4 * i + 1] = p[1]; o[4 * i + 2] = q[0]; o[4 * i + 3] = q[1];
    }
    return o;
}

constexpr int BACK_STEP = 64;                                // values of n per step

// One row of g per workgroup: its largest |g * ws| first, then the float16 rows.  What lies past the first HELD pieces of 8 is read again.
template <typename AT, int HELD>
__global__ __launch_bounds__(256) void row_int8_scale_grad_kernel(const AT *__restrict__ g, const float *__restrict__ ws, _Float16 *__restrict__ to,
                                                                  int32_t *__restrict__ gs, int N, int64_t ldg) {
    constexpr int TERMS = sizeof(AT) == 4 ? 2 : 1;
    typedef AT v8 __attribute__((ext_vector_type(8)));
    __shared__ uint32_t part[4];
    const int t = threadIdx.x;
    const int64_t m = blockIdx.x;
    const AT *const from = g + m * N;
    _Float16 *const row = to + m * TERMS * ldg;
    // g * ws times a power of two, which goes to the smaller of the two first: products below float32's normal numbers keep their bits
    auto load = [&](int n, float (&v)[8], float pre) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
        auto times = [&](float a, float s) {
            if (pre == 1.0f) return a * s;
            return __builtin_fabsf(a) < __builtin_fabsf(s) ? a * pre * s : s * pre * a;
        };
        if (n + 8 <= N) {
            v8 u;
            __builtin_memcpy(&u, from + n, sizeof(u));       // (rows may start at odd places)
            f32x4 s[2];
            __builtin_memcpy(s, ws + n, sizeof(s));
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = times((float)u[j], s[j / 4][j & 3]);
        } else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < N) v[j] = times((float)from[n + j], ws[n + j]);
    };
    float v[HELD][8];
    auto look = [&](float pre) __attribute__((always_inline)) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < HELD; i++) load((i * 256 + t) * 8, v[i], pre);
#pragma unroll
        for (int i = 0; i < HELD; i++) most = max_u32(most, largest_of(v[i]));
        for (int n = (HELD * 256 + t) * 8; n < N; n += 2048) {
            float more[8];
            load(n, more, pre);
            most = max_u32(most, largest_of(more));
        }
        most = max_of_wave(most);
        if ((t & 63) == 0) part[t >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) most = max_u32(most, part[i]);
        return most;
    };
    uint32_t most = look(1.0f);
    int raised = 0;                                          // what the products have been multiplied by already, 2^64 where all are tiny
    if (most < (67u << 23)) {                                // (2^-60; the same for the whole workgroup)
        __syncthreads();
        raised = 64;
        most = look(0x1p64f);
    }
    const float pre = raised ? 0x1p64f : 1.0f;
    const bool finite = most < INFINITE_BITS;
    // e = 14 - exponent of the largest; of products below 2^-64 after the raise (2^-128 before) as of those: up is 2^78 there at most
    const int exponent = (int)((finite ? most : 0u) >> 23) - 127, e = 14 - (exponent < -64 ? -64 : exponent);
    const float up = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
    auto put = [&](int n, const float (&u)[8]) {
        if (n >= ldg) return;
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float s = finite ? u[j] * up : 0.0f;
            hi[j] = (_Float16)s;
            lo[j] = (_Float16)(s - (float)hi[j]);
        }
        *(f16x8 *)(row + n) = hi;
        if constexpr (TERMS == 2) *(f16x8 *)(row + ldg + n) = lo;
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) put((i * 256 + t) * 8, v[i]);
    for (int n = (HELD * 256 + t) * 8; n < ldg; n += 2048) {
        float more[8];
        load(n, more, pre);
        put(n, more);
    }
    if (t == 0) gs[m] = finite ? -e - raised : NOT_FINITE;
}

// WM x WK waves of TM * 16 rows of g by TK * 16 columns of the weight; S buffers.
template <typename OT, bool PART, int TM, int TK, int WM, int WK, int S, int MIN_WAVES>
__global__ __launch_bounds__(64 * WM * WK, MIN_WAVES) void row_int8_back_kernel(const Int8Back p) {
    constexpr int WAVES = WM * WK, BM = WM * TM * 16, BK = WK * TK * 16, PX = BM / 8 / WAVES, PW = BK / 128 * 8 / WAVES, PIECES = PX + PW;
    static_assert(BM / 8 % WAVES == 0 && BK / 128 * 8 % WAVES == 0 && BK % 128 == 0 && 128 % (TK * 16) == 0 && S > 2, "whole pieces per wave");
    constexpr uint32_t GBYTES = BM * 128, BUFFER = GBYTES + BK * BACK_STEP;
    __shared__ __attribute__((aligned(16))) uint8_t lds[S * BUFFER];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int wm = wave / WK, wk = wave % WK;

    // (runs of tiles to the XCDs in turn, as in the forward)
    const uint32_t units = (uint32_t)(p.tiles_m * p.tiles_k * p.splits), xcd = blockIdx.x & 7;
    const uint32_t unit = (uint32_t)((uint64_t)units * xcd >> 3) + (blockIdx.x >> 3);
    if (unit >= (uint32_t)((uint64_t)units * (xcd + 1) >> 3)) return;
    const int tile = (int)(unit / p.splits), split = (int)(unit - (uint32_t)tile * p.splits);
    const int per = 8 * p.tiles_k, band = tile / per, at = tile - band * per, band_rows = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
    const int tk = at / band_rows, m0 = (band * 8 + at - tk * band_rows) * BM, k0 = tk * BK;
    const int s0 = split * p.split_steps, s1 = PART && s0 + p.split_steps < p.all_steps ? s0 + p.split_steps : p.all_steps, last = s1 - 1;

    // ---- sources of this wave's pieces of 8 rows of 128 bytes.  Weights: 64 rows of n for each 128 columns
    const int piece_row = lane >> 3;
    const int64_t row_bytes = (int64_t)p.ldg * 2 * (p.all_steps / p.steps);
    const uint64_t gbase = (uint64_t)(uintptr_t)p.g + (uint64_t)m0 * row_bytes;
    uint32_t goff[PX], wcol[PW];
    int wrow[PW];
#pragma unroll
    for (int j = 0; j < PX; j++) {
        const int row = (wave * PX + j) * 8 + piece_row, m = m0 + row < p.M ? row : p.M - 1 - m0;
        goff[j] = (uint32_t)m * (uint32_t)row_bytes + ((lane & 7) ^ swizzle(row)) * 16;
    }
#pragma unroll
    for (int j = 0; j < PW; j++) {
        const int piece = wave * PW + j, row = piece % 8 * 8 + piece_row, col = piece / 8 * 128 + ((lane & 7) ^ swizzle(row)) * 16;
        wrow[j] = row;
        wcol[j] = k0 + col < p.K ? col : 0;                  // columns past K: the tile's first ones, for results that are not stored
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const uint32_t lds_g = lds0 + wave * PX * 1024, lds_w = lds0 + GBYTES + wave * PW * 1024;
    auto fetch = [&](int step, int which, int q) __attribute__((always_inline)) {
        const uint32_t buffer = which * BUFFER;
        if (q < PX) dma16(goff[q], gbase + (uint64_t)step * (BACK_STEP * 2), lds_g + buffer + q * 1024);     // (the second term lies behind the first)
        else {
            // rows past N: the last one, which g multiplies by zero
            const int j = q - PX, n0 = (step < p.steps ? step : step - p.steps) * BACK_STEP, row = n0 + wrow[j] < p.N ? wrow[j] : p.N - 1 - n0;
            dma16((uint32_t)row * (uint32_t)p.K + wcol[j], (uint64_t)(uintptr_t)p.w + (uint64_t)n0 * p.K + k0, lds_w + buffer + j * 1024);
        }
    };

    // ---- operands of 32 values of n: g's chunk 4 ks + g of row r; of the weight rows 32 ks + 8 g .. of column r of a tile
    const int gread = (wm * TM * 16 + r) * 128, gslot = g ^ swizzle(r);
    auto read_g = [&](int buffer, int ks, int i) __attribute__((always_inline)) {
        return *(const f16x8 *)(lds + buffer + gread + i * 2048 + (gslot ^ (4 * ks)) * 16);
    };
    const int tr = 8 * g + (r >> 1), column = wk * TK * 16;  // (the 16 lanes of a transposing read: 8 rows of two 8-byte halves)
    const int wread = GBYTES + column / 128 * (BACK_STEP * 128) + tr * 128 + (r & 1) * 8, wslot = (column % 128 / 16) ^ swizzle(tr);
    auto read_w = [&](int buffer, int ks, int t) __attribute__((always_inline)) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        // (32 rows on leave the swizzle as it is; the tile turns bits of the slot)
        uint8_t *const from = lds + buffer + wread + ks * 32 * 128 + ((wslot ^ t) * 16);
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2 *)from));
    };

    constexpr int COUNT = 2 * TK * TM, PER = (PIECES + COUNT - 1) / COUNT, IN_FLIGHT = (S - 2) * PIECES;
    static_assert(IN_FLIGHT < 64, "vmcnt has 6 bits");
    f32x4 acc[TK][TM] = {};
    f16x8 b[2][TM];
    u32x2 a[2];
    auto fetch_slot = [&](int step, int which, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int q = slot * PER; q < (slot + 1) * PER && q < PIECES; q++) fetch(step < last ? step : last, which, q);
    };
#pragma unroll
    for (int v = 0; v < S - 1; v++)
#pragma unroll
        for (int q = 0; q < PIECES; q++) fetch(s0 + v < last ? s0 + v : last, v, q);
    wait_loads_but<IN_FLIGHT>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int which = 0;
#pragma unroll
    for (int i = 0; i < TM; i++) b[0][i] = read_g(0, 0, i);
    a[0] = read_w(0, 0, 0);
#pragma unroll
    for (int i = 0; i < TM; i++) fetch_slot(s0 + S - 1, S - 1, i);
    for (int st = s0; st < s1; st++) {
        const int buffer = which * BUFFER, then = which + 1 < S ? which + 1 : 0, other = then * BUFFER, behind = which > 0 ? which - 1 : S - 1;
        f16x8 v;
#pragma unroll
        for (int o = 0; o < COUNT; o++) {
            const int ks = o / (TK * TM), t = o / TM % TK, i = o % TM, tile = o / TM;
            if (o == COUNT - TM) {
                wait_loads_but<IN_FLIGHT>();
                wait_lds();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == 0) {
                v = codes_f16(a[tile & 1]);
                a[(tile + 1) & 1] = tile + 1 < 2 * TK ? read_w(buffer, (tile + 1) / TK, (tile + 1) % TK) : read_w(other, 0, 0);
            }
            if (tile == 0) b[1][i] = read_g(buffer, 1, i);
            if (tile == 2 * TK - 1) b[0][i] = read_g(other, 0, i);
            acc[t][i] = mfma16(v, b[ks][i], acc[t][i]);
            if (o < COUNT - TM) fetch_slot(st + S - 1, behind, TM + o);
            else fetch_slot(st + S, which, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        which = then;
    }
    wait_all_loads();

    // results: lane = row r of g's tile i, columns 4 g .. of tile t
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + (wm * TM + i) * 16 + r;
        if (m >= p.M) continue;
        const int32_t by = PART ? 0 : p.gs[m];
#pragma unroll
        for (int t = 0; t < TK; t++) {
            const int k = k0 + column + t * 16 + g * 4;
            if (k >= p.K) continue;
            if constexpr (PART) *(f32x4 *)(p.part + ((int64_t)split * p.M + m) * p.K + k) = acc[t][i];
            else {
                typedef OT out4 __attribute__((ext_vector_type(4)));
                out4 o;
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = Stored<OT>::of(lowered(acc[t][i][j], by));
                *(out4 *)((OT *)p.gx + (int64_t)m * p.K + k) = o;
            }
        }
    }
}

// gx = 2^-e * sum of the splits' sums, in their order; four columns per thread
template <typename OT>
__global__ __launch_bounds__(256) void row_int8_back_reduce_kernel(const f32x4 *__restrict__ part, const int32_t *__restrict__ gs, OT *__restrict__ gx, int M,
                                                                   int quads, int splits) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)M * quads) return;
    f32x4 v = part[id];
    for (int s = 1; s < splits; s++) v += part[id + s * (int64_t)M * quads];
    const int32_t by = gs[id / quads];
    typedef OT out4 __attribute__((ext_vector_type(4)));
    out4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = Stored<OT>::of(lowered(v[j], by));
    *(out4 *)(gx + id * 4) = o;
}

static int cdiv(int a, int b) { return (a + b - 1) / b; }

// Rows and columns of a tile, workgroups that a CU holds, and a step's time (us) with the GPU full and with one workgroup on a CU.  In the first
// three each wave takes all rows of its tile and 32 columns of it, so that a weight is widened once; the larger ones (waves of 64 x 64, 128 x 64 and
// 96 x 64) read fewer operands from LDS for a product: 2048 x 4096 (N) x 11008 188 us in tiles of 128 x 256, 163 in 192 x 256, 8192 x 4096 x 4096 232 and
// 210 in 256 x 256.  Fitted to 63 sizes, 16 to 8192 rows by 64 to 28672 (N) by 128 to 16384: the pick is 1.1 % above the fastest form and split on
// average, 16 % at worst.
struct Int8BackForm {
    int rows, cols, per_cu;
    float step_us, alone_us;
};
enum { BACK_128, BACK_64, BACK_32, BACK_128_128, BACK_256, BACK_192, BACK_COUNT };
static const Int8BackForm BACK_FORMS[BACK_COUNT] = {{128, 256, 1, 0.786f, 0.736f}, {64, 128, 2, 0.515f, 0.382f}, {32, 128, 2, 0.475f, 0.347f},
                                                    {128, 128, 2, 0.814f, 0.615f}, {256, 256, 1, 1.35f, 1.32f}, {192, 256, 1, 1.093f, 1.068f}};

struct Int8BackPlan {
    int form, splits;
};
static Int8BackPlan back_plan(int M, int steps, int K) {
    Int8BackPlan best = {BACK_128, 1};
    float least = 0.0f;
    for (int form = 0; form < BACK_COUNT; form++) {
        const Int8BackForm &f = BACK_FORMS[form];
        // (a tile's rows of g lie within 2^31 bytes, 64 of them whatever their length: from 2^21 columns of float32 on, 2^22 of 16 bits, not 256)
        if ((int64_t)f.rows * steps * (BACK_STEP * 2) > (int64_t)1 << 31) continue;
        static const int tried[] = {1, 2, 3, 4, 6, 8};
        const int64_t tiles = (int64_t)cdiv(M, f.rows) * cdiv(K, f.cols);
        for (int splits : tried) {
            if (splits > 1 && (steps < 2 * splits || tiles >= 512 || (size_t)splits * M * K * 4 > (size_t)256 << 20)) break;
            float us = tiled_walk_us(f.step_us, f.alone_us, f.per_cu, tiles * splits, cdiv(steps, splits)) + 3.4f + 0.83e-6f * M * K;
            us += 0.16f * ((tiles * splits - 1) / (256 * f.per_cu));
            if (splits > 1) us += 2.6f + (float)splits * M * K * 8.0f / 5.2e6f;
            if (least == 0.0f || us < least) {
                least = us;
                best = {form, splits};
            }
        }
    }
    best.splits = cdiv(steps, cdiv(steps, best.splits));     // (every split has a step)
    return best;
}

static int back_steps(int dtype, int N) { return cdiv(N, BACK_STEP) * (dtype == DT_F32 ? 2 : 1); }

void row_int8_back_plan(int dtype, int M, int N, int K, int *plan4) {
    const Int8BackPlan plan = back_plan(M, back_steps(dtype, N), K);
    plan4[0] = BACK_FORMS[plan.form].rows;
    plan4[1] = BACK_FORMS[plan.form].cols;
    plan4[2] = plan.splits;
    plan4[3] = 1;
}

// rows of g, their scales, a split's sums
struct BackSpace {
    size_t gs, part, bytes;
};
static BackSpace back_space(int dtype, int M, int N, int K, const Int8BackPlan &plan) {
    auto whole = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    BackSpace s;
    s.gs = whole((size_t)M * back_steps(dtype, N) * BACK_STEP * 2);
    s.part = s.gs + whole((size_t)M * 4);
    s.bytes = s.part + (plan.splits > 1 ? (size_t)plan.splits * M * K * 4 : 0);
    return s;
}

size_t row_int8_back_workspace_bytes(int dtype, int M, int N, int K) {
    return back_space(dtype, M, N, K, back_plan(M, back_steps(dtype, N), K)).bytes;
}

template <typename OT, bool PART> static void launch_back(const Int8Back &p, int form, hipStream_t st) {
    const uint32_t units = (uint32_t)(p.tiles_m * p.tiles_k * p.splits);
    const dim3 grid((units + 7) / 8 * 8);
    if (form == BACK_128) hipLaunchKernelGGL((row_int8_back_kernel<OT, PART, 8, 2, 1, 8, 4, 2>), grid, dim3(512), 0, st, p);
    else if (form == BACK_64) hipLaunchKernelGGL((row_int8_back_kernel<OT, PART, 4, 2, 1, 4, 4, 2>), grid, dim3(256), 0, st, p);
    else if (form == BACK_32) hipLaunchKernelGGL((row_int8_back_kernel<OT, PART, 2, 2, 1, 4, 5, 2>), grid, dim3(256), 0, st, p);
    else if (form == BACK_128_128) hipLaunchKernelGGL((row_int8_back_kernel<OT, PART, 4, 4, 2, 2, 3, 2>), grid, dim3(256), 0, st, p);
    else if (form == BACK_256) hipLaunchKernelGGL((row_int8_back_kernel<OT, PART, 8, 4, 2, 4, 3, 2>), grid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((row_int8_back_kernel<OT, PART, 6, 4, 2, 4, 3, 2>), grid, dim3(512), 0, st, p);
}

int launch_row_int8_back(const void *grad, const uint8_t *w, const float *ws, void *gx, int dtype, int M, int N, int K, uint8_t *space, hipStream_t st) {
    const int all_steps = back_steps(dtype, N), steps = cdiv(N, BACK_STEP);
    const Int8BackPlan plan = back_plan(M, all_steps, K);
    const BackSpace at = back_space(dtype, M, N, K, plan);
    const Int8BackForm &f = BACK_FORMS[plan.form];
    Int8Back p = {space, (int32_t *)(space + at.gs), w, gx, (float *)(space + at.part), (int64_t)steps * BACK_STEP, M, N, K, steps, all_steps,
                  cdiv(M, f.rows), cdiv(K, f.cols), plan.splits, cdiv(all_steps, plan.splits)};
    if ((int64_t)p.tiles_m * p.tiles_k * p.splits > most_groups(512)) return -3;
    auto go = [&](auto *typed) {
        using AT = typename std::remove_cv<typename std::remove_pointer<decltype(typed)>::type>::type;
        if (p.ldg <= 2048) hipLaunchKernelGGL((row_int8_scale_grad_kernel<AT, 1>), dim3(M), dim3(256), 0, st, typed, ws, (_Float16 *)space, (int32_t *)(space + at.gs), N, p.ldg);
        else hipLaunchKernelGGL((row_int8_scale_grad_kernel<AT, 4>), dim3(M), dim3(256), 0, st, typed, ws, (_Float16 *)space, (int32_t *)(space + at.gs), N, p.ldg);
        if (plan.splits == 1) return launch_back<AT, false>(p, plan.form, st);
        launch_back<float, true>(p, plan.form, st);
        const int quads = K / 4;
        hipLaunchKernelGGL((row_int8_back_reduce_kernel<AT>), dim3((uint32_t)(((int64_t)M * quads + 255) / 256)), dim3(256), 0, st, (const f32x4 *)p.part, p.gs,
                           (AT *)gx, M, quads, plan.splits);
    };
    if (dtype == DT_F16) go((const _Float16 *)grad);
    else if (dtype == DT_BF16) go((const __bf16 *)grad);
    else if (dtype == DT_F32) go((const float *)grad);
    else return -4;
    return 0;
}

}  // namespace lowbit
