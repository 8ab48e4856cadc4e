// The gradient that flows on below a product with a weight in e4m3 and a scale for each block of 128 (block_fp8.h):
//     gx[m, k] = sum_nb ws[nb, k / 128] * sum_{n in nb} g[m, n] * wc[n, k]
//
// g stays in 16 bits: codes are exact in either 16-bit type, so the products are exact, the sums float32 and the result is rounded once.
//
// The sum runs along N, across the rows of the weight, and an MFMA operand needs eight values of n per lane: codes go to LDS row by row
// by LDS-DMA, and ds_read_b64_tr_b8 hands lane i of 16 lanes byte i of eight rows; four conversions make them an operand.  g's rows lie in
// LDS 64 values at a time, as codes of x do in the forward (block_fp8_gemm.h has the layout, the order of loads and the barrier ahead
// of the last tile, which are the same here).  A step is 64 values of n; two steps, a block, are summed from zero by the MFMA and
// then added to the float32 sums times the block's scale, while the next block's first products run.
//
// Bound by the issue of MFMAs between barriers: 8192^3 975 to 1020 us, 1.1 PFLOP/s, where the library's dense product takes 850; 2048 x 4096
// (N) x 11008 in 187, of which a tenth is the third round of 688 tiles.  Three buffers or five make no difference.
#include "block_fp8_tiled.h"

namespace lowbit {

struct BackArgs {
    const void *g;                                           // [M, N] in rows of ldg values, 16-byte aligned; zeros from N up to ldg, if any
    const uint8_t *w;
    const float *ws;
    void *gx;
    float *part;                                             // sums of a split: [split][M][K]
    int64_t ldg;
    int M, N, K, NB, KB;
    int tiles_m, tiles_k, splits, split_blocks;
};

__device__ const __attribute__((aligned(16))) uint32_t NOTHING[4] = {0, 0, 0, 0};

template <typename AT> struct Widen;
template <> struct Widen<__bf16> {
    static __device__ bf16x8 of(u32x2 c) { return widen8(c[0], c[1]); }
};
template <> struct Widen<_Float16> {
    static __device__ f16x8 of(u32x2 c) {
        const f16x2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], 1.0f, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], 1.0f, true);
        const f16x2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], 1.0f, false), s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], 1.0f, true);
        return {p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
    }
};

constexpr int BACK_STEP = 64;                                // values of n per step

// WM x WK waves of TM * 16 rows of g by TK * 16 columns of the weight; S buffers.
template <typename AT, bool PART, int TM, int TK, int WM, int WK, int S, int MIN_WAVES>
__global__ __launch_bounds__(64 * WM * WK, MIN_WAVES) void block_fp8_back_kernel(const BackArgs p) {
    using V8 = typename Vec8<AT>::type;
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
    const int b0 = split * p.split_blocks, b1 = PART && b0 + p.split_blocks < p.NB ? b0 + p.split_blocks : p.NB;

    // ---- sources of this wave's pieces of 8 rows of 128 bytes.  Weights: 64 rows of n for each 128 columns
    const int piece_row = lane >> 3;
    const uint64_t gbase = (uint64_t)(uintptr_t)p.g + (uint64_t)m0 * p.ldg * 2;
    const uint64_t zeros = (uint64_t)(uintptr_t)NOTHING;
    uint32_t goff[PX], wcol[PW];
    int wrow[PW];
#pragma unroll
    for (int j = 0; j < PX; j++) {
        const int row = (wave * PX + j) * 8 + piece_row, m = m0 + row < p.M ? row : p.M - 1 - m0;
        goff[j] = (uint32_t)m * (uint32_t)(p.ldg * 2) + ((lane & 7) ^ swizzle(row)) * 16;
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
        const int n0 = step * BACK_STEP;
        if (q < PX) {
            const uint64_t from = gbase + (uint64_t)n0 * 2;
            if (n0 + BACK_STEP > p.ldg) {                    // values past N: zeros
                const int row = (wave * PX + q) * 8 + piece_row, chunk = (lane & 7) ^ swizzle(row);
                dma16_at(n0 + chunk * 8 < p.ldg ? from + goff[q] : zeros, lds_g + buffer + q * 1024);
            } else dma16(goff[q], from, lds_g + buffer + q * 1024);
        } else {
            // rows past N: the last one, which g multiplies by zero (a NaN of its own is in the result anyway)
            const int j = q - PX, first = n0 < p.N ? n0 : p.N - 1, row = n0 + wrow[j] < p.N ? n0 + wrow[j] - first : p.N - 1 - first;
            dma16((uint32_t)row * (uint32_t)p.K + wcol[j], (uint64_t)(uintptr_t)p.w + (uint64_t)first * p.K + k0, lds_w + buffer + j * 1024);
        }
    };

    // ---- scales of up to 64 blocks in the lanes of a register
    const int kblock = (k0 + wk * TK * 16) / FP8_BLOCK;
    const float *const wscale = p.ws + (kblock < p.KB ? kblock : p.KB - 1);
    float wheld;
    auto hold = [&](int nb) __attribute__((always_inline)) {
        wheld = wscale[(int64_t)(nb + lane < p.NB ? nb + lane : p.NB - 1) * p.KB];
        asm volatile("" : "+v"(wheld));                      // (waited for here and not in every step)
    };
    auto scale_of = [&](int nb) __attribute__((always_inline)) {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wheld), (nb - b0) & 63));
    };

    // ---- operands of 32 values of n: g's chunk 4 ks + g of row r; of the weight rows 32 ks + 8 g .. of column r of a tile
    const int gread = (wm * TM * 16 + r) * 128, gslot = g ^ swizzle(r);
    auto read_g = [&](int buffer, int ks, int i) __attribute__((always_inline)) {
        return *(const V8 *)(lds + buffer + gread + i * 2048 + (gslot ^ (4 * ks)) * 16);
    };
    const int tr = 8 * g + (r >> 1), column = wk * TK * 16;  // (the 16 lanes of a transposing read: 8 rows of two 8-byte halves)
    const int wread = GBYTES + column / 128 * (BACK_STEP * 128) + tr * 128 + (r & 1) * 8, wslot = (column % 128 / 16) ^ swizzle(tr);
    auto read_w = [&](int buffer, int ks, int t) __attribute__((always_inline)) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        // (32 rows on leave the swizzle as it is; the tile turns bits of the slot)
        uint8_t *const from = lds + buffer + wread + ks * 32 * 128 + ((wslot ^ t) * 16);
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2 *)from));
    };

    constexpr int TILE = TM, COUNT = 2 * TK * TM, PER = (PIECES + COUNT - 1) / COUNT, IN_FLIGHT = (S - 2) * PIECES;
    static_assert(IN_FLIGHT < 64, "vmcnt has 6 bits");
    f32x4 acc[TK][TM] = {}, part[TK][TM];
    V8 b[2][TM];
    u32x2 a[2];
    const int s0 = b0 * 2, s1 = b1 * 2, last = s1 - 1;       // steps (the last may lie past N: zeros)
    auto fetch_slot = [&](int step, int which, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int q = slot * PER; q < (slot + 1) * PER && q < PIECES; q++) fetch(step < last ? step : last, which, q);
    };
    float s = 0.0f;
    auto add = [&](int t, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; j++) acc[t][i][j] = fmaf(s, part[t][i][j], acc[t][i][j]);
        asm volatile("" : "+v"(acc[t][i]));
    };

    hold(b0);
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
    for (int i = 0; i < TILE; i++) fetch_slot(s0 + S - 1, S - 1, i);
    // FRESH: the first step of a block, whose first products start from zero once the last block's sums are added
    auto step = [&](int st, auto fresh) __attribute__((always_inline)) {
        constexpr bool FRESH = decltype(fresh)::value;
        const int buffer = which * BUFFER, then = which + 1 < S ? which + 1 : 0, other = then * BUFFER, behind = which > 0 ? which - 1 : S - 1;
        V8 v;
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
                v = Widen<AT>::of(a[tile & 1]);
                a[(tile + 1) & 1] = tile + 1 < 2 * TK ? read_w(buffer, (tile + 1) / TK, (tile + 1) % TK) : read_w(other, 0, 0);
            }
            if (tile == 0) b[1][i] = read_g(buffer, 1, i);
            if (tile == 2 * TK - 1) b[0][i] = read_g(other, 0, i);
            if (FRESH && ks == 0) {
                add(t, i);
                part[t][i] = mfma16(v, b[ks][i], f32x4{});
            } else part[t][i] = mfma16(v, b[ks][i], part[t][i]);
            if (o < COUNT - TM) fetch_slot(st + S - 1, behind, TM + o);
            else fetch_slot(st + S, which, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        which = then;
    };
#pragma unroll
    for (int t = 0; t < TK; t++)
#pragma unroll
        for (int i = 0; i < TM; i++) part[t][i] = f32x4{};
    for (int nb = b0; nb < b1; nb++) {
        if (((nb - b0) & 63) == 0 && nb != b0) {
            s = scale_of(nb - 1);                            // (of the last block that the register holds)
            hold(nb);
        } else if (nb != b0) s = scale_of(nb - 1);
        step(nb * 2, std::true_type());
        step(nb * 2 + 1, std::false_type());
    }
    s = scale_of(b1 - 1);
#pragma unroll
    for (int t = 0; t < TK; t++)
#pragma unroll
        for (int i = 0; i < TM; i++) add(t, i);
    wait_all_loads();

    // results: lane = row r of g's tile i, columns 4 g .. of tile t
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + (wm * TM + i) * 16 + r;
        if (m >= p.M) continue;
#pragma unroll
        for (int t = 0; t < TK; t++) {
            const int k = k0 + column + t * 16 + g * 4;
            if (k >= p.K) continue;
            if constexpr (PART) *(f32x4 *)(p.part + ((int64_t)split * p.M + m) * p.K + k) = acc[t][i];
            else {
                typedef AT out4 __attribute__((ext_vector_type(4)));
                out4 o;
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = to_at<AT>(acc[t][i][j]);
                *(out4 *)((AT *)p.gx + (int64_t)m * p.K + k) = o;
            }
        }
    }
}

// Rows of g that do not start at 16-byte boundaries: a copy in rows of ldg values, zeros past N.
__global__ __launch_bounds__(256) void block_fp8_pad_kernel(const uint16_t *__restrict__ g, uint16_t *__restrict__ to, int N, int ldg) {
    const int n = (blockIdx.x * 256 + threadIdx.x) * 8;
    if (n >= ldg) return;
    const uint16_t *const from = g + (int64_t)blockIdx.y * N + n;
    u32x4 v = {};
    if (n + 8 <= N) __builtin_memcpy(&v, from, sizeof(v));   // (rows start at odd places)
    else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (n + j < N) v[j / 2] |= (uint32_t)from[j] << (16 * (j & 1));
    }
    *(u32x4 *)(to + (int64_t)blockIdx.y * ldg + n) = v;
}

static int cdiv(int a, int b) { return (a + b - 1) / b; }

// Rows and columns of a tile, workgroups that a CU holds, and a block's time (us) with the GPU full and with one workgroup on a CU.  Each wave
// takes all rows of its tile and 32 columns of it, so that a weight is widened once: at 2048 x 4096 (N) x 11008 waves of 64 x 64 in the
// first form take 195 us where these take 189.
struct BackForm {
    int rows, cols, per_cu;
    float block_us, alone_us;
};
enum { BACK_128, BACK_64, BACK_32, BACK_COUNT };
static const BackForm BACK_FORMS[BACK_COUNT] = {{128, 256, 1, 1.85f, 1.74f}, {64, 128, 2, 1.10f, 0.71f}, {32, 128, 2, 0.85f, 0.64f}};

// The form and the splits of N with the smallest estimate: rounds of workgroups over the GPU, and the sum of the splits, written and read in
// float32.  The constants are fitted to 15000 timed launches of 775 sizes, 1 to 8192 rows by 256 to 16384 (N, K); on as many others the pick
// is 0.5 % above the fastest form and split on average, 34 % at worst (1.5 us).
struct BackPlan {
    int form, splits;
};
static BackPlan back_plan(int M, int N, int K) {
    const int NB = fp8_blocks(N);
    BackPlan best = {BACK_128, 1};
    float least = 0.0f;
    for (int form = 0; form < BACK_COUNT; form++) {
        const BackForm &f = BACK_FORMS[form];
        static const int tried[] = {1, 2, 3, 4, 6, 8};
        const int64_t tiles = (int64_t)cdiv(M, f.rows) * cdiv(K, f.cols);
        for (int splits : tried) {
            if (splits > 1 && (NB < splits || tiles >= 512 || (size_t)splits * M * K * 4 > (size_t)256 << 20)) break;
            float us = tiled_walk_us(f.block_us, f.alone_us, f.per_cu, tiles * splits, cdiv(NB, splits)) + 6.3f;
            if (splits > 1) us += 1.6f + (float)splits * M * K * 8.0f / 5.0e6f;
            if (least == 0.0f || us < least) {
                least = us;
                best = {form, splits};
            }
        }
    }
    best.splits = cdiv(NB, cdiv(NB, best.splits));           // (every split has a block)
    return best;
}

void block_fp8_back_plan(int M, int N, int K, int *plan4) {
    const BackPlan plan = back_plan(M, N, K);
    plan4[0] = BACK_FORMS[plan.form].rows;
    plan4[1] = BACK_FORMS[plan.form].cols;
    plan4[2] = plan.splits;
    plan4[3] = 1;
}

static bool padded(int N) { return N % 8 != 0; }
static size_t padded_bytes(int M, int N) { return padded(N) ? ((size_t)M * (cdiv(N, BACK_STEP) * BACK_STEP) * 2 + 255) & ~(size_t)255 : 0; }

size_t block_fp8_back_workspace_bytes(int dtype, int M, int N, int K) {
    const BackPlan plan = back_plan(M, N, K);
    return padded_bytes(M, N) + (plan.splits > 1 ? (size_t)plan.splits * M * K * 4 : 0);
}

void launch_block_fp8_reduce(const float *part, const void *bias, void *y, int dtype, int M, int N, int splits, hipStream_t st);

template <typename AT, bool PART> static void launch_back(const BackArgs &p, int form, hipStream_t st) {
    const uint32_t units = (uint32_t)(p.tiles_m * p.tiles_k * p.splits);
    const dim3 grid((units + 7) / 8 * 8);
    if (form == BACK_128) hipLaunchKernelGGL((block_fp8_back_kernel<AT, PART, 8, 2, 1, 8, 4, 2>), grid, dim3(512), 0, st, p);
    else if (form == BACK_64) hipLaunchKernelGGL((block_fp8_back_kernel<AT, PART, 4, 2, 1, 4, 4, 2>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((block_fp8_back_kernel<AT, PART, 2, 2, 1, 4, 5, 2>), grid, dim3(256), 0, st, p);
}

int launch_block_fp8_back(const void *grad, const uint8_t *w, const float *ws, void *gx, int dtype, int M, int N, int K, uint8_t *space,
                          hipStream_t st) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    const BackPlan plan = back_plan(M, N, K);
    BackArgs p = {grad, w, ws, gx, (float *)(space + padded_bytes(M, N)), N, M, N, K, fp8_blocks(N), fp8_blocks(K),
                  cdiv(M, BACK_FORMS[plan.form].rows), cdiv(K, BACK_FORMS[plan.form].cols), plan.splits, cdiv(fp8_blocks(N), plan.splits)};
    if ((int64_t)p.tiles_m * p.tiles_k * p.splits > most_groups(512)) return -3;
    if (padded(N)) {
        p.ldg = cdiv(N, BACK_STEP) * BACK_STEP;
        for (int m = 0; m < M; m += 65535) {
            const dim3 grid(cdiv((int)p.ldg, 2048), M - m < 65535 ? M - m : 65535);
            hipLaunchKernelGGL(block_fp8_pad_kernel, grid, dim3(256), 0, st, (const uint16_t *)grad + (int64_t)m * N, (uint16_t *)space + m * p.ldg, N, (int)p.ldg);
        }
        p.g = space;
    }
    if (plan.splits > 1) {
        if (dtype == DT_F16) launch_back<_Float16, true>(p, plan.form, st);
        else launch_back<__bf16, true>(p, plan.form, st);
        launch_block_fp8_reduce(p.part, nullptr, gx, dtype, M, K, plan.splits, st);
    } else if (dtype == DT_F16) launch_back<_Float16, false>(p, plan.form, st);
    else launch_back<__bf16, false>(p, plan.form, st);
    return 0;
}

}  // namespace lowbit
