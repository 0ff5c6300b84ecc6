// Products of 8-bit integers with a scale per row of A and per row of B, and
// the rows' quantisation.  Compiled into hip_gemm.hip.
//
//   x = v (NaN -> 0, magnitudes saturate at FLT_MAX)
//   a = max |x| of a row, s = a / 127 (0 where a < 2^-100), code = rne(x / s)
//   C[m][n] = (as[m] bs[n]) sum_k A[m][k] B[n][k]
// Division, scale and the product of two scales are rounded to fp32; the sums
// are int32 and exact (K <= 131,071: |code| <= 128, so |sum| <= 2^14 K < 2^31),
// so their order, and how K is split, cannot change a result.  The sum's
// conversion to fp32 (exact below 2^24) and its product with the scales round
// once each: 1.5 steps of fp32 in all, far below a code's own error.
#ifndef QH_INT8_KERNELS_H
#define QH_INT8_KERNELS_H

#include <float.h>

#include "gemm_common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));

#define I8_TINY 0x1p-100f
#define I8_MAX_K 131071

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
// a value as its code stands for it: finite
__device__ __forceinline__ float i8_held(float x) {
    x = x == x ? x : 0.0f;
    return fminf(fmaxf(x, -FLT_MAX), FLT_MAX);
}

// rint(x / s), both rounded to fp32 first as the definition has it, without the
// division where it cannot matter: with y = 1 / s rounded (2^-107 <= s < 2^122),
// x y is off x / s by 2^-23 of it, 2^-16 at most, and the quotient's own rounding
// moves it by half of that.  Only a product within 2^-14 of n + 1/2 is divided.
__device__ __forceinline__ int i8_code(float x, float s, float y) {
    float q = x * y, n = rintf(q);
    if (fabsf(fabsf(q - n) - 0.5f) < 0x1p-14f) n = rintf(x / s);
    return (int)n;
}

// eight values from x on, `left` of them there: 16 bytes a load, wherever they
// begin.  ONCE: past the caches
typedef unsigned int i8_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float i8_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint64_t i8_u64 __attribute__((aligned(1)));
template <bool BF, bool ONCE>
__device__ __forceinline__ void i8_eight(float *v, const void *x, size_t i, int left) {
    if (left >= 8) {
        if constexpr (BF) {
            const i8_u32x4 *p = (const i8_u32x4 *)((const uint16_t *)x + i);
            const u32x4 w = ONCE ? __builtin_nontemporal_load(p) : *p;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[2 * j] = bf16_lo(w[j]);
                v[2 * j + 1] = bf16_hi(w[j]);
            }
        } else {
            const i8_f32x4 *p = (const i8_f32x4 *)((const float *)x + i);
            const f32x4 lo = ONCE ? __builtin_nontemporal_load(p) : *p;
            const f32x4 hi = ONCE ? __builtin_nontemporal_load(p + 1) : p[1];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = lo[j];
                v[4 + j] = hi[j];
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        v[j] = j >= left ? 0.0f : BF ? bf16_lo(((const uint16_t *)x)[i + j]) : ((const float *)x)[i + j];
}

// TPR threads a row, in turns of 8 values each.  The first KEEP turns' values stay
// in registers between the maximum and the codes; a longer row's others are read
// again.  Bound by memory: 65,536 x 1,024 fp32 57.4 us (5.8 TB/s; 60.9 through the
// caches), 4,096 x 4,096 16.8 (18.3), bf16 12.8 (15.2); below some MB by the launch
// and two latencies: one row 2.4, 1,999 x 2,048 bf16 6.3.  Many rows: as few threads
// a row as hold it in registers, 30,000 x 64 5.6 us on 16 threads and 13.8 on 64, 30,000
// x 1,500 bf16 36 on 64 with four turns and 60 on 256, 8,000 x 5,000 39 on 256 and 52
// on 1,024.  Few: one turn a thread, a shorter chain, 64 x 1,024 bf16 2.8 us on 256
// threads and 3.3 on 64 (2,000 rows 4.9 and 3.9), 64 x 256 2.7 on 64 and 3.2 on 16, 64 x
// 8,192 4.1 on 1,024 and 4.9 on 256 (1,024 rows 9.9 and 7.2).
template <bool BF, int TPR, int KEEP, bool ONCE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_rows_int8(int8_t *__restrict__ q, size_t ldq, float *__restrict__ scale,
                                                                   const void *__restrict__ x, size_t ldx, int K, int rows) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    const size_t row = (size_t)blockIdx.x * RPB + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    if (TPR <= WAVE && row >= (size_t)rows) return;       // all lanes of a row
    const size_t from = row * ldx;
    float v[KEEP][8], a = 0.0f;
#pragma unroll
    for (int u = 0; u < KEEP; u++) {
        const int k = 8 * (t + u * TPR);
        i8_eight<BF, ONCE>(v[u], x, from + k, K - k);
    }
    for (int k = 8 * (t + KEEP * TPR); k < K; k += 8 * TPR) {
        float w[8];
        i8_eight<BF, ONCE>(w, x, from + k, K - k);
#pragma unroll
        for (int j = 0; j < 8; j++) a = fmaxf(a, fabsf(i8_held(w[j])));
    }
#pragma unroll
    for (int u = 0; u < KEEP; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[u][j] = i8_held(v[u][j]);
            a = fmaxf(a, fabsf(v[u][j]));
        }
#pragma unroll
    for (int m = (TPR < WAVE ? TPR : WAVE) / 2; m >= 1; m >>= 1) a = fmaxf(a, __shfl_xor(a, m));
    if constexpr (TPR > WAVE) {
        __shared__ float red[TPR / WAVE];
        if ((t & 63) == 0) red[t >> 6] = a;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < TPR / WAVE; w++) a = fmaxf(a, red[w]);
    }
    const float s = a < I8_TINY ? 0.0f : a / 127.0f;
    const float y = s == 0.0f ? 0.0f : 1.0f / s;
    if (t == 0) scale[row] = s;
    auto store = [&](const float *w, int k) {
        if (k >= K) return;
        int8_t *to = q + row * ldq + k;
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = s == 0.0f ? 0 : i8_code(w[j], s, y);
        if (k + 8 <= K) {
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                lo |= (uint32_t)(c[j] & 0xFF) << (8 * j);
                hi |= (uint32_t)(c[4 + j] & 0xFF) << (8 * j);
            }
            const uint64_t w8 = lo | (uint64_t)hi << 32;
            if constexpr (ONCE) __builtin_nontemporal_store(w8, (i8_u64 *)to);
            else *(i8_u64 *)to = w8;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k + j < K) to[j] = (int8_t)c[j];
        }
    };
#pragma unroll
    for (int u = 0; u < KEEP; u++) store(v[u], 8 * (t + u * TPR));
    for (int k = 8 * (t + KEEP * TPR); k < K; k += 8 * TPR) {
        float w[8];
        i8_eight<BF, ONCE>(w, x, from + k, K - k);
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = i8_held(w[j]);
        store(w, k);
    }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
struct I8Args {
    void *c;
    size_t ldc;                        // elements
    const int8_t *a;
    size_t lda;                        // bytes
    const float *as;
    const int8_t *b, *b2;              // b2: the up weights of a gated product
    size_t ldb;
    const float *bs, *bs2;
    int M, K, N;
    int whole;                         // pieces of 32 of a row of C are whole lines
};

template <bool CBF>
__device__ __forceinline__ void i8_store(void *c, size_t i, float v) {
    if constexpr (CBF) ((__bf16 *)c)[i] = (__bf16)v;
    else ((float *)c)[i] = v;
}

// silu(g) u = g / (1 + exp(-g)) u, for |g| < I8_SILU_FAR by the hardware's power of two
// of -g log2 e and its reciprocal, in a third of the instructions that the library's
// exponential and division take (1,999 x 1,024 x 2,816 15.4 us, with those 17.4; in bf16
// 14.1 and 16.8).
// For fp32 results the power's remainder is put back and the quotient corrected by its
// own: e is off by 3 half steps of 2^-24, sum, quotient and product by one each, 6 in
// all.  bf16 results go without, which adds 1.23 |g| 2^-24, at most 2^-17.2 where a half
// step of theirs is 2^-8.
#define I8_SILU_FAR 87.0f
template <bool CBF>
__device__ __forceinline__ float i8_silu_near(float g, float u) {
    if constexpr (CBF) return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504e+00f)) * u;
    const float hi = g * -1.44269504e+00f, lo = fmaf(g, -1.92596299e-08f, fmaf(g, -1.44269504e+00f, -hi));
    float e = __builtin_amdgcn_exp2f(hi);
    e = fmaf(e, lo * 6.93147182e-01f, e);
    const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d), q = g * r;
    return fmaf(fmaf(-d, q, g), r, q) * u;
}
// For |g| from there on, where exp(-g) or the reciprocal leaves fp32's range: g u, or,
// 1 + exp(g) being 1, g exp(g) u with half of the exponent on either side of u, so that
// only a result that is subnormal itself passes through subnormal values: 7 half steps.
// exp(g / 2), off by 2 of them, is subnormal for g < -174; that loses less than 2^-244 |u|.
__device__ __forceinline__ float i8_silu_far(float g, float u) {
    const float h = expf(0.5f * fminf(g, 0.0f));
    return g * h * u * h;
}
template <bool CBF>
__device__ __forceinline__ float i8_silu_mul(float g, float u) {
    return fabsf(g) >= I8_SILU_FAR ? i8_silu_far(g, u) : i8_silu_near<CBF>(g, u);
}

// Any strides and addresses: 64 x 64 outputs a block, 64 codes of K a step through
// LDS, four a load wherever they begin, 4 x 4 outputs a thread by v_dot4.
#define I8_ANY 64
template <bool GATED, bool CBF>
__global__ __launch_bounds__(NTHREADS) void k_i8_any(I8Args p, unsigned nt) {
    __shared__ int sa[I8_ANY][I8_ANY / 4 + 1], sb[GATED ? 2 : 1][I8_ANY][I8_ANY / 4 + 1];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const size_t m0 = (size_t)(blockIdx.x / nt) * I8_ANY, n0 = (size_t)(blockIdx.x % nt) * I8_ANY;
    auto four = [&](const int8_t *x, size_t ld, size_t row, int rows, int k) {
        typedef int any_i32 __attribute__((aligned(1)));
        if (row >= (size_t)rows) return 0;
        if (k + 4 <= p.K) return *(const any_i32 *)(x + row * ld + k);
        int w = 0;
        for (int j = 0; j < 3; j++)
            if (k + j < p.K) w |= (int)(uint8_t)x[row * ld + k + j] << (8 * j);
        return w;
    };
    int acc[GATED ? 2 : 1][4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += I8_ANY) {
        for (int i = tid; i < I8_ANY * I8_ANY / 4; i += NTHREADS) {
            const int r = i / (I8_ANY / 4), c = i % (I8_ANY / 4);
            sa[r][c] = four(p.a, p.lda, m0 + r, p.M, k0 + 4 * c);
            sb[0][r][c] = four(p.b, p.ldb, n0 + r, p.N, k0 + 4 * c);
            if constexpr (GATED) sb[GATED][r][c] = four(p.b2, p.ldb, n0 + r, p.N, k0 + 4 * c);
        }
        __syncthreads();
        for (int c = 0; c < I8_ANY / 4; c++)
#pragma unroll
            for (int g = 0; g < (GATED ? 2 : 1); g++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[g][i][j] = __builtin_amdgcn_sdot4(sa[ty + 16 * i][c], sb[g][tx + 16 * j][c], acc[g][i][j], false);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++) {
        const size_t m = m0 + ty + 16 * i;
        if (m >= (size_t)p.M) continue;
        for (int j = 0; j < 4; j++) {
            const size_t n = n0 + tx + 16 * j;
            if (n >= (size_t)p.N) continue;
            float v = (float)acc[0][i][j] * (p.as[m] * p.bs[n]);
            if constexpr (GATED) v = i8_silu_mul<CBF>(v, (float)acc[GATED][i][j] * (p.as[m] * p.bs2[n]));
            i8_store<CBF>(p.c, m * p.ldc + n, v);
        }
    }
}

typedef int i32x16 __attribute__((ext_vector_type(16)));

// What the kernels below take: 16-byte aligned codes in rows of a multiple of
// 16 bytes, so that a row's last piece of 16 may be read whole.  What lies in it
// behind K may be anything: A's bytes there are cleared, and B's then count for
// nothing.  Rows behind M and columns behind N repeat the last ones and are not
// stored.
__device__ __forceinline__ i32x4 i8_keep(i32x4 v, int left) {     // the first `left` of 16 codes, the others 0
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = left - 4 * j;
        v[j] = n >= 4 ? v[j] : n <= 0 ? 0 : (int)((uint32_t)v[j] & ((1u << (8 * n)) - 1));
    }
    return v;
}
__device__ __forceinline__ i32x4 i8_load(const int8_t *p) { return *(const i32x4 *)p; }

// ---------------------------------------------------------------------------
// Few rows, few columns: 16 columns and 16 MT rows a block, K split over its W
// waves
// ---------------------------------------------------------------------------
// D = W X^T with 16x16x64 MFMAs: lane (r, g) = (lane % 16, lane / 16) holds codes
// 16 g .. 16 g + 15 of weight row r (A operand) and of row r of x (B operand),
// and gets rows 4 g + i (columns of C) of column r (a row of C).  Operands come
// straight from memory, a wave's pieces of 128 bytes of each row.  Sums are
// integers, so the waves' may be added in any order.
// Bound by the launch, two latencies and the waves' exchange: 16 x 1024 x 4096 2.9
// us (operands in no cache 3.6), 64 x 2048 x 1024 3.9, where an empty launch takes
// 2.3; for one row by memory, 1 x 1024 x 151936 30.1 us (5.2 TB/s).  4 or 16 waves
// are as fast at K = 1,024 to 8,192.
template <int MT, int W, bool GATED, bool CBF>
__global__ __launch_bounds__(WAVE *W) void k_i8_narrow(I8Args p) {
    constexpr int G = GATED ? 2 : 1;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MT), cols = p.N - n0, rows = p.M - m0;
    const int8_t *wp[G], *xp[MT];
    wp[0] = p.b + (size_t)(n0 + min(r, cols - 1)) * p.ldb;
    if constexpr (GATED) wp[G - 1] = p.b2 + (size_t)(n0 + min(r, cols - 1)) * p.ldb;
#pragma unroll
    for (int t = 0; t < MT; t++) xp[t] = p.a + (size_t)(m0 + min(16 * t + r, rows - 1)) * p.lda;
    struct Set { i32x4 w[2][G], x[2][MT]; };
    auto load = [&](Set &s, int c) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int k = 128 * c + 64 * u + 16 * g, at = k < p.K ? k : 0;
#pragma unroll
            for (int q = 0; q < G; q++) s.w[u][q] = i8_load(wp[q] + at);
#pragma unroll
            for (int t = 0; t < MT; t++) s.x[u][t] = i8_load(xp[t] + at);
        }
    };
    i32x4 acc[G][MT] = {};
    auto multiply = [&](Set &s, int c) {
        if (128 * c + 128 > p.K) {                        // the last piece, not whole
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int t = 0; t < MT; t++) s.x[u][t] = i8_keep(s.x[u][t], p.K - (128 * c + 64 * u + 16 * g));
        }
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int q = 0; q < G; q++)
                    acc[q][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.w[u][q], s.x[u][t], acc[q][t], 0, 0, 0);
    };
    const int pieces = (p.K + 127) / 128;
    Set s0, s1;
    int c = wave;
    if (c < pieces) load(s0, c);
    for (; c < pieces; c += 2 * W) {
        if (c + W < pieces) load(s1, c + W);
        multiply(s0, c);
        if (c + W >= pieces) break;
        if (c + 2 * W < pieces) load(s0, c + 2 * W);
        multiply(s1, c + W);
    }
    __shared__ i32x4 red[W][G][MT][WAVE];
#pragma unroll
    for (int q = 0; q < G; q++)
#pragma unroll
        for (int t = 0; t < MT; t++) red[wave][q][t][lane] = acc[q][t];
    __syncthreads();
    const int *flat = (const int *)red;
    constexpr int OUT = MT * WAVE * 4;                    // sums of one product
    for (int o = tid; o < OUT; o += W * WAVE) {
        const int mo = o / (WAVE * 4) * 16 + (o >> 2 & 15), no = (o >> 6 & 3) * 4 + (o & 3);
        int v[G] = {};
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int q = 0; q < G; q++) v[q] += flat[(w * G + q) * OUT + o];
        if (mo >= rows || no >= cols) continue;
        const int m = m0 + mo, n = n0 + no;
        const float sm = p.as[m];
        float y = (float)v[0] * (sm * p.bs[n]);
        if constexpr (GATED) y = i8_silu_mul<CBF>(y, (float)v[G - 1] * (sm * p.bs2[n]));
        i8_store<CBF>(p.c, (size_t)m * p.ldc + n, y);
    }
}

// ---------------------------------------------------------------------------
// Many rows: tiles through LDS
// ---------------------------------------------------------------------------
// BM x BN outputs a block of WM x WN waves, 32x32x32 MFMAs: lane (c, h) = (lane %
// 32, lane / 32) gives codes 16 h .. 16 h + 15 of row c of either operand and
// holds rows 8 (e / 4) + 4 h + e % 4 of column c of the result.  Stages of 128
// codes of each row are copied from memory straight into one of ST places in LDS,
// 1,024 bytes an instruction; piece c of 16 codes of row r lies at place c ^ f(r)
// of its row, f such that the rows of a fragment meet different banks (the
// conflict counter reads 0), and with a period of 32 rows so that a wave's
// fragments differ by constants.
// A stage is four steps of 32 codes; a step's MFMAs run while the next step's
// fragments are read.  A stage's last step runs behind the barrier: its fragments
// are in registers by then, so the copies of stage kt + ST may start into the same
// place and the first fragments of stage kt + 1 be read while the matrix cores
// still have work (4096 x 4096 x 8192 132 us with the barrier between stages, 124
// so).
// What bounds it: 4096 x 4096 x 8192, bf16 results, 121 us on 256 x 256 tiles, 2.3
// POP/s; without the copies 109, the copies alone 75 to 105.  The matrix cores
// alone reach 3.3 POP/s on such data (the clock falls to two thirds under it; on
// zeros 4.9).  64 x 64 tiles take in 16 KB a stage and are bound by that: 2048 x
// 8192 x 1024 34.3 us, the copies alone 35.  Splitting a stage's codes over waves,
// which halves what is read from LDS, and more stages in flight gained nothing.
// B_AUX: how B is read (2: past the caches)
template <int BM_, int BN_, int WM_, int WN_, int ST_, int B_AUX_ = 0>
struct I8Tile {
    static constexpr int B_AUX = B_AUX_;
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = 128, ST = ST_;
    static constexpr int NW = WM * WN, CPR = BK / 16, RPI = 64 / CPR;    // pieces of a row; rows that a copy instruction fills
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32, KS = BK / 32;
    static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES;
    static constexpr int A_DMA = A_BYTES / 1024 / NW, B_DMA = B_BYTES / 1024 / NW, DMA = A_DMA + B_DMA;
    static_assert(A_DMA * NW * 1024 == A_BYTES && B_DMA * NW * 1024 == B_BYTES, "whole copies a wave");
    static_assert(TM >= 1 && TN >= 1 && ST >= 2 && ST * STAGE <= 160 * 1024, "tile");
    static_assert(STAGE >= 12 * 256, "the scales of a tile in a stage's place");
};
__device__ __forceinline__ int i8_swz(int row) { return (row ^ (row >> 3 & 3)) & 7; }
// 16 bytes a lane from byte at + k0 of a buffer to 1,024 of LDS.  (The host's pass
// knows the builtin, but not the size, and would drop the kernels that use it.)
typedef __attribute__((address_space(3))) void i8_lds;
template <int AUX>
__device__ __forceinline__ void i8_copy(__amdgpu_buffer_rsrc_t from, unsigned char *to, int at, int k0) {
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (i8_lds *)to, 16, at, k0, 0, AUX);
#endif
}
// The compiler moves no LDS access across a barrier.
__device__ __forceinline__ void i8_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
#define I8_VMCNT(n) (0x0070 | ((n) & 15) | ((n) >> 4 << 14))      // s_waitcnt vmcnt(n) lgkmcnt(0)

// The order of a step's instructions in a wave: MFMAs with the next step's
// fragments, and the copies, between them.
template <int I, int PER, int FR, int DMA>
struct I8Order {
    static __device__ __forceinline__ void run() {
        if constexpr (I < PER) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                           // an MFMA
            constexpr int n = (I + 1) * FR / PER - I * FR / PER, m = (I + 1) * DMA / PER - I * DMA / PER;
            if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x100, n, 0);      // LDS reads
            if constexpr (m > 0) __builtin_amdgcn_sched_group_barrier(0x020, m, 0);      // copies
            I8Order<I + 1, PER, FR, DMA>::run();
        }
    }
};

template <typename T, bool GATED, bool CBF>
__global__ __launch_bounds__(WAVE *T::NW, T::NW / 4) void k_i8_tile(I8Args p, int MT, int NT, int per) {
    constexpr int BNO = GATED ? T::BN / 2 : T::BN, ES = CBF ? 2 : 4;
    __shared__ __align__(1024) unsigned char smem[T::ST * T::STAGE];
    // tiles in the order of the XCDs, which get workgroups in turn: each a run of
    // `per` tiles, walked in groups of 8 tile rows, so that what runs together on
    // an XCD shares its L2
    const int local = blockIdx.x >> 3, idx = (blockIdx.x & 7) * per + local;
    if (idx >= MT * NT) return;
    const int first = idx / (8 * NT) * 8, gs = min(MT - first, 8), in = idx - first * NT;
    const int m0 = (first + in % gs) * T::BM, n0 = in / gs * BNO;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int wm = wave / T::WN, wn = wave % T::WN;
    const int rows = min(p.M - m0, T::BM), cols = min(p.N - n0, BNO);
    const auto ra = buf_rsrc(p.a + (size_t)m0 * p.lda, (size_t)rows * p.lda);
    const auto rb = buf_rsrc(p.b + (size_t)n0 * p.ldb, (size_t)cols * p.ldb);
    const auto rb2 = buf_rsrc((GATED ? p.b2 : p.b) + (size_t)n0 * p.ldb, (size_t)cols * p.ldb);
    // row and piece that copy instruction i of the wave brings to this lane's place
    auto a_row = [&](int i) { return (wave * T::A_DMA + i) * T::RPI + lane / T::CPR; };
    auto b_row = [&](int i) { return (wave * T::B_DMA + i) * T::RPI + lane / T::CPR; };
    auto piece = [&](int row) { return ((lane % T::CPR) ^ i8_swz(row)) * 16; };
    auto a_at = [&](int i) { return min(a_row(i), rows - 1) * (int)p.lda; };
    auto b_at = [&](int i) { return min(GATED && b_row(i) >= BNO ? b_row(i) - BNO : b_row(i), cols - 1) * (int)p.ldb; };
    int va[T::A_DMA], vb[T::B_DMA];
#pragma unroll
    for (int i = 0; i < T::A_DMA; i++) va[i] = a_at(i) + piece(a_row(i));
#pragma unroll
    for (int i = 0; i < T::B_DMA; i++) vb[i] = b_at(i) + piece(b_row(i));
    // WHOLE 0: the last stage, of fewer than BK codes.  A's come through registers, those
    // behind K cleared; of pieces that lie behind K the stage's first is read instead
    auto issue = [&](int kt, auto WHOLE) {
        unsigned char *slot = smem + kt % T::ST * T::STAGE;
        const int k0 = kt * T::BK, room = p.K - k0;
#pragma unroll
        for (int i = 0; i < T::A_DMA; i++) {
            unsigned char *to = slot + (wave * T::A_DMA + i) * 1024;
            if constexpr (decltype(WHOLE)::value) {
                i8_copy<0>(ra, to, va[i], k0);
            } else {
                const int pc = piece(a_row(i)), at = a_at(i) + (pc < room ? pc : 0);
                const i32x4 v = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, at, k0, 0));
                *(i32x4 *)(to + lane * 16) = i8_keep(v, room - pc);
            }
        }
#pragma unroll
        for (int i = 0; i < T::B_DMA; i++) {
            const bool up = GATED && (wave * T::B_DMA + i) * T::RPI >= BNO;
            const int at = decltype(WHOLE)::value || piece(b_row(i)) < room ? vb[i] : b_at(i);
            i8_copy<T::B_AUX>(up ? rb2 : rb, slot + T::A_BYTES + (wave * T::B_DMA + i) * 1024, at, k0);
        }
    };
    // this lane's first fragment of A and of B in each step of a stage; the others lie 32 rows on
    const int fr = lane & 31, fh = lane >> 5;
    constexpr int NEXT = 32 * T::BK, UP = (BNO - 32 * (T::TN / 2)) * T::BK;
    int fa_at[T::KS], fb_at[T::KS];
#pragma unroll
    for (int s = 0; s < T::KS; s++) {
        const int pc = ((2 * s + fh) ^ i8_swz(fr)) * 16;
        fa_at[s] = (wm * (T::BM / T::WM) + fr) * T::BK + pc;
        fb_at[s] = T::A_BYTES + (wn * (BNO / T::WN) + fr) * T::BK + pc;
    }
    i32x16 acc[T::TM][T::TN] = {};
    i32x4 fa[2][T::TM], fb[2][T::TN];
    auto read = [&](int kt, int s) {
        const unsigned char *slot = smem + kt % T::ST * T::STAGE;
#pragma unroll
        for (int j = 0; j < T::TN; j++)
            fb[s & 1][j] = *(const i32x4 *)(slot + fb_at[s] + j * NEXT + (GATED && j >= T::TN / 2 ? UP : 0));
#pragma unroll
        for (int i = 0; i < T::TM; i++) fa[s & 1][i] = *(const i32x4 *)(slot + fa_at[s] + i * NEXT);
    };
    auto multiply = [&](int s) {
#pragma unroll
        for (int i = 0; i < T::TM; i++)
#pragma unroll
            for (int j = 0; j < T::TN; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[s & 1][i], fb[s & 1][j], acc[i][j], 0, 0, 0);
    };
    constexpr int PER = T::TM * T::TN, FR = T::TM + T::TN;
    // all but the last step of stage kt, each with the next one's fragments on their way
    auto most = [&](int kt) {
#pragma unroll
        for (int s = 0; s + 1 < T::KS; s++) {
            read(kt, s + 1);
            multiply(s);
            I8Order<0, PER, FR, 0>::run();
        }
    };
    const int nk = (p.K + T::BK - 1) / T::BK, whole = p.K / T::BK;
    auto issue_any = [&](int kt) {
        if (kt < whole) issue(kt, IC<1>{});
        else issue(kt, IC<0>{});
    };
    for (int t = 0; t < T::ST; t++)
        if (t < nk) issue_any(t);
    int kt = 0;
    if (whole >= T::ST) __builtin_amdgcn_s_waitcnt(I8_VMCNT((T::ST - 1) * T::DMA));
    else __builtin_amdgcn_s_waitcnt(I8_VMCNT(0));
    i8_barrier();
    read(0, 0);
    for (; kt + T::ST < whole; kt++) {
        most(kt);
        // this wave has read all of stage kt and its copies of the next are there: after the
        // barrier every wave's
        __builtin_amdgcn_s_waitcnt(I8_VMCNT((T::ST - 2) * T::DMA));
        i8_barrier();
        issue(kt + T::ST, IC<1>{});
        read(kt + 1, 0);
        multiply(T::KS - 1);
        I8Order<0, PER, FR, T::DMA>::run();
        __builtin_amdgcn_sched_barrier(0);
    }
    for (; kt < nk; kt++) {
        most(kt);
        __builtin_amdgcn_s_waitcnt(I8_VMCNT(0));
        i8_barrier();
        if (kt + T::ST < nk) issue_any(kt + T::ST);
        if (kt + 1 < nk) read(kt + 1, 0);
        multiply(T::KS - 1);
        __builtin_amdgcn_sched_barrier(0);
    }

    // the tile's scales through LDS; stores behind M and N fall out of the buffer's range.
    // Whole lines go through the L2 at once: kept there they are written back when the
    // launch ends (2048 x 1024 x 4096 16.6 -> 14.0 us, 4096 x 1024 x 8192 44.6 -> 42.7;
    // past the caches altogether 52).  Rows of C whose pieces of 32 are not whole lines
    // are left to the L2, which joins them (597 x 413 x 100827 91 us, through it 136).
    __syncthreads();
    float *sm = (float *)smem, *sn = sm + T::BM, *su = sn + BNO;
    for (int i = tid; i < T::BM; i += WAVE * T::NW) sm[i] = p.as[m0 + min(i, rows - 1)];
    for (int i = tid; i < BNO; i += WAVE * T::NW) {
        sn[i] = p.bs[n0 + min(i, cols - 1)];
        if constexpr (GATED) su[i] = p.bs2[n0 + min(i, cols - 1)];
    }
    __syncthreads();
    constexpr int TNO = GATED ? T::TN / 2 : T::TN;
    const auto rc = buf_rsrc((char *)p.c + ((size_t)m0 * p.ldc + n0) * ES, ((size_t)(rows - 1) * p.ldc + cols) * ES);
    const int ldc = (int)p.ldc * ES;
    // a row's columns one after another, so that its lines fill up at once
    float s[TNO], s2[TNO];
    unsigned at[TNO];
#pragma unroll
    for (int j = 0; j < TNO; j++) {
        const int n = wn * (BNO / T::WN) + 32 * j + fr;
        s[j] = sn[n];
        s2[j] = GATED ? su[n] : 0.0f;
        at[j] = (n < cols ? n * ES : BUF_OOB) + 4 * fh * ldc;
    }
    float far = 0.0f;                                     // the largest |g| of the wave's gated results
    auto finish = [&](auto AUX, auto FAR) {
#pragma unroll
        for (int i = 0; i < T::TM; i++)
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
                const int m = wm * (T::BM / T::WM) + 32 * i + 8 * e4;
                const f32x4 r = *(const f32x4 *)(sm + m + 4 * fh);
                float y[TNO][4];
#pragma unroll
                for (int j = 0; j < TNO; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) y[j][e] = (float)acc[i][j][4 * e4 + e] * (r[e] * s[j]);
                if constexpr (GATED) {
#pragma unroll
                    for (int j = 0; j < TNO; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float u = (float)acc[i][j + TNO][4 * e4 + e] * (r[e] * s2[j]);
                            if constexpr (!decltype(FAR)::value) far = fmaxf(far, fabsf(y[j][e]));
                            y[j][e] = decltype(FAR)::value ? i8_silu_mul<CBF>(y[j][e], u) : i8_silu_near<CBF>(y[j][e], u);
                        }
                }
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int j = 0; j < TNO; j++) {
                        const unsigned to = at[j] + (m + e) * ldc;
                        if constexpr (CBF) {
                            const uint32_t two = pack_bf16x2(y[j][e & ~1], y[j][e | 1]);
                            __builtin_amdgcn_raw_buffer_store_b16((short)(e & 1 ? two >> 16 : two), rc, to, 0, decltype(AUX)::value);
                        } else {
                            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, y[j][e]), rc, to, 0, decltype(AUX)::value);
                        }
                    }
            }
    };
    auto finish_all = [&](auto FAR) {
        if (p.whole) finish(IC<AUX_SC1>{}, FAR);
        else finish(IC<0>{}, FAR);
    };
    finish_all(IC<0>{});
    // rare, so out of the way: all of the lane's results again (a look at each step's in its
    // place, with these instructions among the others, cost 2 to 4% of a call)
    if constexpr (GATED)
        if (far >= I8_SILU_FAR) finish_all(IC<1>{});
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
static inline bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
#define I8_MAX_LD ((size_t)1 << 40)
#define I8_MAX_NEAR ((size_t)1 << 22)     // 256 rows within 2^31 bytes

extern "C" int qh_rows_int8(int8_t *q, size_t ldq, float *scale, const void *x, size_t ldx, int bf16, int rows, int K) {
    if (rows < 0 || K < 0 || ldq < (size_t)K || ldx < (size_t)K) return QH_EINVAL;
    if (rows == 0) return QH_OK;
    if (!scale || !aligned(scale, 4) || (K > 0 && (!q || !x)) || !aligned(x, bf16 ? 2 : 4)) return QH_EINVAL;
    if (K > I8_MAX_K || ldq > I8_MAX_LD || ldx > I8_MAX_LD) return QH_ETOOBIG;
    if (!g_inited) return QH_ESTATE;
    const bool few = rows <= 1024;
    // more than the L2s hold is read and written past them; few rows' kernels never have as much
    const bool once = (size_t)rows * K * (bf16 ? 2 : 4) >= (size_t)32 << 20;
#define ROWS_AS(BF, TPR, KEEP, O)                                                                            \
    hipLaunchKernelGGL((k_rows_int8<BF, TPR, KEEP, O>), dim3((unsigned)(((size_t)some * TPR + 255) / (TPR < 256 ? 256 : TPR))), \
                       dim3(TPR < 256 ? 256 : TPR), 0, g_stream, q, ldq, scale, x, ldx, K, some)
#define ROWS(BF, O)                                        \
    do {                                                   \
        if (K <= 256 && !few) ROWS_AS(BF, 16, 2, O);    \
        else if (K <= 512) ROWS_AS(BF, 64, 1, O);       \
        else if (K <= 1024 && !few) ROWS_AS(BF, 64, 2, O); \
        else if (K <= 2048 && few) ROWS_AS(BF, 256, 1, false); \
        else if (K <= 2048 && rows >= 4096) ROWS_AS(BF, 64, 4, O); \
        else if (K <= 4096) ROWS_AS(BF, 256, 2, O);     \
        else if (K <= 8192 && rows <= 256) ROWS_AS(BF, 1024, 1, false); \
        else if (K <= 8192) ROWS_AS(BF, 256, 4, O);     \
        else ROWS_AS(BF, 1024, 2, O);                   \
    } while (0)
    // 2^31 threads a launch at most
    for (int done = 0;;) {
        const int some = rows - done < 1 << 21 ? rows - done : 1 << 21;
        if (bf16) {
            if (once) ROWS(true, true);
            else ROWS(true, false);
        } else {
            if (once) ROWS(false, true);
            else ROWS(false, false);
        }
        HCHECK(hipGetLastError(), QH_ELAUNCH);
        if ((done += some) >= rows) return QH_OK;
        q += (size_t)some * ldq;
        scale += some;
        x = (const char *)x + (size_t)some * ldx * (bf16 ? 2 : 4);
    }
#undef ROWS
#undef ROWS_AS
}

enum { I8_ANY_PLAN, I8_NARROW1, I8_NARROW2, I8_TILE64, I8_TILE64X128, I8_TILE64X128_ONCE, I8_TILE128, I8_TILE128_ALONE, I8_TILE192X256, I8_TILE256 };

// Few blocks of 16 columns: as long as there is at most one on each of the 256
// CUs (two of 16 rows), against tiles: 64 x 1024 x 1024 3.2 us and 4.8, 128 x 4096 x
// 1024 7.8 and 9.7; with 512 blocks 64 x 1024 x 4096 5.3 and 4.9.  Rows are read
// by every block, so blocks of 16 rows until 256 of them, then of 32.  Up to four
// rows always: they are read once a block, 1 x 4096 x 20000 18.2 and 21.1 us.
// Tiles: the least of an estimate, us = fixed + rounds * tile + stages * (rounds *
// stage + tiles / 256 * shared), rounds = tiles / 256 rounded up: what a CU does one
// after the other, and what all of them share.  Fitted to 1,497 measurements (M 16
// to 4,096, N 512 to 20,000, K 512 to 4,096), of whose best it takes 0.3% longer on
// average.  A gated product has two weights' columns.  128 x 128 tiles that have a
// CU each take three places for stages instead of two: operands that are in no
// cache 1000 x 4096 x 2816 30.2 -> 22.5 us (in a cache 23.1 and 20.6), 2048 x 1024 x
// 2048 11.7 -> 10.8 (10.0 and 10.4); with two tiles a CU 2048 x 1024 x 4096 15.2 and
// 18.7.
// Weights of 64 MB and more that every tile reads for itself are read past the
// caches, which they would empty, on three blocks a CU: 64 x 1024 x 151936 38.2 ->
// 35.8 us, 16 rows 33.4 -> 31.2 (the other way 32.0 and 35.4 where nothing else is
// read between two calls, so that 155 MB stay in the last cache).
static int i8_plan_of(const I8Args &p, bool gated) {
    if (!p.K || !aligned16(p.a) || !aligned16(p.b) || !aligned16(p.b2) || p.lda % 16 || p.ldb % 16 || p.lda > I8_MAX_NEAR ||
        p.ldb > I8_MAX_NEAR)
        return I8_ANY_PLAN;
    const long cols = ((long)p.N + 15) / 16;
    if (p.M <= 4 || cols * ((p.M + 15l) / 16) <= (p.M <= 16 ? 512 : 256)) return I8_NARROW1;
    if (cols * ((p.M + 31l) / 32) <= 256) return I8_NARROW2;
    // tiles' stores have 32-bit offsets: a tile's rows of C, as fp32, within 2^31 bytes.  Rows further apart
    // than the lowest tile takes go to the narrow kernel, whose addresses have 64 bits (4096 x 1024 x (2^20 + 16)
    // 7.1 ms on tiles, 60.7 there)
    const auto near = [&](int bm) { return (size_t)bm * p.ldc <= (size_t)1 << 29; };
    if (!near(64)) return p.M <= 65535 * 32 ? I8_NARROW2 : I8_ANY_PLAN;
    static const struct { int plan, bm, bn; float fixed, tile, stage, shared; } T[] = {
        {I8_TILE64, 64, 64, 2.41f, 0.67f, 0.201f, 0.012f},      {I8_TILE64X128, 64, 128, 2.59f, 0.79f, 0.300f, 0.062f},
        {I8_TILE128, 128, 128, 0.72f, 1.88f, 0.345f, 0.190f},   {I8_TILE128_ALONE, 128, 128, 4.0f, 0.0f, 0.404f, 0.210f},
        {I8_TILE192X256, 192, 256, 0.76f, 4.33f, 0.821f, 0.591f}, {I8_TILE256, 256, 256, 0.31f, 5.63f, 1.004f, 0.753f}};
    const double stages = (p.K + 127) / 128;
    double best = 1e30;
    int plan = I8_TILE64;
    for (const auto &t : T) {
        const double tiles = ceil(p.M / (double)t.bm) * ceil(p.N * (gated ? 2.0 : 1.0) / t.bn);
        if (t.plan == (tiles > 256 ? I8_TILE128_ALONE : I8_TILE128) || !near(t.bm)) continue;
        const double rounds = ceil(tiles / 256);
        const double us = t.fixed + rounds * t.tile + stages * (rounds * t.stage + tiles / 256 * t.shared);
        if (us < best) {
            best = us;
            plan = t.plan;
        }
    }
    if (plan == I8_TILE64X128 && p.M <= 64 && p.ldb * p.N * (gated ? 2 : 1) >= (size_t)64 << 20) plan = I8_TILE64X128_ONCE;
    return plan;
}

// the plan of codes that are aligned as the fast kernels want them
extern "C" const char *qh_int8_plan(int M, int K, int N, int gated) {
    static const char *const names[] = {"any", "narrow16", "narrow32", "tile64", "tile64x128", "tile64x128-once", "tile128", "tile128-alone",
                                        "tile192x256", "tile256"};
    if (M <= 0 || N <= 0 || K < 0 || K > I8_MAX_K) return "none";
    const size_t ld = ((size_t)K + 15) / 16 * 16;
    return names[i8_plan_of(I8Args{nullptr, (size_t)N, nullptr, ld, nullptr, nullptr, nullptr, ld, nullptr, nullptr, M, K, N, 0}, gated)];
}

// a launch has fewer than 2^32 threads along x
#define I8_GO(KERNEL, X, Y, THREADS, ...)                                                     \
    do {                                                                                      \
        const unsigned long x_ = (X);                                                         \
        if (x_ * (THREADS) >= 1ul << 32) return QH_ETOOBIG;                                   \
        if (!g_inited) return QH_ESTATE;                                                      \
        hipLaunchKernelGGL(KERNEL, dim3((unsigned)x_, Y), dim3(THREADS), 0, g_stream, __VA_ARGS__); \
        HCHECK(hipGetLastError(), QH_ELAUNCH);                                                \
        return QH_OK;                                                                         \
    } while (0)

template <int MT, int W, bool GATED, bool CBF>
static int i8_narrow(const I8Args &p) {
    I8_GO((k_i8_narrow<MT, W, GATED, CBF>), (p.N + 15l) / 16, (unsigned)((p.M + 16 * MT - 1l) / (16 * MT)), WAVE *W, p);
}
// any number of columns, 2^26 a launch
template <bool GATED, bool CBF>
static int i8_narrow_any(I8Args p) {
    const int most = 1 << 26, N = p.N;
    for (int n = 0;; n += most) {
        p.N = N - n < most ? N - n : most;
        const int rc = i8_narrow<2, 8, GATED, CBF>(p);
        if (rc != QH_OK || N - n <= most) return rc;
        p.b += (size_t)most * p.ldb;
        p.bs += most;
        if (GATED) {
            p.b2 += (size_t)most * p.ldb;
            p.bs2 += most;
        }
        p.c = (char *)p.c + (size_t)most * (CBF ? 2 : 4);
    }
}
template <typename T, bool GATED, bool CBF>
static int i8_tile(const I8Args &p) {
    const long bno = GATED ? T::BN / 2 : T::BN, mt = (p.M + T::BM - 1l) / T::BM, nt = (p.N + bno - 1) / bno;
    const long per = (mt * nt + 7) / 8;
    I8_GO((k_i8_tile<T, GATED, CBF>), 8 * per, 1, WAVE *T::NW, p, (int)mt, (int)nt, (int)per);
}
template <bool GATED, bool CBF>
static int i8_any(const I8Args &p) {
    const long mt = (p.M + I8_ANY - 1l) / I8_ANY, nt = (p.N + I8_ANY - 1l) / I8_ANY;
    I8_GO((k_i8_any<GATED, CBF>), mt * nt, 1, NTHREADS, p, (unsigned)nt);
}

template <bool GATED, bool CBF>
static int i8_launch(const I8Args &p) {
    switch (i8_plan_of(p, GATED)) {
    case I8_NARROW1: return i8_narrow<1, 8, GATED, CBF>(p);
    case I8_NARROW2: return i8_narrow_any<GATED, CBF>(p);
    case I8_TILE64: return i8_tile<I8Tile<64, 64, 2, 2 - GATED, 4>, GATED, CBF>(p);
    case I8_TILE64X128: return i8_tile<I8Tile<64, 128, 2, 2, 3>, GATED, CBF>(p);
    case I8_TILE64X128_ONCE: return i8_tile<I8Tile<64, 128, 2, 2, 2, 2>, GATED, CBF>(p);
    case I8_TILE128: return i8_tile<I8Tile<128, 128, 2, 2, 2>, GATED, CBF>(p);
    case I8_TILE128_ALONE: return i8_tile<I8Tile<128, 128, 2, 2, 3>, GATED, CBF>(p);
    case I8_TILE192X256: return i8_tile<I8Tile<192, 256, 2, 4, 2>, GATED, CBF>(p);
    case I8_TILE256: return i8_tile<I8Tile<256, 256, 2, 4, 2>, GATED, CBF>(p);
    default: return i8_any<GATED, CBF>(p);
    }
}

static int i8_common(I8Args p, bool gated, int bf16) {
    if (p.M < 0 || p.N < 0 || p.K < 0) return QH_EINVAL;
    if (p.lda < (size_t)p.K || p.ldb < (size_t)p.K || p.ldc < (size_t)p.N) return QH_EINVAL;
    if (p.M == 0 || p.N == 0) return QH_OK;
    if (!p.c || !p.as || !p.bs || (gated && !p.bs2)) return QH_EINVAL;
    if (p.K > 0 && (!p.a || !p.b || (gated && !p.b2))) return QH_EINVAL;
    if (!aligned(p.c, bf16 ? 2 : 4) || !aligned(p.as, 4) || !aligned(p.bs, 4) || !aligned(p.bs2, 4)) return QH_EINVAL;
    if (p.K > I8_MAX_K || p.lda > I8_MAX_LD || p.ldb > I8_MAX_LD || p.ldc > I8_MAX_LD) return QH_ETOOBIG;
    p.whole = p.ldc % 32 == 0 && aligned(p.c, bf16 ? 64 : 128);
    if (gated) return bf16 ? i8_launch<true, true>(p) : i8_launch<true, false>(p);
    return bf16 ? i8_launch<false, true>(p) : i8_launch<false, false>(p);
}

extern "C" int qh_gemm_int8(void *c, size_t ldc, int bf16, const int8_t *a, size_t lda, const float *as, const int8_t *b,
                            size_t ldb, const float *bs, int M, int K, int N) {
    return i8_common(I8Args{c, ldc, a, lda, as, b, nullptr, ldb, bs, nullptr, M, K, N, 0}, false, bf16);
}

extern "C" int qh_gemm_int8_gate_up_silu(void *h, size_t ldh, int bf16, const int8_t *x, size_t ldx, const float *xs,
                                         const int8_t *wg, const float *gs, const int8_t *wu, const float *us, size_t ldw,
                                         int M, int K, int N) {
    return i8_common(I8Args{h, ldh, x, ldx, xs, wg, wu, ldw, gs, us, M, K, N, 0}, true, bf16);
}

#endif  // QH_INT8_KERNELS_H
