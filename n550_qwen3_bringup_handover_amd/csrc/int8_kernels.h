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

template <bool BF>
__device__ __forceinline__ float i8_value(const void *x, size_t i) {
    return BF ? bf16_lo(((const uint16_t *)x)[i]) : ((const float *)x)[i];
}

template <bool BF>
__global__ __launch_bounds__(NTHREADS) void k_rows_int8(int8_t *__restrict__ q, size_t ldq, float *__restrict__ scale,
                                                       const void *__restrict__ x, size_t ldx, int K) {
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x;
    float a = 0.0f;
    for (int k = tid; k < K; k += NTHREADS) a = fmaxf(a, fabsf(i8_held(i8_value<BF>(x, row * ldx + k))));
    __shared__ float red[NTHREADS / WAVE];
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) a = fmaxf(a, __shfl_xor(a, m));
    if ((tid & 63) == 0) red[tid >> 6] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NTHREADS / WAVE; w++) a = fmaxf(a, red[w]);
    const float s = a < I8_TINY ? 0.0f : a / 127.0f;
    if (tid == 0) scale[row] = s;
    for (int k = tid; k < K; k += NTHREADS) {
        const float v = i8_held(i8_value<BF>(x, row * ldx + k));
        q[row * ldq + k] = s == 0.0f ? 0 : (int8_t)(int)rintf(v / s);
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
};

template <bool CBF>
__device__ __forceinline__ void i8_store(void *c, size_t i, float v) {
    if constexpr (CBF) ((__bf16 *)c)[i] = (__bf16)v;
    else ((float *)c)[i] = v;
}

// Any K, strides and addresses: 64 x 64 outputs a block, 64 bytes of K a step
// through LDS, read byte by byte, 4 x 4 outputs a thread by v_dot4.
#define I8_ANY 64
template <bool GATED, bool CBF>
__global__ __launch_bounds__(NTHREADS) void k_i8_any(I8Args p) {
    __shared__ int sa[I8_ANY][I8_ANY / 4 + 1], sb[GATED ? 2 : 1][I8_ANY][I8_ANY / 4 + 1];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const size_t m0 = (size_t)blockIdx.y * I8_ANY, n0 = (size_t)blockIdx.x * I8_ANY;
    auto four = [&](const int8_t *x, size_t ld, size_t row, int rows, int k) {
        int w = 0;
        for (int j = 0; j < 4; j++)
            if (row < (size_t)rows && k + j < p.K) w |= (int)(uint8_t)x[row * ld + k + j] << (8 * j);
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
            if constexpr (GATED) v = silu_mul(v, (float)acc[GATED][i][j] * (p.as[m] * p.bs2[n]));
            i8_store<CBF>(p.c, m * p.ldc + n, v);
        }
    }
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
static inline bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
#define I8_MAX_LD ((size_t)1 << 40)

extern "C" int qh_rows_int8(int8_t *q, size_t ldq, float *scale, const void *x, size_t ldx, int bf16, int rows, int K) {
    if (rows < 0 || K < 0 || ldq < (size_t)K || ldx < (size_t)K) return QH_EINVAL;
    if (rows == 0) return QH_OK;
    if (!scale || !aligned(scale, 4) || (K > 0 && (!q || !x)) || !aligned(x, bf16 ? 2 : 4)) return QH_EINVAL;
    if (K > I8_MAX_K || ldq > I8_MAX_LD || ldx > I8_MAX_LD) return QH_ETOOBIG;
    if (!g_inited) return QH_ESTATE;
    if (bf16) hipLaunchKernelGGL(k_rows_int8<true>, dim3(rows), dim3(NTHREADS), 0, g_stream, q, ldq, scale, x, ldx, K);
    else hipLaunchKernelGGL(k_rows_int8<false>, dim3(rows), dim3(NTHREADS), 0, g_stream, q, ldq, scale, x, ldx, K);
    HCHECK(hipGetLastError(), QH_ELAUNCH);
    return QH_OK;
}

template <bool GATED, bool CBF>
static int i8_launch(const I8Args &p) {
    const dim3 any((p.N + I8_ANY - 1) / I8_ANY, (p.M + I8_ANY - 1) / I8_ANY);
    if (any.y > 65535) return QH_ETOOBIG;
    hipLaunchKernelGGL((k_i8_any<GATED, CBF>), any, dim3(NTHREADS), 0, g_stream, p);
    HCHECK(hipGetLastError(), QH_ELAUNCH);
    return QH_OK;
}

static int i8_common(const I8Args &p, bool gated, int bf16) {
    if (p.M < 0 || p.N < 0 || p.K < 0) return QH_EINVAL;
    if (p.lda < (size_t)p.K || p.ldb < (size_t)p.K || p.ldc < (size_t)p.N) return QH_EINVAL;
    if (p.M == 0 || p.N == 0) return QH_OK;
    if (!p.c || !p.as || !p.bs || (gated && !p.bs2)) return QH_EINVAL;
    if (p.K > 0 && (!p.a || !p.b || (gated && !p.b2))) return QH_EINVAL;
    if (!aligned(p.c, bf16 ? 2 : 4) || !aligned(p.as, 4) || !aligned(p.bs, 4) || !aligned(p.bs2, 4)) return QH_EINVAL;
    if (p.K > I8_MAX_K || p.lda > I8_MAX_LD || p.ldb > I8_MAX_LD || p.ldc > I8_MAX_LD) return QH_ETOOBIG;
    if (!g_inited) return QH_ESTATE;
    if (gated) return bf16 ? i8_launch<true, true>(p) : i8_launch<true, false>(p);
    return bf16 ? i8_launch<false, true>(p) : i8_launch<false, false>(p);
}

extern "C" int qh_gemm_int8(void *c, size_t ldc, int bf16, const int8_t *a, size_t lda, const float *as, const int8_t *b,
                            size_t ldb, const float *bs, int M, int K, int N) {
    return i8_common(I8Args{c, ldc, a, lda, as, b, nullptr, ldb, bs, nullptr, M, K, N}, false, bf16);
}

extern "C" int qh_gemm_int8_gate_up_silu(void *h, size_t ldh, int bf16, const int8_t *x, size_t ldx, const float *xs,
                                         const int8_t *wg, const float *gs, const int8_t *wu, const float *us, size_t ldw,
                                         int M, int K, int N) {
    return i8_common(I8Args{h, ldh, x, ldx, xs, wg, wu, ldw, gs, us, M, K, N}, true, bf16);
}

#endif  // QH_INT8_KERNELS_H
