// What the kernels of the 8-bit rows and products read and write, on the CPU:
// launched by their own launchers, one lane after the other, every buffer
// against an unreadable page, every lane's accesses as the unoptimised build
// makes them.  No address depends on what lanes exchange, so exchanges and
// matrix products are left out.  Copies into LDS have to lie in the buffer they
// are made from, results in their rows and columns; padding keeps its marks.
// Rules on logits run with a thread for each of a block's and are held to their
// definition as well.
#include <float.h>
#include <math.h>
#include <pthread.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <algorithm>
#include <thread>
#include <vector>

// ---- what the headers take from the HIP runtime and the units they are compiled into
#define QH_GEMM_COMMON_H
#define __HIP_DEVICE_COMPILE__ 1
#define __device__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __align__(n) __attribute__((aligned(n)))
struct dim3 {
    unsigned x, y, z;
    dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
static thread_local dim3 threadIdx, blockIdx;
struct uint4 { unsigned x, y, z, w; };
static inline uint4 make_uint4(unsigned a, unsigned b, unsigned c, unsigned d) { return uint4{a, b, c, d}; }
using std::max;
using std::min;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
#define WAVE 64
#define NTHREADS 256
#define NTH 256
#define AUX_SC1 16
#define BUF_OOB 0x80000000u
template <int V> struct IC { static constexpr int value = V; };
static inline float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
static inline float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xFFFF0000u); }
static inline uint32_t pack_bf16x2(float, float) { return 0; }
extern "C" __bf16 __truncsfbf2(float f) { return __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, f) >> 16)); }
static bool g_threads_run;
static pthread_barrier_t g_block;
static inline void __syncthreads() { if (g_threads_run) pthread_barrier_wait(&g_block); }
template <typename T> static inline T __shfl_xor(T v, int) { return v; }
template <typename T> static inline void atomicOr(T *p, T v) { __atomic_fetch_or(p, v, __ATOMIC_RELAXED); }
template <typename T> static inline void atomicAdd(T *p, T v) { __atomic_fetch_add(p, v, __ATOMIC_RELAXED); }
template <typename T> static inline void atomicMax(T *p, T v) {
    for (T o = *p; o < v && !__atomic_compare_exchange_n(p, &o, v, false, __ATOMIC_RELAXED, __ATOMIC_RELAXED);) {}
}
struct rsrc { char *p; size_t bytes; };
#define __amdgpu_buffer_rsrc_t rsrc
static inline rsrc buf_rsrc(const void *p, size_t bytes) { return rsrc{(char *)p, bytes}; }
static volatile char g_seen;
static void copied(rsrc r, unsigned at, unsigned k0) {            // into LDS: always inside
    if ((size_t)at + k0 + 16 > r.bytes) { printf("a copy from %u + %u of %zu bytes\n", at, k0, r.bytes); exit(1); }
    for (int i = 0; i < 16; i++) g_seen = r.p[(size_t)at + k0 + i];
}
static u32x4 loaded(rsrc r, unsigned at, unsigned k0) {
    copied(r, at, k0);
    return u32x4{};
}
template <typename T> static void stored(T v, rsrc r, unsigned at) {   // past its size a store does nothing
    if ((size_t)at + sizeof v <= r.bytes) memcpy(r.p + at, &v, sizeof v);
}
#define __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, n, at, k0, o, a) copied(r, at, k0)
#define __builtin_amdgcn_raw_buffer_load_b128(r, at, k0, a) loaded(r, at, k0)
#define __builtin_amdgcn_raw_buffer_store_b16(v, r, at, s, a) stored((short)(v), r, at)
#define __builtin_amdgcn_raw_buffer_store_b32(v, r, at, s, a) stored((int)(v), r, at)
#define __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_sdot4(a, b, c, d) (c)
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_sched_group_barrier(a, b, c) ((void)0)
#define __builtin_amdgcn_s_waitcnt(x) ((void)0)
#define __builtin_amdgcn_s_barrier() ((void)0)

template <typename F> static void run_grid(dim3 grid, unsigned threads, F f) {
    for (unsigned y = 0; y < grid.y; y++)
        for (unsigned x = 0; x < grid.x; x++) {
            auto lane = [&](unsigned t) {
                blockIdx = dim3(x, y);
                threadIdx.x = t;
                f();
            };
            if (!g_threads_run) {
                for (unsigned t = 0; t < threads; t++) lane(t);
                continue;
            }
            pthread_barrier_init(&g_block, nullptr, threads);
            std::vector<std::thread> all;
            for (unsigned t = 0; t < threads; t++) all.emplace_back(lane, t);
            for (auto &t : all) t.join();
            pthread_barrier_destroy(&g_block);
        }
}
#define hipLaunchKernelGGL(K, GRID, BLOCK, SHM, STREAM, ...) run_grid(GRID, (BLOCK).x, [&] { K(__VA_ARGS__); })
enum { hipSuccess };
static inline int hipGetLastError() { return hipSuccess; }
#define HCHECK(expr, code) do { if ((expr) != hipSuccess) return code; } while (0)
typedef void *hipStream_t;
static const int g_inited = 1;
static hipStream_t g_stream;
static inline hipStream_t stream() { return (hipStream_t)&g_block; }
static inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }
#include "hip_shim.h"
#include "model_shim.h"
#include "int8_kernels.h"
#include "rules_kernels.h"

// ---- buffers against an unreadable page
static bool g_front;                                  // the page before the start, not behind the end
static std::vector<std::pair<void *, size_t>> g_maps;
static char *guarded(size_t bytes, int fill) {
    const size_t page = 4096, n = (bytes + page - 1) / page * page;
    char *p = (char *)mmap(nullptr, n + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (p == MAP_FAILED || mprotect(p + page, n, PROT_READ | PROT_WRITE)) abort();
    g_maps.push_back({p, n + 2 * page});
    memset(p + page, fill, n);
    return g_front ? p + page : p + page + (n - bytes);
}
static void release() {
    for (auto &m : g_maps) munmap(m.first, m.second);
    g_maps.clear();
}
static void want(bool ok, const char *what) {
    if (!ok) { printf("%s\n", what); exit(1); }
}

static void rows_case(int rows, int K, bool bf, size_t ldx, size_t ldq) {
    printf("rows %d x %d, %s, %zu, %zu\n", rows, K, bf ? "bf16" : "fp32", ldx, ldq);
    const int es = bf ? 2 : 4;
    // the last row ends with its last value, as a caller's may
    const char *x = guarded(((rows - 1) * ldx + K) * es, 0);
    char *q = guarded((rows - 1) * ldq + K, 77), *s = guarded(4 * rows, 77);
    want(qh_rows_int8((int8_t *)q, ldq, (float *)s, x, ldx, bf, rows, K) == QH_OK, "refused");
    for (int r = 0; r < rows; r++) {
        want(*(float *)(s + 4 * r) == 0.0f, "a scale is missing");
        for (size_t k = 0; k < (r + 1 < rows ? ldq : K); k++) want(q[r * ldq + k] == (k < (size_t)K ? 0 : 77), "a code");
    }
    release();
}

template <bool G, bool CB, typename F> static void product_case(const char *name, int M, int K, int N, size_t lda, size_t ldb, F go) {
    printf("%s %d x %d x %d, %zu, %zu, %s%s\n", name, M, K, N, lda, ldb, G ? "gated " : "", CB ? "bf16" : "fp32");
    const size_t es = CB ? 2 : 4, ldc = N + 3;
    I8Args p = {};
    p.a = (int8_t *)guarded(M * lda, 1);
    p.b = (int8_t *)guarded(N * ldb, 1);
    p.b2 = G ? (int8_t *)guarded(N * ldb, 1) : nullptr;
    p.as = (float *)guarded(4 * M, 0);
    p.bs = (float *)guarded(4 * N, 0);
    p.bs2 = G ? (float *)guarded(4 * N, 0) : nullptr;
    char *c = guarded(((M - 1) * ldc + N) * es, 77);
    p.c = c;
    p.lda = lda;
    p.ldb = ldb;
    p.ldc = ldc;
    p.M = M;
    p.K = K;
    p.N = N;
    want(go(p) == QH_OK, "refused");
    for (int m = 0; m < M; m++)
        for (size_t n = 0; n < (m + 1 < M ? ldc : N); n++)
            for (size_t i = 0; i < es; i++)
                want((c[(m * ldc + n) * es + i] == 77) == (n >= (size_t)N), "a result is missing, or padding is written");
    release();
}
template <bool G, bool CB> static void products() {
    auto any = [](const I8Args &p) { return i8_launch<G, CB>(p); };
    for (int K : {1, 16, 100, 129, 300})
        for (int M : {1, 17}) {
            const size_t up = (K + 15) / 16 * 16;
            product_case<G, CB>("narrow", M, K, 21, up, up + 16, [](const I8Args &p) { return i8_narrow<1, 8, G, CB>(p); });
            product_case<G, CB>("narrow 32", M, K, 21, up, up, [](const I8Args &p) { return i8_narrow<2, 8, G, CB>(p); });
            product_case<G, CB>("any", M, K, 21, K, K + 1, any);
        }
    product_case<G, CB>("any", 3, 0, 5, 0, 0, any);
#define TILE(BM, BN, WM, WN, ...)                                                                                  \
    for (int K : {16, 120, 128, 530, 641})                                                                         \
        for (int full = 0; full < 2; full++)                                                                       \
            product_case<G, CB>("tile " #BM " x " #BN, full ? BM : BM + 1, K, full ? (G ? BN / 2 : BN) : BN / 2 + 5, (K + 15) / 16 * 16, \
                                (K + 15) / 16 * 16, [](const I8Args &p) { return i8_tile<I8Tile<BM, BN, WM, WN, __VA_ARGS__>, G, CB>(p); })
    TILE(64, 64, 2, 2 - G, 4);
    TILE(64, 128, 2, 2, 3);
    TILE(64, 128, 2, 2, 2, 2);
    TILE(128, 128, 2, 2, 2);
    TILE(128, 128, 2, 2, 3);
    TILE(192, 256, 2, 4, 2);
    TILE(256, 256, 2, 4, 2);
#undef TILE
}

// PIECE: of a row, for those that the launcher keeps for many rows; 0: its choice
template <int PIECE>
static void rules_launch(float *o, size_t ld, const float *x, int vocab, int n, const qm_rules_t &t) {
    const dim3 grid((vocab + PIECE - 1) / PIECE, n);
    if (o == x) hipLaunchKernelGGL((k_logits_rules<true, PIECE>), grid, dim3(RULES_NT), 0, stream(), o, ld, x, ld, vocab, t);
    else hipLaunchKernelGGL((k_logits_rules<false, PIECE>), grid, dim3(RULES_NT), 0, stream(), o, ld, x, ld, vocab, t);
}

template <int PIECE = 0>
static void rules_case(int n, int vocab, int pad, int history, int shift, bool masks, bool in_place) {
    printf("rules %d x %d + %d, %d tokens + %d, %d %d\n", n, vocab, pad, history, shift, masks, in_place);
    const size_t ld = vocab + pad, words = (vocab + 31) / 32;
    float *x = (float *)guarded(((n - 1) * ld + vocab) * 4, 0);
    float *o = in_place ? x : (float *)guarded(((n - 1) * ld + vocab) * 4, 77);
    const float mark = in_place ? 0.0f : *(o + vocab - 1);
    int *tok = (int *)guarded(4 * (size_t)n * history, 0), *len = (int *)guarded(4 * n, 0), *from = (int *)guarded(4 * n, 0);
    float *pen = (float *)guarded(12 * n, 0);
    int *row = (int *)guarded(4 * (n + 1), 0), *btok = (int *)guarded(4 * 3 * n, 0), *of = (int *)guarded(4 * n, 0);
    float *bias = (float *)guarded(4 * 3 * n, 0);
    uint32_t *mask = (uint32_t *)guarded(4 * words * n, 0x5F);
    unsigned st = 1;
    auto rnd = [&](int below) { return (int)((st = st * 1664525u + 1013904223u) >> 8) % below; };
    for (int i = 0; i < n; i++) {
        for (int v = 0; v < vocab; v++) x[i * ld + v] = (rnd(2001) - 1000) / 64.0f;
        for (int j = 0; j < history; j++) tok[i * history + j] = rnd(vocab + 2) - 1;
        len[i] = i % 3 == 2 ? history : rnd(history + 1);
        from[i] = rnd(history + 1);
        pen[i] = 2.0f;
        pen[n + i] = 0.5f;
        pen[2 * n + i] = 0.25f;
        row[i + 1] = row[i] + 3;
        for (int j = 0; j < 3; j++) { btok[3 * i + j] = rnd(j == 2 ? vocab + 1 : min(vocab, 3)); bias[3 * i + j] = rnd(9) + 1.0f; }
        of[i] = i % 4 == 3 ? -1 : rnd(n);
    }
    std::vector<float> y(n * (size_t)vocab);
    for (int i = 0; i < n; i++)
        for (int v = 0; v < vocab; v++) {
            float w = x[i * ld + v];
            int seen = 0, count = 0, last = -1;
            for (int j = 0; j < len[i]; j++)
                if (tok[i * history + j] == v) { seen = 1; count += j >= from[i]; }
            if (seen) w = w > 0 ? w / 2 : w * 2;
            if (count) w = w - 0.25f * count - 0.5f;
            for (int j = row[i]; j < row[i + 1]; j++)
                if (btok[j] == v) last = j;
            if (last >= 0) w += bias[last];
            if (masks && of[i] >= 0 && !(mask[of[i] * words + v / 32] >> v % 32 & 1)) w = -INFINITY;
            y[i * (size_t)vocab + v] = w;
        }
    const qm_rules_t t = {tok, history, from, len, pen, pen + n, pen + 2 * n, row, btok, bias, 3 * n,
                          masks ? mask : nullptr, words, masks ? n : 0, masks ? of : nullptr};
    if constexpr (PIECE > 0) rules_launch<PIECE>(o, ld, x, vocab, n, t);
    else want(qm_logits_rules(o, ld, x, ld, vocab, n, &t) == QH_OK, "refused");
    for (int i = 0; i < n; i++)
        for (size_t v = 0; v < (i + 1 < n ? ld : vocab); v++)
            want(o[i * ld + v] == (v < (size_t)vocab ? y[i * (size_t)vocab + v] : mark), "a logit");
    release();
}

int main(int argc, char **argv) {
    if (argc < 2) { printf("10\n"); return 0; }
    const int which = atoi(argv[1]);
    g_front = which & 1;
    switch (which / 2) {
    case 0:
        for (bool bf : {false, true})
            for (int K : {1, 7, 8, 255, 256, 257, 1000, 1024, 1025, 4096, 4104, 8192, 9000, 17000})
                for (int rows : {1, 5, 18}) {
                    rows_case(rows, K, bf, (K + 7) / 8 * 8, (K + 15) / 16 * 16);
                    rows_case(rows, K, bf, K + 1, K);
                }
        rows_case(2100, 4000, false, 4000, 4000);         // past the caches
        for (auto [rows, K] : {std::pair{1030, 200}, {1030, 1001}, {1030, 2047}, {4100, 1500}, {260, 8190}})
            rows_case(rows, K, rows & 2, K, K);           // enough rows for other kernels
        break;
    case 1: products<false, false>(); break;
    case 2: products<true, false>(); break;
    case 3: products<false, true>(); products<true, true>(); break;
    case 4:
        g_threads_run = true;
        for (bool in_place : {false, true})
            for (bool masks : {false, true}) {
                rules_case(2, 1, 0, 3, 0, masks, in_place);
                rules_case(3, 33, 1, 5, 0, masks, in_place);
                rules_case(5, 8190, 2, 70, 0, masks, in_place);
                rules_case(2, 8193, 3, 2600, 0, masks, in_place);
                rules_case(1, 9000, 0, 5003, 0, masks, in_place);
                rules_case<4096>(3, 4099, 1, 4100, 0, masks, in_place);
                rules_case<8192>(3, 8190, 2, 70, 0, masks, in_place);
                rules_case<8192>(2, 8195, 3, 2600, 0, masks, in_place);
            }
        break;
    }
    printf("every access inside\n");
    return 0;
}
