// kv8_kernels.h compiled for the host: what it takes from the HIP runtime and
// from hip_model.hip.  A block is a host thread for each of its own, or, with
// KV8_ONE_LANE defined, one lane after the other, which leaves the exchanges
// between lanes out; matrix products are empty.  So the store's kernels can be
// run for their values, and both for what they read and write: no address
// depends on what lanes exchange.
#include <math.h>
#include <float.h>
#include <pthread.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <algorithm>
#include <thread>
#include <vector>

// ---- what the header takes from the HIP runtime and hip_model.hip
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
static dim3 gridDim;
struct uint2 { unsigned x, y; };
struct uint4 { unsigned x, y, z, w; };
static inline uint4 make_uint4(unsigned a, unsigned b, unsigned c, unsigned d) { return uint4{a, b, c, d}; }
using std::max;
using std::min;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
#define WAVE 64
#define NTH 256
#define HD 128
#define NKV 8
#define GRP 2
#define QKV_LD 4096
static inline float bf16f(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
static pthread_barrier_t g_block, g_wave[16];
#ifdef KV8_ONE_LANE
static inline void __syncthreads() {}
template <typename F> static inline float over_wave(float v, F) { return v; }
#else
static float g_lane[16][WAVE];
static inline void __syncthreads() { pthread_barrier_wait(&g_block); }
template <typename F> static inline float over_wave(float v, F f) {
    const int w = threadIdx.x / WAVE, l = threadIdx.x % WAVE;
    g_lane[w][l] = v;
    pthread_barrier_wait(&g_wave[w]);
    float r = g_lane[w][0];
    for (int i = 1; i < WAVE; i++) r = f(r, g_lane[w][i]);
    pthread_barrier_wait(&g_wave[w]);
    return r;
}
#endif
static inline float wave_sum(float v) { return over_wave(v, [](float a, float b) { return a + b; }); }
static inline float wave_max(float v) { return over_wave(v, [](float a, float b) { return fmaxf(a, b); }); }
static inline float sumsq2(float a, float b) { return a * a + b * b; }
static inline void rope_pair(float y0, float y1, float c, float sn, float &o0, float &o1) {
    o0 = y0 * c - y1 * sn;
    o1 = y1 * c + y0 * sn;
}
extern "C" __bf16 __truncsfbf2(float f) {             // RNE; the host's runtime may have none
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    u = (u & 0x7FFFFFFF) > 0x7F800000 ? u | 0x400000 : u + 0x7FFF + ((u >> 16) & 1);
    return __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
}
static inline f32x2 swap16(float x) { return f32x2{x, x}; }
static inline f32x2 swap32(float x) { return f32x2{x, x}; }
static inline float mul_add(float a, float b, float c) { return a * b + c; }
static inline uint2 pack4(f32x4) { return uint2{}; }
// a buffer's loads past its size return zeros and read nothing, stores past it do nothing
struct rsrc { char *p; size_t bytes; };
#define __amdgpu_buffer_rsrc_t rsrc
static inline rsrc buf_rsrc(const void *p, size_t bytes) { return rsrc{(char *)p, bytes}; }
static inline u32x4 buf_load(rsrc r, size_t at) {
    u32x4 v = {};
    if (at + 16 <= r.bytes) memcpy(&v, r.p + at, 16);
    return v;
}
static inline void buf_store(u32x4 v, rsrc r, size_t at) {
    if (at + 16 <= r.bytes) memcpy(r.p + at, &v, 16);
}
#define BUF_OOB 0x80000000u
static inline int __umulhi(unsigned a, unsigned b) { return (int)((uint64_t)a * b >> 32); }
static inline bool __any(bool b) { return b; }
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_s_waitcnt(x) ((void)0)
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, hi) (old)
#define __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, hi) bf16x2{}
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_raw_buffer_load_b128(r, o, s, a) buf_load(r, o)
#define __builtin_amdgcn_raw_buffer_store_b128(v, r, o, s, a) buf_store(v, r, o)
#define __hip_atomic_fetch_add(p, v, o, s) ((*(p) += (v)) - (v))
#define __hip_atomic_store(p, v, o, s) (*(p) = (v))
#ifndef hipLaunchKernelGGL
#define hipLaunchKernelGGL(...) ((void)0)
#endif
enum { hipSuccess };
static inline int hipGetLastError() { return hipSuccess; }
typedef void *hipStream_t;
static inline hipStream_t stream() { return (hipStream_t)&g_block; }
#include "hip_shim.h"
#include "model_shim.h"
#include "kv8_kernels.h"

// ---- buffers against an unreadable page
static bool g_front;                                  // the page before the start, not behind the end
static std::vector<std::pair<void *, size_t>> g_maps;
static void *guarded(size_t bytes) {
    const size_t page = 4096, n = (bytes + page - 1) / page * page;
    char *p = (char *)mmap(nullptr, n + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (p == MAP_FAILED || mprotect(p + page, n, PROT_READ | PROT_WRITE)) abort();
    g_maps.push_back({p, n + 2 * page});
    return g_front ? p + page : p + page + (n - bytes);
}
static void release() {
    for (auto &m : g_maps) munmap(m.first, m.second);
    g_maps.clear();
}
