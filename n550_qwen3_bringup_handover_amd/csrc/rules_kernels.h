// Rules on logits: penalties for repeated tokens, biases and masks, in one
// pass.  Compiled into hip_model.hip.
//
//   y = x; seen in the row's history:       y = y > 0 ? y / r : y r
//   c times behind the row's prompt, c > 0: y = y - f c, y = y - p
//   named by the row's biases:              y = y + b (of the last entry)
//   mask bit 0:                             y = -inf
// each step rounded to fp32, without fused multiply-adds.
//
// A block takes RULES_PIECE tokens of a row and reads the row's whole history
// for those that lie there: a count and a "seen" bit for each token in LDS,
// which integer atomics fill in any order with the same result.  So there is
// no bound on the history's length, no table of n x vocab counts in memory and
// nothing to clear between calls.

#define RULES_PIECE 4096
#define RULES_GROUPS (RULES_PIECE / 4 / NTH)  // of four tokens a thread: tid, tid + NTH, ...
#define RULES_SEEN 0x80000000u

// e: a token's word of the table
__device__ __forceinline__ float rules_penalised(float x, uint32_t e, float r, float f, float p) {
#pragma clang fp contract(off)
    if (e & RULES_SEEN) x = x > 0.0f ? x / r : x * r;
    const uint32_t c = e & ~RULES_SEEN;
    if (c) {
        x = x - f * (float)c;
        x = x - p;
    }
    return x;
}

// four tokens from x on, `left` of them there
template <bool VEC>
__device__ __forceinline__ f32x4 rules_load(const float *x, int left) {
    if (VEC && left >= 4) return *(const f32x4 *)x;
    f32x4 v = {};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < left) v[e] = x[e];
    return v;
}
template <bool VEC>
__device__ __forceinline__ void rules_store(float *x, f32x4 v, int left) {
    if (VEC && left >= 4) {
        *(f32x4 *)x = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < left) x[e] = v[e];
}

// INPLACE: what a rule does not touch is neither read nor written.
// Every load that does not wait for another one goes out first: the logits, the
// first tokens of the history (whose number is then not known yet), the row's
// numbers.
template <bool VEC, bool INPLACE, bool BIAS>
__global__ __launch_bounds__(NTH) void k_logits_rules(float *out, size_t ldo, const float *in, size_t ldx, int vocab,
                                                     qm_rules_t t) {
    __shared__ __align__(16) uint32_t tab[RULES_PIECE];          // occurrences behind the prompt, RULES_SEEN
    __shared__ __align__(16) int last[BIAS ? RULES_PIECE : 4];   // 1 + the last bias entry that names the token
    const int i = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * RULES_PIECE, nv = min(vocab - v0, RULES_PIECE);
    const float *x = in + (size_t)i * ldx + v0;
    float *o = out + (size_t)i * ldo + v0;
    f32x4 y[RULES_GROUPS];
    if constexpr (!INPLACE) {
#pragma unroll
        for (int u = 0; u < RULES_GROUPS; u++) y[u] = rules_load<VEC>(x + 4 * (tid + u * NTH), nv - 4 * (tid + u * NTH));
    }
    const int *h = t.token + (size_t)i * t.ld_token;
    int early[4];
#pragma unroll
    for (int u = 0; u < 4; u++) early[u] = tid + u * NTH < t.ld_token && t.token ? h[tid + u * NTH] : -1;
    int len = t.token ? t.n_token[i] : 0;
    if (len > t.ld_token) len = 0;
    const int prompt = t.n_prompt ? t.n_prompt[i] : 0;
    int b0 = 0, b1 = 0;
    if constexpr (BIAS) {
        b0 = t.bias_row[i];
        b1 = t.bias_row[i + 1];
        if (b0 < 0 || b1 > t.n_bias) b1 = b0;
    }
    const float r = t.repetition ? t.repetition[i] : 1.0f, f = t.frequency ? t.frequency[i] : 0.0f;
    const float p = t.presence ? t.presence[i] : 0.0f;
    const int mi = !t.mask ? -1 : t.mask_of ? t.mask_of[i] : i;
    const uint32_t *mask = mi >= 0 && mi < t.n_mask ? t.mask + (size_t)mi * t.ld_mask + v0 / 32 : nullptr;

#pragma unroll
    for (int u = 0; u < RULES_GROUPS; u++) {
        ((uint4 *)tab)[tid + u * NTH] = make_uint4(0, 0, 0, 0);
        if constexpr (BIAS) ((uint4 *)last)[tid + u * NTH] = make_uint4(0, 0, 0, 0);
    }
    uint32_t words[RULES_GROUPS];
#pragma unroll
    for (int u = 0; u < RULES_GROUPS; u++)
        words[u] = mask && 4 * (tid + u * NTH) < nv ? mask[(tid + u * NTH) / 8] >> (tid % 8 * 4) & 15 : 15;
    __syncthreads();
    auto count = [&](int token, int j) {
        const unsigned v = (unsigned)token - (unsigned)v0;
        if (v >= (unsigned)nv) return;
        atomicOr(&tab[v], RULES_SEEN);
        if (j >= prompt) atomicAdd(&tab[v], 1u);
    };
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (tid + u * NTH < len) count(early[u], tid + u * NTH);
    for (int j = tid + 4 * NTH; j < len; j += 4 * NTH) {
        int v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] = h[min(j + u * NTH, len - 1)];
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (j + u * NTH < len) count(v[u], j + u * NTH);
    }
    if constexpr (BIAS)
        for (int j = b0 + tid; j < b1; j += NTH) {
            const unsigned v = (unsigned)t.bias_token[j] - (unsigned)v0;
            if (v < (unsigned)nv) atomicMax(&last[v], j + 1);
        }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < RULES_GROUPS; u++) {
        const int g = tid + u * NTH, left = nv - 4 * g;
        if (left <= 0) continue;
        const uint4 e = ((const uint4 *)tab)[g];
        const uint4 l = BIAS ? ((const uint4 *)last)[g] : make_uint4(0, 0, 0, 0);
        const bool touched = (e.x | e.y | e.z | e.w | l.x | l.y | l.z | l.w) != 0;
        if constexpr (INPLACE) {
            if (!touched && words[u] == 15) continue;
            if (words[u]) y[u] = rules_load<VEC>(x + 4 * g, left);
        }
        if (touched) {
            const uint32_t ee[4] = {e.x, e.y, e.z, e.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                y[u][k] = rules_penalised(y[u][k], ee[k], r, f, p);
                if (BIAS && ll[k]) y[u][k] += t.bias[ll[k] - 1];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (!(words[u] >> k & 1)) y[u][k] = -INFINITY;
        rules_store<VEC>(o + 4 * g, y[u], left);
    }
}

// ---------------------------------------------------------------------------
// launcher
// ---------------------------------------------------------------------------
extern "C" int qm_logits_rules(float *out, size_t ldo, const float *logits, size_t ld, int vocab, int n, const qm_rules_t *t) {
    if (!t || n < 0 || vocab < 1 || ldo < (size_t)vocab || ld < (size_t)vocab) return QH_EINVAL;
    if (n == 0) return QH_OK;
    if (!out || !logits || (out == logits && ldo != ld) || (((uintptr_t)out | (uintptr_t)logits) & 3)) return QH_EINVAL;
    if (n > QM_RULES_MAX_ROWS || vocab > QM_RULES_MAX_VOCAB || ldo > (size_t)1 << 40 || ld > (size_t)1 << 40) return QH_ETOOBIG;
    // rows must not reach into other rows of the other buffer
    const uintptr_t o = (uintptr_t)out, x = (uintptr_t)logits;
    const uintptr_t oe = o + ((size_t)(n - 1) * ldo + vocab) * sizeof(float), xe = x + ((size_t)(n - 1) * ld + vocab) * sizeof(float);
    if (o != x && o < xe && x < oe) return QH_EINVAL;
    if (t->ld_token < 0 || t->n_bias < 0 || t->n_mask < 0) return QH_EINVAL;
    if (t->token && !t->n_token) return QH_EINVAL;
    if (!t->token && (t->repetition || t->presence || t->frequency)) return QH_EINVAL;
    if (t->ld_token > QM_RULES_MAX_TOKENS) return QH_ETOOBIG;
    if (t->bias_row && t->n_bias > 0 && (!t->bias_token || !t->bias)) return QH_EINVAL;
    if (!t->bias_row && t->n_bias > 0) return QH_EINVAL;
    if (t->mask && t->ld_mask < ((size_t)vocab + 31) / 32) return QH_EINVAL;
    if (t->mask && !t->mask_of && t->n_mask < n) return QH_EINVAL;
    if (t->mask_of && !t->mask) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    const dim3 grid((vocab + RULES_PIECE - 1) / RULES_PIECE, n);
    const bool vec = aligned16(out) && aligned16(logits) && ldo % 4 == 0 && ld % 4 == 0;
#define RULES_AS(V, I, B) \
    hipLaunchKernelGGL((k_logits_rules<V, I, B>), grid, dim3(NTH), 0, stream(), out, ldo, logits, ld, vocab, *t)
#define RULES(V, I)                           \
    do {                                      \
        if (t->n_bias > 0) RULES_AS(V, I, true); \
        else RULES_AS(V, I, false);           \
    } while (0)
    if (out == logits) {
        if (vec) RULES(true, true);
        else RULES(false, true);
    } else {
        if (vec) RULES(true, false);
        else RULES(false, false);
    }
#undef RULES
#undef RULES_AS
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}
