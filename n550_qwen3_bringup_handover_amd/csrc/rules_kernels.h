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
#define RULES_SEEN 0x80000000u

// e: a token's word of `tab`
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

__global__ __launch_bounds__(NTH) void k_logits_rules(float *out, size_t ldo, const float *x, size_t ldx, int vocab,
                                                     qm_rules_t t) {
    __shared__ uint32_t tab[RULES_PIECE];     // occurrences behind the prompt, RULES_SEEN
    __shared__ int last[RULES_PIECE];         // 1 + the last bias entry that names the token
    const int i = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * RULES_PIECE, nv = min(vocab - v0, RULES_PIECE);
    for (int v = tid; v < RULES_PIECE; v += NTH) {
        tab[v] = 0;
        last[v] = 0;
    }
    __syncthreads();
    if (t.token) {
        const int len = t.n_token[i], prompt = t.n_prompt ? t.n_prompt[i] : 0;
        const int *h = t.token + (size_t)i * t.ld_token;
        if (len >= 0 && len <= t.ld_token)
            for (int j = tid; j < len; j += NTH) {
                const unsigned v = (unsigned)h[j] - (unsigned)v0;
                if (v < (unsigned)nv) {
                    atomicOr(&tab[v], RULES_SEEN);
                    if (j >= prompt) atomicAdd(&tab[v], 1u);
                }
            }
    }
    if (t.bias_row) {
        const int b0 = t.bias_row[i], b1 = t.bias_row[i + 1];
        if (b0 >= 0 && b1 <= t.n_bias)
            for (int j = b0 + tid; j < b1; j += NTH) {
                const unsigned v = (unsigned)t.bias_token[j] - (unsigned)v0;
                if (v < (unsigned)nv) atomicMax(&last[v], j + 1);
            }
    }
    __syncthreads();
    const float r = t.repetition ? t.repetition[i] : 1.0f, f = t.frequency ? t.frequency[i] : 0.0f;
    const float p = t.presence ? t.presence[i] : 0.0f;
    const uint32_t *mask = nullptr;
    if (t.mask) {
        const int m = t.mask_of ? t.mask_of[i] : i;
        if (m >= 0 && m < t.n_mask) mask = t.mask + (size_t)m * t.ld_mask;
    }
    for (int v = tid; v < nv; v += NTH) {
        float y = rules_penalised(x[(size_t)i * ldx + v0 + v], tab[v], r, f, p);
        if (last[v]) y += t.bias[last[v] - 1];
        if (mask && !(mask[(v0 + v) >> 5] >> ((v0 + v) & 31) & 1)) y = -INFINITY;
        out[(size_t)i * ldo + v0 + v] = y;
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
    hipLaunchKernelGGL(k_logits_rules, dim3((vocab + RULES_PIECE - 1) / RULES_PIECE, n), dim3(NTH), 0, stream(), out, ldo,
                       logits, ld, vocab, *t);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}
