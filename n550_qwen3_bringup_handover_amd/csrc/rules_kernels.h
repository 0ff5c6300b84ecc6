// Rules on logits: penalties for repeated tokens, biases and masks, in one
// pass.  Compiled into hip_model.hip.
//
//   y = x; seen in the row's history:       y = y > 0 ? y / r : y r
//   c times behind the row's prompt, c > 0: y = y - f c, y = y - p
//   named by the row's biases:              y = y + b (of the last entry)
//   mask bit 0:                             y = -inf
// each step rounded to fp32, without fused multiply-adds.
//
// A block takes PIECE tokens of a row and reads the row's whole history for
// those that lie there: a count and a "seen" bit for each token in LDS, which
// integer atomics fill in any order with the same result.  So there is no bound
// on the history's length, no table of n x vocab counts in memory and nothing to
// clear between calls.
// Many copied rows are bound by memory, 64 of 151,936 under penalties, biases and
// masks 18.9 us (20.4 from no cache; a copy of as much 15.0); many in place by the
// scans of the histories, 64 behind 2,048 tokens 11.3; few by a block's chain of
// latencies, which is shorter the fewer tokens a thread has: one row behind 700
// tokens 3.3 us in pieces of 2,048, 3.8 of 4,096 and 4.9 of 8,192, in place 3.5, 4.3
// and 6.1; 16 rows 5.9, 5.6 and 6.5.  Small pieces scan the histories more often, and
// more of them than the CUs hold at once (four on each) take turns: 34 rows 10.0 us
// in pieces of 4,096 and 8.6 of 8,192, 24 behind 8,000 tokens 10.8 in pieces of 2,048
// and 8.1 of 4,096.

#define RULES_NT 512
#define RULES_AT_ONCE 1024
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

// four tokens from x on, `left` of them there, wherever they begin.  ONCE: past the caches, for rows that
// are copied (64 rows of 151,936 that are in no cache 23.9 -> 20.5 us, 128 of 32,000
// 10.8 -> 7.8; in a cache the same)
typedef float rules_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int rules_u32x4 __attribute__((ext_vector_type(4), aligned(4)));
template <bool ONCE>
__device__ __forceinline__ f32x4 rules_load(const float *x, int left) {
    if (left >= 4) return ONCE ? __builtin_nontemporal_load((const rules_f32x4 *)x) : *(const rules_f32x4 *)x;
    f32x4 v = {};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < left) v[e] = x[e];
    return v;
}
template <bool ONCE>
__device__ __forceinline__ void rules_store(float *x, f32x4 v, int left) {
    if (left >= 4) {
        if constexpr (ONCE) __builtin_nontemporal_store((rules_f32x4)v, (rules_f32x4 *)x);
        else *(rules_f32x4 *)x = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < left) x[e] = v[e];
}

// four tokens of the history from j on, below n
__device__ __forceinline__ uint4 rules_tokens(const int *h, int j, int n) {
    if (j + 4 <= n) {
        const rules_u32x4 v = *(const rules_u32x4 *)(h + j);
        return make_uint4(v[0], v[1], v[2], v[3]);
    }
    uint4 v = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (j < n) v.x = h[j];
    if (j + 1 < n) v.y = h[j + 1];
    if (j + 2 < n) v.z = h[j + 2];
    if (j + 3 < n) v.w = h[j + 3];
    return v;
}

// INPLACE: what a rule does not touch is neither read nor written.
// Every load that does not wait for another one goes out first: the logits, the
// first tokens of the history (whose number is then not known yet), the row's
// numbers.  The biases take the table's place once the penalties are done with it.
template <bool INPLACE, int PIECE>
__global__ __launch_bounds__(RULES_NT) void k_logits_rules(float *out, size_t ldo, const float *in, size_t ldx, int vocab,
                                                          qm_rules_t t) {
    constexpr int NT = RULES_NT, GROUPS = PIECE / 4 / NT;    // of four tokens a thread: tid, tid + NT, ...
    __shared__ __align__(16) uint32_t tab[PIECE];   // occurrences behind the prompt, RULES_SEEN; then 1 + a bias entry
    const int i = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * PIECE, nv = min(vocab - v0, PIECE);
    const float *x = in + (size_t)i * ldx + v0;
    float *o = out + (size_t)i * ldo + v0;
    f32x4 y[GROUPS];
    if constexpr (!INPLACE) {
#pragma unroll
        for (int u = 0; u < GROUPS; u++) y[u] = rules_load<!INPLACE>(x + 4 * (tid + u * NT), nv - 4 * (tid + u * NT));
    }
    const int *h = t.token + (size_t)i * t.ld_token;
    const uint4 early = rules_tokens(h, 4 * tid, t.token ? t.ld_token : 0);
    int len = t.token ? t.n_token[i] : 0;
    if (len > t.ld_token) len = 0;
    const int prompt = t.n_prompt ? t.n_prompt[i] : 0;
    int b0 = 0, b1 = 0;
    if (t.bias_row) {
        b0 = t.bias_row[i];
        b1 = t.bias_row[i + 1];
        if (b0 < 0 || b1 > t.n_bias) b1 = b0;
    }
    const float r = t.repetition ? t.repetition[i] : 1.0f, f = t.frequency ? t.frequency[i] : 0.0f;
    const float p = t.presence ? t.presence[i] : 0.0f;
    const int mi = !t.mask ? -1 : t.mask_of ? t.mask_of[i] : i;
    const uint32_t *mask = mi >= 0 && mi < t.n_mask ? t.mask + (size_t)mi * t.ld_mask + v0 / 32 : nullptr;

    auto clear = [&] {
#pragma unroll
        for (int u = 0; u < GROUPS; u++) ((uint4 *)tab)[tid + u * NT] = make_uint4(0, 0, 0, 0);
    };
    clear();
    uint32_t words[GROUPS];
#pragma unroll
    for (int u = 0; u < GROUPS; u++)
        words[u] = mask && 4 * (tid + u * NT) < nv ? mask[(tid + u * NT) / 8] >> (tid % 8 * 4) & 15 : 15;
    __syncthreads();
    auto count = [&](uint32_t token, int j) {
        const uint32_t v = token - (uint32_t)v0;
        if (j >= len || v >= (uint32_t)nv) return;
        atomicOr(&tab[v], RULES_SEEN);
        if (j >= prompt) atomicAdd(&tab[v], 1u);
    };
    auto count4 = [&](uint4 v, int j) {
        count(v.x, j);
        count(v.y, j + 1);
        count(v.z, j + 2);
        count(v.w, j + 3);
    };
    count4(early, 4 * tid);
    for (int j = 4 * (tid + NT); j < len; j += 8 * NT) {
        const uint4 one = rules_tokens(h, j, len), two = rules_tokens(h, j + 4 * NT, len);
        count4(one, j);
        count4(two, j + 4 * NT);
    }
    __syncthreads();
    uint32_t have = 0;                                    // groups whose values are in y
#pragma unroll
    for (int u = 0; u < GROUPS; u++) {
        const int g = tid + u * NT, left = nv - 4 * g;
        const uint4 e = ((const uint4 *)tab)[g];
        if ((e.x | e.y | e.z | e.w) == 0) continue;
        if constexpr (INPLACE) y[u] = rules_load<!INPLACE>(x + 4 * g, left);
        have |= 1u << u;
        const uint32_t ee[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int k = 0; k < 4; k++) y[u][k] = rules_penalised(y[u][k], ee[k], r, f, p);
    }
    if (b0 < b1) {                                        // the same for the whole block
        __syncthreads();
        clear();
        __syncthreads();
        for (int j = b0 + tid; j < b1; j += NT) {
            const uint32_t v = (uint32_t)t.bias_token[j] - (uint32_t)v0;
            if (v < (uint32_t)nv) atomicMax(&tab[v], (uint32_t)j + 1);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < GROUPS; u++) {
            const int g = tid + u * NT, left = nv - 4 * g;
            const uint4 e = ((const uint4 *)tab)[g];
            if ((e.x | e.y | e.z | e.w) == 0) continue;
            if (INPLACE && !(have >> u & 1)) y[u] = rules_load<!INPLACE>(x + 4 * g, left);
            have |= 1u << u;
            const uint32_t ee[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (ee[k]) y[u][k] += t.bias[ee[k] - 1];
        }
    }
#pragma unroll
    for (int u = 0; u < GROUPS; u++) {
        const int g = tid + u * NT, left = nv - 4 * g;
        if (left <= 0) continue;
        if constexpr (INPLACE) {
            if (!(have >> u & 1) && words[u] == 15) continue;
            if (!(have >> u & 1) && words[u]) y[u] = rules_load<!INPLACE>(x + 4 * g, left);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (!(words[u] >> k & 1)) y[u][k] = -INFINITY;
        rules_store<!INPLACE>(o + 4 * g, y[u], left);
    }
}

// a sequence's text after a step: the token that is fed next, at its position
__global__ __launch_bounds__(NTH) void k_rules_note(int *__restrict__ text, int ld, int *__restrict__ n_text,
                                                   const int *__restrict__ tok, const int *__restrict__ pos, int n) {
    const int i = blockIdx.x * NTH + threadIdx.x;
    if (i >= n || pos[i] < 0 || pos[i] >= ld) return;
    text[(size_t)i * ld + pos[i]] = tok[i];
    n_text[i] = pos[i] + 1;
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
extern "C" int qm_rules_note(int *text, int ld, int *n_text, const int *tok, const int *pos, int n) {
    if (!text || !n_text || !tok || !pos || ld <= 0 || n <= 0) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    hipLaunchKernelGGL(k_rules_note, dim3((n + NTH - 1) / NTH), dim3(NTH), 0, stream(), text, ld, n_text, tok, pos, n);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

extern "C" int qm_logits_rules(float *out, size_t ldo, const float *logits, size_t ld, int vocab, int n, const qm_rules_t *t) {
    if (!t || n < 0 || vocab < 1 || ldo < (size_t)vocab || ld < (size_t)vocab) return QH_EINVAL;
    if (n == 0) return QH_OK;
    if (!out || !logits || (out == logits && ldo != ld) || (((uintptr_t)out | (uintptr_t)logits) & 3)) return QH_EINVAL;
    if (n > QM_RULES_MAX_ROWS || vocab > QM_RULES_MAX_VOCAB || ldo > (size_t)1 << 40 || ld > (size_t)1 << 40) return QH_ETOOBIG;
    const size_t es = sizeof(float);
    if (out != logits && qh_rows_meet(out, ldo * es, vocab * es, logits, ld * es, vocab * es, n)) return QH_EINVAL;
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
    // the smallest piece that takes a row, or whose blocks all run at once
    auto fits = [&](int piece) { return vocab <= piece || (size_t)((vocab + piece - 1) / piece) * n <= RULES_AT_ONCE; };
#define RULES(INPLACE, PIECE)                                                                                     \
    hipLaunchKernelGGL((k_logits_rules<INPLACE, PIECE>), dim3((vocab + PIECE - 1) / PIECE, n), dim3(RULES_NT), 0, \
                       stream(), out, ldo, logits, ld, vocab, *t)
#define RULES_OF(PIECE)                         \
    do {                                        \
        if (out == logits) RULES(true, PIECE);  \
        else RULES(false, PIECE);               \
    } while (0)
    if (fits(2048)) RULES_OF(2048);
    else if (fits(4096)) RULES_OF(4096);
    else RULES_OF(8192);
#undef RULES_OF
#undef RULES
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}
