// The 8-bit KV cache: storing rows into it and attention over it.  Compiled
// into hip_model.hip.
//
// One layer's cache (qm_kv8_t): pages of B = 16, 32 or 64 tokens.  A finished
// block lies in a page as one byte per value with one fp32 scale per kv head
// for K and one for V; the unfinished block of a sequence lies in its tail as
// bf16.  A block is quantised once, when its last row arrives, from the same
// bf16 values whatever calls brought them, and never changes again, so beams
// can share pages.
//   x = bf16(row)           RNE; NaN -> 0, magnitudes saturate at the largest bf16
//   a = max |x| over B x D, s = a / qmax (0 where a < 2^-100)
//   code = rne(x / s)       e4m3 (qmax 448) or int8 (qmax 127); division and
//                           scale rounded to fp32
// K rows lie [slot][dim], V columns [dim][slot]: both products of attention
// then read 8 or 16 contiguous bytes per lane in the order their MFMA wants.

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

#define KV8_TINY 0x1p-100f
#define KV8_BF16_MAX 3.38953139e38f       // 0x7F7F as bf16

template <int FMT>
struct kv8_qmax { static constexpr float v = FMT == QM_KV8_E4M3 ? 448.0f : 127.0f; };

// what a call says about entry e: its rows in the call's buffers and the
// position of the first; false (the entry is left out) where these do not fit
struct kv8_entry { int r0, cnt, pos; };
__device__ __forceinline__ bool kv8_get(kv8_entry &t, const qm_kv8_t &c, const int *row, const int *pos, int e,
                                        int rows, int max_rows) {
    t.r0 = row ? row[e] : e;
    const int r1 = row ? row[e + 1] : e + 1;
    t.pos = pos[e];
    if (t.r0 < 0 || r1 <= t.r0 || r1 > rows || r1 - t.r0 > max_rows) return false;
    t.cnt = r1 - t.r0;
    return t.pos >= 0 && t.pos <= c.max_blocks * c.block - t.cnt;
}

// ---------------------------------------------------------------------------
// The model's q and k rows before they meet the cache: QK-norm and RoPE
// (qwen3.c:298-305, ops_scalar.c:21-35) of one head's 128 values, two a lane
// ---------------------------------------------------------------------------
typedef struct {
    float *qkv;                        // rows of QKV_LD: 16 query heads, 8 key heads, 8 value heads
    const uint16_t *qn, *kn;           // norm weights
    const float *rcos, *rsin;          // [max_seq][64]
    int max_seq;
    float eps;
} kv8_rope;
__device__ __forceinline__ void kv8_rope_head(const kv8_rope &a, const float *x, const uint16_t *w, int pos, int lane,
                                              float &o0, float &o1) {
    const float x0 = x[lane], x1 = x[lane + 64];
    const float c = a.rcos[(size_t)pos * (HD / 2) + lane], sn = a.rsin[(size_t)pos * (HD / 2) + lane];
    const float sc = 1.0f / sqrtf(wave_sum(sumsq2(x0, x1)) / (float)HD + a.eps);
    rope_pair((x0 * sc) * bf16f(w[lane]), (x1 * sc) * bf16f(w[lane + 64]), c, sn, o0, o1);
}

// A prompt's pass: row i at position *pos + i.  k in place; q in place or, where
// qb is set, as bf16 [nt][2048].  grid = (nt, 6): wave w of block (i, b) takes
// head 4 b + w of q's 16 and k's 8.  (A decode step's rows: k_kv8_append.)
__global__ __launch_bounds__(NTH) void k_qk_rope(kv8_rope a, uint16_t *__restrict__ qb, const int *__restrict__ pos_d) {
    constexpr int QH = NKV * GRP;
    const int i = blockIdx.x, lane = threadIdx.x & 63, hd = blockIdx.y * 4 + (threadIdx.x >> 6);
    const int pos = *pos_d + i;
    if (pos < 0 || pos >= a.max_seq) return;
    float *x = a.qkv + (size_t)i * QKV_LD + hd * HD;         // k's heads lie behind q's
    float o0, o1;
    kv8_rope_head(a, x, hd < QH ? a.qn : a.kn, pos, lane, o0, o1);
    if (qb && hd < QH) {
        __bf16 *o = (__bf16 *)qb + (size_t)i * (QH * HD) + hd * HD;
        o[lane] = (__bf16)o0;
        o[lane + 64] = (__bf16)o1;
    } else {
        x[lane] = o0;
        x[lane + 64] = o1;
    }
}

// blocks of sequence s that are not finished (from pos[s] / block on; all where
// pos is NULL) get its own pages, s * max_blocks + block index
__global__ __launch_bounds__(NTH) void k_kv8_own(int *__restrict__ table, const int *__restrict__ pos, int block,
                                                int max_blocks) {
    const int s = blockIdx.y, b = blockIdx.x * NTH + threadIdx.x;
    if (b < max_blocks && (!pos || b >= pos[s] / block)) table[(size_t)s * max_blocks + b] = s * max_blocks + b;
}

// ---------------------------------------------------------------------------
// store
// ---------------------------------------------------------------------------
// a row's value as the cache holds it: bf16, finite
__device__ __forceinline__ __bf16 kv8_held(float x) {
    x = x == x ? x : 0.0f;
    return (__bf16)fminf(fmaxf(x, -KV8_BF16_MAX), KV8_BF16_MAX);
}

// A block's scale s = a / qmax and what divides by it: x / s rounded to fp32, as
// the definition has it, in three instructions for the compiler's ten.  With
// y = 1 / s rounded, q = x y is off by a last place or two, and q plus its
// remainder x - q s times y rounds to the quotient -- for every
// pair of 8-bit significands of x and a, which is all there are (the tests
// divide each).  Small blocks are scaled up first, so that no remainder
// underflows.
struct kv8_div { float s, y, up; };
template <int FMT>
__device__ __forceinline__ kv8_div kv8_scale(float a) {
    kv8_div d;
    d.up = a < 0x1p-40f ? 0x1p64f : 1.0f;
    d.s = a < KV8_TINY ? 0.0f : a / kv8_qmax<FMT>::v;
    d.y = d.s == 0.0f ? 0.0f : 1.0f / (d.s * d.up);
    return d;
}
__device__ __forceinline__ float kv8_quotient(float x, kv8_div d) {
    x *= d.up;
    const float q = x * d.y, s = d.s * d.up;
    return fmaf(fmaf(-q, s, x), d.y, q);
}

template <int FMT>
__device__ __forceinline__ uint32_t kv8_codes4(float a, float b, float c, float d, kv8_div s) {
    a = kv8_quotient(a, s);
    b = kv8_quotient(b, s);
    c = kv8_quotient(c, s);
    d = kv8_quotient(d, s);
    if constexpr (FMT == QM_KV8_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    } else {
        // |x / s| is at most 127 (1 + 2^-23): it rounds to a byte
        auto i = [](float x) { return (uint32_t)(int)rintf(x) & 0xFFu; };
        return i(a) | i(b) << 8 | i(c) << 16 | i(d) << 24;
    }
}

// sixteen consecutive values, 16-byte aligned, as they lie and as the cache holds them
template <bool BF>
struct kv8_16 {
    f32x4 v[BF ? 2 : 4];
    __device__ __forceinline__ void load(const void *p, size_t i) {
        const f32x4 *q = (const f32x4 *)(BF ? (const void *)((const __bf16 *)p + i) : (const void *)((const float *)p + i));
#pragma unroll
        for (int j = 0; j < (BF ? 2 : 4); j++) v[j] = q[j];
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (BF) return (float)__builtin_bit_cast(bf16x8, v[j >> 3])[j & 7];
        else return v[j >> 2][j & 3];
    }
};

// Block (h, e, z): kv head h of entry e, the z-th block its rows touch; B D / 16
// threads, so that a finished block is one unit of 16 values of K (of a row)
// and one of V (of a column: 16 rows of one dim) a thread, in registers from
// the load to the codes: all loads of a block in flight at once, its largest
// magnitudes the only exchange.  Rows that earlier calls brought come from the
// tail.  The rows behind the last finished block go to the tail, by z = 0
// alone and after it has read the tail: two blocks of one launch must not meet
// there.
// Bound by latencies: position, rows and tail, exchange, codes.  A row each of
// 64 sequences (3 % of which finish a block) 5.9 us, 3.1 where none does; 1,999
// rows (20.5 MB) 7.7 us, 16 x 300 5.9, where a copy of as much takes 3.9 and
// 1.2.  With the loads in the compiler's order, conversions between them, and
// the tail's values one a thread and turn, 9.9 and 7.7; in two passes over
// memory 18.5.
// ROPE: a row of each of the model's sequences, as its product left them (kn and
// vn point into rope.qkv).  The block's waves normalise and rotate its key head,
// handed on in LDS, and its query heads, in place; a launch of its own for that
// cost a layer 2 us.
template <int FMT, int D, int B, bool BF, bool ROPE>
__global__ __launch_bounds__(B *D / 16) void k_kv8_append(qm_kv8_t c, const void *kn, const void *vn, size_t ldk, size_t ldv,
                                                         const int *__restrict__ row, const int *__restrict__ pos, int rows,
                                                         int max_rows, kv8_rope rope) {
    constexpr int NT = B * D / 16, NWV = NT / WAVE;
    const int h = blockIdx.x, e = blockIdx.y, z = blockIdx.z, tid = threadIdx.x;
    kv8_entry t;
    if (!kv8_get(t, c, row, pos, e, rows, max_rows)) return;
    if (ROPE && t.pos >= rope.max_seq) return;
    __shared__ __align__(16) float krow[ROPE ? D : 4];
    auto rotate = [&] {
        if constexpr (ROPE) {
            const int lane = tid & 63;
            float *x = rope.qkv + (size_t)e * QKV_LD;
            for (int hd = tid >> 6; hd < 1 + GRP; hd += NWV) {
                float *q = x + (h * GRP + hd - 1) * HD, o0, o1;
                kv8_rope_head(rope, hd == 0 ? x + (NKV * GRP + h) * HD : q, hd == 0 ? rope.kn : rope.qn, t.pos, lane, o0, o1);
                float *o = hd == 0 ? krow : q;
                o[lane] = o0;
                o[lane + 64] = o1;
            }
            __syncthreads();
        }
    };
    const int end = t.pos + t.cnt, b0 = t.pos / B, bl = end / B, b = b0 + z;
    if (b >= bl && z > 0) return;
    const int kr = tid / (D / 16), kd = tid % (D / 16) * 16;           // the thread's K: slot and dims
    const int vd = tid % D, vr = tid / D * 16;                         // and V: dim and slots
    __bf16 *kt = (__bf16 *)c.k_tail + ((size_t)e * c.heads + h) * (B * D);
    __bf16 *vt = (__bf16 *)c.v_tail + ((size_t)e * c.heads + h) * (B * D);

    if (b < bl) {
        const int page = c.table[(size_t)e * c.max_blocks + b];
        const int have = max(t.pos - b * B, 0);           // rows in the tail, < B
        const int p0 = t.r0 + b * B - t.pos;              // row of the block's slot 0 (before r0 where some are in the tail)
        // every load first, the tail's too where some of the rows lie there
        kv8_16<true> kold = {}, vold = {};
        if (have > 0) {
            kold.load(kt, kr * D + kd);
            vold.load(vt, vd * B + vr);
        }
        kv8_16<BF> knew;
        float vnew[16];
        if constexpr (!ROPE) knew.load(kn, (size_t)(p0 + max(kr, have)) * ldk + h * D + kd);
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const size_t i = (size_t)(p0 + max(vr + j, have)) * ldv + h * D + vd;
            vnew[j] = BF ? (float)((const __bf16 *)vn)[i] : ((const float *)vn)[i];
        }
        __builtin_amdgcn_sched_barrier(0);                // all in flight before the first is waited for
        if constexpr (ROPE) {
            rotate();
            knew.load(krow, kd);
        }
        __bf16 x[16], y[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x[j] = kv8_held(kr < have ? kold.at(j) : knew.at(j));
            y[j] = kv8_held(vr + j < have ? vold.at(j) : vnew[j]);
        }
        float ak = 0.0f, av = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            ak = fmaxf(ak, fabsf((float)x[j]));
            av = fmaxf(av, fabsf((float)y[j]));
        }
        __shared__ float red[2][NWV];
        ak = wave_max(ak);
        av = wave_max(av);
        if ((tid & 63) == 0) { red[0][tid >> 6] = ak; red[1][tid >> 6] = av; }
        __syncthreads();                                  // the tail has been read, too
#pragma unroll
        for (int w = 0; w < NWV; w++) {
            ak = fmaxf(ak, red[0][w]);
            av = fmaxf(av, red[1][w]);
        }
        const kv8_div ks = kv8_scale<FMT>(ak), vs = kv8_scale<FMT>(av);
        if (page >= 0 && page < c.n_page) {               // the same for the whole block
            const size_t at = (size_t)page * c.heads + h;
            uint32_t u[4], w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                u[j] = kv8_codes4<FMT>((float)x[4 * j], (float)x[4 * j + 1], (float)x[4 * j + 2], (float)x[4 * j + 3], ks);
                w[j] = kv8_codes4<FMT>((float)y[4 * j], (float)y[4 * j + 1], (float)y[4 * j + 2], (float)y[4 * j + 3], vs);
            }
            *(uint4 *)(c.k + at * (B * D) + kr * D + kd) = make_uint4(u[0], u[1], u[2], u[3]);
            *(uint4 *)(c.v + at * (B * D) + vd * B + vr) = make_uint4(w[0], w[1], w[2], w[3]);
            if (tid == 0) {
                c.k_scale[at] = ks.s;
                c.v_scale[at] = vs.s;
            }
        }
    }
    // slots lo .. hi - 1 of the tail, which begin with row p0 + lo.  None where the
    // rows end with a block: p0 + lo is then the row behind them
    const int lo = max(t.pos - bl * B, 0), hi = end - bl * B, p0 = t.r0 + bl * B - t.pos;
    if (z > 0 || hi <= lo) return;
    if (ROPE || hi - lo <= NT / D) {                      // a row or few: a value of K and of V a thread
        const int slot = lo + tid / D;
        const bool in = slot < hi;
        const size_t r = p0 + (in ? slot : lo);
        float a = 0.0f;
        if constexpr (!ROPE) a = BF ? (float)((const __bf16 *)kn)[r * ldk + h * D + vd] : ((const float *)kn)[r * ldk + h * D + vd];
        const float o = BF ? (float)((const __bf16 *)vn)[r * ldv + h * D + vd] : ((const float *)vn)[r * ldv + h * D + vd];
        if constexpr (ROPE) {
            __builtin_amdgcn_sched_barrier(0);            // V's values on their way meanwhile
            rotate();
            a = krow[vd];
        }
        if (!in) return;
        kt[slot * D + vd] = kv8_held(a);
        vt[vd * B + slot] = kv8_held(o);
        return;
    }
    // the units of a block again, all loads first (of the nearest row that is there)
    kv8_16<BF> kx;
    float vx[16];
    kx.load(kn, (size_t)(p0 + min(max(kr, lo), hi - 1)) * ldk + h * D + kd);
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const size_t i = (size_t)(p0 + min(max(vr + j, lo), hi - 1)) * ldv + h * D + vd;
        vx[j] = BF ? (float)((const __bf16 *)vn)[i] : ((const float *)vn)[i];
    }
    __builtin_amdgcn_sched_barrier(0);
    if (kr >= lo && kr < hi) {
        __bf16 *o = kt + kr * D + kd;
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
            bf16x8 u;
#pragma unroll
            for (int n = 0; n < 8; n++) u[n] = kv8_held(kx.at(j + n));
            *(bf16x8 *)(o + j) = u;
        }
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
        if (vr + j >= lo && vr + j < hi) vt[vd * B + vr + j] = kv8_held(vx[j]);
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// S^T = K Q^T and O^T += V^T P^T with 16x16x32 bf16 MFMAs, the columns being
// query rows (row r, query head g of the kv head: column r G + g), 64 keys a
// step.  8-bit codes are exact in bf16, so the scales stay outside: K's
// multiplies the scores, V's the weights.
// fp32 rows keep fp32 accuracy: q and the weights go through the matrix cores
// as three bf16 pieces each (8 bits apiece: x - x1 - x2 - x3 < 2^-24 x).  bf16
// rows are one piece, and their weights two: in one, 16 to 21 % faster in a prompt,
// the weights' roundings would add as much error as the results' own, or more
// where few keys weigh (1.5 times the results' alone over short prompts).
//   S^T tile t, row m <-> key 16 (m / 4) + 4 t + m % 4 of the step, so that
//   lane (c, h) = (lane % 16, lane / 16) ends up with keys 16 h + 4 t + i of
//   column c: four tiles are 16 consecutive keys, which lie in one page (one
//   scale) and, in V's columns, in 16 consecutive bytes.  The weights of
//   tiles 2 s and 2 s + 1 are then, as they lie, the B operand of the MFMA
//   over keys 16 h + 8 s .. + 7, and 8 bytes of V's column its A operand.
template <int FMT>
__device__ __forceinline__ bf16x8 kv8_bf16(uint32_t a, uint32_t b) {      // eight codes
    union { bf16x2 p[4]; bf16x8 v; } r;
    if constexpr (FMT == QM_KV8_E4M3) {
        r.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
        r.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
        r.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
        r.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    } else {
        // a code's byte is sign-extended by the conversion itself: three instructions for two codes
        auto pair = [](uint32_t x, int n) {
            const f32x2 t = {(float)(int)(signed char)(x >> n), (float)(int)(signed char)(x >> (n + 8))};
            return __builtin_convertvector(t, bf16x2);
        };
        r.p[0] = pair(a, 0);
        r.p[1] = pair(a, 16);
        r.p[2] = pair(b, 0);
        r.p[3] = pair(b, 16);
    }
    return r.v;
}

typedef float f32x8 __attribute__((ext_vector_type(8)));

// x as NP bf16 pieces
template <int NP>
__device__ __forceinline__ void kv8_pieces(f32x8 x, bf16x8 (&p)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        p[i] = __builtin_convertvector(x, bf16x8);
        if (i + 1 < NP) x -= __builtin_convertvector(p[i], f32x8);
    }
}

__device__ __forceinline__ f32x4 kv8_mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// eight values of a query row, and their pieces
template <bool BF>
struct kv8_row {
    f32x4 a, b;
    __device__ __forceinline__ void load(const void *q, size_t i) {
        if constexpr (BF) {
            a = *(const f32x4 *)((const __bf16 *)q + i);
        } else {
            a = *(const f32x4 *)((const float *)q + i);
            b = *(const f32x4 *)((const float *)q + i + 4);
        }
    }
    template <int NP>
    __device__ __forceinline__ void pieces(bf16x8 (&p)[NP]) const {
        if constexpr (BF) {
            static_assert(NP == 1, "bf16 rows are one piece");
            p[0] = __builtin_bit_cast(bf16x8, a);
        } else {
            kv8_pieces<NP>(f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, p);
        }
    }
};

// max and sum over the four lanes that share a column
__device__ __forceinline__ float col_max(float v) {
    f32x2 p = swap16(v);
    v = fmaxf(p.x, p.y);
    p = swap32(v);
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float col_sum(float v) {
    f32x2 p = swap16(v);
    v = p.x + p.y;
    p = swap32(v);
    return p.x + p.y;
}

// 1 / sum of weights; a row of which nothing was left (pages that are none) is 0
__device__ __forceinline__ float kv8_inverse(float den) { return den == 0.0f ? 0.0f : 1.0f / den; }

// the running softmax of one column tile: raw products s (masked ones -inf), of
// which k > 0 times each is the score in units of log2, become weights; returns
// what the sums so far are to be multiplied by
__device__ __forceinline__ float kv8_softmax(f32x4 (&s)[4], float k, float &m, float &l) {
    auto mx2 = [](float a, float b) { return __builtin_elementwise_maximum(a, b); };
    float mx = s[0].x;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = t ? 0 : 1; i < 4; i++) mx = mx2(mx, s[t][i]);
    const float nm = fmaxf(m, col_max(mx * k));
    const float ref = nm == -INFINITY ? 0.0f : nm;       // nothing seen yet: every weight is 0
    const float r = __builtin_amdgcn_exp2f(m - ref);
    m = nm;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // the product rounded as the maximum's was: at 1e31 a fused one is off by 1e24
            s[t][i] = __builtin_amdgcn_exp2f(mul_add(s[t][i], k, -ref));
            sum += s[t][i];
        }
    l = l * r + sum;
    return r;
}

// A block has CG x KG waves on COLS = 16 CT CG columns of one kv head: wave
// (cg, kg) takes 16 CT of the columns and, of the steps of 64 keys, in turn
// with the other groups of keys and the other splits, its own; each operand
// goes from memory straight into its MFMA's registers, converted on the way
// (K of the next step is in flight during this step's V product), so that
// waves never wait for one another until the groups' sums meet in LDS at the
// end.  The unfinished block is one more step.  With several splits (blocks on
// the same columns) each block writes a partial {m, l, -, -, o[D]} per column
// with agent-scope (write-through) stores, waits for them, and takes a ticket
// of its columns; the block that draws the last one reads all partials, merges
// them in split order and resets the counter.  No block waits for another; a
// launch of its own for the merge cost 4 us.
//   few columns (decode, a few rows): CT = CG = 1, the keys split over four or
//   eight waves and over blocks
//   many (a prompt): two groups of keys, two of columns; the column tiles with
//   the longest contexts first, or, where all blocks fit the CUs at once, so
//   that the two blocks of a CU are a long and a short one
// Few columns are bound by the bytes: 64 sequences at 2,048 positions (238 MB)
// 44.5 us, 5.3 TB/s, where a copy reaches 5.3; with fewer blocks than CUs by
// the chain of latencies of a block and the merge (700 positions 7.5 us, 6 x
// 8,000 of int8, 48 MB, 15).
// Prompts are bound by the vector instructions that make operands and weights,
// behind which the two waves a SIMD has registers for hide the products only in
// part: of 96 products (19 cycles each) and about 570 others a step of a wave,
// 128 convert codes (6), 32 are exponentials (9) and 96 split the weights.  2,048
// rows behind 6,000 186 us, 630 TFLOP/s; 1,999 behind nothing 38 us, 425, where
// the columns with the most keys end alone.  int8, whose conversions are three
// instructions for two codes, 226 and 44; fp32 rows, three products for one, 57
// (e4m3) and 68 (1,999 rows: 42.6 at a large product's rate).
#define KV8_MAX_SPLITS 32
template <bool NT>
__device__ __forceinline__ uint4 kv8_read(const uint8_t *p) {
    if constexpr (NT) return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u32x4 *)p));
    return *(const uint4 *)p;
}
enum { KV8_LONG_FIRST, KV8_PAIRED };
#define KV8_SC1 16                     // agent scope: past this XCD's L2
// one per kv head, sequence and column tile of a launch that splits its keys;
// zero between launches, which run one after the other on the library stream
#define KV8_TICKETS 128
__device__ unsigned kv8_tickets[KV8_TICKETS];
template <int FMT, int D, bool BF, int CT, int CG, int KG>
__global__ __launch_bounds__(WAVE *CG *KG, 2) void k_kv8_attend(qm_kv8_t c, void *__restrict__ out,
                                                               const void *__restrict__ q, size_t ldo, size_t ldq,
                                                               const int *__restrict__ row, const int *__restrict__ pos,
                                                               int rows, int max_rows, int G, unsigned inv_G, float f,
                                                               int nsplit,
                                                               int order, float *__restrict__ part) {
    constexpr int NP = BF ? 1 : 3, NW = BF ? 2 : 3;         // pieces of q, and of a weight
    constexpr int KS = D / 32, DT = D / 16, LD = D + 4, COLS = 16 * CT * CG, NT = WAVE * CG * KG;
    const int e = blockIdx.y, split = blockIdx.x % nsplit, x = blockIdx.x / nsplit, head = x % c.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cg = wave % CG, kg = wave / CG;
    const int cl = lane & 15, h = lane >> 4;
    const int gk = (lane >> 2) & 3;                                        // the group of 16 keys its K row lies in
    const int B = c.block, lb = __builtin_ctz(B);
    const int *table = c.table + (size_t)e * c.max_blocks;
    // table entry of a key, and the page it stands for, -1 where there is none.
    // Entries are read two steps ahead, the first before anything says how long
    // the sequence is, so that no address waits for one
    auto entry_of = [&](int key) { return table[min(key >> lb, c.max_blocks - 1)]; };
    int s = KG * split + kg;
    int pk = entry_of(64 * s + 16 * gk), pv = entry_of(64 * s + 16 * h);
    int ek = entry_of(64 * (s + KG * nsplit) + 16 * gk), ev = entry_of(64 * (s + KG * nsplit) + 16 * h);
    kv8_entry t;
    if (!kv8_get(t, c, row, pos, e, rows, max_rows)) return;
    // column / G, exact up to 2^26 columns of up to 64 a row
    auto row_of = [&](int col) { return inv_G ? (int)__umulhi((unsigned)col, inv_G) : col; };
    const int ncol = t.cnt * G, tiles = (ncol + COLS - 1) / COLS, at_ = x / c.heads;
    if (at_ >= tiles) return;
    const int tile = order == KV8_LONG_FIRST || at_ < (tiles + 1) / 2 ? tiles - 1 - at_ : at_ - (tiles + 1) / 2;
    const int col0 = tile * COLS, w0 = col0 + 16 * CT * cg;                // the block's and the wave's first column
    const int full = (t.pos + t.cnt) >> lb << lb;                          // keys in finished blocks
    const int wlast = w0 < ncol ? t.pos + min(t.cnt - 1, row_of(w0 + 16 * CT - 1)) : -1;   // the last key the wave sees
    const int wfirst = w0 < ncol ? t.pos + row_of(w0) : -1;                    // and the last that all its columns see
    const int ns = (min(full, wlast + 1) + 63) >> 6, stride = KG * nsplit;

    // the lane's dims of the MFMA over the j-th 32: 16 consecutive ones of each 64,
    // so that the four lanes of a row read 64 consecutive bytes of K
    auto dim_of = [&](int j) { return 64 * (j >> 1) + 16 * h + 8 * (j & 1); };
    int last[CT];                                                          // the column's last key
    kv8_row<BF> qr_[CT][KS];
#pragma unroll
    for (int n = 0; n < CT; n++) {
        const int col = w0 + 16 * n + cl;
        const bool in = col < ncol;
        const int qr = in ? row_of(col) : 0, qg = in ? col - qr * G : 0;   // a lane without a column reads the first's
        last[n] = in ? t.pos + qr : -1;
#pragma unroll
        for (int j = 0; j < KS; j++)
            qr_[n][j].load(q, (size_t)(t.r0 + qr) * ldq + (size_t)(head * G + qg) * D + dim_of(j));
    }
    // -1: no finished block.  Its lanes read page 0, without a branch, and do not
    // use what they read
    auto page_of = [&](int key, int p) { return key < full && (unsigned)p < (unsigned)c.n_page ? p : -1; };
    uint4 kk[4][D / 64], vv[DT];
    float ksn = 0.0f, vsn = 0.0f;                                          // the next step's scales
    auto load_k = [&](int s, int p) {
        const int key = 64 * s + 16 * gk;
        const uint8_t *b = c.k + (((size_t)max(p, 0) * c.heads + head) * B + ((key & (B - 1)) + (lane & 3))) * D + 16 * h;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int u = 0; u < D / 64; u++)
                kk[i][u] = kv8_read<CT == 1 && CG == 1 && KG == 4>(b + (size_t)4 * i * D + 64 * u);
    };
    auto load_v = [&](int s, int p) {
        const int key = 64 * s + 16 * h;
        const uint8_t *b = c.v + (((size_t)max(p, 0) * c.heads + head) * D + cl) * B + (key & (B - 1));
#pragma unroll
        for (int i = 0; i < DT; i++) vv[i] = kv8_read<CT == 1 && CG == 1 && KG == 4>(b + (size_t)16 * i * B);
    };
    if (s < ns) {
        pk = page_of(64 * s + 16 * gk, pk);
        pv = page_of(64 * s + 16 * h, pv);
        load_k(s, pk);
        const size_t at = (size_t)max(pv, 0) * c.heads + head;
        ksn = c.k_scale[at];
        vsn = c.v_scale[at];
    }
    bf16x8 qf[CT][KS][NP];
    float m[CT], l[CT];
    f32x4 o[CT][DT], s4[CT][4];
#pragma unroll
    for (int n = 0; n < CT; n++) {
#pragma unroll
        for (int j = 0; j < KS; j++) qr_[n][j].pieces(qf[n][j]);
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; i++) o[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // one tile of 16 keys' products
    auto score = [&](int i, const bf16x8 (&kf)[KS]) {
#pragma unroll
        for (int n = 0; n < CT; n++) {
            s4[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int u = 0; u < NP; u++) s4[n][i] = kv8_mma(kf[j], qf[n][j][u], s4[n][i]);
        }
    };
    auto softmax = [&](float k) {
#pragma unroll
        for (int n = 0; n < CT; n++) {
            const float r = kv8_softmax(s4[n], k, m[n], l[n]);
            if (__any(r != 1.0f)) {                                        // a maximum grew
#pragma unroll
                for (int i = 0; i < DT; i++) o[n][i] *= r;
            }
        }
    };
    // weights (times the page's V scale) as B operands of key half s2
    auto weights = [&](int s2, float vs, bf16x8 (&pf)[CT][NW]) {
#pragma unroll
        for (int n = 0; n < CT; n++) {
            const f32x4 a = s4[n][2 * s2] * vs, b = s4[n][2 * s2 + 1] * vs;
            kv8_pieces<NW>(f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, pf[n]);
        }
    };
    auto add_v = [&](int i, bf16x8 vf, const bf16x8 (&pf)[CT][NW]) {
#pragma unroll
        for (int n = 0; n < CT; n++)
#pragma unroll
            for (int u = 0; u < NW; u++) o[n][i] = kv8_mma(vf, pf[n][u], o[n][i]);
    };

    for (; s < ns; s += stride) {
        // In this order, and without a branch, so that nothing below waits for
        // loads behind those it needs
        load_v(s, pv);
        const int nx = s + stride, pkn = page_of(64 * nx + 16 * gk, ek), pvn = page_of(64 * nx + 16 * h, ev);
        ek = entry_of(64 * (nx + stride) + 16 * gk);
        ev = entry_of(64 * (nx + stride) + 16 * h);
        float ks = ksn * f, vs = vsn;
        const size_t at = (size_t)max(pvn, 0) * c.heads + head;
        ksn = c.k_scale[at];
        vsn = c.v_scale[at];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            bf16x8 kf[KS];
#pragma unroll
            for (int j = 0; j < KS; j++) {
                const uint4 w = kk[i][j >> 1];
                kf[j] = (j & 1) ? kv8_bf16<FMT>(w.z, w.w) : kv8_bf16<FMT>(w.x, w.y);
            }
            score(i, kf);
        }
        load_k(nx, pkn);
        __builtin_amdgcn_sched_barrier(0);                // V's codes are not converted before they are needed
        if (64 * s + 63 > wfirst || 64 * s + 64 > full || __any(pv < 0)) {
#pragma unroll
            for (int n = 0; n < CT; n++) {
                const int lim = pv >= 0 ? last[n] - (64 * s + 16 * h) : -1;        // the group's last key that is seen
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s4[n][i][r] = 4 * i + r <= lim ? s4[n][i][r] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < DT; i++) vv[i] = pv >= 0 ? vv[i] : uint4{};
            ks = pv >= 0 ? ks : 1.0f;
            vs = pv >= 0 ? vs : 0.0f;
        }
        // (a scale of 0, a block of zeros, would make 0 x -inf of a masked key)
        softmax(fmaxf(ks, FLT_MIN));
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
            bf16x8 pf[CT][NW];
            weights(s2, vs, pf);
#pragma unroll
            for (int i = 0; i < DT; i++)
                add_v(i, s2 ? kv8_bf16<FMT>(vv[i].z, vv[i].w) : kv8_bf16<FMT>(vv[i].x, vv[i].y), pf);
            __builtin_amdgcn_sched_barrier(0);
        }
        pv = pvn;
    }

    // the unfinished block, as one more step of the turn.  Its rows are read
    // whether they are there or not (within the tail): scores of keys that are
    // not are masked, and V is cleared where they lie, as it may hold anything
    if (wlast >= full && (full + 63) / 64 % stride == KG * split + kg) {
        const int nt = t.pos + t.cnt - full;                               // rows it holds, < B <= 64
        const __bf16 *kt = (const __bf16 *)c.k_tail + ((size_t)e * c.heads + head) * ((size_t)B * D);
        const __bf16 *vt = (const __bf16 *)c.v_tail + ((size_t)e * c.heads + head) * ((size_t)B * D);
        bf16x8 tk[4][KS], tv[2][DT];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < KS; j++)
                tk[i][j] = *(const bf16x8 *)(kt + (size_t)min(16 * gk + 4 * i + (lane & 3), B - 1) * D + dim_of(j));
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++)
#pragma unroll
            for (int i = 0; i < DT; i++)
                tv[s2][i] = *(const bf16x8 *)(vt + (size_t)(16 * i + cl) * B + min(16 * h + 8 * s2, B - 8));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            score(i, tk[i]);
#pragma unroll
            for (int n = 0; n < CT; n++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int k = 16 * h + 4 * i + r;
                    s4[n][i][r] = k < nt && full + k <= last[n] ? s4[n][i][r] : -INFINITY;
                }
        }
        softmax(f);
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
            bf16x8 pf[CT][NW];
            weights(s2, 1.0f, pf);
            const int there = nt - (16 * h + 8 * s2);
            // 32 bits, two keys, at a time
            typedef unsigned int u4 __attribute__((ext_vector_type(4)));
            u4 mask;
#pragma unroll
            for (int n = 0; n < 4; n++) mask[n] = there > 2 * n + 1 ? ~0u : there == 2 * n + 1 ? 0xFFFFu : 0u;
#pragma unroll
            for (int i = 0; i < DT; i++)
                add_v(i, __builtin_bit_cast(bf16x8, __builtin_bit_cast(u4, tv[s2][i]) & mask), pf);
        }
    }

    // the groups' sums, and the splits' partials
    __shared__ __align__(16) float so[KG][COLS][LD];
    __shared__ float sm[KG][COLS], sl[KG][COLS];
#pragma unroll
    for (int n = 0; n < CT; n++) {
        const int cc = 16 * (CT * cg + n) + cl;
        l[n] = col_sum(l[n]);
#pragma unroll
        for (int i = 0; i < DT; i++) *(f32x4 *)&so[kg][cc][16 * i + 4 * h] = o[n][i];
        if (h == 0) { sm[kg][cc] = m[n]; sl[kg][cc] = l[n]; }
    }
    __syncthreads();
    constexpr int TPC = D / 4;                            // threads of a column
    constexpr int PER = (COLS * TPC + NT - 1) / NT;       // quads of the block's output a thread
    auto store = [&](int col, int d, f32x4 num, float den) {
        num *= kv8_inverse(den);
        const int qr = row_of(col);
        const size_t at = (size_t)(t.r0 + qr) * ldo + (size_t)(head * G + col - qr * G) * D + d;
        if constexpr (BF) *(uint2 *)((uint16_t *)out + at) = pack4(num);
        else *(f32x4 *)((float *)out + at) = num;
    };
    // this block's partials, [split][column][LD]
    constexpr unsigned BYTES = COLS * LD * 4;
    const unsigned mine = (unsigned)e * (gridDim.x / nsplit) + x;          // of its kv head, sequence and tile
    const __amdgpu_buffer_rsrc_t rp = buf_rsrc((char *)part + (size_t)mine * nsplit * BYTES, (size_t)nsplit * BYTES);
#pragma unroll 1
    for (int u = 0; u < PER; u++) {
        const int i = tid + NT * u, cc = i / TPC, d = i % TPC * 4, col = col0 + cc;
        if (i >= COLS * TPC || col >= ncol) continue;
        float mx = sm[0][cc];
#pragma unroll
        for (int g = 1; g < KG; g++) mx = fmaxf(mx, sm[g][cc]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float den = 0.0f;
        f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < KG; g++) {
            // a wave without keys weighs 0 (its sums are 0); one whose scores were all NaN keeps its NaN
            const float w = __builtin_amdgcn_exp2f(sm[g][cc] - ref);
            den += w * sl[g][cc];
            num += *(const f32x4 *)&so[g][cc][d] * w;
        }
        if (nsplit == 1) {
            store(col, d, num, den);
        } else {
            const unsigned at = split * BYTES + (cc * LD + 4 + d) * 4;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, num), rp, at, 0, KV8_SC1);
            if (d == 0)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{mx, den, 0.f, 0.f}), rp, at - 16, 0,
                                                       KV8_SC1);
        }
    }
    if (nsplit == 1) return;
    __shared__ unsigned drawn;
    __builtin_amdgcn_s_waitcnt(0);                        // this thread's sums have landed
    __syncthreads();                                      // ... and every thread's
    if (tid == 0) drawn = __hip_atomic_fetch_add(&kv8_tickets[mine], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (drawn != (unsigned)nsplit - 1u) return;           // uniform over the block
#pragma unroll 1
    for (int u = 0; u < PER; u++) {
        const int i = tid + NT * u, cc = i / TPC, d = i % TPC * 4, col = col0 + cc;
        if (i >= COLS * TPC || col >= ncol) continue;
        float mx = -INFINITY, den = 0.0f;
        f32x4 num = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < nsplit; s0 += 8) {          // eight splits' reads in flight
            f32x4 ml[8], o8[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const unsigned at = s0 + k < nsplit ? (s0 + k) * BYTES + cc * LD * 4 : BUF_OOB;
                ml[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, at, 0, KV8_SC1));
                o8[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, at + 16 + d * 4, 0, KV8_SC1));
                if (s0 + k >= nsplit) ml[k].x = -INFINITY;
            }
            float nm = mx;
#pragma unroll
            for (int k = 0; k < 8; k++) nm = fmaxf(nm, ml[k].x);
            const float ref = nm == -INFINITY ? 0.0f : nm, r = __builtin_amdgcn_exp2f(mx - ref);
            den *= r;
            num *= r;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float w = __builtin_amdgcn_exp2f(ml[k].x - ref);
                den += w * ml[k].y;
                num += o8[k] * w;
            }
            mx = nm;
        }
        store(col, d, num, den);
    }
    if (tid == 0) __hip_atomic_store(&kv8_tickets[mine], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

static int kv8_sizes(const qm_kv8_t *c) {
    if (c->format != QM_KV8_E4M3 && c->format != QM_KV8_INT8) return QH_EINVAL;
    if (c->head_dim != 64 && c->head_dim != 128) return QH_EINVAL;
    if (c->block != 16 && c->block != 32 && c->block != 64) return QH_EINVAL;
    if (c->heads < 1 || c->heads > QM_KV8_MAX_HEADS || c->n_page < 1 || c->n_seq < 1 || c->max_blocks < 1) return QH_EINVAL;
    return (long)c->max_blocks * c->block > QM_KV8_MAX_CTX ? QH_ETOOBIG : QH_OK;
}
static int kv8_check(const qm_kv8_t *c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !c->table) return QH_EINVAL;
    const int rc = kv8_sizes(c);
    if (rc) return rc;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_tail) || !aligned16(c->v_tail)) return QH_EINVAL;
    return QH_OK;
}
// rows of `cols` values at stride ld, loaded 16 bytes at a time
static bool kv8_rows_ok(const void *p, size_t ld, int cols, int bf16) {
    return p && aligned16(p) && ld >= (size_t)cols && ld % (bf16 ? 8 : 4) == 0;
}
static int kv8_call_check(const qm_kv8_t *c, const int *row, const int *pos, int n, int rows, int max_rows) {
    if (n < 0 || n > c->n_seq || n > QM_KV8_MAX_SEQS || !pos || rows < 0 || max_rows < 1) return QH_EINVAL;
    if (!row && (rows != n || max_rows != 1)) return QH_EINVAL;
    if ((long)max_rows > (long)c->max_blocks * c->block) return QH_EINVAL;
    return QH_OK;
}

#define KV8_SWITCH(CALL)                                                        \
    do {                                                                        \
        if (c->format == QM_KV8_E4M3) {                                         \
            if (c->head_dim == 128) { if (bf16) CALL(QM_KV8_E4M3, 128, true); else CALL(QM_KV8_E4M3, 128, false); } \
            else { if (bf16) CALL(QM_KV8_E4M3, 64, true); else CALL(QM_KV8_E4M3, 64, false); }                      \
        } else {                                                                \
            if (c->head_dim == 128) { if (bf16) CALL(QM_KV8_INT8, 128, true); else CALL(QM_KV8_INT8, 128, false); } \
            else { if (bf16) CALL(QM_KV8_INT8, 64, true); else CALL(QM_KV8_INT8, 64, false); }                      \
        }                                                                       \
    } while (0)

extern "C" size_t qm_kv8_bytes(const qm_kv8_t *c) {
    if (!c || kv8_sizes(c)) return 0;
    const size_t values = 2 * (size_t)c->heads * c->block * c->head_dim;       // K and V of a block
    return c->n_page * (values + 2 * (size_t)c->heads * sizeof(float)) +
           c->n_seq * (2 * values + (size_t)c->max_blocks * sizeof(int));
}

extern "C" int qm_qk_rope(float *qkv, uint16_t *qb, const uint16_t *qn, const uint16_t *kn, const float *rcos,
                          const float *rsin, const int *pos, int nt, int max_seq, float eps) {
    if (!qkv || !qn || !kn || !rcos || !rsin || !pos || nt <= 0 || max_seq <= 0) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    const kv8_rope a = {qkv, qn, kn, rcos, rsin, max_seq, eps};
    hipLaunchKernelGGL(k_qk_rope, dim3(nt, (NKV * GRP + NKV) / 4), dim3(NTH), 0, stream(), a, qb, pos);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

extern "C" int qm_kv8_rope_append(const qm_kv8_t *c, float *qkv, const uint16_t *qn, const uint16_t *kn, const float *rcos,
                                  const float *rsin, const int *pos, int n, int max_seq, float eps) {
    int rc = kv8_check(c);
    if (!rc) rc = kv8_call_check(c, NULL, pos, n, n, 1);
    if (rc) return rc;
    if (c->heads != NKV || c->head_dim != HD || c->block != 32) return QH_EINVAL;
    if (n == 0) return QH_OK;
    if (!qkv || !aligned16(qkv) || !qn || !kn || !rcos || !rsin || max_seq <= 0) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    const kv8_rope a = {qkv, qn, kn, rcos, rsin, max_seq, eps};
    const float *k = qkv + NKV * GRP * HD, *v = k + NKV * HD;
    if (c->format == QM_KV8_E4M3)
        hipLaunchKernelGGL((k_kv8_append<QM_KV8_E4M3, HD, 32, false, true>), dim3(NKV, n), dim3(2 * HD), 0, stream(), *c, k, v,
                           QKV_LD, QKV_LD, NULL, pos, n, 1, a);
    else
        hipLaunchKernelGGL((k_kv8_append<QM_KV8_INT8, HD, 32, false, true>), dim3(NKV, n), dim3(2 * HD), 0, stream(), *c, k, v,
                           QKV_LD, QKV_LD, NULL, pos, n, 1, a);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

extern "C" int qm_kv8_own(int *table, const int *pos, int n_seq, int block, int max_blocks) {
    if (!table || n_seq <= 0 || n_seq > 65535 || block <= 0 || max_blocks <= 0) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    hipLaunchKernelGGL(k_kv8_own, dim3((max_blocks + NTH - 1) / NTH, n_seq), dim3(NTH), 0, stream(), table, pos, block,
                       max_blocks);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

extern "C" int qm_kv8_append(const qm_kv8_t *c, const void *k, const void *v, size_t ldk, size_t ldv, int bf16,
                             const int *row, const int *pos, int n, int rows, int max_rows) {
    int rc = kv8_check(c);
    if (!rc) rc = kv8_call_check(c, row, pos, n, rows, max_rows);
    if (rc) return rc;
    if (n == 0 || rows == 0) return QH_OK;
    if (!kv8_rows_ok(k, ldk, c->heads * c->head_dim, bf16) || !kv8_rows_ok(v, ldv, c->heads * c->head_dim, bf16))
        return QH_EINVAL;
    // blocks that an entry's rows touch at most, wherever they start
    const dim3 grid(c->heads, n, ((max_rows < rows ? max_rows : rows) + c->block - 2) / c->block + 1);
    if (grid.z > 65535) return QH_ETOOBIG;
    if (!stream()) return QH_ESTATE;
#define APPEND_B(F, D_, B_, BF_) \
    hipLaunchKernelGGL((k_kv8_append<F, D_, B_, BF_, false>), grid, dim3(B_ *D_ / 16), 0, stream(), *c, k, v, ldk, ldv, row, \
                       pos, rows, max_rows, kv8_rope{})
#define APPEND(F, D_, BF_)                                  \
    do {                                                    \
        if (c->block == 16) APPEND_B(F, D_, 16, BF_);       \
        else if (c->block == 32) APPEND_B(F, D_, 32, BF_);  \
        else APPEND_B(F, D_, 64, BF_);                      \
    } while (0)
    KV8_SWITCH(APPEND);
#undef APPEND
#undef APPEND_B
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

// The launch for max_rows x G columns a kv head and sequence.
//   CT: two column tiles a wave where rows are bf16 and there are more than 16
//     columns (fp32 rows take the registers for their pieces).
//   Prompts that fill the CUs: blocks of two groups of keys and two of columns,
//     which share what they read, against four groups of keys.  From 960 blocks
//     of the latter, where they come even: a prompt of 1,700 bf16 rows (856
//     blocks) 34.9 us against 32.8, of 1,999 (1,000) 38.2 against 40.5; fp32 700
//     rows (704) 18.6 against 17.1, 1,000 (1,008) 21.1 against 25.7.  From four
//     tiles a sequence: 30 x 61 rows 13.0 against 17.5, behind 2,048 positions
//     64.7 against 65.6; 8 x 250 16.7 against 20.8; with three tiles, the fourth
//     a block's half that is idle, 40 x 45 behind 2,048 81.6 against 66.9.  At
//     head_dim 64, whose steps are half the products, only many short prompts
//     would gain (16 x 120 9.5 against 11.1) and long ones lose (1,999 26.5
//     against 25.1, 2,500 41.8 against 34.5): never.
//   Few blocks: the keys split over blocks of four waves, a step a wave, up to
//     128 blocks (one head of a kv head's, 700 positions: 8.0 us against 9.7 on
//     one block of eight waves and 9.9 on two, 1,500 8.3 against 10.1); with 17
//     to 64 blocks up to 192 to 256 (5 x 960 positions 8.1 us against 9.8 on
//     blocks of eight waves, 17 rows behind 6,000 14.2 against 16.2, 6 x 8,000
//     15.0 against 16.4; 24 blocks by ten are slower than by eight, 15.7, since
//     a multiple of eight keeps the tiles of the same keys on one XCD).  Two
//     blocks a CU, by 16, are slower still: 24 blocks at 8,000 18.7, 20 17.1
//     against 14.1, 32 19.8 against 16.3.
//   Between: four groups of keys where a wave of eight would have a step or two
//     (32 x 700 positions 10.8 against 11.5 us, 60 x 700 17.6 against 20.1) or
//     where columns see different numbers of keys and there is a block for each
//     CU (1,000 tokens 18.0 against 20.5, fp32 500 behind 1,499 28.9 against
//     33.5); eight elsewhere, which read ahead further (16 x 700 positions 9.1
//     us against 10.2, 40 x 2,000 34.4 against 36.7), with the keys of long
//     contexts split over blocks as long as there is a CU for each (8 heads at
//     8,000: 11.5 us on 128 blocks).
struct kv8_plan { int ct, cg, kg, splits, order, cols, tiles; };
static kv8_plan kv8_plan_of(const qm_kv8_t *c, int G, int n, int max_rows, int max_ctx, int bf16) {
    const long cols = (long)max_rows * G;
    kv8_plan p = {bf16 && cols > 16 ? 2 : 1, 1, 4, 1, KV8_LONG_FIRST, 0, 0};
    p.cols = 16 * p.ct;
    p.tiles = (int)((cols + p.cols - 1) / p.cols);
    const long blocks = (long)p.tiles * c->heads * n;
    if (blocks >= 960 && p.tiles >= 4 && c->head_dim == 128) {
        p.cg = p.kg = 2;
        p.cols *= 2;
        p.tiles = (p.tiles + 1) / 2;
        if ((long)p.tiles * c->heads * n <= 512) p.order = KV8_PAIRED;
    } else if (blocks < 512) {
        const int steps = (max_ctx + 63) / 64 + 1;       // the unfinished block's among them
        static_assert(KV8_TICKETS >= 256 / 2, "a ticket for each block that is split");
        const bool cu_each = blocks >= 256;
        if (blocks * ((steps + 3) / 4) <= 128) {
            p.splits = (steps + 3) / 4;
        } else if (blocks > 16 && blocks <= 64) {
            p.splits = blocks <= 21 ? 12 : blocks <= 32 ? 8 : blocks <= 42 ? 6 : 4;
            if (p.splits > (steps + 3) / 4) p.splits = (steps + 3) / 4;
        } else if (steps > (p.tiles > 1 || cu_each ? 16 : 12) && !(p.tiles > 1 && cu_each)) {
            p.kg = 8;
            const long room = 256 / blocks, want = (steps + 7) / 8;
            if (steps > 16) p.splits = (int)(want < room ? want : room);
        }
        if (p.splits > KV8_MAX_SPLITS) p.splits = KV8_MAX_SPLITS;
        if (p.splits < 1) p.splits = 1;
    }
    return p;
}
// Bytes of partials that calls of at most these sizes need: a program asks for
// its largest once.  Of all launches above that split, with blocks of 16
// columns, splits <= (steps + 3) / 4 and blocks x splits <= 256; with 32 columns
// a block, there are as many blocks or fewer.
extern "C" size_t qm_kv8_attention_work(const qm_kv8_t *c, int q_heads, int n, int max_rows, int max_ctx) {
    if (!c || kv8_sizes(c) || q_heads < c->heads || n < 1 || max_rows < 1 || max_ctx < 1) return 0;
    const size_t cols = (size_t)max_rows * (q_heads / c->heads), split = ((size_t)(max_ctx - 1) / 64 + 2 + 3) / 4;
    const size_t most = (size_t)n * c->heads * ((cols + 15) / 16) * split;
    return split == 1 ? 0 : (most < 256 ? most : 256) * (cols > 16 ? 32 : 16) * (c->head_dim + 4) * sizeof(float);
}

extern "C" int qm_kv8_attention(const qm_kv8_t *c, void *out, const void *q, size_t ldo, size_t ldq, int bf16, int q_heads,
                                const int *row, const int *pos, int n, int rows, int max_rows, int max_ctx, float scale,
                                void *work, size_t work_bytes) {
    int rc = kv8_check(c);
    if (!rc) rc = kv8_call_check(c, row, pos, n, rows, max_rows);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % c->heads || q_heads / c->heads > QM_KV8_MAX_GROUP) return QH_EINVAL;
    if (max_ctx < 1 || max_ctx > c->max_blocks * c->block || !(scale > 0.0f && scale < INFINITY)) return QH_EINVAL;
    if (n == 0 || rows == 0) return QH_OK;
    if (!kv8_rows_ok(q, ldq, q_heads * c->head_dim, bf16) || !kv8_rows_ok(out, ldo, q_heads * c->head_dim, bf16))
        return QH_EINVAL;
    const int G = q_heads / c->heads;
    const unsigned inv_G = G == 1 ? 0 : (unsigned)(((1ull << 32) + G - 1) / G);
    const float f = scale * 1.44269504088896340736f;     // the softmax runs on powers of two
    const size_t need = qm_kv8_attention_work(c, q_heads, n, max_rows, max_ctx);
    if (need && (!work || !aligned16(work))) return QH_EINVAL;
    if (work_bytes < need) return QH_ETOOBIG;
    const kv8_plan p = kv8_plan_of(c, G, n, max_rows < rows ? max_rows : rows, max_ctx, bf16);
    const long blocks = (long)p.tiles * c->heads * p.splits;
    if (blocks * 512 >= 1L << 32) return QH_ETOOBIG;
    if (!stream()) return QH_ESTATE;
    const dim3 grid((unsigned)blocks, n);
#define ATTEND_AS(F, D_, BF_, CT_, CG_, KG_)                                                                           \
    hipLaunchKernelGGL((k_kv8_attend<F, D_, BF_, CT_, CG_, KG_>), grid, dim3(WAVE *CG_ *KG_), 0, stream(), *c, out, q, ldo, \
                       ldq, row, pos, rows, max_rows, G, inv_G, f, p.splits, p.order, (float *)work)
#define ATTEND_KG(F, D_, BF_, CT_)                            \
    do {                                                      \
        if (p.kg == 4) ATTEND_AS(F, D_, BF_, CT_, 1, 4);      \
        else ATTEND_AS(F, D_, BF_, CT_, 1, 8);                \
    } while (0)
    // (two groups of columns only at head_dim 128, and with bf16 rows only two tiles a wave)
#define ATTEND(F, D_, BF_)                                    \
    do {                                                      \
        if (p.cg == 2) ATTEND_AS(F, 128, BF_, (BF_ ? 2 : 1), 2, 2); \
        else if (p.ct == 2) ATTEND_KG(F, D_, BF_, (BF_ ? 2 : 1)); \
        else ATTEND_KG(F, D_, BF_, 1);                        \
    } while (0)
    KV8_SWITCH(ATTEND);
#undef ATTEND
#undef ATTEND_KG
#undef ATTEND_AS
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}
