// Beam search: the choice of each group's continuations and the reordering of
// the beams' states.  Compiled into hip_model.hip.

// ---------------------------------------------------------------------------
// choice
// ---------------------------------------------------------------------------
// Group g holds W beams (rows g W ..).  Beam w continues with token v at
//   score_w + x_wv - log sum_u e^(x_wu)
// (a finished beam with one candidate, the end token at score_w); the best W
// of them all, in order, ties to the lowest w V + v.
//
// Within a row the scores are ordered as the logits are, so one pass over the
// logits finds each piece's maximum, sum of e^(x - max) and W best logits; a
// second launch joins the pieces' sums and lists.  Rows' sums are joined, and
// scores of different beams compared, in 64 bits: in fp32 scores, which grow
// with the text, would tie at 2^-24 of their size.  The exponentials and their
// sums over a piece are fp32 (roundings of arguments, of the function and of 32
// values a lane and 6 levels: below 64 x 2^-24 of the sum, 2^-18 in its
// logarithm).
// Bound by the logits' bytes for many beams and by two launches' latencies for
// few: 8 x 8 beams over 151,936 logits (38.9 MB) 15.2 us, of which the first
// launch takes 10 (a copy of as much 7.4), 1 x 4 9.0 (two empty launches 4.6).
#define BEAM_MAX QM_BEAM_MAX_WIDTH     // beams of a group
#define BEAM_PIECE 2048                // logits of a wave: 32 a lane
#define BEAM_V (BEAM_PIECE / WAVE)
#define BEAM_NONE 0x7FFFFFFF           // the index of no candidate
#define BEAM_E 8                       // list entries a lane of the second launch has in flight

struct beam_cand { float v; int i; };
struct beam_sum { float m, s; };

// workspace: sums [row][piece], lists [row][W][piece] (by rank: the lanes of the
// second launch then hold entries of like ranks)
static size_t beam_pieces(int vocab) { return ((size_t)vocab + BEAM_PIECE - 1) / BEAM_PIECE; }

template <int CTRL>
__device__ __forceinline__ int dpp_int(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false); }
__device__ __forceinline__ int wave_min_int(int v) {
    v = min(v, dpp_int<0xB1>(v));
    v = min(v, dpp_int<0x4E>(v));
    v = min(v, dpp_int<0x141>(v));
    v = min(v, dpp_int<0x140>(v));
    auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = min((int)p[0], (int)p[1]);
    p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return min((int)p[0], (int)p[1]);
}

// a comes before b: larger, or equal with the lower index
__device__ __forceinline__ bool beam_before(float av, int ai, float bv, int bi) {
    return (av > bv) | ((av == bv) & (ai < bi));          // no branch: loops over it keep their reads in flight
}

// A wave's choice of W among what its lanes hold: a threshold that W of the
// lanes' maxima reach, so that at least W values do and hardly more; they go to
// LDS, where each finds its rank by counting who comes before it.  Where more
// than a lane each reach it (equal values), or fewer than W are finite, the
// callers choose one at a time.
#define BEAM_CAP WAVE
// found bit by bit over the order of floats, until W lanes are left: about
// twelve rounds of a compare and a count whatever W is, where W rounds of a
// wave-wide maximum take 200 cycles each
__device__ __forceinline__ float beam_threshold(float lane_max, int W) {
    const unsigned b = __float_as_uint(lane_max), key = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
    unsigned t = 0;
    for (int bit = 31; bit >= 0; bit--) {
        const unsigned c = t | 1u << bit;
        const int n = __popcll(__ballot(key >= c));
        if (n >= W) t = c;
        if (n == W) break;
    }
    if (t <= 0x007FFFFFu) return -INFINITY;               // the place of -inf in that order
    return __uint_as_float(t & 0x80000000u ? t ^ 0x80000000u : ~t);
}
__device__ __forceinline__ void beam_collect(beam_cand *cand, int &n, bool in, float v, int i) {
    const unsigned long long mask = __ballot(in);
    if (mask) {
        const int at = n + __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
        if (in && at < BEAM_CAP) cand[at] = beam_cand{v, i};
        n += __popcll(mask);
    }
}
__device__ __forceinline__ int beam_rank(const beam_cand *cand, int n, beam_cand t) {
    int rank = 0;
#pragma unroll 4
    for (int u = 0; u < n; u++) {
        const beam_cand o = cand[u];
        rank += beam_before(o.v, o.i, t.v, t.i);
    }
    return rank;
}

// Wave: one piece of one row, 32 logits a lane in registers.
template <bool VEC>
__global__ __launch_bounds__(NTH) void k_beam_pieces(const float *__restrict__ logits, size_t ld, int vocab, int rows,
                                                    int W, int pieces, const float *__restrict__ score,
                                                    const int *__restrict__ done, beam_sum *__restrict__ sums,
                                                    beam_cand *__restrict__ lists) {
    __shared__ beam_cand cands[NTH / WAVE][BEAM_CAP];
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.y, piece = blockIdx.x * (NTH / WAVE) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dn = *(done ? done + r : (const int *)score);     // both reads at once
    const float sc = score[r];
    if (piece >= pieces) return;
    beam_cand *out = lists + (size_t)r * pieces * W + piece;             // entry w at w * pieces
    const float *x = logits + (size_t)r * ld;
    const int base = piece * BEAM_PIECE;
    float v[BEAM_V];
    auto at = [&](int k) { return VEC ? base + (k >> 2) * (4 * WAVE) + 4 * lane + (k & 3) : base + k * WAVE + lane; };
    // a finished beam's row is not read; a beam that is not in use offers its
    // first tokens, in case nothing else is left
    const bool over = done && dn != 0;
    if (over || !(fabsf(sc) < INFINITY)) {
        if (lane < W) out[(size_t)lane * pieces] = beam_cand{-INFINITY, !over && piece == 0 && lane < vocab ? lane : BEAM_NONE};
        if (lane == 0) sums[(size_t)r * pieces + piece] = beam_sum{-INFINITY, 0.0f};
        return;
    }
    if (VEC && base + BEAM_PIECE <= vocab) {
#pragma unroll
        for (int k = 0; k < BEAM_V; k += 4) {
            const f32x4 t = *(const f32x4 *)(x + at(k));
#pragma unroll
            for (int u = 0; u < 4; u++) v[k + u] = t[u];
        }
    } else {
#pragma unroll
        for (int k = 0; k < BEAM_V; k++) {
            const float t = x[min(at(k), vocab - 1)];
            v[k] = at(k) < vocab ? t : -INFINITY;
        }
    }
    float lm = -INFINITY;
#pragma unroll
    for (int k = 0; k < BEAM_V; k++) {
        v[k] = fmaxf(v[k], -INFINITY);                    // a NaN is never chosen
        lm = fmaxf(lm, v[k]);
    }
    const float mx = wave_max(lm);
    float sum = 0.0f;
    if (mx > -INFINITY) {
        // +inf gives NaN: a row without probabilities, which the maximum tells
#pragma unroll
        for (int k = 0; k < BEAM_V; k++) sum += __builtin_amdgcn_exp2f((v[k] - mx) * 1.44269504088896340736f);
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[(size_t)r * pieces + piece] = beam_sum{mx, sum};

    const float thr = beam_threshold(lm, W);
    beam_cand *cand = cands[threadIdx.x >> 6];
    int n = 0;
    if (thr > -INFINITY) {
#pragma unroll
        for (int k = 0; k < BEAM_V; k++) beam_collect(cand, n, v[k] >= thr, v[k], at(k));
        if (n <= BEAM_CAP) {
            if (lane < n) {
                const beam_cand t = cand[lane];
                const int rank = beam_rank(cand, n, t);
                if (rank < W) out[(size_t)rank * pieces] = t;
            }
            return;
        }
    }
    // one at a time: the first that comes behind the last one taken
    float pv = INFINITY;
    int pi = -1;
    for (int w = 0; w < W; w++) {
        float bv = -INFINITY;
        int bi = BEAM_NONE;
#pragma unroll
        for (int k = 0; k < BEAM_V; k++) {
            const int i = at(k);
            if (i < vocab && beam_before(pv, pi, v[k], i) && beam_before(v[k], i, bv, bi)) { bv = v[k]; bi = i; }
        }
        pv = wave_max(bv);
        pi = wave_min_int(bv == pv ? bi : BEAM_NONE);
        if (lane == 0) out[(size_t)w * pieces] = beam_cand{pv, pi};
    }
}

// Block: one group.  Wave w joins row w's sums and finds the row's best W in
// its pieces' lists; then the W x W are ranked.
__global__ __launch_bounds__(WAVE *BEAM_MAX) void k_beam_pick(int vocab, int W, int pieces, const float *score,
                                                             const int *done, int end0, int end1,
                                                             const beam_sum *__restrict__ sums,
                                                             const beam_cand *__restrict__ lists, float *score_out,
                                                             int *done_out, int *__restrict__ token_out,
                                                             int *__restrict__ parent_out) {
    const int g = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __shared__ double cv[BEAM_MAX * BEAM_MAX];
    __shared__ long cid[BEAM_MAX * BEAM_MAX];             // w V + token, BEAM_NOWHERE for no candidate
    __shared__ beam_cand cands[BEAM_MAX][BEAM_CAP];
    __shared__ int sdone[BEAM_MAX], ranks[BEAM_MAX * BEAM_MAX];
    constexpr long BEAM_NOWHERE = 0x7FFFFFFFFFFFFFFFL;
    const int r = g * W + w;                              // launched with W waves
    const beam_sum *ps = sums + (size_t)r * pieces;
    const beam_cand *pl = lists + (size_t)r * pieces * W;
    const int entries = pieces * W;
    // the first reads of everything at once, without branches around them: each
    // costs the kernel a microsecond if it waits for another
    const int dn = *(done ? done + r : (const int *)ps);
    const float sc = score[r];
    beam_cand first[BEAM_E];
    beam_sum sum0[2];
    auto entry = [&](int i) {
        const beam_cand t = pl[min(i, entries - 1)];
        return beam_cand{i < entries ? t.v : -INFINITY, i < entries ? t.i : BEAM_NONE};
    };
#pragma unroll
    for (int k = 0; k < 2; k++) sum0[k] = ps[min(lane + WAVE * k, pieces - 1)];
#pragma unroll
    for (int k = 0; k < BEAM_E; k++) first[k] = entry(lane + WAVE * k);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 2; k++)
        if (lane + WAVE * k >= pieces) sum0[k].m = -INFINITY;
    const bool over = done && dn != 0;
    const double base = fabsf(sc) < INFINITY ? (double)sc : -INFINITY;
    if (lane == 0) sdone[w] = over;
    for (int i = threadIdx.x; i < W * W; i += W * WAVE) ranks[i] = 0;
    if (over) {
        if (lane < W) {
            cv[w * W + lane] = lane == 0 ? base : -INFINITY;
            cid[w * W + lane] = lane == 0 ? (long)w * vocab + end0 : BEAM_NOWHERE;
        }
    } else {
        float mx = fmaxf(sum0[0].m, sum0[1].m);
        for (int p = lane + 2 * WAVE; p < pieces; p += WAVE) mx = fmaxf(mx, ps[p].m);
        mx = wave_max(mx);
        // log of the sum of e^x over the row
        double sum = 0.0;
        auto add = [&](beam_sum t) {
            if (t.m > -INFINITY) sum += (double)t.s * exp((double)t.m - (double)mx);
        };
        add(sum0[0]);
        add(sum0[1]);
        for (int p = lane + 2 * WAVE; p < pieces; p += WAVE) add(ps[p]);
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) sum += __shfl_xor(sum, s);
        const double lse = (double)mx + log(sum);
        auto put = [&](int k, float v, int i) {
            const double t = base + ((double)v - lse);
            cv[w * W + k] = t == t ? t : -INFINITY;       // -inf of a row of -inf
            cid[w * W + k] = i == BEAM_NONE ? BEAM_NOWHERE : (long)w * vocab + i;
        };
        // twice over the lists, eight entries a lane in flight: unrolled over all
        // of them, in registers, the kernel spends its time fetching instructions
        float lm = -INFINITY;
#pragma unroll
        for (int k = 0; k < BEAM_E; k++) lm = fmaxf(lm, first[k].v);
        for (int i0 = lane + BEAM_E * WAVE; i0 < entries; i0 += BEAM_E * WAVE) {
            float v[BEAM_E];
#pragma unroll
            for (int k = 0; k < BEAM_E; k++) v[k] = entry(i0 + WAVE * k).v;
#pragma unroll
            for (int k = 0; k < BEAM_E; k++) lm = fmaxf(lm, v[k]);
        }
        const float thr = beam_threshold(lm, W);
        beam_cand *cand = cands[w];
        int n = 0;
        if (thr > -INFINITY) {
#pragma unroll
            for (int k = 0; k < BEAM_E; k++) beam_collect(cand, n, first[k].v >= thr, first[k].v, first[k].i);
            for (int i0 = lane + BEAM_E * WAVE; i0 - lane < entries; i0 += BEAM_E * WAVE) {
                beam_cand t[BEAM_E];
#pragma unroll
                for (int k = 0; k < BEAM_E; k++) t[k] = entry(i0 + WAVE * k);
#pragma unroll
                for (int k = 0; k < BEAM_E; k++) beam_collect(cand, n, t[k].v >= thr, t[k].v, t[k].i);
            }
        }
        if (mx == INFINITY) {                             // no probabilities: as a beam that is not in use
            if (lane < W) put(lane, -INFINITY, lane);
        } else if (n > 0 && n <= BEAM_CAP) {
            if (lane < n) {
                const beam_cand t = cand[lane];
                const int rank = beam_rank(cand, n, t);
                if (rank < W) put(rank, t.v, t.i);
            }
        } else {
            float pv = INFINITY;
            int pi = -1;
            for (int k = 0; k < W; k++) {
                float bv = -INFINITY;
                int bi = BEAM_NONE;
                for (int i = lane; i < entries; i += WAVE) {
                    const beam_cand t = pl[i];
                    if (beam_before(pv, pi, t.v, t.i) && beam_before(t.v, t.i, bv, bi)) { bv = t.v; bi = t.i; }
                }
                pv = wave_max(bv);
                pi = wave_min_int(bv == pv ? bi : BEAM_NONE);
                if (lane == 0) put(k, pv, pi);
            }
        }
    }
    __syncthreads();
    // each of the W x W counts who comes before it: a thread for each of them
    // and each beam
    const int n2 = W * W;
    for (int task = threadIdx.x; task < n2 * W; task += W * WAVE) {
        const int i = task % n2, from = task / n2 * W;
        const double v = cv[i];
        const long id = cid[i];
        int before = 0;
#pragma unroll 4
        for (int u = 0; u < W; u++) {
            const double a = cv[from + u];
            const long b = cid[from + u];
            before += (a > v) | ((a == v) & (b < id));    // no branch: the reads stay in flight
        }
        if (before) atomicAdd(&ranks[i], before);
    }
    __syncthreads();                                      // the group's inputs have been read: outputs may lie there
    const int i = threadIdx.x;
    if (i >= n2) return;
    const double v = cv[i];
    const long id = cid[i];
    const int rank = ranks[i];
    if (rank < W && id != BEAM_NOWHERE) {
        const int par = i / W, tok = (int)(id - (long)par * vocab);
        score_out[g * W + rank] = (float)v;
        token_out[g * W + rank] = tok;
        parent_out[g * W + rank] = par;
        done_out[g * W + rank] = sdone[par] != 0 || tok == end0 || tok == end1;
    }
}

// ---------------------------------------------------------------------------
// reordering
// ---------------------------------------------------------------------------
// dst row w of every group = src row parent[w], over `slabs` states of
// n_group * W rows, each row `runs` stretches of `run_bytes` used bytes.  A
// thread owns two units of T, a block's width apart, at the same place of all W
// rows: it reads every row it needs before it writes any, so dst may be src,
// and rows that stay where they are are then not touched.  Bound by the
// memory's rate: the tails of 8 x 8 beams (235 MB, of which a random choice of
// parents reads two thirds) 78 us, where a copy of as much takes 89; 108 with
// one unit a thread, 85 with four, 116 with stores through the caches.
#define REORDER_UNITS 2
template <typename T, int WT>
__global__ __launch_bounds__(NTH) void k_beam_reorder(uint8_t *dst, const uint8_t *src, const int *__restrict__ parent,
                                                     int W, unsigned units, unsigned runs, size_t slab_stride,
                                                     size_t seq_stride, size_t run_stride) {
    const int g = blockIdx.y;
    const bool same = dst == src;
    int p[WT];
#pragma unroll
    for (int w = 0; w < WT; w++) {
        p[w] = w < W ? parent[g * W + w] : -1;
        if (p[w] >= W || (same && p[w] == w)) p[w] = -1;
    }
    constexpr int NU = REORDER_UNITS;
    T v[NU][WT];
    size_t at[NU];
    bool in[NU];
#pragma unroll
    for (int k = 0; k < NU; k++) {
        const unsigned u = (blockIdx.x * NU + k) * NTH + threadIdx.x, run = u / units;
        in[k] = run < runs;
        at[k] = (size_t)blockIdx.z * slab_stride + (size_t)g * W * seq_stride + (size_t)run * run_stride +
                (size_t)(u - run * units) * sizeof(T);
    }
#pragma unroll
    for (int k = 0; k < NU; k++)
#pragma unroll
        for (int w = 0; w < WT; w++)
            if (in[k] && p[w] >= 0) v[k][w] = *(const T *)(src + at[k] + (size_t)p[w] * seq_stride);
#pragma unroll
    for (int k = 0; k < NU; k++)
#pragma unroll
        for (int w = 0; w < WT; w++)
            if (in[k] && p[w] >= 0) __builtin_nontemporal_store(v[k][w], (T *)(dst + at[k] + (size_t)w * seq_stride));
}

// ---------------------------------------------------------------------------
// A search's bookkeeping.  Start: the first beam of each group alone is in use.
// Step: the choice goes to row `step` of the history {token, parent}[n], and
// positions advance by adv.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(NTH) void k_beam_start(float *score, int *done, int n, int W) {
    const int i = blockIdx.x * NTH + threadIdx.x;
    if (i < n) {
        score[i] = i % W ? -INFINITY : 0.0f;
        done[i] = 0;
    }
}
__global__ __launch_bounds__(NTH) void k_beam_record(int *hist, const int *token, const int *parent, int *pos, int n, int step,
                                                    int adv) {
    const int i = blockIdx.x * NTH + threadIdx.x;
    if (i < n) {
        hist[((size_t)step * n + i) * 2] = token[i];
        hist[((size_t)step * n + i) * 2 + 1] = parent[i];
        pos[i] += adv;
    }
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
extern "C" int qm_beam_start(float *score, int *done, int n, int width) {
    if (!score || !done || n <= 0 || width <= 0) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    hipLaunchKernelGGL(k_beam_start, dim3((n + NTH - 1) / NTH), dim3(NTH), 0, stream(), score, done, n, width);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}
extern "C" int qm_beam_record(int *hist, const int *token, const int *parent, int *pos, int n, int step, int adv) {
    if (!hist || !token || !parent || !pos || n <= 0 || step < 0) return QH_EINVAL;
    if (!stream()) return QH_ESTATE;
    hipLaunchKernelGGL(k_beam_record, dim3((n + NTH - 1) / NTH), dim3(NTH), 0, stream(), hist, token, parent, pos, n, step,
                       adv);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

extern "C" size_t qm_beam_select_work(int vocab, int n_group, int width) {
    if (vocab < 1 || n_group < 1 || width < 1 || width > BEAM_MAX) return 0;
    const size_t lists = (size_t)n_group * width * beam_pieces(vocab);
    return lists * (sizeof(beam_sum) + (size_t)width * sizeof(beam_cand));
}

extern "C" int qm_beam_select(const float *logits, size_t ld, int vocab, int n_group, int width, const float *score,
                              const int *done, int end0, int end1, float *score_out, int *done_out, int *token_out,
                              int *parent_out, void *work, size_t work_bytes) {
    if (n_group < 0 || width < 1 || width > BEAM_MAX || vocab < width || ld < (size_t)vocab) return QH_EINVAL;
    if (end0 >= vocab || end1 >= vocab || (done && end0 < 0)) return QH_EINVAL;
    if (n_group == 0) return QH_OK;
    if (!logits || !score || !score_out || !done_out || !token_out || !parent_out || !work || ((uintptr_t)work & 7)) return QH_EINVAL;
    const size_t pieces = beam_pieces(vocab);
    if (pieces > QM_BEAM_MAX_PIECES || (long)n_group * width > 65535) return QH_ETOOBIG;
    if (work_bytes < qm_beam_select_work(vocab, n_group, width)) return QH_ETOOBIG;
    if (!stream()) return QH_ESTATE;
    const int rows = n_group * width;
    beam_sum *sums = (beam_sum *)work;
    beam_cand *lists = (beam_cand *)(sums + (size_t)rows * pieces);
    const dim3 grid((unsigned)((pieces + NTH / WAVE - 1) / (NTH / WAVE)), rows);
    if (aligned16(logits) && ld % 4 == 0)
        hipLaunchKernelGGL(k_beam_pieces<true>, grid, dim3(NTH), 0, stream(), logits, ld, vocab, rows, width, (int)pieces,
                           score, done, sums, lists);
    else
        hipLaunchKernelGGL(k_beam_pieces<false>, grid, dim3(NTH), 0, stream(), logits, ld, vocab, rows, width, (int)pieces,
                           score, done, sums, lists);
    if (hipGetLastError() != hipSuccess) return QH_ELAUNCH;
    hipLaunchKernelGGL(k_beam_pick, dim3(n_group), dim3(WAVE * width), 0, stream(), vocab, width, (int)pieces, score, done,
                       end0, end1, sums, lists, score_out, done_out, token_out, parent_out);
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}

extern "C" int qm_beam_reorder(void *dst, const void *src, const int *parent, int n_group, int width, int slabs,
                               size_t slab_stride, size_t seq_stride, int runs, size_t run_stride, size_t run_bytes) {
    if (n_group < 0 || width < 1 || width > BEAM_MAX || slabs < 0 || runs < 0) return QH_EINVAL;
    if (n_group == 0 || slabs == 0 || runs == 0 || run_bytes == 0) return QH_OK;
    if (!dst || !src || !parent) return QH_EINVAL;
    if (run_bytes % 4 || (runs > 1 && run_stride % 4) || seq_stride % 4 || (slabs > 1 && slab_stride % 4) ||
        (((uintptr_t)dst | (uintptr_t)src) & 3))
        return QH_EINVAL;
    // rows, and the states, must not reach into one another
    if (n_group > 65535 || slabs > 65535 || runs > 1 << 24 || run_bytes > (size_t)1 << 40 || seq_stride > (size_t)1 << 44 ||
        slab_stride > (size_t)1 << 46 || run_stride > (size_t)1 << 40)
        return QH_ETOOBIG;
    const size_t row = (size_t)(runs - 1) * run_stride + run_bytes;
    const size_t slab = ((size_t)n_group * width - 1) * seq_stride + row;
    if ((runs > 1 && run_stride < run_bytes) || seq_stride < row || (slabs > 1 && slab_stride < slab)) return QH_EINVAL;
    const size_t all = (size_t)(slabs - 1) * (slabs > 1 ? slab_stride : 0) + slab;
    const uintptr_t d = (uintptr_t)dst, s = (uintptr_t)src;
    if (d != s && d < s + all && s < d + all) return QH_EINVAL;
    if (width == 1 && d == s) return QH_OK;
    const bool wide = !((run_bytes | seq_stride | (runs > 1 ? run_stride : 0) | (slabs > 1 ? slab_stride : 0) | d | s) & 15);
    const size_t units = run_bytes / (wide ? 16 : 4);
    if (units * runs >= (size_t)1 << 31) return QH_ETOOBIG;
    if (!stream()) return QH_ESTATE;
    const dim3 grid((unsigned)((units * runs + NTH * REORDER_UNITS - 1) / (NTH * REORDER_UNITS)), n_group, slabs);
#define REORDER(T, WT)                                                                                               \
    hipLaunchKernelGGL((k_beam_reorder<T, WT>), grid, dim3(NTH), 0, stream(), (uint8_t *)dst, (const uint8_t *)src,  \
                       parent, width, (unsigned)units, (unsigned)runs, slab_stride, seq_stride, run_stride)
#define REORDER_W(T)                          \
    do {                                      \
        if (width <= 4) REORDER(T, 4);        \
        else if (width <= 8) REORDER(T, 8);   \
        else REORDER(T, 16);                  \
    } while (0)
    if (wide) REORDER_W(u32x4);
    else REORDER_W(uint32_t);
#undef REORDER_W
#undef REORDER
    return hipGetLastError() == hipSuccess ? QH_OK : QH_ELAUNCH;
}
