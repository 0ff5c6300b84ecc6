/* Host side of the device-resident Qwen3-0.6B forward, in C11.
 *
 * The forward follows fpga_bringup/src/src/qwen3.c:455-576 op for op; what
 * changes is where the data lives and how ops are grouped into launches:
 *
 *   chunk (prefill, n tokens)           decode step (1 token, graph-replayed)
 *   ------------------------------     --------------------------------------
 *   embed + rmsnorm        rows_norm    [rmsnorm prologue + qkv GEMV]  (layer 0
 *   qkv GEMM (q|k|v, N=4096)  gemm       gathers the embedding row itself)
 *   qk-norm, rope, KV write,            [qk-norm, rope, KV write, attention]
 *     attention            attention    [o GEMV]
 *   o GEMM                 gemm         [residual + rmsnorm prologue +
 *   residual + rmsnorm     rows_norm     gate/up GEMV + silu*up]
 *   gate/up GEMM + silu*up gemm (gated) [down GEMV]
 *   down GEMM              gemm         ... next layer's prologue adds down
 *   (next layer's rows_norm adds down)  [residual + final norm + lm_head GEMV]
 *   residual + final norm + lm_head     [argmax + token/pos/out bookkeeping]
 *     GEMV on the last row
 *
 * The residual stream of a decode step ping-pongs between x0 and x1: each
 * prologue reads one and its single writer stores x + r into the other.
 */
#define _POSIX_C_SOURCE 200809L   /* clock_gettime under -std=c11 */
#include "qwen3_hip_model.h"
#include "qwen3_hip.h"
#include "hip_shim.h"
#include "model_shim.h"
#include "qw3m.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>
#include <time.h>

#define H QW3M_HIDDEN
#define QKV_N (QW3M_Q_DIM + 2 * QW3M_KV_DIM)
#define NL QW3M_N_LAYERS
#define V QW3M_VOCAB
#define DEFAULT_MAX_SEQ 4096

typedef struct {
    uint16_t *in_norm, *wqkv, *qn, *kn, *wo, *post_norm, *wg, *wu, *wd;
} layer_t;

struct qwen3_hip_model {
    int max_seq;
    uint16_t *wbuf;                    /* all weights, one allocation */
    uint16_t *embed, *final_norm;
    layer_t L[NL];
    float *kc, *vc;                    /* [NL][KVH][..] see hip_model.hip */
    float *rcos, *rsin;                /* [max_seq][64] */
    float *x, *x0, *x1, *xb, *qkv, *att, *ob, *hb, *dn, *logits;
    float *apart;                      /* decode attention partials [QM_ATT_LONG_PART_FLOATS] */
    float *cpart;                      /* chunk attention partials [QM_ATT_CHUNK_PART_FLOATS] */
    int *tok_in;                       /* [prefill_rows(max_seq)] */
    int *state;                        /* [0] token, [1] position, [2] step */
    int *out_tok;                      /* [max_seq + 1] */
    int use_graph;
    int use_persist;                   /* decode layers as one persistent launch */
    int graph_id[2];                   /* the decode step (1: long context), -1 until captured */
    qwen3_hip_dump_fn dump;            /* chunk-path intermediate dumps (NULL = off) */
    void *dump_ctx;
    float *dump_host;                  /* staging for dumps */
    int have_logits;
    double t_prefill_ms, t_decode_ms;
    /* the head's weights as int8 rows, and a step's rows before it; NULL until a batch asks for them */
    int8_t *embed8, *row8;
    float *embed8_scale, *row8_scale;
    struct qwen3_hip_batch *batches;   /* open batches on this model (linked by next) */
};

static void detach_batches(qwen3_hip_model *m);

static double now_ms(void) {
    struct timespec ts;
    clock_gettime(CLOCK_MONOTONIC, &ts);
    return (double)ts.tv_sec * 1e3 + (double)ts.tv_nsec * 1e-6;
}

/* ---- QW3M -------------------------------------------------------------------- */

size_t qwen3_hip_qw3m_size(int layout) { return qw3m_size(layout); }

int qwen3_hip_qw3m_write_random(void *blob, size_t size, uint64_t seed, int layout, int threads) {
    return qw3m_write_random(blob, size, seed, layout, threads) == 0 ? QWEN3_HIP_OK : QWEN3_HIP_EINVAL;
}

int qwen3_hip_qw3m_check(const void *blob, size_t size) { return qw3m_parse(blob, size, NULL); }

/* ---- open / close ------------------------------------------------------------ */

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

/* rows of the chunk buffers: the tokens one pass of the layers takes at most
 * (forward() takes up to QM_MAX_CHUNK per call, which a smaller cache does
 * not lower) */
static int prefill_rows(int max_seq) {
    const int n = max_seq < QM_PREFILL_ROWS ? max_seq : QM_PREFILL_ROWS;
    return n > QM_MAX_CHUNK ? n : QM_MAX_CHUNK;
}

/* bytes of each device tensor, in allocation order */
static size_t dev_weight_bytes(void) {
    size_t b = up256((size_t)V * H * 2) + up256(H * 2);
    const size_t per = up256(H * 2) + up256((size_t)QKV_N * H * 2) + 2 * up256(QW3M_HEAD_DIM * 2) +
                       up256((size_t)H * QW3M_Q_DIM * 2) + up256(H * 2) +
                       2 * up256((size_t)QW3M_INTER * H * 2) + up256((size_t)H * QW3M_INTER * 2);
    return b + (size_t)NL * per;
}

/* upload tensor t of the blob into dst (row-major [rows][cols]); tile-major
 * matrices go through stage and are re-laid on the device */
static int upload(const uint8_t *blob, const qw3m_info_t *info, int t, uint16_t *dst, uint16_t *stage) {
    int rows, cols, mat;
    qw3m_tensor_shape(t, &rows, &cols, &mat);
    const size_t bytes = (size_t)rows * cols * 2;
    const void *src = blob + info->offset[t];
    if (info->layout == QW3M_LAYOUT_TILE && mat) {
        int rc = qh_h2d(stage, src, bytes);
        if (!rc) rc = qh_tile_to_row(dst, stage, rows, cols, info->tile_n, info->tile_k);
        /* the next upload overwrites stage: wait here (pageable source too) */
        const int rc2 = qh_sync();
        return rc ? rc : rc2;
    }
    int rc = qh_h2d(dst, src, bytes);
    if (!rc) rc = qh_sync();
    return rc;
}

static void rope_tables(float *c, float *s, int max_seq) {
    /* ops_scalar.c:21-35: inv_freq = 1 / theta^(2i / head_dim), angle = pos * inv_freq */
    const int half = QW3M_HEAD_DIM / 2;
    for (int i = 0; i < half; i++) {
        const float inv_freq = 1.0f / powf(QW3M_ROPE_THETA, (float)(2 * i) / (float)QW3M_HEAD_DIM);
        for (int p = 0; p < max_seq; p++) {
            const float ang = (float)p * inv_freq;
            c[(size_t)p * half + i] = cosf(ang);
            s[(size_t)p * half + i] = sinf(ang);
        }
    }
}

void qwen3_hip_model_close(qwen3_hip_model *m) {
    if (!m) return;
    (void)qh_sync();
    detach_batches(m);
    for (int g = 0; g < 2; g++)
        if (m->graph_id[g] >= 0) (void)qh_graph_destroy(m->graph_id[g]);
    void *bufs[] = {m->wbuf, m->kc, m->vc, m->rcos, m->rsin, m->x, m->x0, m->x1, m->xb, m->qkv,
                    m->att, m->ob, m->hb, m->dn, m->logits, m->apart, m->cpart, m->tok_in, m->state, m->out_tok,
                    m->embed8, m->row8, m->embed8_scale, m->row8_scale};
    for (size_t i = 0; i < sizeof bufs / sizeof bufs[0]; i++) (void)qh_free(bufs[i]);
    free(m->dump_host);
    free(m);
}

int qwen3_hip_model_open(qwen3_hip_model **out, const void *blob, size_t size, int max_seq) {
    if (!out) return QWEN3_HIP_EINVAL;
    *out = NULL;
    qw3m_info_t info;
    int rc = qw3m_parse(blob, size, &info);
    if (rc) return rc;
    if (max_seq == 0) max_seq = DEFAULT_MAX_SEQ;
    if (max_seq < 1 || max_seq > QM_MAX_SEQ) return QWEN3_HIP_EINVAL;
    rc = qwen3_hip_init(-1);
    if (rc) return rc;

    qwen3_hip_model *m = (qwen3_hip_model *)calloc(1, sizeof *m);
    if (!m) return QWEN3_HIP_ENOMEM;
    m->max_seq = max_seq;
    m->use_graph = 1;
    m->graph_id[0] = m->graph_id[1] = -1;
    {
        /* the persistent decode launch, opt-in: measured slower than the
         * per-layer launches (1,720-1,750 against 1,780-1,805 tok/s).  Its
         * buffers, shared by every model, are allocated when first wanted;
         * failing to get them only leaves it off. */
        const char *env = getenv("QWEN3_HIP_MODEL_PERSIST");
        m->use_persist = env && strcmp(env, "1") == 0 && qm_persist_init() == 0 && qm_persist_supported();
    }

#define DEV(ptr, bytes)                                                   \
    do {                                                                  \
        if ((rc = qh_malloc((void **)&(ptr), (bytes))) != 0) goto fail;   \
    } while (0)
    DEV(m->wbuf, dev_weight_bytes());
    const size_t kv_bytes = (size_t)NL * QW3M_N_KV_HEADS * max_seq * QW3M_HEAD_DIM * sizeof(float);
    DEV(m->kc, kv_bytes);
    DEV(m->vc, kv_bytes);
    const size_t rope_bytes = (size_t)max_seq * (QW3M_HEAD_DIM / 2) * sizeof(float);
    DEV(m->rcos, rope_bytes);
    DEV(m->rsin, rope_bytes);
    const size_t B = (size_t)prefill_rows(max_seq);
    DEV(m->x, B * H * 4);
    DEV(m->x0, H * 4);
    DEV(m->x1, H * 4);
    DEV(m->xb, B * H * 4);
    DEV(m->qkv, B * QKV_N * 4);
    DEV(m->att, B * QW3M_Q_DIM * 4);
    DEV(m->ob, B * H * 4);
    DEV(m->hb, B * QW3M_INTER * 4);
    DEV(m->dn, B * H * 4);
    DEV(m->logits, (size_t)V * 4);
    DEV(m->apart, (size_t)QM_ATT_LONG_PART_FLOATS * 4);
    DEV(m->cpart, QM_ATT_CHUNK_PART_FLOATS * 4);
    DEV(m->tok_in, B * sizeof(int));
    DEV(m->state, 4 * sizeof(int));
    DEV(m->out_tok, ((size_t)max_seq + 1) * sizeof(int));
#undef DEV

    /* carve the weight allocation */
    {
        uint8_t *p = (uint8_t *)m->wbuf;
#define CARVE(dst, bytes) do { (dst) = (uint16_t *)p; p += up256(bytes); } while (0)
        CARVE(m->embed, (size_t)V * H * 2);
        CARVE(m->final_norm, H * 2);
        for (int l = 0; l < NL; l++) {
            layer_t *L = &m->L[l];
            CARVE(L->in_norm, H * 2);
            CARVE(L->wqkv, (size_t)QKV_N * H * 2);
            CARVE(L->qn, QW3M_HEAD_DIM * 2);
            CARVE(L->kn, QW3M_HEAD_DIM * 2);
            CARVE(L->wo, (size_t)H * QW3M_Q_DIM * 2);
            CARVE(L->post_norm, H * 2);
            CARVE(L->wg, (size_t)QW3M_INTER * H * 2);
            CARVE(L->wu, (size_t)QW3M_INTER * H * 2);
            CARVE(L->wd, (size_t)H * QW3M_INTER * 2);
        }
#undef CARVE
    }

    /* upload; the tile stage holds the largest matrix (6 MiB) */
    {
        uint16_t *stage = NULL;
        if (info.layout == QW3M_LAYOUT_TILE &&
            (rc = qh_malloc((void **)&stage, (size_t)QW3M_INTER * H * 2)) != 0)
            goto fail;
        const uint8_t *b = (const uint8_t *)blob;
        rc = upload(b, &info, 0, m->embed, stage);
        for (int l = 0; l < NL && !rc; l++) {
            const int t0 = 1 + 11 * l;
            layer_t *L = &m->L[l];
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_IN_NORM, L->in_norm, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WQ, L->wqkv, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WK, L->wqkv + (size_t)QW3M_Q_DIM * H, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WV, L->wqkv + (size_t)(QW3M_Q_DIM + QW3M_KV_DIM) * H, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_QNORM, L->qn, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_KNORM, L->kn, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WO, L->wo, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_POST_NORM, L->post_norm, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WGATE, L->wg, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WUP, L->wu, stage);
            if (!rc) rc = upload(b, &info, t0 + QW3M_T_WDOWN, L->wd, stage);
        }
        if (!rc) rc = upload(b, &info, QW3M_N_TENSORS - 1, m->final_norm, stage);
        if (stage) (void)qh_free(stage);
        if (rc) goto fail;
    }

    /* rope tables */
    {
        float *c = (float *)malloc(rope_bytes), *s = (float *)malloc(rope_bytes);
        if (!c || !s) { free(c); free(s); rc = QWEN3_HIP_ENOMEM; goto fail; }
        rope_tables(c, s, max_seq);
        rc = qh_h2d(m->rcos, c, rope_bytes);
        if (!rc) rc = qh_h2d(m->rsin, s, rope_bytes);
        const int rc2 = qh_sync();     /* copies read these tables, whatever happened */
        if (!rc) rc = rc2;
        free(c);
        free(s);
        if (rc) goto fail;
    }
    *out = m;
    return QWEN3_HIP_OK;
fail:
    qwen3_hip_model_close(m);
    return rc;
}

int qwen3_hip_model_max_seq(const qwen3_hip_model *m) { return m ? m->max_seq : 0; }

int qwen3_hip_model_set_dump(qwen3_hip_model *m, qwen3_hip_dump_fn fn, void *ctx) {
    if (!m) return QWEN3_HIP_EINVAL;
    if (fn && !m->dump_host) {
        m->dump_host = (float *)malloc((size_t)QM_MAX_CHUNK * QKV_N * sizeof(float));
        if (!m->dump_host) return QWEN3_HIP_ENOMEM;
    }
    m->dump = fn;
    m->dump_ctx = ctx;
    return QWEN3_HIP_OK;
}

/* copy rows x cols floats at column col0 of a [rows][ld] device matrix to the
 * host and hand them to the dump callback (same names as qwen3.c's EMITs) */
static int dump_dev(qwen3_hip_model *m, int layer, const char *name, const float *dev, int rows,
                    int ld, int col0, int cols) {
    float *h = m->dump_host;
    int rc = qh_d2h(h, dev, (size_t)rows * ld * sizeof(float));
    if (!rc) rc = qh_sync();
    if (rc) return rc;
    if (col0 != 0 || cols != ld)
        for (int r = 0; r < rows; r++) memmove(h + (size_t)r * cols, h + (size_t)r * ld + col0, cols * sizeof(float));
    m->dump(m->dump_ctx, layer, name, h, (size_t)rows * cols);
    return QWEN3_HIP_OK;
}

int qwen3_hip_model_set_graph(qwen3_hip_model *m, int on) {
    if (!m) return QWEN3_HIP_EINVAL;
    m->use_graph = on ? 1 : 0;
    return QWEN3_HIP_OK;
}

int qwen3_hip_model_set_persistent(qwen3_hip_model *m, int on) {
    if (!m) return QWEN3_HIP_EINVAL;
    if (on) {
        const int rc = qm_persist_init();   /* once: the launch's buffers and the residency check */
        if (rc) return rc;
        if (!qm_persist_supported()) return QWEN3_HIP_ENODEV;
    }
    if ((on ? 1 : 0) != m->use_persist && m->graph_id[0] >= 0) {   /* the captured step is the other kind */
        int rc = qh_sync();
        if (!rc) rc = qh_graph_destroy(m->graph_id[0]);
        if (rc) return rc;
        m->graph_id[0] = -1;
    }
    m->use_persist = on ? 1 : 0;
    return QWEN3_HIP_OK;
}

int qwen3_hip_model_persistent(const qwen3_hip_model *m) { return m ? m->use_persist : 0; }

int qwen3_hip_model_persist_errors(qwen3_hip_model *m, unsigned *flags) {
    if (!m || !flags) return QWEN3_HIP_EINVAL;
    *flags = 0;
    return qm_persist_supported() ? qm_persist_errors(flags) : QWEN3_HIP_OK;
}

/* ---- forward ----------------------------------------------------------------- */

static size_t kv_layer_floats(const qwen3_hip_model *m) {
    return (size_t)QW3M_N_KV_HEADS * m->max_seq * QW3M_HEAD_DIM;
}

/* a batch's 8-bit caches: layer 0's, and what to add for the next layer's */
#define KV8_BLOCK 32
typedef struct {
    qm_kv8_t c;
    size_t codes, scales, tails;       /* per layer: bytes of K, floats, bf16 values */
    int *row;                          /* [2]: a prompt pass's row offsets 0, nt */
    void *work;
    size_t work_bytes;
} kv8_t;

static qm_kv8_t kv8_layer(const kv8_t *k, int l) {
    qm_kv8_t c = k->c;
    c.k += l * k->codes;
    c.v += l * k->codes;
    c.k_scale += l * k->scales;
    c.v_scale += l * k->scales;
    c.k_tail += l * k->tails;
    c.v_tail += l * k->tails;
    return c;
}
/* the cache of sequence seq alone */
static kv8_t kv8_seq(const kv8_t *k, int seq) {
    kv8_t s = *k;
    const size_t tail = (size_t)k->c.heads * k->c.block * k->c.head_dim;
    s.c.table += (size_t)seq * k->c.max_blocks;
    s.c.k_tail += seq * tail;
    s.c.v_tail += seq * tail;
    s.c.n_seq = 1;
    return s;
}

/* where a chunk's K/V go: layer l's cache of one sequence starts at
 * kc + l * layer_stride (layout in hip_model.hip, max_seq positions), or the
 * 8-bit cache kv8 of that sequence */
typedef struct {
    float *kc, *vc;
    size_t layer_stride;
    int max_seq;
    const kv8_t *kv8;
} kv_t;

static kv_t model_kv(qwen3_hip_model *m) {
    const kv_t kv = {m->kc, m->vc, kv_layer_floats(m), m->max_seq, NULL};
    return kv;
}

/* 1 / sqrt(head_dim), the constant of qwen3.c:311 */
#define ATT_SCALE 0.08838834764831845f

/* attention of nt rows of m->qkv over an 8-bit cache: q and k are normalised
 * and rotated, k and v stored, then read back through the cache.  n sequences
 * of one row (pos[i]), or one sequence's nt rows at *pos ... */
static int attend_kv8(qwen3_hip_model *m, const kv8_t *k, int l, const layer_t *L, int n, int nt, const int *pos,
                      int ctx, int bf16) {
    const qm_kv8_t c = kv8_layer(k, l);
    const int each = n == nt;          /* a row of each sequence */
    /* bf16 rows: the output takes the first half of the buffer, q the second */
    uint16_t *qb = bf16 ? (uint16_t *)m->att + (size_t)nt * QW3M_Q_DIM : NULL;
    int rc;
    if (each) {
        rc = qm_kv8_rope_append(&c, m->qkv, L->qn, L->kn, m->rcos, m->rsin, pos, n, m->max_seq, QW3M_RMS_EPS);
    } else {
        rc = qm_qk_rope(m->qkv, qb, L->qn, L->kn, m->rcos, m->rsin, pos, nt, m->max_seq, QW3M_RMS_EPS);
        if (!rc) rc = qm_kv8_append(&c, m->qkv + QW3M_Q_DIM, m->qkv + QW3M_Q_DIM + QW3M_KV_DIM, QKV_N, QKV_N, 0, k->row,
                                    pos, n, nt, nt);
    }
    if (!rc) rc = qm_kv8_attention(&c, m->att, bf16 ? (const void *)qb : m->qkv, QW3M_Q_DIM, bf16 ? QW3M_Q_DIM : QKV_N,
                                   bf16, QW3M_N_HEADS, each ? NULL : k->row, pos, n, nt, each ? 1 : nt, ctx,
                                   ATT_SCALE, k->work, k->work_bytes);
    return rc;
}

/* attention of a chunk of nt tokens at pos0, the cache's entries written */
static int attend_chunk(qwen3_hip_model *m, const kv_t *kv, int l, const layer_t *L, int nt, int pos0, int bf16) {
    if (kv->kv8) return attend_kv8(m, kv->kv8, l, L, 1, nt, m->state + 1, pos0 + nt, bf16);
    float *kc = kv->kc + l * kv->layer_stride, *vc = kv->vc + l * kv->layer_stride;
    return bf16 ? qm_attention_bf16(m->qkv, (uint16_t *)m->att, m->cpart, kc, vc, L->qn, L->kn, m->rcos, m->rsin,
                                    m->state + 1, nt, kv->max_seq, pos0 + nt, QW3M_RMS_EPS)
                : qm_attention(m->qkv, m->att, m->cpart, kc, vc, L->qn, L->kn, m->rcos, m->rsin, m->state + 1, nt,
                               kv->max_seq, pos0 + nt, QW3M_RMS_EPS);
}

/* the layers of a chunk of more than BF16_ROWS tokens with the inputs of all
 * four products stored as bf16: their producers round what the products would
 * round on loading, so the values are the same and the products read half the
 * bytes of A (up to 64 rows the small-batch kernels read fp32 A).  Measured on
 * MI355X: forward of 128 tokens 1,557 -> 1,420 us, 16 prompts of up to 200 tokens
 * and 24 batched steps 54.9 -> 52.3 ms, 1,800-token prompt and 32 greedy tokens
 * 32.7 -> 31.9 ms */
#define BF16_ROWS 64
static int run_layers_bf16(qwen3_hip_model *m, const kv_t *kv, int nt, int pos0) {
    const float eps = QW3M_RMS_EPS;
    uint16_t *xb = (uint16_t *)m->xb, *att = (uint16_t *)m->att, *hb = (uint16_t *)m->hb;
    const float *opart = NULL, *dpart = NULL;
    int oks = 0, dks = 0, rc = QWEN3_HIP_OK;
    for (int l = 0; l < NL && !rc; l++) {
        const layer_t *L = &m->L[l];
        rc = qm_rows_norm_bf16(m->x, l == 0 || dks ? NULL : m->dn, l == 0 ? m->embed : NULL, m->tok_in, V, L->in_norm,
                               xb, nt, H, eps, dpart, dks);
        if (!rc) rc = qh_gemm_bf16a(m->qkv, xb, L->wqkv, nt, H, QKV_N);
        if (!rc) rc = attend_chunk(m, kv, l, L, nt, pos0, 1);
        if (!rc) rc = qh_gemm_split_bf16a(m->ob, att, L->wo, nt, QW3M_Q_DIM, H, &opart, &oks);
        if (!rc) rc = qm_rows_norm_bf16(m->x, oks ? NULL : m->ob, NULL, NULL, 0, L->post_norm, xb, nt, H, eps, opart,
                                        oks);
        if (!rc) rc = qh_gemm_gate_up_silu_bf16ac(hb, xb, L->wg, L->wu, nt, H, QW3M_INTER);
        dks = 0;
        if (!rc) rc = l == NL - 1 ? qh_gemm_bf16a(m->dn, hb, L->wd, nt, QW3M_INTER, H)
                                  : qh_gemm_split_bf16a(m->dn, hb, L->wd, nt, QW3M_INTER, H, &dpart, &dks);
    }
    return rc;
}

/* nt tokens already in tok_in at positions pos0.. (pos0 also set by the
 * caller in state[1]) of the sequence whose cache is kv; logits of the last
 * row when want_logits */
static int run_chunk(qwen3_hip_model *m, const kv_t *kv, int nt, int pos0, int want_logits) {
    int rc = QWEN3_HIP_OK;
    const float eps = QW3M_RMS_EPS;
    /* with a dump callback the residual add of down_proj is done at the end
       of its layer (to materialise "layer_out"), not in the next prologue */
    const int dumping = m->dump != NULL;
#define DUMP(layer, name, ptr, ld, col0, cols) \
    do { if (!rc && dumping) rc = dump_dev(m, (layer), (name), (ptr), nt, (ld), (col0), (cols)); } while (0)
    /* without dumps, the o and down projections may leave split-K slice sums
       (qh_gemm_split) that the next residual + RMSNorm adds itself; the last
       layer's down is written out for the lm_head GEMV's prologue */
    const float *opart = NULL, *dpart = NULL;
    int oks = 0, dks = 0;
    const int bf16 = !dumping && nt > BF16_ROWS;
    if (bf16 && (rc = run_layers_bf16(m, kv, nt, pos0)) != 0) return rc;
    for (int l = 0; l < NL && !bf16; l++) {
        const layer_t *L = &m->L[l];
        if (l == 0) {
            rc = qm_rows_norm(m->x, NULL, m->embed, m->tok_in, V, L->in_norm, m->xb, nt, H, eps);
            DUMP(-1, "embed_out", m->x, H, 0, H);
        } else {
            rc = qm_rows_norm_split(m->x, dumping || dks ? NULL : m->dn, NULL, NULL, 0, L->in_norm, m->xb, nt, H,
                                    eps, dpart, dks);
        }
        DUMP(l, "input_layernorm_out", m->xb, H, 0, H);
        if (!rc) rc = qh_gemm(m->qkv, m->xb, L->wqkv, nt, H, QKV_N);
        DUMP(l, "q_proj_out", m->qkv, QKV_N, 0, QW3M_Q_DIM);
        DUMP(l, "k_proj_out", m->qkv, QKV_N, QW3M_Q_DIM, QW3M_KV_DIM);
        DUMP(l, "v_proj_out", m->qkv, QKV_N, QW3M_Q_DIM + QW3M_KV_DIM, QW3M_KV_DIM);
        if (!rc) rc = attend_chunk(m, kv, l, L, nt, pos0, 0);
        DUMP(l, "attn_out", m->att, QW3M_Q_DIM, 0, QW3M_Q_DIM);
        if (!rc) rc = dumping ? qh_gemm(m->ob, m->att, L->wo, nt, QW3M_Q_DIM, H)
                              : qh_gemm_split(m->ob, m->att, L->wo, nt, QW3M_Q_DIM, H, &opart, &oks);
        DUMP(l, "o_proj_out", m->ob, H, 0, H);
        if (!rc) rc = qm_rows_norm_split(m->x, oks ? NULL : m->ob, NULL, NULL, 0, L->post_norm, m->xb, nt, H, eps,
                                         opart, oks);
        DUMP(l, "x_after_attn_residual", m->x, H, 0, H);
        DUMP(l, "post_attn_norm_out", m->xb, H, 0, H);
        if (!rc) rc = qh_gemm_gate_up_silu(m->hb, m->xb, L->wg, L->wu, nt, H, QW3M_INTER);
        DUMP(l, "silu_gate_mul_up", m->hb, QW3M_INTER, 0, QW3M_INTER);
        dks = 0;
        if (!rc) rc = (dumping || l == NL - 1) ? qh_gemm(m->dn, m->hb, L->wd, nt, QW3M_INTER, H)
                                               : qh_gemm_split(m->dn, m->hb, L->wd, nt, QW3M_INTER, H, &dpart, &dks);
        DUMP(l, "down_proj_out", m->dn, H, 0, H);
        if (!rc && dumping) {
            /* x += down (xb is scratch here; the next layer recomputes it) */
            rc = qm_rows_norm(m->x, m->dn, NULL, NULL, 0, L->in_norm, m->xb, nt, H, eps);
            DUMP(l, "layer_out", m->x, H, 0, H);
        }
        if (rc) return rc;
    }
#undef DUMP
    if (!want_logits) return QWEN3_HIP_OK;
    const qh_gemv_pro_t pro = {m->x + (size_t)(nt - 1) * H, NULL, NULL, 0,
                               dumping ? NULL : m->dn + (size_t)(nt - 1) * H, m->final_norm, NULL, eps};
    rc = qh_gemv_pro(m->logits, &pro, m->embed, NULL, H, V, 0);
    if (!rc && dumping) {
        rc = qh_d2h(m->dump_host, m->logits, (size_t)V * sizeof(float));
        if (!rc) rc = qh_sync();
        if (!rc) m->dump(m->dump_ctx, -1, "logits", m->dump_host, V);
    }
    return rc;
}

/* the logits of token state[0] at position state[1], its K and V appended to
 * the cache; the layers as one launch when persist, except behind a long
 * context (more than QM_LONG_CTX positions, the new one included), whose
 * attention is split finer than that launch does */
static int decode_logits(qwen3_hip_model *m, int persist, int lng) {
    int rc = QWEN3_HIP_OK;
    persist = persist && !lng;
    const float eps = QW3M_RMS_EPS;
    if (persist) {
        /* the 28 layers in one launch: x0 and dn as the per-layer launches leave them */
        const uint16_t *w[NL * 9];
        for (int l = 0; l < NL; l++) {
            const layer_t *L = &m->L[l];
            const uint16_t *lw[9] = {L->in_norm, L->wqkv, L->qn, L->kn, L->wo, L->post_norm, L->wg, L->wu, L->wd};
            memcpy(w + 9 * l, lw, sizeof lw);
        }
        rc = qm_decode_layers_persist(w, NL, m->embed, V, m->state, m->kc, m->vc, kv_layer_floats(m), m->rcos,
                                      m->rsin, m->max_seq, eps, m->x0, m->dn);
    }
    for (int l = 0; l < NL && !rc && !persist; l++) {
        const layer_t *L = &m->L[l];
        qh_gemv_pro_t pro = {m->x0, NULL, NULL, 0, m->dn, L->in_norm, m->x1, eps};
        if (l == 0) { pro.x = NULL; pro.r = NULL; pro.emb = m->embed; pro.tok = m->state; pro.emb_rows = V; }
        rc = qh_gemv_pro(m->qkv, &pro, L->wqkv, NULL, H, QKV_N, 0);
        float *kc = m->kc + l * kv_layer_floats(m), *vc = m->vc + l * kv_layer_floats(m);
        if (lng) {
            if (!rc) rc = qm_attention_decode_long(m->qkv, m->att, m->apart, kc, vc, L->qn, L->kn, m->rcos, m->rsin,
                                                   m->state + 1, m->max_seq, eps);
            if (!rc) rc = qh_gemm(m->ob, m->att, L->wo, 1, QW3M_Q_DIM, H);
        } else {
            /* attention as split-softmax partials, merged in the o GEMV's prologue */
            if (!rc) rc = qm_attention_decode_part(m->qkv, m->apart, kc, vc, L->qn, L->kn, m->rcos, m->rsin,
                                                   m->state + 1, m->max_seq, eps);
            if (!rc) rc = qh_gemv_merge(m->ob, m->apart, L->wo, QW3M_Q_DIM, H);
        }
        const qh_gemv_pro_t pro2 = {m->x1, NULL, NULL, 0, m->ob, L->post_norm, m->x0, eps};
        if (!rc) rc = qh_gemv_pro(m->hb, &pro2, L->wg, L->wu, H, QW3M_INTER, 1);
        if (!rc) rc = qh_gemm(m->dn, m->hb, L->wd, 1, QW3M_INTER, H);
    }
    const qh_gemv_pro_t fin = {m->x0, NULL, NULL, 0, m->dn, m->final_norm, NULL, eps};
    if (!rc) rc = qh_gemv_pro(m->logits, &fin, m->embed, NULL, H, V, 0);
    return rc;
}

/* one greedy decode step on the device: token state[0] at position
 * state[1]; appends the next token to out_tok[state[2]] */
static int decode_step(qwen3_hip_model *m, int lng) {
    int rc = decode_logits(m, m->use_persist, lng);
    if (!rc) rc = qh_argmax_step(m->state, m->out_tok, m->state + 2, m->max_seq + 1, m->state + 1, 1,
                                 m->logits, V);
    return rc;
}

static int check_tokens(const int *t, int n) {
    for (int i = 0; i < n; i++)
        if (t[i] < 0 || t[i] >= V) return QWEN3_HIP_EINVAL;
    return QWEN3_HIP_OK;
}

/* tokens -> tok_in and pos0 -> state[1].  Up to QM_MAX_CHUNK tokens travel as
 * kernel arguments: no copy and no wait (a copy from the caller's pageable
 * memory has to be waited for).  Refused while the caller records a graph: its
 * replays would feed these tokens again */
static int load_chunk(qwen3_hip_model *m, const int *tokens, int nt, int pos0) {
    if (qh_capturing()) return QWEN3_HIP_ERUNTIME;
    if (nt <= QM_MAX_CHUNK) return qm_set_tokens(m->tok_in, tokens, nt, m->state + 1, pos0);
    int rc = qh_h2d(m->tok_in, tokens, (size_t)nt * sizeof(int));
    if (!rc) rc = qm_set_i32(m->state + 1, pos0);
    const int rc2 = qh_sync();         /* the copy reads the caller's tokens, whatever happened */
    return rc ? rc : rc2;
}

/* a whole prompt at positions 0 .. n - 1 into the sequence whose cache is kv,
 * in equal passes of at most prefill_rows tokens (QM_MAX_CHUNK while a dump
 * callback wants each pass's tensors); logits of the last token.  *last: the
 * tokens of the last pass. */
static int prefill(qwen3_hip_model *m, const kv_t *kv, const int *prompt, int n, int *last) {
    const int most = m->dump ? QM_MAX_CHUNK : prefill_rows(m->max_seq);
    const int passes = (n + most - 1) / most, each = (n + passes - 1) / passes;
    int rc = QWEN3_HIP_OK;
    for (int p0 = 0; p0 < n && !rc; p0 += each) {
        *last = n - p0 < each ? n - p0 : each;
        rc = load_chunk(m, prompt + p0, *last, p0);
        if (!rc && kv->kv8) rc = qm_set_i32(kv->kv8->row + 1, *last);
        if (!rc) rc = run_chunk(m, kv, *last, p0, p0 + *last == n);
    }
    return rc;
}

int qwen3_hip_model_forward(qwen3_hip_model *m, const int *tokens, int n_token, int pos0) {
    if (!m || !tokens) return QWEN3_HIP_EINVAL;
    if (n_token < 1 || n_token > QM_MAX_CHUNK || pos0 < 0 || pos0 + n_token > m->max_seq)
        return QWEN3_HIP_EINVAL;
    int rc = check_tokens(tokens, n_token);
    if (!rc && n_token == 1 && !m->dump) {
        /* one token is a decode step whose next token the caller picks: five
           launches per layer on the GEMV kernels instead of a chunk's eight
           (measured on MI355X behind 700 positions, the copy of the logits
           included: 1,640 -> 745 to 800 us a call) */
        rc = qh_capturing() ? QWEN3_HIP_ERUNTIME : qm_set_tokens(m->state, tokens, 1, m->state + 1, pos0);
        if (!rc) rc = decode_logits(m, 0, pos0 + 1 > QM_LONG_CTX);
    } else if (!rc) {
        const kv_t kv = model_kv(m);
        rc = load_chunk(m, tokens, n_token, pos0);
        if (!rc) rc = run_chunk(m, &kv, n_token, pos0, 1);
    }
    m->have_logits = rc == 0;
    return rc;
}

int qwen3_hip_model_logits(qwen3_hip_model *m, float *out) {
    if (!m || !out || !m->have_logits) return QWEN3_HIP_EINVAL;
    int rc = qh_d2h(out, m->logits, (size_t)V * sizeof(float));
    if (!rc) rc = qh_sync();
    return rc;
}

int qwen3_hip_model_argmax(qwen3_hip_model *m, int *token) {
    if (!m || !token || !m->have_logits) return QWEN3_HIP_EINVAL;
    int rc = qh_argmax(m->state + 3, m->logits, V);
    if (!rc) rc = qh_d2h(token, m->state + 3, sizeof(int));
    if (!rc) rc = qh_sync();
    return rc;
}

int qwen3_hip_model_generate(qwen3_hip_model *m, const int *prompt, int n_prompt, int n_decode,
                             int stop_at_eos, int *out, int *n_out) {
    if (!m || !prompt || !out || !n_out) return QWEN3_HIP_EINVAL;
    *n_out = 0;
    if (n_prompt < 1 || n_decode < 0 || (long)n_prompt + n_decode > m->max_seq) return QWEN3_HIP_EINVAL;
    int rc = check_tokens(prompt, n_prompt);
    if (rc) return rc;

    const kv_t kv = model_kv(m);
    const double t0 = now_ms();
    int nt = 0;
    rc = prefill(m, &kv, prompt, n_prompt, &nt);
    /* first token; state[1] = pos0 of the last chunk + nt = n_prompt */
    if (!rc) rc = qm_set_i32(m->state + 2, 0);
    if (!rc) rc = qh_argmax_step(m->state, m->out_tok, m->state + 2, m->max_seq + 1, m->state + 1, nt,
                                 m->logits, V);
    if (!rc) rc = qh_sync();
    const double t1 = now_ms();
    if (rc) return rc;

    for (int s = 0; s < n_decode && !rc; s++) {
        const int lng = n_prompt + s + 1 > QM_LONG_CTX;
        if (m->use_graph && m->graph_id[lng] < 0) {
            rc = qh_capture_begin();
            if (rc) break;
            const int rc2 = decode_step(m, lng);
            int gid = -1;
            rc = qh_capture_end(&gid);
            if (!rc) rc = rc2;
            if (rc) {
                if (gid >= 0) (void)qh_graph_destroy(gid);
                break;
            }
            m->graph_id[lng] = gid;
        }
        rc = m->use_graph ? qh_graph_launch(m->graph_id[lng]) : decode_step(m, lng);
    }
    if (rc) {
        (void)qh_sync();               /* steps already launched */
        return rc;
    }
    if (!rc) rc = qh_sync();
    const double t2 = now_ms();
    if (rc) return rc;
    m->have_logits = 1;

    rc = qh_d2h(out, m->out_tok, ((size_t)n_decode + 1) * sizeof(int));
    if (!rc) rc = qh_sync();
    if (rc) return rc;
    int n = n_decode + 1;
    if (stop_at_eos)
        for (int i = 0; i < n; i++)
            if (out[i] == QW3M_EOS0 || out[i] == QW3M_EOS1) { n = i + 1; break; }
    *n_out = n;
    m->t_prefill_ms = t1 - t0;
    m->t_decode_ms = t2 - t1;
    return QWEN3_HIP_OK;
}

int qwen3_hip_model_timing(const qwen3_hip_model *m, double *prefill_ms, double *decode_ms) {
    if (!m) return QWEN3_HIP_EINVAL;
    if (prefill_ms) *prefill_ms = m->t_prefill_ms;
    if (decode_ms) *decode_ms = m->t_decode_ms;
    return QWEN3_HIP_OK;
}

/* ---- multi-sequence batched decode ------------------------------------------ */

#define MASK_WORDS ((V + 31) / 32)
/* what is asked of a sequence's tokens; of the batch's masks two are a sequence's, so
 * that a new one leaves the one in use whole */
typedef struct {
    int on, mask, n_bias;              /* mask: its place, 2 seq or 2 seq + 1; -1: none */
    float repetition, presence, frequency;
    int *bias_token;
    float *bias;
} seq_rules_t;

struct qwen3_hip_batch {
    qwen3_hip_model *m;
    int n_seq, max_ctx, out_ld;
    size_t kv_seq;                     /* floats of one sequence's cache in one layer */
    float *kc, *vc;                    /* [NL][n_seq][kv_seq]; NULL with 8-bit caches */
    kv8_t kv8;                         /* c.k NULL with fp32 caches */
    int *table;                        /* kv8.c.table */
    float *logits;                     /* [n_seq][V] of the last decode step */
    float *part;                       /* [n_seq][QM_BATCH_PART_FLOATS] */
    int *tok, *pos, *plen;             /* [n_seq]: next token fed, its position, prompt length */
    int *out;                          /* [n_seq][out_ld]: token i of a sequence at i = pos - plen + 1 */
    int *h_next;                       /* host: position of each sequence's next fed token (-1: empty) */
    int *h_plen;                       /* host: prompt length of each sequence */
    int *h_out;                        /* host staging of out */
    int use_graph;
    int graph_id[3];                   /* the greedy step, the beams' forward, the step under rules; -1 until captured */
    int ruled;                         /* a step under rules has run eagerly since the graphs went */
    int have_logits;
    int head8;                         /* the head's product in 8-bit integers */
    double t_decode_ms;
    /* rules on logits, allocated by the first: the texts [n_seq][out_ld] and their
     * lengths, kept up while a sequence is under rules; penalties [3][n_seq]; the
     * sequences' biases one after another, room for bias_room; two masks each.
     * torn: an upload failed, and what is here is no one's until the next succeeds */
    int *h_text;                       /* host: every prefilled sequence's prompt */
    seq_rules_t *h_rules;
    int n_rules;                       /* sequences under rules */
    int *text, *n_text, *bias_row, *bias_token, *mask_of;
    float *penalty, *bias;
    uint32_t *mask;
    int bias_room, torn;
    /* beam search, allocated by the first: per sequence score, finished, parent;
     * {token, parent} of every step; the choice's workspace */
    float *score;
    int *done, *parent, *hist;
    void *swork;
    size_t swork_bytes;
    qwen3_hip_batch *next;             /* the model's list of open batches */
};

/* A batch's graphs hold the model's device addresses: when the model closes
 * first, its batches lose the graphs and the model, and later calls on them
 * return QWEN3_HIP_ESTATE instead of touching freed memory. */
static void drop_graphs(qwen3_hip_batch *b) {
    for (int g = 0; g < 3; g++) {
        if (b->graph_id[g] >= 0) (void)qh_graph_destroy(b->graph_id[g]);
        b->graph_id[g] = -1;
    }
    b->ruled = 0;
}

static void detach_batches(qwen3_hip_model *m) {
    for (qwen3_hip_batch *b = m->batches; b; b = b->next) {
        drop_graphs(b);
        b->m = NULL;
    }
    m->batches = NULL;
}

void qwen3_hip_batch_close(qwen3_hip_batch *b) {
    if (!b) return;
    (void)qh_sync();
    if (b->m) {
        qwen3_hip_batch **pp = &b->m->batches;
        while (*pp && *pp != b) pp = &(*pp)->next;
        if (*pp) *pp = b->next;
    }
    drop_graphs(b);
    void *bufs[] = {b->kc, b->vc, b->logits, b->part, b->tok, b->pos, b->plen, b->out, b->kv8.c.k, b->kv8.c.k_scale,
                    b->kv8.c.k_tail, b->table, b->kv8.row, b->kv8.work, b->score, b->done, b->parent, b->hist, b->swork,
                    b->text, b->n_text, b->bias_row, b->bias_token, b->mask_of, b->penalty, b->bias, b->mask};
    for (size_t i = 0; i < sizeof bufs / sizeof bufs[0]; i++) (void)qh_free(bufs[i]);
    for (int s = 0; b->h_rules && s < b->n_seq; s++) {
        free(b->h_rules[s].bias_token);
        free(b->h_rules[s].bias);
    }
    free(b->h_rules);
    free(b->h_text);
    free(b->h_next);
    free(b->h_plen);
    free(b->h_out);
    free(b);
}

/* the 8-bit caches of a batch: pages s * max_blocks .. of sequence s, its
 * tails one allocation [K, V][layer][sequence] so that beams reorder them in
 * one call.  Blocks of 32 tokens: 131 KB of tail per sequence and layer and a
 * scale for 4,096 values; 16 halves the one and doubles the scales, 64 the
 * other way, with no other cost in the kernels. */
static int open_kv8(qwen3_hip_batch *b, int format) {
    qm_kv8_t *c = &b->kv8.c;
    c->format = format;
    c->heads = QW3M_N_KV_HEADS;
    c->head_dim = QW3M_HEAD_DIM;
    c->block = KV8_BLOCK;
    c->n_seq = b->n_seq;
    c->max_blocks = (b->max_ctx + KV8_BLOCK - 1) / KV8_BLOCK;
    c->n_page = b->n_seq * c->max_blocks;
    const size_t unit = (size_t)c->heads * c->block * c->head_dim;      /* values of a block */
    b->kv8.codes = c->n_page * unit;
    b->kv8.scales = (size_t)c->n_page * c->heads;
    b->kv8.tails = b->n_seq * unit;
    int rc = qh_malloc((void **)&c->k, 2 * NL * b->kv8.codes);
    if (!rc) rc = qh_malloc((void **)&c->k_scale, 2 * NL * b->kv8.scales * sizeof(float));
    if (!rc) rc = qh_malloc((void **)&c->k_tail, 2 * NL * b->kv8.tails * sizeof(uint16_t));
    if (!rc) rc = qh_malloc((void **)&b->table, (size_t)c->n_page * sizeof(int));
    if (!rc) rc = qh_malloc((void **)&b->kv8.row, 2 * sizeof(int));
    if (rc) return rc;
    c->v = c->k + NL * b->kv8.codes;
    c->v_scale = c->k_scale + NL * b->kv8.scales;
    c->v_tail = c->k_tail + NL * b->kv8.tails;
    c->table = b->table;
    /* of a step of every sequence, and of a prompt's pass */
    b->kv8.work_bytes = qm_kv8_attention_work(c, QW3M_N_HEADS, b->n_seq, 1, b->max_ctx);
    const size_t pass = qm_kv8_attention_work(c, QW3M_N_HEADS, 1, b->max_ctx, b->max_ctx);
    if (pass > b->kv8.work_bytes) b->kv8.work_bytes = pass;
    rc = qh_malloc(&b->kv8.work, b->kv8.work_bytes);
    if (!rc) rc = qm_zero_i32(b->kv8.row, 2);
    if (!rc) rc = qm_kv8_own(b->table, NULL, b->n_seq, c->block, c->max_blocks);
    return rc;
}

/* format: QM_KV8_*, or -1 for fp32 caches */
static int batch_open(qwen3_hip_batch **out, qwen3_hip_model *m, int n_seq, int max_ctx, int format) {
    if (!out) return QWEN3_HIP_EINVAL;
    *out = NULL;
    if (!m || n_seq < 1 || n_seq > QM_MAX_CHUNK || max_ctx < 2 || max_ctx > m->max_seq) return QWEN3_HIP_EINVAL;
    qwen3_hip_batch *b = (qwen3_hip_batch *)calloc(1, sizeof *b);
    if (!b) return QWEN3_HIP_ENOMEM;
    b->m = m;
    b->n_seq = n_seq;
    b->max_ctx = max_ctx;
    b->out_ld = max_ctx + 1;
    b->kv_seq = (size_t)QW3M_N_KV_HEADS * max_ctx * QW3M_HEAD_DIM;
    b->use_graph = 1;
    b->graph_id[0] = b->graph_id[1] = b->graph_id[2] = -1;
    int rc = QWEN3_HIP_ENOMEM;
    b->h_next = (int *)malloc((size_t)n_seq * sizeof(int));
    b->h_plen = (int *)calloc((size_t)n_seq, sizeof(int));
    b->h_out = (int *)malloc((size_t)n_seq * b->out_ld * sizeof(int));
    b->h_text = (int *)malloc((size_t)n_seq * b->out_ld * sizeof(int));
    b->h_rules = (seq_rules_t *)calloc((size_t)n_seq, sizeof *b->h_rules);
    if (!b->h_next || !b->h_plen || !b->h_out || !b->h_text || !b->h_rules) goto fail;
    for (int s = 0; s < n_seq; s++) b->h_next[s] = -1;
#define DEV(ptr, bytes)                                                   \
    do {                                                                  \
        if ((rc = qh_malloc((void **)&(ptr), (bytes))) != 0) goto fail;   \
    } while (0)
    if (format >= 0) {
        if ((rc = open_kv8(b, format)) != 0) goto fail;
    } else {
        const size_t kv_bytes = (size_t)NL * n_seq * b->kv_seq * sizeof(float);
        DEV(b->kc, kv_bytes);
        DEV(b->vc, kv_bytes);
        DEV(b->part, (size_t)n_seq * QM_BATCH_PART_FLOATS * sizeof(float));
    }
    DEV(b->logits, (size_t)n_seq * V * sizeof(float));
    DEV(b->tok, (size_t)n_seq * sizeof(int));
    DEV(b->pos, (size_t)n_seq * sizeof(int));
    DEV(b->plen, (size_t)n_seq * sizeof(int));
    DEV(b->out, (size_t)n_seq * b->out_ld * sizeof(int));
#undef DEV
    rc = qm_zero_i32(b->tok, n_seq);
    if (!rc) rc = qm_zero_i32(b->pos, n_seq);
    if (!rc) rc = qm_zero_i32(b->plen, n_seq);
    if (!rc) rc = qh_sync();
    if (rc) goto fail;
    b->next = m->batches;
    m->batches = b;
    *out = b;
    return QWEN3_HIP_OK;
fail:
    qwen3_hip_batch_close(b);
    return rc;
}

int qwen3_hip_batch_open(qwen3_hip_batch **out, qwen3_hip_model *m, int n_seq, int max_ctx) {
    return batch_open(out, m, n_seq, max_ctx, -1);
}

int qwen3_hip_batch_open_kv8(qwen3_hip_batch **out, qwen3_hip_model *m, int n_seq, int max_ctx, int format) {
    if (out) *out = NULL;
    if (format != QM_KV8_E4M3 && format != QM_KV8_INT8) return QWEN3_HIP_EINVAL;
    return batch_open(out, m, n_seq, max_ctx, format);
}

int qwen3_hip_batch_set_graph(qwen3_hip_batch *b, int on) {
    if (!b) return QWEN3_HIP_EINVAL;
    if (!b->m) return QWEN3_HIP_ESTATE;
    b->use_graph = on ? 1 : 0;
    return QWEN3_HIP_OK;
}

/* a prompt into sequence seq's cache; its last row's logits in the model's
 * buffer */
static int batch_prompt(qwen3_hip_batch *b, int seq, const int *prompt, int n_prompt) {
    const int has8 = b->kv8.c.k != NULL;
    kv8_t k8 = b->kv8;
    if (has8) k8 = kv8_seq(&b->kv8, seq);
    const kv_t kv = {has8 ? NULL : b->kc + (size_t)seq * b->kv_seq, has8 ? NULL : b->vc + (size_t)seq * b->kv_seq,
                     (size_t)b->n_seq * b->kv_seq, b->max_ctx, has8 ? &k8 : NULL};
    b->m->have_logits = 0;             /* the model's logits buffer is reused */
    int nt = 0;
    return prefill(b->m, &kv, prompt, n_prompt, &nt);
}

/* the rules on the rows of logits of sequences seq .. */
static qm_rules_t rules_from(const qwen3_hip_batch *b, int seq) {
    const int n = b->n_seq;
    const qm_rules_t r = {b->text + (size_t)seq * b->out_ld, b->out_ld, b->plen + seq, b->n_text + seq, b->penalty + seq,
                          b->penalty + n + seq, b->penalty + 2 * n + seq, b->bias_row + seq, b->bias_token, b->bias,
                          b->bias_room, b->mask, MASK_WORDS, 2 * n, b->mask_of + seq};
    return r;
}

/* the texts of all sequences as they stand, from the prompts and what the steps
 * have put out: kept up by the steps from here on while there are rules.  n [n_seq]
 * is read until the stream is waited for */
static int rules_texts(qwen3_hip_batch *b, int *n) {
    const size_t all = (size_t)b->n_seq * b->out_ld;
    int rc = qh_d2h(b->h_out, b->out, all * sizeof(int));
    if (!rc) rc = qh_sync();
    for (int s = 0; s < b->n_seq && !rc; s++) {
        const size_t row = (size_t)s * b->out_ld;
        n[s] = b->h_next[s] < 0 ? 0 : b->h_next[s] + 1;       /* the token that is fed next is the last */
        for (int i = b->h_plen[s]; i < n[s]; i++) b->h_text[row + i] = b->h_out[row + i - b->h_plen[s]];
    }
    if (!rc) rc = qh_h2d(b->text, b->h_text, all * sizeof(int));
    if (!rc) rc = qh_h2d(b->n_text, n, (size_t)b->n_seq * sizeof(int));
    return rc;
}

/* device room for the rules, `biases` in all */
static int rules_room(qwen3_hip_batch *b, int biases) {
    const size_t n = (size_t)b->n_seq;
    int rc = QWEN3_HIP_OK;
    if (!b->text) rc = qh_malloc((void **)&b->text, n * b->out_ld * sizeof(int));
    if (!rc && !b->n_text) rc = qh_malloc((void **)&b->n_text, n * sizeof(int));
    if (!rc && !b->penalty) rc = qh_malloc((void **)&b->penalty, 3 * n * sizeof(float));
    if (!rc && !b->bias_row) rc = qh_malloc((void **)&b->bias_row, (n + 1) * sizeof(int));
    if (!rc && !b->mask_of) rc = qh_malloc((void **)&b->mask_of, n * sizeof(int));
    if (!rc && !b->mask) rc = qh_malloc((void **)&b->mask, 2 * n * MASK_WORDS * sizeof(uint32_t));
    if (rc || (b->bias_room && biases <= b->bias_room)) return rc;
    const int room = biases < 512 ? 1024 : 2 * biases;
    int *tok = NULL;
    float *val = NULL;
    rc = qh_malloc((void **)&tok, (size_t)room * sizeof(int));
    if (!rc) rc = qh_malloc((void **)&val, (size_t)room * sizeof(float));
    if (!rc) rc = qh_sync();           /* steps that read the old ones */
    if (rc) {
        (void)qh_free(tok);
        (void)qh_free(val);
        return rc;
    }
    if (b->graph_id[2] >= 0) (void)qh_graph_destroy(b->graph_id[2]);
    b->graph_id[2] = -1;
    b->torn = 1;                       /* the biases are in neither until they are uploaded */
    (void)qh_free(b->bias_token);
    (void)qh_free(b->bias);
    b->bias_token = tok;
    b->bias = val;
    b->bias_room = room;
    return rc;
}

/* penalties, biases and which sequences have masks, with `next` in the place of sequence
 * seq's rules.  stage: 5 n_seq + 1 + 2 biases words, read until the stream is waited for */
static int rules_upload(qwen3_hip_batch *b, int seq, const seq_rules_t *next, int biases, int *stage) {
    const int n = b->n_seq;
    float *pen = (float *)stage, *val = (float *)(stage + 5 * n + 1 + biases);
    int *of = stage + 3 * n, *row = of + n, *tok = row + n + 1;
    row[0] = 0;
    for (int s = 0; s < n; s++) {
        const seq_rules_t *r = s == seq ? next : &b->h_rules[s];
        pen[s] = r->on ? r->repetition : 1.0f;
        pen[n + s] = r->on ? r->presence : 0.0f;
        pen[2 * n + s] = r->on ? r->frequency : 0.0f;
        of[s] = r->on ? r->mask : -1;
        const int k = r->on ? r->n_bias : 0;
        if (k) {
            memcpy(tok + row[s], r->bias_token, (size_t)k * sizeof(int));
            memcpy(val + row[s], r->bias, (size_t)k * sizeof(float));
        }
        row[s + 1] = row[s] + k;
    }
    b->torn = 1;
    int rc = qh_h2d(b->penalty, pen, 3 * (size_t)n * sizeof(float));
    if (!rc) rc = qh_h2d(b->mask_of, of, (size_t)n * sizeof(int));
    if (!rc) rc = qh_h2d(b->bias_row, row, ((size_t)n + 1) * sizeof(int));
    if (!rc && biases) rc = qh_h2d(b->bias_token, tok, (size_t)biases * sizeof(int));
    if (!rc && biases) rc = qh_h2d(b->bias, val, (size_t)biases * sizeof(float));
    return rc;
}

int qwen3_hip_batch_set_rules(qwen3_hip_batch *b, int seq, const qwen3_hip_batch_rules *r) {
    if (!b || seq < 0 || seq >= b->n_seq) return QWEN3_HIP_EINVAL;
    if (!b->m) return QWEN3_HIP_ESTATE;
    seq_rules_t *now = &b->h_rules[seq];
    if (!r && !now->on && !(b->torn && b->n_rules)) return QWEN3_HIP_OK;
    if (r) {
        if (!(r->repetition > 0.0f) || !isfinite(r->repetition) || !isfinite(r->presence) || !isfinite(r->frequency))
            return QWEN3_HIP_EINVAL;
        if (r->n_bias < 0 || (r->n_bias && (!r->bias_token || !r->bias))) return QWEN3_HIP_EINVAL;
        if (r->n_bias > QWEN3_HIP_BATCH_MAX_BIAS) return QWEN3_HIP_ETOOBIG;
        for (int i = 0; i < r->n_bias; i++)
            if (r->bias_token[i] < 0 || r->bias_token[i] >= V || isnan(r->bias[i])) return QWEN3_HIP_EINVAL;
    }
    if (qh_capturing()) return QWEN3_HIP_ERUNTIME;   /* rules come from the host */

    const int n = b->n_seq;
    int biases = r ? r->n_bias : 0, rc = QWEN3_HIP_OK;
    for (int s = 0; s < n; s++)
        if (s != seq && b->h_rules[s].on) biases += b->h_rules[s].n_bias;
    seq_rules_t next = {0};
    int *stage = (int *)malloc((6 * (size_t)n + 1 + 2 * (size_t)biases) * sizeof(int));
    if (!stage) rc = QWEN3_HIP_ENOMEM;
    if (r) {
        const int place = now->on && now->mask == 2 * seq ? 2 * seq + 1 : 2 * seq;
        next = (seq_rules_t){1, r->mask ? place : -1, r->n_bias, r->repetition, r->presence, r->frequency, NULL, NULL};
        if (!rc && r->n_bias) {
            next.bias_token = (int *)malloc((size_t)r->n_bias * sizeof(int));
            next.bias = (float *)malloc((size_t)r->n_bias * sizeof(float));
            if (!next.bias_token || !next.bias) rc = QWEN3_HIP_ENOMEM;
            else {
                memcpy(next.bias_token, r->bias_token, (size_t)r->n_bias * sizeof(int));
                memcpy(next.bias, r->bias, (size_t)r->n_bias * sizeof(float));
            }
        }
        if (!rc) rc = rules_room(b, biases);
        if (!rc && b->n_rules == 0) rc = rules_texts(b, stage + 5 * n + 1 + 2 * biases);
        if (!rc && r->mask) rc = qh_h2d(b->mask + (size_t)place * MASK_WORDS, r->mask, MASK_WORDS * sizeof(uint32_t));
    }
    if (!rc) rc = rules_upload(b, seq, &next, biases, stage);
    if (stage) {
        const int rc2 = qh_sync();     /* copies read the staging and the caller's mask, whatever happened */
        if (!rc) rc = rc2;
    }
    free(stage);
    if (rc) {                          /* the rules stay as they were, torn or whole */
        free(next.bias_token);
        free(next.bias);
        return rc;
    }
    b->torn = 0;
    b->n_rules += next.on - now->on;
    free(now->bias_token);
    free(now->bias);
    *now = next;
    return rc;
}

int qwen3_hip_batch_set_int8_head(qwen3_hip_batch *b, int on) {
    if (!b) return QWEN3_HIP_EINVAL;
    if (!b->m) return QWEN3_HIP_ESTATE;
    on = on ? 1 : 0;
    if (on == b->head8) return QWEN3_HIP_OK;
    if (qh_capturing()) return QWEN3_HIP_ERUNTIME;   /* allocates, and drops graphs */
    qwen3_hip_model *m = b->m;
    if (on && !m->embed8) {
        int8_t *w = NULL;
        int rc = QWEN3_HIP_OK;
        if (!m->embed8_scale) rc = qh_malloc((void **)&m->embed8_scale, (size_t)V * sizeof(float));
        if (!rc && !m->row8) rc = qh_malloc((void **)&m->row8, (size_t)QM_MAX_CHUNK * H);
        if (!rc && !m->row8_scale) rc = qh_malloc((void **)&m->row8_scale, (size_t)QM_MAX_CHUNK * sizeof(float));
        if (!rc) rc = qh_malloc((void **)&w, (size_t)V * H);
        if (!rc) rc = qh_rows_int8(w, H, m->embed8_scale, m->embed, H, 1, V, H);
        if (!rc) rc = qh_sync();
        if (rc) {
            (void)qh_free(w);
            return rc;
        }
        m->embed8 = w;
    }
    const int rc = qh_sync();          /* steps of the graphs that go */
    if (rc) return rc;
    drop_graphs(b);
    b->head8 = on;
    return QWEN3_HIP_OK;
}

int qwen3_hip_batch_prefill(qwen3_hip_batch *b, int seq, const int *prompt, int n_prompt) {
    if (!b || !prompt || seq < 0 || seq >= b->n_seq || n_prompt < 1 || n_prompt >= b->max_ctx)
        return QWEN3_HIP_EINVAL;
    if (!b->m || (b->n_rules && b->torn)) return QWEN3_HIP_ESTATE;
    int rc = check_tokens(prompt, n_prompt);
    if (rc) return rc;
    qwen3_hip_model *m = b->m;
    b->h_next[seq] = -1;
    if ((rc = batch_prompt(b, seq, prompt, n_prompt)) != 0) return rc;
    /* first token: out[seq][0] at pos - plen + 1 = 0, then pos = n_prompt */
    rc = qm_set_i32(b->pos + seq, n_prompt - 1);
    if (!rc) rc = qm_set_i32(b->plen + seq, n_prompt);
    int *text = b->h_text + (size_t)seq * b->out_ld;
    memcpy(text, prompt, (size_t)n_prompt * sizeof(int));
    if (!rc && b->n_rules) rc = qh_h2d(b->text + (size_t)seq * b->out_ld, text, (size_t)n_prompt * sizeof(int));
    if (!rc && b->n_rules) rc = qm_set_i32(b->n_text + seq, n_prompt);
    if (!rc && b->h_rules[seq].on) {
        const qm_rules_t r = rules_from(b, seq);
        rc = qm_logits_rules(m->logits, V, m->logits, V, V, 1, &r);
    }
    if (!rc) rc = qm_argmax_rows(m->logits, V, 1, b->tok + seq, b->pos + seq, b->plen + seq,
                                 b->out + (size_t)seq * b->out_ld, b->out_ld);
    if (!rc && b->n_rules)
        rc = qm_rules_note(b->text + (size_t)seq * b->out_ld, b->out_ld, b->n_text + seq, b->tok + seq, b->pos + seq, 1);
    const int rc2 = qh_sync();         /* the text's copy reads h_text, whatever happened */
    if (!rc) rc = rc2;
    if (!rc) {
        b->h_next[seq] = n_prompt;
        b->h_plen[seq] = n_prompt;
    }
    return rc;
}

/* the logits of one decode step of every sequence: token tok[s] at position
 * pos[s], K and V appended.  When
 * the o and down projections split K (the skinny kernel up to 16 sequences,
 * the ring tiles above 64 and, for down, from 17), their
 * slice sums are added by the residual + RMSNorm kernel that consumes them
 * (the sums a reduction launch would form), one launch fewer each. */
static int batch_forward(qwen3_hip_batch *b) {
    qwen3_hip_model *m = b->m;
    const int n = b->n_seq;
    const float eps = QW3M_RMS_EPS;
    const size_t lstride = (size_t)n * b->kv_seq;
    int rc = QWEN3_HIP_OK;
    const float *dpart = NULL, *opart = NULL;
    int dks = 0, oks = 0;
    for (int l = 0; l < NL && !rc; l++) {
        const layer_t *L = &m->L[l];
        if (l == 0) rc = qm_rows_norm(m->x, NULL, m->embed, b->tok, V, L->in_norm, m->xb, n, H, eps);
        else rc = qm_rows_norm_split(m->x, dks ? NULL : m->dn, NULL, NULL, 0, L->in_norm, m->xb, n, H, eps, dpart, dks);
        if (!rc) rc = qh_gemm(m->qkv, m->xb, L->wqkv, n, H, QKV_N);
        if (!rc && b->kv8.c.k) rc = attend_kv8(m, &b->kv8, l, L, n, n, b->pos, b->max_ctx, 0);
        else if (!rc) rc = qm_attention_decode_batch(m->qkv, m->att, b->part, b->kc + l * lstride, b->vc + l * lstride,
                                                     b->kv_seq, L->qn, L->kn, m->rcos, m->rsin, b->pos, n,
                                                     b->max_ctx, eps);
        if (!rc) rc = qh_gemm_split(m->ob, m->att, L->wo, n, QW3M_Q_DIM, H, &opart, &oks);
        if (!rc) rc = qm_rows_norm_split(m->x, oks ? NULL : m->ob, NULL, NULL, 0, L->post_norm, m->xb, n, H, eps,
                                         opart, oks);
        if (!rc) rc = qh_gemm_gate_up_silu(m->hb, m->xb, L->wg, L->wu, n, H, QW3M_INTER);
        if (!rc) rc = qh_gemm_split(m->dn, m->hb, L->wd, n, QW3M_INTER, H, &dpart, &dks);
    }
    if (!rc) rc = qm_rows_norm_split(m->x, dks ? NULL : m->dn, NULL, NULL, 0, m->final_norm, m->xb, n, H, eps,
                                     dpart, dks);
    if (!b->head8) return rc ? rc : qh_gemm(b->logits, m->xb, m->embed, n, H, V);
    if (!rc) rc = qh_rows_int8(m->row8, H, m->row8_scale, m->xb, H, 0, n, H);
    if (!rc) rc = qh_gemm_int8(b->logits, V, 0, m->row8, H, m->row8_scale, m->embed8, H, m->embed8_scale, n, H, V);
    return rc;
}

/* the forward and the greedy choice of every sequence's next token, without
 * rules (0) or under them (2), or the forward alone (1) */
static int batch_step(qwen3_hip_batch *b, int which) {
    int rc = batch_forward(b);
    if (!rc && which == 2) {
        const qm_rules_t r = rules_from(b, 0);
        rc = qm_logits_rules(b->logits, V, b->logits, V, V, b->n_seq, &r);
    }
    if (!rc && which != 1) rc = qm_argmax_rows(b->logits, V, b->n_seq, b->tok, b->pos, b->plen, b->out, b->out_ld);
    if (!rc && which == 2) rc = qm_rules_note(b->text, b->out_ld, b->n_text, b->tok, b->pos, b->n_seq);
    return rc;
}

/* step i of a call: with graphs on, a first step runs eagerly (any workspace
 * its GEMM plans need is allocated then, outside capture); later steps replay
 * the one captured step.  Steps under rules are called for one by one where a
 * mask follows each: their first call's stays the only eager one */
static int batch_run(qwen3_hip_batch *b, int i, int which) {
    int *id = &b->graph_id[which];
    if (!b->use_graph || (*id < 0 && i == 0 && !(which == 2 && b->ruled))) {
        if (which == 2) b->ruled = 1;
        return batch_step(b, which);
    }
    if (*id < 0) {
        int rc = qh_capture_begin();
        if (rc) return rc;
        const int rc2 = batch_step(b, which);
        int gid = -1;
        rc = qh_capture_end(&gid);
        if (!rc) rc = rc2;
        if (rc) {
            if (gid >= 0) (void)qh_graph_destroy(gid);
            return rc;
        }
        *id = gid;
    }
    return qh_graph_launch(*id);
}

int qwen3_hip_batch_decode(qwen3_hip_batch *b, int n_decode, int *out) {
    if (!b || !out || n_decode < 0) return QWEN3_HIP_EINVAL;
    if (!b->m || (b->n_rules && b->torn)) return QWEN3_HIP_ESTATE;
    for (int s = 0; s < b->n_seq; s++)
        if (b->h_next[s] < 0 || (long)b->h_next[s] + n_decode > b->max_ctx) return QWEN3_HIP_EINVAL;
    int rc = QWEN3_HIP_OK;
    const double t0 = now_ms();
    for (int i = 0; i < n_decode && !rc; i++) rc = batch_run(b, i, b->n_rules ? 2 : 0);
    if (!rc) rc = qh_sync();
    b->t_decode_ms = now_ms() - t0;
    if (rc) return rc;
    if (n_decode > 0) b->have_logits = 1;
    rc = qh_d2h(b->h_out, b->out, (size_t)b->n_seq * b->out_ld * sizeof(int));
    if (!rc) rc = qh_sync();
    if (rc) return rc;
    for (int s = 0; s < b->n_seq; s++) {
        /* the token fed at position h_next sits at out index h_next - plen */
        const int *row = b->h_out + (size_t)s * b->out_ld + (b->h_next[s] - b->h_plen[s]);
        memcpy(out + (size_t)s * (n_decode + 1), row, ((size_t)n_decode + 1) * sizeof(int));
        b->h_next[s] += n_decode;
    }
    return QWEN3_HIP_OK;
}

/* ---- beam search ------------------------------------------------------------ */

static int beam_buffers(qwen3_hip_batch *b, int width) {
    const size_t n = (size_t)b->n_seq;
    const size_t need = qm_beam_select_work(V, b->n_seq / width, width);
    int rc = QWEN3_HIP_OK;
    if (!b->score) rc = qh_malloc((void **)&b->score, n * sizeof(float));
    if (!rc && !b->done) rc = qh_malloc((void **)&b->done, n * sizeof(int));
    if (!rc && !b->parent) rc = qh_malloc((void **)&b->parent, n * sizeof(int));
    if (!rc && !b->hist) rc = qh_malloc((void **)&b->hist, 2 * n * b->max_ctx * sizeof(int));
    if (!rc && need > b->swork_bytes) {
        rc = qh_sync();
        if (!rc) rc = qh_free(b->swork);
        b->swork = NULL;
        b->swork_bytes = 0;
        if (!rc) rc = qh_malloc(&b->swork, need);
        if (!rc) b->swork_bytes = need;
    }
    return rc;
}

/* every sequence's state after its parent's, `rows` positions of the longest:
 * fp32 caches move; of 8-bit ones the tables and the unfinished blocks do,
 * finished blocks are shared, and a sequence's next ones are its own again */
static int beam_states(qwen3_hip_batch *b, int width, int rows) {
    const int n = b->n_seq, g = n / width;
    if (b->kv8.c.k) {
        const qm_kv8_t *c = &b->kv8.c;
        const size_t tail = (size_t)c->heads * c->block * c->head_dim * sizeof(uint16_t);
        const size_t line = (size_t)c->max_blocks * sizeof(int);
        int rc = qm_beam_reorder(c->k_tail, c->k_tail, b->parent, g, width, 2 * NL, n * tail, tail, 1, tail, tail);
        if (!rc) rc = qm_beam_reorder(b->table, b->table, b->parent, g, width, 1, n * line, line, 1, line, line);
        if (!rc) rc = qm_kv8_own(b->table, b->pos, n, c->block, c->max_blocks);
        return rc;
    }
    const size_t seq = b->kv_seq * sizeof(float), ctx = (size_t)b->max_ctx;
    int rc = qm_beam_reorder(b->kc, b->kc, b->parent, g, width, NL, n * seq, seq, QW3M_KV_DIM / 4, ctx * 16,
                             (size_t)rows * 16);
    if (!rc) rc = qm_beam_reorder(b->vc, b->vc, b->parent, g, width, NL, n * seq, seq, QW3M_N_KV_HEADS,
                                  ctx * QW3M_HEAD_DIM * 4, (size_t)rows * QW3M_HEAD_DIM * 4);
    return rc;
}

int qwen3_hip_batch_beam(qwen3_hip_batch *b, int width, const int *prompts, const int *n_prompt, int n_tokens,
                         int stop_at_eos, int *out, float *scores) {
    if (!b || !prompts || !n_prompt || !out || !scores || n_tokens < 1) return QWEN3_HIP_EINVAL;
    if (!b->m) return QWEN3_HIP_ESTATE;
    if (width < 1 || width > QM_BEAM_MAX_WIDTH || b->n_seq % width) return QWEN3_HIP_EINVAL;
    if (b->n_rules) return QWEN3_HIP_ESTATE;
    const int n = b->n_seq, groups = n / width;
    int longest = 0, rc = QWEN3_HIP_OK;
    size_t total = 0;
    for (int g = 0; g < groups; g++) {
        if (n_prompt[g] < 1 || n_prompt[g] >= b->max_ctx || (long)n_prompt[g] + n_tokens - 1 > b->max_ctx)
            return QWEN3_HIP_EINVAL;
        if (n_prompt[g] > longest) longest = n_prompt[g];
        if ((rc = check_tokens(prompts + total, n_prompt[g])) != 0) return rc;
        total += (size_t)n_prompt[g];
    }
    if (qh_capturing()) return QWEN3_HIP_ERUNTIME;   /* prompts come from the host */
    if ((rc = beam_buffers(b, width)) != 0) return rc;
    int *hist = (int *)malloc((size_t)n_tokens * n * 2 * sizeof(int));
    if (!hist) return QWEN3_HIP_ENOMEM;

    const double t0 = now_ms();
    double t1 = t0;
    for (int s = 0; s < n; s++) b->h_next[s] = -1;   /* whatever happens, the sequences are the search's now */
    b->have_logits = 0;
    const int *p = prompts;
    for (int g = 0; g < groups && !rc; p += n_prompt[g++]) {
        rc = batch_prompt(b, g * width, p, n_prompt[g]);
        if (!rc) rc = qh_d2d(b->logits + (size_t)g * width * V, b->m->logits, (size_t)V * sizeof(float));
        for (int w = 0; w < width && !rc; w++) rc = qm_set_i32(b->pos + g * width + w, n_prompt[g]);
    }
    if (!rc) rc = qm_beam_start(b->score, b->done, n, width);
    if (!rc) rc = qh_sync();
    t1 = now_ms();
    for (int t = 0; t < n_tokens && !rc; t++) {
        rc = qm_beam_select(b->logits, V, V, groups, width, b->score, stop_at_eos ? b->done : NULL,
                            stop_at_eos ? QW3M_EOS0 : -1, stop_at_eos ? QW3M_EOS1 : -1, b->score, b->done, b->tok, b->parent,
                            b->swork, b->swork_bytes);
        if (!rc) rc = qm_beam_record(b->hist, b->tok, b->parent, b->pos, n, t, t > 0);
        if (rc || t + 1 == n_tokens) break;
        rc = beam_states(b, width, longest + t);
        if (!rc) rc = batch_run(b, t, 1);
    }
    if (!rc) rc = qh_sync();
    else (void)qh_sync();              /* steps already launched */
    b->t_decode_ms = now_ms() - t1;
    if (b->kv8.c.k) {                  /* every sequence has its own pages again */
        const int rc2 = qm_kv8_own(b->table, NULL, n, b->kv8.c.block, b->kv8.c.max_blocks);
        if (!rc) rc = rc2;
    }
    if (!rc) rc = qh_d2h(hist, b->hist, (size_t)n_tokens * n * 2 * sizeof(int));
    if (!rc) rc = qh_d2h(scores, b->score, (size_t)n * sizeof(float));
    const int rc3 = qh_sync();         /* copies write hist and the caller's scores, whatever happened */
    if (!rc) rc = rc3;
    for (int s = 0; s < n && !rc; s++)
        for (int t = n_tokens - 1, at = s; t >= 0; t--) {
            const int *h = hist + ((size_t)t * n + at) * 2;
            out[(size_t)s * n_tokens + t] = h[0];
            at = s / width * width + h[1];
        }
    free(hist);
    return rc;
}

int qwen3_hip_batch_logits(qwen3_hip_batch *b, float *out) {
    if (!b || !out || !b->have_logits) return QWEN3_HIP_EINVAL;
    if (!b->m) return QWEN3_HIP_ESTATE;
    int rc = qh_d2h(out, b->logits, (size_t)b->n_seq * V * sizeof(float));
    if (!rc) rc = qh_sync();
    return rc;
}

int qwen3_hip_batch_timing(const qwen3_hip_batch *b, double *decode_ms) {
    if (!b) return QWEN3_HIP_EINVAL;
    if (decode_ms) *decode_ms = b->t_decode_ms;
    return QWEN3_HIP_OK;
}
