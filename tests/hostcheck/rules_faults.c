/* A batch's host code while the device or memory refuses: every allocation, copy,
 * launch and wait of a call fails in turn.  model_hip.c itself, with its mallocs
 * counted, over a stand-in whose copies happen when the stream is waited for: the
 * test generates a stub for each launch (rules_faults_stubs.c).
 *
 * After a call that failed: no copy may be on its way to or from the host, no
 * block may have been freed under one, and every sequence must be under the rules
 * it had, or the batch must refuse decodes and prefills until a call succeeds. */
#define _POSIX_C_SOURCE 200809L
#include "qwen3_hip.h"
#include "qwen3_hip_model.h"
#include "hip_shim.h"
#include "model_shim.h"
#include "qw3m.h"
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <time.h>

static long g_ops, g_fail = -1;                       /* the operation that fails */
int fault_op(void) { return g_ops++ == g_fail; }

#define MOST 64
static struct { char *dst; const char *src; size_t n; int to_host; } g_copy[MOST];
static int g_copies, g_bad;
static int g_only_copies;                             /* the first argument: "copies" or "rules" */
static const char *g_doing = "";
static void found(long k, const char *what) {
    printf("%s, operation %ld: %s\n", g_doing, k, what);
    g_bad++;
}
static void bad_copy(const char *what) { found(g_fail, what); }
static void bad(long k, const char *what) {
    if (!g_only_copies) found(k, what);
}
static int touches(int i, const char *p, size_t n) {
    const char *h = g_copy[i].to_host ? g_copy[i].dst : g_copy[i].src;
    return h < p + n && p < h + g_copy[i].n;
}
/* host blocks carry their size */
static long g_blocks;
static void *fault_malloc(size_t n) {
    if (fault_op()) return NULL;
    size_t *p = (size_t *)malloc(n + 16);
    if (!p) abort();
    *p = n;
    memset(p + 2, 0xA7, n);
    g_blocks++;
    return p + 2;
}
static void *fault_calloc(size_t a, size_t b) {
    void *p = fault_malloc(a * b);
    return p ? memset(p, 0, a * b) : p;
}
static void fault_free(void *q) {
    if (!q) return;
    size_t *p = (size_t *)q - 2;
    for (int i = 0; i < g_copies; i++)
        if (touches(i, (const char *)q, *p)) {
            bad_copy("a block is freed under a copy");
            g_copy[i].n = 0;
        }
    g_blocks--;
    free(p);
}
static int copy(void *dst, const void *src, size_t n, int to_host) {
    if (fault_op()) return 5;
    if (g_copies == MOST) abort();
    g_copy[g_copies].dst = (char *)dst;
    g_copy[g_copies].src = (const char *)src;
    g_copy[g_copies].n = n;
    g_copy[g_copies++].to_host = to_host;
    return 0;
}
int qh_h2d(void *d, const void *s, size_t n) { return copy(d, s, n, 0); }
int qh_d2h(void *d, const void *s, size_t n) { return copy(d, s, n, 1); }
int qh_sync(void) {                                   /* a wait that reports an error has waited all the same */
    for (int i = 0; i < g_copies; i++) memcpy(g_copy[i].dst, g_copy[i].src, g_copy[i].n);
    g_copies = 0;
    return fault_op() ? 5 : 0;
}
static long g_dev;
int qh_malloc(void **p, size_t n) {
    *p = NULL;
    if (fault_op()) return 2;
    /* of what is large nothing is copied */
    if (n > 1 << 20) n = 1 << 20;
    *p = malloc(n ? n : 1);
    memset(*p, 0xCD, n);
    g_dev++;
    return 0;
}
int qh_free(void *p) {
    if (p) g_dev--;
    free(p);
    return 0;
}
int qh_capturing(void) { return 0; }
int qm_beam_record(int *hist, const int *token, const int *parent, int *pos, int n, int t, int advance) {
    memset(hist + (size_t)2 * t * n, 0, (size_t)2 * n * sizeof(int));
    return fault_op() ? 5 : 0;
}
int qw3m_parse(const void *blob, size_t size, qw3m_info_t *info) {
    if (info) memset(info, 0, sizeof *info);
    return fault_op() ? 5 : 0;
}
void qw3m_tensor_shape(int t, int *rows, int *cols, int *mat) {
    *rows = *cols = 0;
    *mat = 0;
}
size_t qm_beam_select_work(int v, int g, int w) { (void)v; (void)g; (void)w; return 64; }
size_t qm_kv8_attention_work(const qm_kv8_t *c, int h, int n, int r, int x) { (void)c; (void)h; (void)n; (void)r; (void)x; return 64; }

#define malloc fault_malloc
#define calloc fault_calloc
#define free fault_free
#include "model_hip.c"
#undef malloc
#undef calloc
#undef free

#define N 3
#define CTX 300
static uint32_t masks[4][MASK_WORDS];
static int tokens[700];
static float values[700];
static const qwen3_hip_batch_rules SOME[] = {
    {1.5f, 0.25f, 0.5f, 2, tokens, values, masks[0]},
    {2.0f, 0.5f, 0.125f, 5, tokens + 2, values + 2, masks[1]},
    {1.0f, 0.0f, 0.0f, 0, NULL, NULL, masks[2]},
    {3.0f, 1.0f, 0.0f, 600, tokens, values, NULL},    /* more than the first room */
    {1.0f, 2.0f, 0.0f, 1, tokens + 9, values + 9, NULL},
};

static int under(const qwen3_hip_batch *b, const qwen3_hip_batch_rules *const *rules) {
    const qm_rules_t t = rules_from(b, 0);
    int on = 0;
    for (int s = 0; s < N; s++) on += rules[s] != NULL;
    if (b->n_rules != on) return 0;
    for (int s = 0; s < N && on; s++) {
        const qwen3_hip_batch_rules *r = rules[s];
        if (t.repetition[s] != (r ? r->repetition : 1.0f) || t.presence[s] != (r ? r->presence : 0.0f) ||
            t.frequency[s] != (r ? r->frequency : 0.0f))
            return 0;
        const int n = r ? r->n_bias : 0, at = t.bias_row[s];
        if (at < 0 || t.bias_row[s + 1] - at != n || at + n > t.n_bias) return 0;
        for (int i = 0; i < n; i++)
            if (t.bias_token[at + i] != r->bias_token[i] || t.bias[at + i] != r->bias[i]) return 0;
        const int m = t.mask_of[s];
        if ((m >= 0 && m < t.n_mask) != (r && r->mask)) return 0;
        if (r && r->mask && memcmp(t.mask + (size_t)m * t.ld_mask, r->mask, MASK_WORDS * sizeof(uint32_t))) return 0;
        /* the text: the prompt, and what the steps put out, the token that is fed next the last */
        if (t.n_token[s] != 4) return 0;
        for (int i = 0; i < 4; i++)
            if (t.token[s * t.ld_token + i] != (i < 3 ? 10 * s + i : 100 + s)) return 0;
    }
    return 1;
}

static qwen3_hip_batch *opened(qwen3_hip_model *m) {
    qwen3_hip_batch *b = NULL;
    if (qwen3_hip_batch_open(&b, m, N, CTX)) abort();
    qwen3_hip_batch_set_graph(b, 0);
    for (int s = 0; s < N; s++) {
        const int p[] = {10 * s, 10 * s + 1, 10 * s + 2};
        if (qwen3_hip_batch_prefill(b, s, p, 3)) abort();
        b->out[s * b->out_ld] = 100 + s;
    }
    return b;
}

/* the end of a call that may have failed */
static void returned(void) {
    if (g_copies) bad_copy("a copy is on its way when the call returns");
    g_fail = -1;
    (void)qh_sync();
}

/* rules for `seq` of a batch under `before`, each operation failing in turn, then the same call once more */
static void faulty_rules(qwen3_hip_model *m, const char *name, const qwen3_hip_batch_rules *const *before, int seq, int which) {
    static uint32_t mask[MASK_WORDS];
    g_doing = name;
    for (long k = 0;; k++) {
        g_fail = -1;
        qwen3_hip_batch *b = opened(m);
        for (int s = 0; s < N; s++)
            if (before[s] && qwen3_hip_batch_set_rules(b, s, before[s])) abort();
        if (!under(b, before)) { found(k, "the start is not under its rules"); return; }
        const qwen3_hip_batch_rules *after[N] = {before[0], before[1], before[2]};
        after[seq] = which < 0 ? NULL : &SOME[which];
        /* the caller's memory is its own again when the call returns */
        qwen3_hip_batch_rules r = which < 0 ? SOME[0] : SOME[which];
        if (r.mask) r.mask = (uint32_t *)memcpy(mask, r.mask, sizeof mask);
        g_ops = 0;
        g_fail = k;
        const int rc = qwen3_hip_batch_set_rules(b, seq, which < 0 ? NULL : &r);
        const long used = g_ops;
        returned();
        memset(mask, 0x11, sizeof mask);
        int out[N];
        const int p[] = {1};
        if (rc) {
            if (qwen3_hip_batch_decode(b, 0, out) != QWEN3_HIP_ESTATE) {
                if (!under(b, before)) bad(k, "the rules are not those of before, and steps are taken");
            } else if (qwen3_hip_batch_prefill(b, 0, p, 1) != QWEN3_HIP_ESTATE) {
                bad(k, "a prompt is taken where steps are refused");
            }
            if (qwen3_hip_batch_set_rules(b, seq, which < 0 ? NULL : &SOME[which])) bad(k, "the call does not succeed afterwards");
        }
        if (!under(b, after) || qwen3_hip_batch_decode(b, 0, out)) bad(k, "the new rules are not there");
        qwen3_hip_batch_close(b);
        if (!rc && k >= used) break;
        if (!rc) bad(k, "a failure is not reported");
    }
    printf("%s done\n", name);
}

static void faulty_open(void) {
    static uint16_t blob[16];
    g_doing = "a model is opened";
    for (long k = 0;; k++) {
        qwen3_hip_model *m = NULL;
        g_ops = 0;
        g_fail = k;
        const int rc = qwen3_hip_model_open(&m, blob, sizeof blob, CTX);
        const long used = g_ops;
        returned();
        qwen3_hip_model_close(m);
        if (!rc && k >= used) break;
        if (k > 5000) { found(k, "no end"); return; }
    }
    printf("%s done\n", g_doing);
}

/* another call on a batch under rules, each operation failing in turn */
static void faulty_call(qwen3_hip_model *m, const char *name, int which) {
    g_doing = name;
    for (long k = 0;; k++) {
        g_fail = -1;
        qwen3_hip_batch *b = opened(m);
        if (which != 2 && qwen3_hip_batch_set_rules(b, 1, &SOME[0])) abort();
        int out[N * 4], n_prompt[N] = {2, 2, 2}, prompts[200] = {1, 2, 3, 4, 5, 6};
        float score[N];
        g_ops = 0;
        g_fail = k;
        int rc;
        if (which == 0) rc = qwen3_hip_batch_prefill(b, 1, prompts, 5);
        else if (which == 1) rc = qwen3_hip_batch_decode(b, 2, out);
        else if (which == 2) rc = qwen3_hip_batch_beam(b, 1, prompts, n_prompt, 4, 0, out, score);
        else if (which == 3) rc = qwen3_hip_batch_set_int8_head(b, 1);
        else rc = qwen3_hip_batch_prefill(b, 1, prompts, 200);
        const long used = g_ops;
        returned();
        qwen3_hip_batch_close(b);
        if (which == 3) {
            (void)qh_free(m->embed8); (void)qh_free(m->row8); (void)qh_free(m->embed8_scale); (void)qh_free(m->row8_scale);
            m->embed8 = m->row8 = NULL;
            m->embed8_scale = m->row8_scale = NULL;
        }
        if (!rc && k >= used) break;
        if (k > 5000) { found(k, "no end"); return; }
    }
    printf("%s done\n", name);
}

int main(int argc, char **argv) {
    g_only_copies = argc > 1 && !strcmp(argv[1], "copies");
    qwen3_hip_model *m = (qwen3_hip_model *)calloc(1, sizeof *m);
    m->max_seq = CTX;
    m->logits = (float *)malloc(4);
    m->tok_in = (int *)malloc(CTX * sizeof(int));
    for (int i = 0; i < 700; i++) { tokens[i] = 3 * i; values[i] = i / 4.0f; }
    for (int k = 0; k < 4; k++)
        for (int i = 0; i < MASK_WORDS; i++) masks[k][i] = (i + 1) * (k + 3) * 2654435761u;
    const qwen3_hip_batch_rules *none[N] = {0}, *one[N] = {&SOME[0]}, *two[N] = {&SOME[0], &SOME[4], &SOME[2]};
    faulty_rules(m, "the first rules", none, 0, 0);
    faulty_rules(m, "first rules of many biases", none, 2, 3);
    faulty_rules(m, "other rules", one, 0, 1);
    faulty_rules(m, "rules of another sequence", one, 2, 2);
    faulty_rules(m, "more biases than there is room for", two, 1, 3);
    faulty_rules(m, "another mask", two, 2, 1);
    faulty_rules(m, "no mask", two, 0, 4);
    faulty_rules(m, "rules are taken away", two, 1, -1);
    faulty_rules(m, "the last rules are taken away", one, 0, -1);
    faulty_call(m, "a prompt", 0);
    faulty_call(m, "steps", 1);
    faulty_call(m, "a search", 2);
    faulty_call(m, "8-bit head", 3);
    faulty_call(m, "a prompt from the caller's memory", 4);
    faulty_open();
    if (g_blocks) found(-1, "host blocks are left");
    printf("%d faults found\n", g_bad);
    return g_bad != 0;
}
