/* MI355X (gfx950) operators of a serving program — public C ABI of
 * libqwen3_hip (same library as qwen3_hip.h): a KV cache held in 8 bits with
 * the attention that reads it, and beam search.  No counterpart in the
 * reference, whose cache is fp32 and whose only search is the argmax
 * (fpga_bringup/src/src/qwen3.h:62-76, ops_scalar.c:57-62).
 *
 * Device-pointer entry points, as the _dev calls of qwen3_hip.h: pointers
 * ending in _d are device memory, calls are asynchronous on the library
 * stream, return a QWEN3_HIP_* code, never abort, allocate nothing, and may be
 * captured into a graph.  Structures are read before the call returns.  What
 * lies in device memory (positions, rows, tables, parents) cannot be checked
 * on the host: the kernels leave out entries that do not fit, as said below,
 * and never read or write outside the buffers described.
 */
#ifndef QWEN3_HIP_SERVE_H
#define QWEN3_HIP_SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 8-bit KV cache --------------------------------------------------------
 *
 * One layer's cache of n_seq sequences.  Tokens lie in blocks of `block` (16,
 * 32 or 64).  The unfinished block of a sequence, its newest position % block
 * rows, is held as bf16 (the tail).  When its last row arrives the block is
 * stored in a page: per kv head, with x the bf16 rows,
 *   a = max |x| over the block, s = a / 448 (e4m3) or a / 127 (int8) as fp32,
 *   code = x / s (fp32) rounded to the nearest value, ties to even
 * and read back as s * code.  s = 0 and codes of 0 where a < 2^-100.  A page
 * is written once and never changed: sequences may share pages.
 * What a cache holds is finite: a NaN is stored as 0 and magnitudes beyond
 * bf16's range as its largest value. */
#define QWEN3_HIP_KV8_E4M3 0
#define QWEN3_HIP_KV8_INT8 1
typedef struct {
    int format;          /* QWEN3_HIP_KV8_* */
    int kv_heads;        /* 1 .. 256 */
    int head_dim;        /* 64 or 128 */
    int block;           /* 16, 32 or 64 */
    int n_page;          /* pages of the pool */
    int n_seq;           /* sequences: rows of table and tails */
    int max_blocks;      /* columns of table; max_blocks * block <= 2^20 positions */
    uint8_t *k;          /* [n_page][kv_heads][block][head_dim] codes */
    uint8_t *v;          /* [n_page][kv_heads][head_dim][block] codes */
    float *k_scale;      /* [n_page][kv_heads] */
    float *v_scale;      /* [n_page][kv_heads] */
    uint16_t *k_tail;    /* [n_seq][kv_heads][block][head_dim] bf16 */
    uint16_t *v_tail;    /* [n_seq][kv_heads][head_dim][block] bf16 */
    const int *table;    /* [n_seq][max_blocks]: the page of each block */
} qwen3_hip_kv8;         /* k, v and the tails 16-byte aligned */

/* Bytes of the arrays of such a cache, in the order k + v, k_scale + v_scale,
 * k_tail + v_tail, table summed: what a sequence's positions cost in memory.
 * 0 for a description that the calls would refuse for its sizes. */
size_t qwen3_hip_kv8_bytes(const qwen3_hip_kv8 *cache);

/* New rows of n sequences into the cache: entry i is sequence i, its rows are
 * rows row_d[i] .. row_d[i+1] - 1 of k_d and v_d (row_d: n + 1 ints; NULL: one
 * row each, row i) and go to positions pos_d[i], pos_d[i] + 1, ...; whatever
 * was appended before must end at pos_d[i].  Rows are fp32, or bf16 where bf16
 * is set, [kv_heads][head_dim] at a stride of ldk / ldv values (a multiple of
 * 16 bytes; 16-byte aligned pointers).  `rows`: rows of k_d and v_d;
 * max_rows: the most rows of an entry.
 * Where two entries' tables name the same page for a block that this call
 * finishes, the page holds either's rows or a mix.
 * An entry whose rows do not lie in 0 .. rows, exceed max_rows or max_blocks
 * blocks, or whose pos_d is negative is left out (a negative pos_d leaves a
 * sequence out on purpose); a finished block whose table entry is no page is
 * not stored.  Tail rows behind the newest one keep what they held. */
int qwen3_hip_kv8_append_dev(const qwen3_hip_kv8 *cache, const void *k_d, const void *v_d, size_t ldk, size_t ldv,
                             int bf16, const int *row_d, const int *pos_d, int n, int rows, int max_rows);

/* Causal attention of the same rows: row r of entry i, at position
 * pos_d[i] + r, over positions 0 .. pos_d[i] + r of the cache, to which the
 * entry's rows have been appended (qwen3_hip_kv8_append_dev with the same
 * row_d and pos_d):
 *   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j),  scale > 0
 * (p_j up to 1, as the largest is divided out; sums of p_j v_j, which precede the
 * division, have to stay within fp32's range)
 * q_d and out_d: [q_heads][head_dim] per row, both fp32 or, where bf16 is set,
 * both bf16; query head h reads kv head h / (q_heads / kv_heads), at most 64
 * query heads a kv head.  fp32 rows are computed with fp32 accuracy
 * throughout; bf16 rows with weights of 16 bits: results are off by their own
 * rounding to bf16 and by little else (about one in 400 is a neighbour of the
 * value that rounding alone would give).  Strides and alignment as above.  A row
 * that is left out keeps what out_d held; a page that is no page of the pool is
 * left out of the sums, and a row with nothing left is 0.
 * max_ctx: a bound on pos_d[i] + rows of i, which picks the launch (a longer
 * entry is right too).  work_d: qwen3_hip_kv8_attention_work() bytes for the
 * same sizes or larger ones (4.4 MB at most; it never shrinks as n, max_rows or
 * max_ctx grow), 16-byte aligned, written by the call; QWEN3_HIP_ETOOBIG where
 * work_bytes is less.  Calls that share it have to run one after the other, as
 * calls on the library stream do.  out_d must not overlap what the call reads. */
size_t qwen3_hip_kv8_attention_work(const qwen3_hip_kv8 *cache, int q_heads, int n, int max_rows, int max_ctx);
int qwen3_hip_kv8_attention_dev(const qwen3_hip_kv8 *cache, void *out_d, const void *q_d, size_t ldo, size_t ldq,
                                int bf16, int q_heads, const int *row_d, const int *pos_d, int n, int rows,
                                int max_rows, int max_ctx, float scale, void *work_d, size_t work_bytes);

/* ---- beam search ------------------------------------------------------------
 *
 * n_group groups of `width` (1 .. 16) beams; beam w of group g is row
 * g * width + w of every array. */

/* The best `width` continuations of each group.  Beam w continues with token v
 * at score_d[w] + logits[w][v] - log sum_u exp(logits[w][u]); a finished beam
 * (done_d[w] != 0; done_d NULL: none) only with the token end0, at score_d[w].
 * Output row k of a group is its k-th best: its score, token, the beam it
 * continues (parent, 0 .. width - 1) and whether it is finished (its parent
 * was, or its token is end0 or end1; -1: no such token, which end0 may be only
 * where done_d is NULL).  Of one beam the tokens with the largest logits are
 * taken, ties to the lowest; those of all beams are compared by their scores in
 * 64 bits, equal ones in the order of beam and token.  A row's log sum is formed
 * from fp32 exponentials and fp32 sums of 2,048 of them and is off by 2^-18 at
 * most, so continuations of two beams whose scores are closer than 2^-17 may
 * come in either order; score_out_d is the score rounded to fp32.  Where fewer
 * than `width` continuations have a score, the others are taken in the same
 * order, as -inf: those of beams not in use (a score_d that is not finite; -inf
 * before the first token for all beams but the first), of tokens whose logit is
 * -inf or NaN, and of rows with an infinite logit, which have no probabilities.
 * logits_d: fp32 [n_group * width][ld >= vocab]; vocab in width .. 2^21.
 * score_out_d may be score_d and done_out_d done_d.  work_d:
 * qwen3_hip_beam_select_work() bytes, 8-byte aligned. */
size_t qwen3_hip_beam_select_work(int vocab, int n_group, int width);
int qwen3_hip_beam_select_dev(const float *logits_d, size_t ld, int vocab, int n_group, int width, const float *score_d,
                              const int *done_d, int end0, int end1, float *score_out_d, int *done_out_d,
                              int *token_out_d, int *parent_out_d, void *work_d, size_t work_bytes);

/* Rows of the beams' states after their parents: row w of each group of dst_d
 * receives row parent_d[w] (0 .. width - 1; a row with any other parent is left
 * as it is) of the same group of src_d.  dst_d may be src_d; otherwise the two
 * must not overlap.  A state is `slabs` arrays (layers, say), slab_stride bytes
 * apart, of n_group * width rows, seq_stride bytes apart; a row is `runs`
 * stretches of run_bytes used bytes, run_stride apart (a cache [head][position]
 * of which few positions are used).  Everything a multiple of 4 bytes; 16 is
 * faster.  An 8-bit cache is reordered by its table and its tails alone. */
int qwen3_hip_beam_reorder_dev(void *dst_d, const void *src_d, const int *parent_d, int n_group, int width, int slabs,
                               size_t slab_stride, size_t seq_stride, int runs, size_t run_stride, size_t run_bytes);

#ifdef __cplusplus
}
#endif
#endif
