/* Attention between the trunk's q, k, v linears and its o linear on MI355X: a paged key-value cache that quantises what
 * it is given, attention of new tokens over it, and attention over packed prompts.
 *
 * Entry points of their own header, as ijah_exl3.h (reference include/engine.h:11-12); errors, buffers, streams and
 * gpu_ms as there. No reference counterpart: the reference's attention is a sparse one over its own cache
 * (kernels/fn_attn.metal); this is the dense one.
 *
 * Rows: a matrix of rows is [R][heads][dim] with ld elements from one row to the next (0: heads * dim), of NE_F32, NE_BF16
 * or NE_F16; each row starts on a 16-byte boundary of its buffer (offset and ld in bytes are multiples of 16).
 * dim is 64, 128 or 256. Nothing is written behind the rows that the calls name.
 */
#ifndef IJAH_ATTN_H
#define IJAH_ATTN_H
#include "engine.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the paged cache ----
 * One handle holds the keys and values of `layers` layers in pages of NE_KV_PAGE tokens; a page id is the same page number
 * in every layer. dtype: NE_BF16 or NE_F16 (rows rounded to nearest even) or NE_I8: per token and head step = max|x| *
 * f32(1 / 127), the cache holds round(x / step) (f32 division, ties to even, within +-127) and the step; a row with an
 * infinity or a NaN reads back as NaN throughout. The layout inside a page is the library's own: matrix-core operands, one
 * 16-byte load per lane. Everything a call needs is allocated here, so that calls can be captured into a graph. A handle's
 * decode workspace is one: calls on one handle that overlap (other streams than the library's, replayed side by side)
 * race.
 */
#define NE_KV_PAGE 64
typedef struct ne_kv ne_kv;
typedef struct {
  int layers, pages, heads, dim, dtype;
} ne_kv_desc;
NE_API ne_kv *ne_kv_create(const ne_kv_desc *d);
NE_API void ne_kv_free(ne_kv *kv);
/* d: as created (may be NULL); bytes: device memory of the cache itself (may be NULL) */
NE_API int ne_kv_info(const ne_kv *kv, ne_kv_desc *d, uint64_t *bytes);

/* A batch of sequences. Sequence b has lens[b] tokens in the cache after this step; token p is in page table[b][p / 64]
 * at p % 64. rows: i32 [n + 1], ascending; rows[b] .. rows[b + 1] - 1 are the call's rows of sequence b, its newest tokens:
 * the last of them is token lens[b] - 1 (NULL: one row each, row b). All three live on the device and are read by the
 * kernels, so a captured call takes what they hold at the replay. What they hold is bounds-checked there: a length
 * outside 0 .. 64 ldt and rows outside 0 .. R are clamped, a page id outside the handle's pages is a page without
 * tokens (not written, read as zeros, not attended), and a row before token 0 is not written, is zero when read, and
 * attends to nothing. Sequences may share pages that the call does not write. */
typedef struct ne_kv_seqs {
  int n, ldt;                  /* sequences; pages per row of table */
  const ne_buf *table, *lens;  /* i32 [n][ldt], i32 [n] */
  const ne_buf *rows;          /* i32 [n + 1] or NULL */
} ne_kv_seqs;
/* Writes the R rows k and v (heads and dim of the handle) into the cache. */
NE_API int ne_kv_write(ne_kv *kv, int layer, const ne_kv_seqs *s, int R, const ne_buf *k, uint64_t k_off, int ldk,
                       const ne_buf *v, uint64_t v_off, int ldv, int dtype, double *gpu_ms);
/* The same tokens back as rows (for a prompt's next chunk: rows[b] .. rows[b + 1] all lens[b] tokens). */
NE_API int ne_kv_read(const ne_kv *kv, int layer, const ne_kv_seqs *s, int R, ne_buf *k, uint64_t k_off, int ldk, ne_buf *v,
                      uint64_t v_off, int ldv, int dtype, double *gpu_ms);
/* Attention of the R newest tokens over the cache, which holds them already: for the row of token p, query head h (of
 * `heads`, a multiple of the handle's; key head h / (heads / handle's heads)): out = sum_{j <= p} softmax_j(scale q .
 * k_j) v_j. A row that sees no token is zero. out has q's type; it may be q's own rows. One launch for any mixture of
 * lengths (and one that joins the parts of long sequences, where there are more rows than sequences or more than 16 query
 * heads to a key head); results of one call do not vary from run to run (the sums' order follows the batch's lengths).
 * What a row does not see may hold anything, infinities and NaN included; a row that sees a key or a value that is not
 * finite is not finite where that enters it. n tables of ldt pages and R rows of `heads` heads must stay below 2^31 units
 * of work (a page for 16 rows of a key head), all counted as full: larger batches are refused. */
NE_API int ne_attn_decode(ne_kv *kv, int layer, const ne_kv_seqs *s, int R, int heads, const ne_buf *q, uint64_t q_off,
                          int ldq, ne_buf *out, uint64_t out_off, int ldo, int dtype, float scale, double *gpu_ms);

/* ---- packed prompts ----
 * n sequences packed behind one another: rows q_rows[b] .. q_rows[b + 1] - 1 of q and out, rows k_rows[b] .. k_rows[b +
 * 1] - 1 of k and v (i32 [n + 1], ascending, on the device; k_rows NULL: q_rows; values outside 0 .. Rq / Rk are
 * clamped). Causal with the ends aligned: row i of nq sees the keys j <= i + nk - nq; one that sees none is zero. Query
 * head h uses key head h / (heads / kv_heads). Rows of out that no sequence names are left as they were; out may not
 * overlap q, k or v. Masked keys and values may hold anything, as above. 16-bit rows: products of that type summed in
 * f32, the softmax weights rounded to it. 32-bit rows: products exact to f32's rounding. */
typedef struct ne_attn_prompt_desc {
  int n, heads, kv_heads, dim, dtype; /* dtype of q, k, v and out: NE_F32, NE_BF16 or NE_F16 */
  int Rq, Rk;                         /* rows of q and out; of k and v */
  int ldq, ldk, ldv, ldo;             /* 0: packed */
  float scale;
  const ne_buf *q_rows, *k_rows;
  const ne_buf *q, *k, *v;
  uint64_t q_off, k_off, v_off, out_off;
  ne_buf *out;
} ne_attn_prompt_desc;
NE_API int ne_attn_prompt(const ne_attn_prompt_desc *d, double *gpu_ms);

#ifdef __cplusplus
}
#endif
#endif /* IJAH_ATTN_H */
