/*
 * holo_forward.h -- the Llama forward over a prompt of M tokens in one pass:
 * row-batched ops and a driver that runs all M rows through every layer at
 * once.
 *
 * The reference processes a prompt one token at a time: llm_forward runs
 * every layer for token t before token t+1 (src/ai/llm.c:1015-1270, CPU), and
 * the GPU loop does the same with one GEMV per matrix and token
 * (src/ai/llm_cuda.c:574-891).  holo_llama_forward computes the same result
 * for tokens[0..n) at positions pos0..pos0+n-1:
 *   - each matrix multiplies all n rows at once (holo_matmul_rows: the exact
 *     batched product with n >= 3, otherwise one GEMV per row);
 *   - RoPE, the KV-cache writes and the norms take all rows in one launch;
 *   - attention is causal over the prompt (holo_attention_prefill): row m sees
 *     positions 0..pos0+m, as token pos0+m does in the reference.
 * The logits of the last token are written, as after the reference's loop.
 * n = 1 is one decode step.
 *
 * Supported: the Llama layer of llm.c (attention norm, q/k/v/o, SwiGLU FFN,
 * final norm, output head); no QKV biases, QK-norm, post-norms or embedding
 * scaling (the Qwen/Gemma branches of llm.c), head_dim <= 128.
 */
#ifndef HOLO_FORWARD_H
#define HOLO_FORWARD_H

#include "holo_gguf.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- row-batched ops ---------------------------------------------------------
 * rows consecutive vectors; each row as the single-vector op would compute it. */

/* cuda_rms_norm (cuda_ops.h:75) on each of rows rows of n floats.            */
void holo_rms_norm_rows(float *dst, const float *x, const float *weight, int rows, int n, float eps);
/* cuda_rope_apply (cuda_ops.h:117) with row r at position pos0 + r; q rows of
 * n_heads*head_dim floats, k rows of n_kv_heads*head_dim.                    */
void holo_rope_rows(float *q, float *k, int rows, int pos0, int head_dim, int n_heads, int n_kv_heads,
                    float freq_base);
/* cuda_get_embedding_* (cuda_ops.h:121-129) for tokens[0..rows) (a device
 * array of int): F32, F16, Q8_0, Q4_0, Q6_K; and Q4_K, which has no lookup
 * op in the reference, as the bit-exact dequantize_row_q4_k of each row
 * (quant.c:277-311), as llm.c:998-1003 looks Q4_K rows up.                 */
void holo_embedding_rows(float *dst, const void *embeddings, const int *tokens, int rows, int dim, int type);
/* Causal attention: row m of q (position pos0 + m) against positions
 * 0..pos0+m of this layer's caches [pos][n_kv_heads*head_dim], which must
 * already hold those positions; head h reads KV head h / (n_heads /
 * n_kv_heads) (cuda_multi_head_attention, cuda_ops.h:112, per row).           */
void holo_attention_prefill(float *out, const float *q, const float *k_cache, const float *v_cache, int rows,
                            int pos0, int head_dim, int n_heads, int n_kv_heads);
/* Each row of n values to softmax(scale (x - max x)): the logits of several tokens
 * to probabilities, scale 1 / temperature (large for the largest alone).  ldd and
 * ldx are the floats from one row to the next; dst may be x with the same ld.
 * Values of -infinity get 0, a row of nothing else is zeros; a row with NaN or
 * +infinity is NaN.  Returns 0 or HOLO_EINVAL (nothing launched): a scale that is
 * not positive and finite.  (cuda_softmax takes one row, cuda_ops.h:79.)         */
int holo_softmax_rows(float *dst, const float *x, int rows, int n, int ldd, int ldx, float scale);
/* Y[rows][out] = X[rows][in] . W^T for any GEMV type (holo_matmul per row).
 * rows >= 3 with in_dim whole blocks takes the batched MFMA product
 * (holo_matmul_batch) unless `exact` is set.                                  */
void holo_matmul_rows(float *Y, const void *W, const float *X, int rows, int out_dim, int in_dim, int type,
                      int exact);

/* ---- several sequences at once ------------------------------------------------
 * A batch is the new rows of n_seqs sequences, packed: entry s has rows
 * cu_rows[s] .. cu_rows[s + 1] - 1 (one in a decode step, a chunk or a whole
 * prompt otherwise).  cu_rows and seqs are device arrays, so a captured graph
 * follows what they hold at each replay; what they say past `rows` is cut off.
 * rows, max_rows and max_len bound the launch: an entry's rows past its first
 * max_rows are left as they were.  No rows or no entries: nothing is done.
 * No reference counterpart (one sequence, one token at a time: llm.c:1015-1270). */
typedef struct {
    int rows;           /* rows of the call, over all entries */
    int n_seqs;         /* entries, up to 65535 */
    int max_rows;       /* the most rows of an entry */
    int max_len;        /* holo_attention_kv4: the most positions of an entry's sequence */
    const int *cu_rows; /* device, [n_seqs + 1], rising from 0 to rows */
    const int *seqs;    /* device, [n_seqs]: the entry's sequence of the cache, each once; NULL: entry s is sequence s */
} holo_batch_t;

/* Causal attention within each sequence: row i of an entry against its rows 0
 * .. i, softmax(q . k / sqrt(head_dim)) v, head h reading KV head h / (n_heads
 * / n_kv_heads): the prompts of several sequences in one call
 * (holo_attention_prefill at pos0 = 0, entry by entry).  ldo, ldq, ldk and ldv
 * are the floats from one row to the next (q, k and v may lie side by side in
 * one buffer).  head_dim 32, 64, 96 or 128; every pointer 16-byte aligned and
 * every ld a multiple of 4, ldk and ldv below 2^24; max_rows times n_heads /
 * n_kv_heads up to 2097120.  seqs and max_len are not read.  A row is not
 * touched by what the rows behind it hold, infinities and NaN among it.  Any
 * magnitude is right whose scores are floats: a key whose score lies below a
 * float's range has no part, one above it or no key with a part makes the row
 * and head NaN.  Keys or values of 255.9375 and more (and rows of which none
 * reaches 2^-11, where they make up an output) take an fp32 path some thirty
 * times slower; others are held within 2^-22 of themselves, or within 2^-33
 * where that is more.  Returns 0 or HOLO_EINVAL (nothing launched).            */
int holo_attention_packed(float *out, const float *q, const float *k, const float *v, int ldo, int ldq, int ldk,
                          int ldv, int head_dim, int n_heads, int n_kv_heads, const holo_batch_t *b);

/* ---- a cache in pages, four bits a value -------------------------------------------
 * Q4_0 values (16 codes about a block scale, 32 dims a block) in a layout for
 * the matrix cores: a page holds page_len positions of every layer and KV head,
 * in tiles of 32 positions of 36 * head_dim bytes (16 codes bytes a position and
 * 32 dims for keys and for values each, and their f16 scales), 4.5 bits a value.
 * A block's scale is d = -m / 8 of its value m of largest magnitude (the negative
 * one of two), rounded to bfloat16, at most 2720 in magnitude and held in f16;
 * a value is d * c, c the nearest to x / d in -8 .. 7 (ties to the even one).
 * d has 8 significant bits, so d * c is an f16 and the products below are of
 * exact operands (holo_kv4_append writes no other scales).  A block that holds an
 * infinity or NaN reads as NaN; values past 21760 are held as about that.
 *
 * pool, table and len are device memory of the caller.  Entry p of a sequence's
 * row of `table` is the page of its positions p * page_len ..; an entry outside
 * 0 .. n_pages - 1 is no page: nothing is stored there, and attention passes
 * over its positions.  len holds each sequence's positions, the rows of the
 * batch in hand among them: the last of them are the batch's.  Sequences may
 * share pages (holo_kv4_pages_fork).                                           */
typedef struct {
    void *pool;       /* n_pages * holo_kv4_page_bytes bytes, 16-byte aligned */
    const int *table; /* [n_seqs][max_pages] */
    const int *len;   /* [n_seqs] */
    int n_pages;
    int page_len;     /* 32, 64, 128, 256, 512 or 1024 */
    int n_layers, n_kv_heads; /* up to 65535 */
    int head_dim;     /* 32, 64, 96 or 128 */
    int n_seqs, max_pages;
} holo_kv4_t;

/* Bytes of a page, or 0 for a layout outside the set above (only the layout is read). */
size_t holo_kv4_page_bytes(const holo_kv4_t *c);
/* The batch's rows of k and v ([n_kv_heads * head_dim] floats, ldk and ldv from
 * one row to the next) into the pages of one layer, at the last positions of
 * their sequences, shared pages among them (reserve first).  What the other
 * positions hold stays.  0 or HOLO_EINVAL.                                      */
int holo_kv4_append(const holo_kv4_t *c, int layer, const float *k, const float *v, int ldk, int ldv,
                    const holo_batch_t *b);
/* The values that the cache holds for the batch's rows (zeros where there is no page). */
int holo_kv4_read(const holo_kv4_t *c, int layer, float *k, float *v, int ldk, int ldv, const holo_batch_t *b);
/* Attention of the batch's rows over their sequences' pages: row i of an entry
 * of r rows is at position len - r + i and sees the positions up to its own
 * (cuda_multi_head_attention over several sequences, cuda_ops.h:112; with more
 * rows holo_attention_prefill).  A row that sees no position gives zeros; the
 * rows of a sequence longer than max_len give NaN.  q rows of n_heads *
 * head_dim floats; scores past a float's range give NaN, or zeros where every one is
 * below it.  max_rows up to 65535, and its tiles of 16 columns (a row's heads
 * of one KV head) times n_kv_heads too.  Long sequences are cut into ranges, as
 * many as entries of max_rows rows each leave room for: single tokens are faster
 * in a call of their own than beside a chunk of many rows.  0 or HOLO_EINVAL;
 * without memory for its partial sums the hipError_t.                          */
int holo_attention_kv4(const holo_kv4_t *c, int layer, float *out, const float *q, int ldo, int ldq, int n_heads,
                       const holo_batch_t *b);
/* ---- rotary positions of a batch ------------------------------------------------------
 * Pair i of a head's leading `dims` dims turns by t = position * freq[i]: (a, b)
 * becomes scale * (a cos t - b sin t, a sin t + b cos t), in 64 bits, rounded once;
 * the other dims pass as they are.                                              */
typedef struct {
    const double *freq; /* device, [dims / 2]: radians a position, each pair's (holo_rope_freqs) */
    int dims;           /* even, 2 .. head_dim */
    int interleaved;    /* a pair is dims (2 i, 2 i + 1); 0: (i, i + dims / 2), as cuda_rope_apply has it */
    float scale;        /* 1, or what holo_rope_freqs gives */
} holo_rope_t;

/* holo_kv4_append of rotated keys, and the queries rotated beside it.  The
 * cache gets the keys at their rows' places (the last positions of their
 * sequences) and the values; k_out (NULL: none) the rotated keys as floats, for
 * holo_attention_packed; q_out the rotated queries.  q_out may be q and k_out k,
 * with the same ld; otherwise nothing that is written overlaps what is read.  A
 * row turns by len - r + i (row i of an entry of r rows), or with depth (device,
 * [rows]) by len - r + depth[row]: rows of a tree.  n_heads 0: no queries; n_kv_heads
 * times half the query heads of each (rounded up) up to 65535.
 * Rows without a page, or before position 0, are rotated all the same.  0 or
 * HOLO_EINVAL.  (cuda_rope_apply, cuda_ops.h:117, takes one row.)               */
int holo_kv4_append_rope(const holo_kv4_t *c, int layer, const holo_rope_t *r, const float *q, const float *k,
                         const float *v, int ldq, int ldk, int ldv, float *q_out, float *k_out, int ldqo, int ldko,
                         int n_heads, const int *depth, const holo_batch_t *b);

/* Frequencies, on the host: base^(-2 i / dims), each divided by divisors[i] where
 * there are any, and for contexts `factor` times the trained one
 *   PLAIN   as they are (factor and what follows it are not read)
 *   LINEAR  divided by factor
 *   BASE    with base * factor^(dims / (dims - 2)) for base
 *   BANDS   pairs that turn more than `high` times over the `trained` positions as
 *           they are, those that turn less than `low` times divided by factor,
 *           between them the mean weighted by (turns - low) / (high - low)
 *   RAMP    the same, weighted along the pairs' numbers instead, from the one
 *           that turns `high` times (rounded down) to the one that turns `low`
 *           times (up); scale becomes 0.1 ln(factor) + 1, otherwise it is 1
 * freq: host, [dims / 2]; scale may be NULL.  0 or HOLO_EINVAL.                     */
#define HOLO_ROPE_PLAIN 0
#define HOLO_ROPE_LINEAR 1
#define HOLO_ROPE_BASE 2
#define HOLO_ROPE_BANDS 3
#define HOLO_ROPE_RAMP 4
typedef struct {
    int kind, dims;        /* dims: even, up to 128 (BASE: from 4) */
    double base;           /* above 1 */
    double factor;         /* at least 1 */
    double low, high;      /* 0 < low < high */
    int trained;           /* positions */
    const float *divisors; /* host, [dims / 2], positive; NULL: none */
} holo_rope_scaling_t;
int holo_rope_freqs(double *freq, float *scale, const holo_rope_scaling_t *s);

/* ---- drafted tokens ------------------------------------------------------------------
 * A small model drafts what may follow a sequence, the large one runs over all of
 * it in one step.  An entry's row 0 is then the sequence's last token, the others
 * the drafted ones: parent[row] (device, [rows]) is the row of the entry that a
 * row follows, an earlier one, anything else none.  A step:
 *   holo_kv4_pages_reserve   positions for all rows of the entries
 *   holo_draft_plan          once
 *   holo_kv4_append_rope, holo_attention_kv4_draft   in every layer
 *   holo_softmax_rows, holo_draft_verify             on the rows' logits
 *   holo_kv4_keep            the rows that stand to the front, every layer
 *   holo_kv4_pages_trim      the other rows' positions given back
 * All but the pages' calls can be captured.                                     */

/* Of each row: how many rows it follows up the tree, and itself and those rows as
 * bits, bit j & 31 of word j / 32 for row j (mask: device, [rows][words]).  max_rows up
 * to 32 * words, words up to 32.  0 or HOLO_EINVAL.                                */
int holo_draft_plan(const int *parent, int *depth, uint32_t *mask, int words, const holo_batch_t *b);
/* holo_attention_kv4 of rows that see the positions before their entry's rows, and
 * of these the ones whose bits their mask has (any mask, its own row's bit too;
 * rows past the words have none).  A row that sees nothing gives zeros.  max_rows up
 * to 32 * words, words up to 32, otherwise as holo_attention_kv4; n_seqs times the
 * tiles of columns and KV heads up to some 4.29e9.  Ranges go by the lengths themselves, for
 * up to 1024 entries: ragged batches, and long sequences beside short ones, need no calls of their own.  */
int holo_attention_kv4_draft(const holo_kv4_t *c, int layer, float *out, const float *q, int ldo, int ldq,
                             int n_heads, const uint32_t *mask, int words, const holo_batch_t *b);

/* Which drafted tokens stand, so that the tokens have the target's distribution.
 * target and draft: the probabilities of the token behind each row (rows ldt and
 * ldd floats apart); tokens, parent and u, random numbers in [0, 1), of each
 * row.  A walk begins at row 0 and judges the rows in order whose parent it is at,
 * with p and q that row's probabilities, x the judged token, N = 1 and beta = Q = 0:
 *   DRAWN     the tokens behind a row were drawn from its q, each by itself.  It
 *             stands if u q(x) N < max(p(x) - beta q(x), 0) (1 - Q); else beta += N / (1 - Q),
 *             N = sum max(p - beta q, 0)
 *   DISTINCT  they were drawn without repeats: and Q += q(x)
 *   CHOSEN    they were not drawn (the most probable ones, say; draft is not read).
 *             It stands if u N < p(x), p(x) = 0 for a token refused here before; else
 *             N -= p(x)
 * A row that stands is where the walk goes on, with N = 1 and beta = Q = 0.
 * path (device, [rows]) gets the entry's rows that stand, row 0 first, then -1;
 * n_path[s] how many; next[s] the token behind the last of them: the first x at which the
 * sum of w(0 .. x) passes u of row 0 times the sum of all, w = max(p - beta q, 0), or p
 * without the refused tokens (no weight at all: the target's most probable token).  A u
 * outside [0, 1) counts as the nearest number inside, NaN as 0.  Sums are
 * in 64 bits.  target's rows sum to 1; values that are negative or no finite
 * numbers count as 0.  Tokens outside 0 .. vocab - 1 never stand.  An entry without
 * rows beside others that have some: n_path 0, next -1.  A batch whose `rows` is 0
 * writes nothing, as every call: n_path and next keep what an earlier step left
 * there.  vocab up to 2^24, max_rows up to 1024.  0 or HOLO_EINVAL.               */
#define HOLO_DRAFT_CHOSEN 0
#define HOLO_DRAFT_DRAWN 1
#define HOLO_DRAFT_DISTINCT 2
int holo_draft_verify(int *path, int *n_path, int *next, const float *target, const float *draft, int ldt, int ldd,
                      int vocab, const int *tokens, const int *parent, const float *u, int mode, const holo_batch_t *b);
/* Of each entry, row path[i] to the place of row i for i < n_path[s], keys and
 * values, every layer: what holo_kv4_append_rope would have stored of these rows
 * alone.  path rises (device, [rows], as holo_draft_verify leaves it); an entry of
 * it outside the rows, or a place without a page, moves nothing.  What the other positions
 * hold stays.  The pages written must not be shared (holo_kv4_pages_reserve sees to it).
 * 0 or HOLO_EINVAL.                                                             */
int holo_kv4_keep(const holo_kv4_t *c, const int *path, const int *n_path, const holo_batch_t *b);

/* Page dst[i] becomes a copy of page src[i], every layer (host arrays).
 * HOLO_EINVAL, and nothing copied, for a page outside the pool, a page written
 * twice, or one that is read and written.                                      */
int holo_kv4_copy_pages(const holo_kv4_t *c, const int *src, const int *dst, int n);

/* Which pages belong to which sequence, on the host: the lowest free page is
 * taken first, and the device's table and len follow on the library stream.
 * c's device arrays must outlive the handle and be written by it alone; a c
 * without any (pool, table and len NULL) is bookkeeping without a device.  Calls
 * return 0, HOLO_EINVAL (also under graph capture) or HOLO_ENOPAGES (reserve);
 * then nothing has changed.  One handle may be used by several threads.        */
typedef struct holo_kv4_pages holo_kv4_pages_t;
/* Every sequence empty, every page free; NULL with the error latched.          */
holo_kv4_pages_t *holo_kv4_pages_create(const holo_kv4_t *c);
void holo_kv4_pages_destroy(holo_kv4_pages_t *p);
/* Room for rows[i] more positions of sequence seqs[i] (host arrays, a sequence
 * once), len counting them from now on: before a batch's append.  A sequence
 * whose last page is not full and shared gets a copy of it.                    */
int holo_kv4_pages_reserve(holo_kv4_pages_t *p, const int *seqs, const int *rows, int n);
/* The empty sequence dst[i] becomes a copy of src[i], sharing its pages.  Entry
 * by entry: a src may be an earlier dst.                                       */
int holo_kv4_pages_fork(holo_kv4_pages_t *p, const int *src, const int *dst, int n);
/* The last rows[i] positions of sequence seqs[i] (a sequence once) given back, and
 * the pages that hold no others.  HOLO_EINVAL for more than it has.             */
int holo_kv4_pages_trim(holo_kv4_pages_t *p, const int *seqs, const int *rows, int n);
/* Sequences emptied; pages that no other sequence shares are free again.       */
int holo_kv4_pages_free(holo_kv4_pages_t *p, const int *seqs, int n);
/* The pages in use moved to the front of the pool: 0 .. used - 1.              */
int holo_kv4_pages_compact(holo_kv4_pages_t *p);
/* Pages free; positions of a sequence (-1: none such); its pages, at most n of
 * them (host array), and how many it has.                                      */
int holo_kv4_pages_available(holo_kv4_pages_t *p);
int holo_kv4_pages_len(holo_kv4_pages_t *p, int seq);
int holo_kv4_pages_list(holo_kv4_pages_t *p, int seq, int *pages, int n);

/* ---- the model --------------------------------------------------------------- */

typedef struct {
    const float *attn_norm;  /* [dim] F32, or NULL (no norm) */
    const void *wq, *wk, *wv, *wo;
    int wq_type, wk_type, wv_type, wo_type;
    const float *ffn_norm;   /* [dim] F32, or NULL */
    const void *w1, *w2, *w3; /* gate [ffn][dim], down [dim][ffn], up [ffn][dim] */
    int w1_type, w2_type, w3_type;
} holo_llama_layer_t;

typedef struct {
    int n_layers, dim, n_heads, n_kv_heads, head_dim, ffn_dim;
    int vocab;               /* rows of the output head (logits written) */
    int max_seq;             /* positions held by the caches */
    float rms_eps, rope_base;
    const void *tok_emb;     /* [vocab][dim] blocks */
    int emb_type;
    const float *out_norm;   /* [dim] F32, or NULL */
    const void *output;      /* [vocab][dim] */
    int out_type;
    float *key_cache, *value_cache;   /* device, [n_layers][max_seq][n_kv_heads*head_dim] */
    const holo_llama_layer_t *layers; /* host array of n_layers */
} holo_llama_t;

#define HOLO_FORWARD_EXACT 1 /* every matmul as fp32-activation GEMVs (no Q8_0 activations) */

/* Runs tokens[0..n) (host array) at positions pos0..pos0+n-1, writes the
 * caches' rows pos0..pos0+n-1 of every layer and the last token's logits
 * (device, [vocab]).  0, or HOLO_EINVAL for a model or shape outside the
 * supported set (nothing launched).  Scratch is stream-ordered.               */
int holo_llama_forward(const holo_llama_t *m, const int *tokens, int n, int pos0, float *logits, int flags);

/* holo_prefill_prepare for every Q6_K layer matrix of m (q, k, v, o, gate,
 * down, up; the output head runs the GEMV), and holo_prefill_release for
 * them: the prompt forward then reads their repacked copies (1 byte per
 * weight of those matrices) instead of repacking each one per call.  No
 * reference counterpart.  0, or the first failing holo_prefill_prepare's
 * code (the matrices prepared before it are released).                      */
int holo_llama_prepare(const holo_llama_t *m);
void holo_llama_release(const holo_llama_t *m);

/* Fills m and layers[0..n_layers) from an uploaded GGUF file
 * (holo_gguf_upload), with the reference loader's tensor names and model
 * parameters (llm.c:344-533, 617-660): token_embd, blk.N.{attn_norm,
 * attn_q, attn_k, attn_v, attn_output, ffn_norm, ffn_gate, ffn_down,
 * ffn_up}, output_norm, output (tied to token_embd when absent).  vocab is
 * token_embd's row count.  The caller sets max_seq and the caches.
 * 0, or -1 when a required tensor is missing, n_layers > max_layers, or
 * holo_llama_gguf_check rejects the file.                                   */
int holo_llama_from_gguf(const holo_gguf_t *g, holo_llama_t *m, holo_llama_layer_t *layers, int max_layers);
/* 0 when a parsed GGUF file (host-side parse is enough) is the plain Llama
 * body this forward runs; -1 when it needs a branch of the reference's
 * forward that is not built here: a Gemma architecture (general.architecture
 * contains "gemma"), or any blk.N.attn_{q,k,v}.bias, attn_{q,k}_norm.weight,
 * post_attention_norm.weight or post_ffw_norm.weight tensor (the Qwen and
 * Gemma branches of llm.c:451-521, 1037-1133).                               */
int holo_llama_gguf_check(const holo_gguf_t *g);

#ifdef __cplusplus
}
#endif

#endif /* HOLO_FORWARD_H */
