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
