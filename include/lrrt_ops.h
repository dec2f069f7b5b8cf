/*
 * C ABI of the paged-cache operators (liblrrt_ops.so): what a step of serving
 * many sequences from one pool of key-value pages runs besides its matrix
 * products. No counterpart in light-rocm-runtime, whose caches are one
 * contiguous array per stream (benchmarks/qwen_stateful_graph.cpp:730-1118).
 *
 *   lro_rope_append      rotary positions of queries and keys; keys and values
 *                        written to their pages
 *   lro_paged_attention  one new token per sequence over the paged cache
 *   lro_pages_fork       sequences reordered, shared and split copy-on-write,
 *                        freed, and given pages to grow into
 *   lro_pages_compact    live pages moved to the front of the pool
 *   lro_pages_copy       a list of whole pages copied
 *   lro_beam_select      the best continuations over beams and vocabulary
 *
 * The cache. A page holds page_size tokens of every key-value head of one
 * layer; a sequence's token j is row j % page_size of page
 * table[sequence][j / page_size]. Strides are given in elements, so pages may
 * be stored token by token or head by head; the head_dim elements of one row
 * are contiguous. Strides are less than 2^31 elements. A table entry outside
 * [0, page_count) is "no page": its tokens are not read and not written.
 *
 * Calls enqueue their work on the context's queue and return; the device
 * arrays they are given must stay until it is done. The calls of one context
 * share its workspace: use a context from one host thread at a time, and one
 * context per queue. Nothing is kept from one call for the next.
 *
 * Pointers are device pointers unless a comment says otherwise. All functions
 * return lr_status_t; lro_last_error() describes this thread's last failure.
 */
#ifndef LRRT_OPS_H_
#define LRRT_OPS_H_

#include "lrrt/lrrt.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct lro_context_t lro_context_t;

typedef enum lro_type_t { LRO_F32 = 0, LRO_BF16 = 1, LRO_F16 = 2 } lro_type_t;

/* Rows of heads: [row][head][head_dim], strides in elements. */
typedef struct lro_rows_t {
  void *data;
  int64_t row_stride, head_stride;
} lro_rows_t;

/* One layer's pages. */
typedef struct lro_cache_t {
  void *keys, *values;
  int64_t key_page_stride, key_token_stride, key_head_stride;
  int64_t value_page_stride, value_token_stride, value_head_stride;
  uint32_t type; /* lro_type_t */
  uint32_t page_count, page_size, kv_heads, head_dim;
} lro_cache_t;

/* Page numbers [rows][columns] of `rows` sequences. */
typedef struct lro_table_t {
  const int32_t *pages;
  int64_t row_stride;
  uint32_t rows, columns;
} lro_table_t;

/*
 * A context: the operators' module (paged_ops.cubin), the queue they run on
 * (NULL: the device's default queue; it must outlive the context) and a
 * workspace, with counters that blocks meet at. Both grow when a call needs more
 * of them; what they outgrow stays until the context is destroyed, so that CUDA
 * graphs captured before can be replayed after. While its queue is captured a
 * call that would have to grow them fails: make a call of the same sizes before,
 * or reserve. An attention needs a counter for each sequence and key-value head,
 * and each 16 of its query heads; a selection one for each beam and each
 * group; 16384 are there.
 */
LRRT_API lr_status_t lro_context_create(lr_device_t device, lr_queue_t *queue,
                                        const void *module_image, size_t module_image_size,
                                        lro_context_t **context);
LRRT_API lr_status_t lro_context_destroy(lro_context_t *context);
LRRT_API lr_status_t lro_context_reserve(lro_context_t *context, size_t workspace_bytes);
LRRT_API lr_status_t lro_context_reserve_counters(lro_context_t *context, uint64_t counters);

/*
 * cos/sin tables [positions][rotary_dim / 2] (host arrays), computed in 64 bits
 * and rounded once: angle(p, i) = p * f(i), f(i) = theta^(-2 i / rotary_dim).
 * factor > 1 stretches a model trained on `trained_positions`: frequencies
 * that turn fewer than `low_turns` times in them are divided by factor, those
 * with more than `high_turns` are kept, and between the two the scaled and the
 * kept are blended linearly. low_turns = high_turns = 0 divides them all.
 */
LRRT_API lr_status_t lro_rope_tables(uint32_t positions, uint32_t rotary_dim, double theta,
                                     double factor, double low_turns, double high_turns,
                                     double trained_positions, float *cos_table,
                                     float *sin_table);

/*
 * For each token t: rotates the first rotary_dim elements of its query and key
 * heads by the angles of positions[t], passes the others through, writes the
 * queries to q_out (which may be q) and the keys and values to token
 * positions[t] of sequence sequences[t]. Pairs are (i, i + rotary_dim / 2), or
 * (2 i, 2 i + 1) when interleaved. The arithmetic is in 32 bits, rounded once.
 * A token with a sequence or a position out of range of the table or of the
 * cos/sin tables, or with no page, is padding: its queries become zeros and
 * nothing is appended. Two tokens of one call must not share a cache row, nor two
 * rows of the cache or of q_out memory.
 */
typedef struct lro_rope_append_t {
  lro_rows_t q, q_out, k, v;
  lro_cache_t cache; /* its type is that of q, q_out, k and v too */
  lro_table_t table;
  const int32_t *sequences; /* [tokens]; NULL: token t is of sequence t */
  const int32_t *positions; /* [tokens] */
  const float *cos_table, *sin_table; /* [table_positions][rotary_dim / 2] */
  uint32_t tokens, heads, rotary_dim, table_positions;
  uint32_t interleaved, reserved;
} lro_rope_append_t;

LRRT_API lr_status_t lro_rope_append(lro_context_t *context, const lro_rope_append_t *arguments);

/*
 * Attention of one query row per sequence over the first lengths[b] tokens of
 * its pages; query head h reads key-value head h / (heads / kv_heads).
 *   x_j = scale * q . k_j;  with softcap > 0: x_j = softcap * tanh(x_j / softcap)
 *   s_j = x_j - slopes[h] * (lengths[b] - 1 - j)   (slopes may be NULL)
 *   out = sum_j exp(s_j) v_j / sum_j exp(s_j),  lse = log sum_j exp(s_j)
 * over the tokens j that have a page and, with window > 0, are among the last
 * `window`. A row that sees no token, or none with a score above -infinity, has
 * out = 0 and lse = -infinity; lengths are clamped to [0, columns * page_size].
 * An infinite value makes its column infinite (NaN with both signs); a NaN, or
 * a score of infinity, leaves NaN in out and lse. Sums are held in 32 bits;
 * 32-bit products are three TF32 products (about 2^-21 per product).
 * out may be q, and must not lie partly in it, nor may its rows share memory.
 * head_dim: a multiple of 8, at most 256 (128 in 32 bits). Cache pointers and
 * strides: multiples of 16 bytes.
 */
typedef struct lro_paged_attention_t {
  lro_rows_t q, out;
  lro_cache_t cache; /* its type is that of q and out too */
  lro_table_t table;
  const int32_t *lengths; /* [table.rows] */
  const float *slopes;    /* [heads], or NULL */
  float *lse;             /* [table.rows][heads], or NULL */
  uint32_t heads, window;
  float scale, softcap;
} lro_paged_attention_t;

LRRT_API lr_status_t lro_paged_attention(lro_context_t *context,
                                         const lro_paged_attention_t *arguments);

/*
 * The pages of all layers, as the page operators move them. A page of one
 * layer is `segments` runs of page_size rows of row_bytes, one after another
 * (token by token: 1 run of rows of kv_heads * head_dim elements; head by head:
 * kv_heads runs of rows of head_dim elements). Keys and values are alike.
 * row_bytes, strides and pointers: multiples of 4 bytes.
 */
typedef struct lro_pool_t {
  void *keys, *values;
  int64_t layer_stride_bytes, page_stride_bytes;
  uint32_t layers, page_count, page_size, segments, row_bytes;
  uint32_t reserved;
} lro_pool_t;

/*
 * New sequences from old ones: row s of table_out continues sequence
 * parents[s] (a parent out of range: the row is empty), with room for `room`
 * more tokens. Rows share the whole pages of their parent. A last, unfinished
 * page, which the row will write to, is its own: it stays with the lowest row
 * that has it, and every other row gets a copy; where any row holds that page
 * whole, or held[page] is set, all get copies. Then each row gets the pages
 * that `room` needs, as far as the table has columns.
 * New pages are the lowest free ones, in the order of the rows; free are the
 * pages that no row holds and held (may be NULL, [page_count]) does not name.
 * So a sequence that is nobody's parent is freed. Table entries past a row's
 * pages are -1, as are those that found the pool empty.
 *   lengths_out[s] = lengths[parents[s]], 0 for an empty row
 *   status[0] = pages that were missing, status[1] = pages that are left free
 * The outputs must not overlap the inputs (keep two tables and swap them).
 */
typedef struct lro_pages_fork_t {
  lro_pool_t pool;
  lro_table_t table;
  const int32_t *lengths; /* [table.rows] */
  const int32_t *parents; /* [rows_out] */
  const uint8_t *held;
  int32_t *table_out; /* [rows_out][table.columns] */
  int64_t table_out_row_stride;
  int32_t *lengths_out; /* [rows_out] */
  int32_t *status;      /* [2] */
  uint32_t rows_out, room;
} lro_pages_fork_t;

LRRT_API lr_status_t lro_pages_fork(lro_context_t *context, const lro_pages_fork_t *arguments);

/*
 * Moves the live pages (those with a table entry) to the front of the pool:
 * with n pages live or held, the live ones numbered n and above move to the
 * free ones below n, both in rising order, and table_out (which may be the
 * table) holds the new numbers. Held pages stay where they are.
 *   status[0] = n, status[1] = pages moved
 */
typedef struct lro_pages_compact_t {
  lro_pool_t pool;
  lro_table_t table;
  const uint8_t *held; /* [page_count], or NULL */
  int32_t *table_out;
  int64_t table_out_row_stride;
  int32_t *status; /* [2] */
} lro_pages_compact_t;

LRRT_API lr_status_t lro_pages_compact(lro_context_t *context,
                                       const lro_pages_compact_t *arguments);

/* Page sources[i] copied to page targets[i] in every layer, for i < count.
 * No page may be both; pairs with a number out of range are skipped. */
typedef struct lro_pages_copy_t {
  lro_pool_t pool;
  const int32_t *sources, *targets;
  uint32_t count, reserved;
} lro_pages_copy_t;

LRRT_API lr_status_t lro_pages_copy(lro_context_t *context, const lro_pages_copy_t *arguments);

/*
 * The `count` best continuations of each group of beams.
 * Beam k of group g has the score scores[g][k] and the logits row
 * g * beams + k; its continuation by token t scores
 *   scores[g][k] + (logit[t] - log sum_u exp(logit[u]))
 * A finished beam (finished[g][k] != 0; finished may be NULL) has one
 * continuation, the end token at its own score. Candidates are ordered by
 * score, then lower beam, then higher logit, then lower token; NaN counts as
 * -infinity. Continuations of score -infinity are no candidates: where fewer than
 * `count` remain, scores are -infinity, parents and tokens -1, finished 1.
 *   parents_out = g * beams + k, as lro_pages_fork takes them
 *   finished_out = the beam was finished, or the token is end_token
 * With count = beams, scores_out and finished_out may be scores and finished.
 * Outputs are [groups][count]; beams and count: 1 to 64, their product at most
 * 2048; count <= vocab <= 2^21; groups * beams <= 65535.
 */
typedef struct lro_beam_select_t {
  const void *logits; /* [groups * beams][vocab] */
  int64_t logits_row_stride;
  const float *scores;     /* [groups][beams] */
  const uint8_t *finished; /* [groups][beams], or NULL */
  float *scores_out;
  int32_t *parents_out, *tokens_out;
  uint8_t *finished_out; /* or NULL */
  uint32_t type;         /* lro_type_t of the logits */
  uint32_t groups, beams, vocab, count;
  int32_t end_token; /* -1: none */
} lro_beam_select_t;

LRRT_API lr_status_t lro_beam_select(lro_context_t *context, const lro_beam_select_t *arguments);

/* The calling thread's last failure ("" before the first). */
LRRT_API const char *lro_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* LRRT_OPS_H_ */
