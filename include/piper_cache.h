/*
 * piper_cache.h -- C ABI of the quantised paged KV cache and the attention that reads it (gfx950; in
 * libpiper_mi355x.so beside the operators of piper_mi355x.h, whose dtypes, status codes, tensor
 * struct and piper_last_error() it uses).  No counterpart in the reference, which has no cache.
 *
 * Like the rest of the library these functions validate, launch kernels on `stream` (a hipStream_t; NULL:
 * the default stream) of the current device and return: they never allocate, synchronise or keep anything
 * between calls, so they can be captured into a graph, and calls on different streams do not meet unless they
 * share buffers.
 *
 * The cache.  A page holds 64 tokens (PIPER_CACHE_PAGE) of every K/V head.  With P pages, H K/V heads and
 * head size D all arrays are dense and row-major, each 16-byte aligned (bound_scale: 4-byte):
 *
 *   key          8 bit  [P, H, 64, D]
 *   key_scale    float  [P, H, 64]
 *   value        8 bit  [P, H, 8, D, 8]   token 8 a + j of the page, feature d at [a, d, j]: eight tokens of a
 *                                         feature are the eight bytes a matrix instruction takes together
 *   value_scale  float  [P, H, 64]
 *   bounds       int8   [P, H, 2, D]      of a full page: codes of the largest and of the smallest key value
 *                                         per feature
 *   bound_scale  float  [P, H]
 *
 * A row x of D values is held as code = round_half_even(x * (L / a)) and scale = a / L, with a its largest
 * magnitude, L = 127 for INT8 and 448 for FP8 E4M3, every operation in FP32; it stands for code * scale.  A row
 * with a < 2^-118 is held as zeros.  A row with an infinity or a NaN gets a NaN scale and zero codes: what
 * attends to it becomes NaN, nothing else does.  Bounds are held by the same rule (L = 127, a over the 2 D
 * values), taken over the values the page's keys stand for, NaN left out.
 *
 * Where tokens stand.  Sequence b's position p is slot p % 64 of page page_table[b][p / 64].  A call's row i of
 * sequence b, i < counts[b] (NULL: every row), is position starts[b] + i.  All three live in device memory.
 * Positions below 0 or beyond the table and entries outside [0, P) name no page: nothing is written there, reads
 * give zeros and attention does not see it.  Counts are taken as 0 below 0 and as the row count beyond it.
 *
 * A call that would take 2^23 workgroups or more is refused (PIPER_ERROR_UNSUPPORTED).  Workgroups: for a write or a read one
 * per page touched and K/V head; for attention one per K/V head and block of up to 16, 32, 128 or 256 query rows
 * (with selected pages one per token and up to 32); for selection at most one per row, K/V head and 256 pages.
 */
#ifndef PIPER_CACHE_H
#define PIPER_CACHE_H

#include "piper_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PIPER_CACHE_ABI_VERSION 1
#define PIPER_CACHE_PAGE 64

typedef enum piper_cache_code { PIPER_CACHE_INT8 = 0, PIPER_CACHE_FP8 = 1 } piper_cache_code;

typedef struct piper_cache {
  void* key;
  float* key_scale;
  void* value;
  float* value_scale;
  int8_t* bounds;     /* piper_cache_write and piper_cache_select only */
  float* bound_scale; /* likewise */
  int64_t pages;
  int64_t kv_heads;
  int32_t head_dim; /* 64 or 128 */
  int32_t code;     /* piper_cache_code */
} piper_cache;

typedef struct piper_cache_rows {
  const int32_t* page_table; /* [batch, table_width], rows table_stride elements apart */
  const int32_t* starts;     /* [batch] */
  const int32_t* counts;     /* [batch] or NULL */
  int64_t table_stride;
  int64_t table_width;
  int64_t batch;
  int64_t tokens; /* rows per sequence in this call */
} piper_cache_rows;

typedef struct piper_cache_write_args {
  int32_t abi_version;
  int32_t dtype; /* of key and value: PIPER_FLOAT16 or PIPER_BFLOAT16 */
  piper_cache cache;
  piper_cache_rows rows;
  piper_tensor key; /* [batch, kv_heads, tokens, D] */
  piper_tensor value;
} piper_cache_write_args;

typedef struct piper_cache_read_args {
  int32_t abi_version;
  int32_t dtype; /* of the outputs */
  piper_cache cache;
  piper_cache_rows rows;
  void* key; /* dense [batch, kv_heads, tokens, D], 16-byte aligned */
  void* value;
} piper_cache_read_args;

typedef struct piper_cache_attention_args {
  int32_t abi_version;
  int32_t dtype; /* of query and output */
  float scale;   /* finite and positive */
  int32_t reserved;
  int64_t heads; /* query heads, a multiple of cache.kv_heads: head h reads K/V head h / (heads / kv_heads) */
  piper_cache cache;
  piper_cache_rows rows;
  piper_tensor query; /* [batch, heads, tokens, D] */
  /* NULL: row i sees positions <= starts[b] + i.  Else bytes [batch, tokens, tokens], rows mask_stride_row
   * apart, sequences mask_stride_batch (0: one mask for all): row i sees positions < starts[b] and
   * starts[b] + j where mask[b][i][j] != 0 and j < counts[b] */
  const uint8_t* mask;
  int64_t mask_stride_batch;
  int64_t mask_stride_row;
  /* NULL: every page.  Else dense [batch, kv_heads, tokens, budget]: row i sees, of the positions up to its
   * own, those in these pages of its sequence.  Negative entries and such beyond the table name no page; a page
   * named twice counts twice.  Not together with a mask */
  const int32_t* selected;
  int64_t budget;
  void* output; /* dense [batch, heads, tokens, D], 16-byte aligned; rows that see nothing, and rows >= counts[b], are zero */
  void* workspace; /* piper_cache_attention_workspace_bytes, 16-byte aligned; NULL if that is 0 */
  int64_t workspace_bytes;
} piper_cache_attention_args;

typedef struct piper_cache_select_args {
  int32_t abi_version;
  int32_t dtype; /* of the query */
  int64_t heads;
  piper_cache cache; /* key, value and their scales are not read and may be NULL */
  piper_cache_rows rows;
  piper_tensor query;
  int64_t budget;  /* pages per row and K/V head */
  int32_t* output; /* dense [batch, kv_heads, tokens, budget] */
  void* workspace; /* piper_cache_select_workspace_bytes, 16-byte aligned; NULL if that is 0 */
  int64_t workspace_bytes;
} piper_cache_select_args;

int piper_cache_abi_version(void);

/* Quantise the rows into their slots, and take the bounds of every page whose last slot is among them (from the
 * keys that it holds then).  Slots that are no row's keep their bytes.  Two rows of one call must not name the
 * same slot, nor two sequences a page that either fills: what such a slot or page holds afterwards is unspecified. */
int piper_cache_write(const piper_cache_write_args* args, void* stream);

/* The values that the rows' slots stand for, rounded to the output type; rows >= counts[b] are zero. */
int piper_cache_read(const piper_cache_read_args* args, void* stream);

/* softmax(scale q k) v over what each row sees.  Scores, softmax statistics and sums in FP32. */
int piper_cache_attention(const piper_cache_attention_args* args, void* stream);

/* Workspace bytes of piper_cache_attention for these arguments on the current device (pointers are not read). */
int piper_cache_attention_workspace_bytes(const piper_cache_attention_args* args, int64_t* bytes);

/* Per row and K/V head: the page of the row's own position, and the budget - 1 pages before it whose bounds allow
 * the largest scores, ties to the lower page; ascending, then -1.  With the query row of head h held as INT8 codes
 * c_h and scale s_h by the cache's rule, a page's score is
 *     max over the K/V head's query heads of (sum_d max(c_h[d], 0) upper[d] + min(c_h[d], 0) lower[d]) * s_h,  times bound_scale:
 * the sum in integers, both products in FP32, so every order of evaluation gives the same score.  A page that the
 * table does not name has score -inf.  Heads whose query row is not finite are left out of the maximum; where all
 * are, every page has score -inf.  Rows >= counts[b], and rows whose position the table does not reach, are
 * all -1. */
int piper_cache_select(const piper_cache_select_args* args, void* stream);
int piper_cache_select_workspace_bytes(const piper_cache_select_args* args, int64_t* bytes);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* PIPER_CACHE_H */
