/*
 * q3s_decode.h -- C ABI of the decode step's operators beside the sampler
 * (B200, sm_100a): the paged key/value cache's bookkeeping and append, the
 * attention that reads it, and the 8-bit projections.  Same library and
 * conventions as q3s_sampler.h: every pointer in a descriptor is a DEVICE
 * pointer; calls are asynchronous on `stream`, never allocate and never
 * synchronise; arguments are checked on the host before any CUDA call (a bad
 * one returns Q3S_ERR_INVALID_ARGUMENT and launches nothing,
 * q3s_last_error_string() says why); problems only visible on the device are
 * reported in the optional device word `error_word` (Q3S_DECERR_* bits) and
 * the offending entries are skipped.
 *
 * The reference keeps the cache on the host side of its engine
 * (engine/backend/kv_cache_pool.py, engine/backend/prefix_cache.py) and runs
 * attention and projections inside the fused TensorRT engine; these entry
 * points let the steps around the sampler run from device lengths alone.
 *
 * The cache.  `k_cache` / `v_cache` are [blocks, kv_heads, block_size, dim]
 * with any strides whose last is 1 (a [blocks, block_size, kv_heads, dim]
 * allocation is the same view with two axes swapped).  A slot is
 * block * block_size + place in the block.
 */
#ifndef Q3S_DECODE_H
#define Q3S_DECODE_H

#include <stdint.h>

#include "q3s_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

#define Q3S_DECERR_LENGTHS 1   /* a negative length, or offsets that do not ascend (treated as 0 / cut) */
#define Q3S_DECERR_TABLE 2     /* a row outgrew its block table: it got no blocks */
#define Q3S_DECERR_POOL 4      /* the free ring ran out: this row and later ones that need blocks got none */
#define Q3S_DECERR_TOKENS 8    /* more new tokens than max_tokens: the rest have no slot (Q3S_TABLES_WHOLE_ROWS) */
#define Q3S_DECERR_BLOCK_ID 16 /* a block id or slot outside the cache: its tokens read as zeros / are not stored */
#define Q3S_DECERR_WAIT 32     /* a bounded device wait gave up */

/* Element types of the operators' tensors. */
typedef enum q3s_elem { Q3S_ELEM_F32 = 0, Q3S_ELEM_BF16 = 1, Q3S_ELEM_F16 = 2 } q3s_elem;

#define Q3S_MAX_CACHE_ROWS 65536
#define Q3S_MAX_QUERY_GROUP 16 /* query heads per key/value head */

/* q3s_cache_tables_desc.flags: a row whose new tokens end past max_tokens is
 * refused whole, like one that does not fit its table.  Without it such a row
 * is granted, and its length counts tokens that have no slot: a caller that
 * goes on from those lengths would read places that nothing was written to. */
#define Q3S_TABLES_WHOLE_ROWS 1u

/* Block tables, slot map and positions of one step, from the rows' lengths.
 *
 * Row b holds context_lengths[b] tokens (0 when released[b]) in
 * held = ceil(context / block_size) blocks and gets new_lengths[b] more.  In
 * row order, a row that needs blocks takes them from the front of the free
 * ring while the running sum of needs fits what the ring holds; a row whose
 * tokens do not fit its table, or whose blocks the ring no longer has, is
 * refused: it keeps its length and its new tokens have slot -1.  The blocks of
 * released rows go to the back of the ring, in row order, for the next step;
 * a released row may be given to a new request in the same step.
 *
 * New tokens are numbered row by row: row b's are [query_offsets[b],
 * query_offsets[b+1]).  Entries of slot_map / positions past the last token
 * are -1 / 0, so buffers of a fixed size can be bound to a CUDA graph. */
typedef struct q3s_cache_tables_desc {
  uint32_t struct_size;           /* = sizeof(q3s_cache_tables_desc) */
  int32_t batch;                  /* B, 0..Q3S_MAX_CACHE_ROWS */
  int32_t block_size;             /* tokens per block, >= 1 */
  int32_t max_blocks;             /* columns of block_table */
  const int32_t* context_lengths; /* [B] */
  const int32_t* new_lengths;     /* [B] */
  const uint8_t* released;        /* optional [B], non-zero = the row's request has ended */
  int32_t* block_table;           /* [B, block_table_stride], read and updated */
  int64_t block_table_stride;     /* elements, >= max_blocks */
  int32_t* free_blocks;           /* [ring_size] ring of free block ids, read and updated */
  const int32_t* free_state;      /* [2]: first entry, number of entries */
  int32_t* free_state_out;        /* [2], not overlapping any input */
  int32_t* lengths_out;           /* [B] lengths with the new tokens, not overlapping any input */
  int32_t* query_offsets;         /* [B+1] */
  int64_t* slot_map;              /* [max_tokens] */
  int32_t* positions;             /* [max_tokens] place of the token in its row */
  int32_t* error_word;            /* optional, written (not OR-ed) */
  int32_t ring_size;              /* blocks that the ring can hold, >= 1 */
  int32_t max_tokens;             /* >= 0 */
  uint32_t flags;                 /* Q3S_TABLES_*; a struct_size that ends before this field means 0 */
  uint32_t reserved0;
} q3s_cache_tables_desc;

q3s_status q3s_cache_tables(const q3s_cache_tables_desc* desc, void* stream);

/* cache[slot / block_size, h, slot % block_size] = new[t, h] for keys and
 * values of every token t with slot_map[t] >= 0 (distinct slots). */
typedef struct q3s_cache_append_desc {
  uint32_t struct_size;        /* = sizeof(q3s_cache_append_desc) */
  int32_t tokens;              /* T >= 0 */
  int32_t kv_heads;
  int32_t dim;
  int32_t block_size;
  int32_t blocks;              /* blocks in the cache */
  int32_t elem;                /* q3s_elem of all four tensors */
  int32_t reserved0;
  const void* k;               /* [T, kv_heads, dim], strides below (elements), unit last stride */
  const void* v;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
  const int64_t* slot_map;     /* [T]; < 0 = not stored */
  void* k_cache;               /* [blocks, kv_heads, block_size, dim], strides below (elements) */
  void* v_cache;
  int64_t k_block_stride, k_cache_head_stride, k_place_stride;
  int64_t v_block_stride, v_cache_head_stride, v_place_stride;
  int32_t* error_word;         /* optional, OR-ed: Q3S_DECERR_BLOCK_ID */
} q3s_cache_append_desc;

q3s_status q3s_cache_append(const q3s_cache_append_desc* desc, void* stream);

/* Attention of a batch that shares a prefix.
 *
 * Row b's queries are tokens [query_offsets[b], query_offsets[b+1]), n_b of
 * them (0 = idle row).  Each sees all prefix_length tokens of the shared
 * prefix (blocks prefix_blocks[]), and query i of row b the row's own tokens
 * j <= lengths[b] - n_b + i (blocks block_table[b, :]; lengths count the
 * step's own tokens, which are already in the cache).  Query head h reads
 * key/value head h / (q_heads / kv_heads).  A row that q3s_cache_tables refused
 * has queries but not their keys: with the step's slot_map they see nothing
 * (without, they would be taken for the row's last stored tokens).
 *   out = softmax(scale * q . k) v,   lse = log sum exp(scale * q . k)
 * with 0 and -inf for a query that sees nothing.  Softmax statistics and sums
 * are 32-bit.  For the product with v, as the tensor cores take it,
 * probabilities over the prefix of a large batch are rounded to the cache's
 * type (and divided by the sum of what was rounded: with U its unit roundoff,
 * that moves out by U sum p |v - out| at most), the others held as the sum of
 * two such values.  A key that a query does
 * not see has no part in its result, whatever k and v hold there; an infinity
 * in v of one that it sees makes out that infinity (NaN where the key's
 * probability underflows). */
typedef struct q3s_prefix_attention_desc {
  uint32_t struct_size;        /* = sizeof(q3s_prefix_attention_desc) */
  int32_t batch;               /* B, 0..Q3S_MAX_CACHE_ROWS */
  int32_t tokens;              /* T >= 0: queries in the packed batch */
  int32_t q_heads;
  int32_t kv_heads;            /* divides q_heads, q_heads / kv_heads <= Q3S_MAX_QUERY_GROUP */
  int32_t dim;                 /* 64 or 128 */
  int32_t block_size;          /* 16, 32, 64 or 128 */
  int32_t blocks;              /* blocks in the cache */
  int32_t elem;                /* Q3S_ELEM_BF16 or Q3S_ELEM_F16: q, caches and out */
  int32_t max_blocks;          /* columns of block_table */
  int32_t prefix_length;       /* >= 0 */
  float scale;
  const void* q;               /* [T, q_heads, dim], 16-byte aligned rows */
  int64_t q_token_stride, q_head_stride;
  const void* k_cache;         /* [blocks, kv_heads, block_size, dim]: strides multiples of 8 elements, base 16-byte aligned */
  const void* v_cache;
  int64_t k_block_stride, k_head_stride, k_place_stride;
  int64_t v_block_stride, v_head_stride, v_place_stride;
  const int32_t* query_offsets; /* [B+1] */
  const int32_t* block_table;   /* [B, block_table_stride] */
  int64_t block_table_stride;
  const int32_t* lengths;       /* [B] */
  const int32_t* prefix_blocks; /* [ceil(prefix_length / block_size)]; may be NULL when prefix_length is 0 */
  void* out;                    /* [T, q_heads, dim], 16-byte aligned rows */
  int64_t out_token_stride, out_head_stride;
  float* lse;                   /* optional [T, q_heads] */
  void* workspace;              /* q3s_prefix_attention_workspace() bytes, 16-byte aligned; needs no initial value */
  int64_t workspace_bytes;
  int32_t* error_word;          /* optional, OR-ed */
  const int64_t* slot_map;      /* optional [T]: a query whose slot is negative sees nothing (a struct_size that ends before this field: none) */
} q3s_prefix_attention_desc;

/* Workspace bytes for a descriptor's sizes (its pointers are not read). */
q3s_status q3s_prefix_attention_workspace(const q3s_prefix_attention_desc* desc, int64_t* bytes);
q3s_status q3s_prefix_attention(const q3s_prefix_attention_desc* desc, void* stream);

/* Per-row quantisation: a = max |x_m|, scales[m] = a / 127,
 * values[m] = round to nearest even of x_m * (127 / a), IEEE in 32 bits.  A
 * row with a < 2^-100 gets values 0 and scale 0; one that holds an infinity
 * or a NaN gets values 0 and scale NaN, so that what is made of it is NaN. */
typedef struct q3s_quantize_rows_desc {
  uint32_t struct_size;        /* = sizeof(q3s_quantize_rows_desc) */
  int32_t rows;                /* M >= 0 */
  int32_t cols;                /* K >= 1 */
  int32_t elem;                /* q3s_elem of x */
  const void* x;               /* [M, x_row_stride] */
  int64_t x_row_stride;
  int8_t* values;              /* [M, values_row_stride] */
  int64_t values_row_stride;
  float* scales;               /* [M] */
} q3s_quantize_rows_desc;

q3s_status q3s_quantize_rows(const q3s_quantize_rows_desc* desc, void* stream);

/* y[m, n] = (sum_k a[m, k] * w[n, k]) * a_scales[m] * w_scales[n] (+ bias[n]):
 * 8-bit integers and exact 32-bit sums; the sum's conversion, the two products
 * and the bias are fp32 operations (four roundings of 2^-24, which for fp32 y are
 * the whole error), then y is rounded to its type.  Any operand, the weight too,
 * may be what the call before on the stream writes. */
typedef struct q3s_int8_matmul_desc {
  uint32_t struct_size;        /* = sizeof(q3s_int8_matmul_desc) */
  int32_t rows;                /* M >= 0 */
  int32_t inputs;              /* K: a positive multiple of 16, <= 131056 (so that no sum reaches 2^31) */
  int32_t outputs;             /* N >= 1 */
  int32_t elem;                /* q3s_elem of y */
  int32_t reserved0;
  const int8_t* a;             /* [M, a_row_stride], 16-byte aligned rows */
  int64_t a_row_stride;        /* elements, >= K, a multiple of 16 */
  const float* a_scales;       /* [M] */
  const int8_t* w;             /* [N, w_row_stride]: the Linear's weight (out x in), 16-byte aligned rows */
  int64_t w_row_stride;
  const float* w_scales;       /* [N] */
  const float* bias;           /* optional [N] */
  void* y;                     /* [M, y_row_stride] */
  int64_t y_row_stride;        /* elements, >= N */
  int32_t* error_word;         /* optional, OR-ed: Q3S_DECERR_WAIT */
} q3s_int8_matmul_desc;

q3s_status q3s_int8_matmul(const q3s_int8_matmul_desc* desc, void* stream);

/* A Linear: quantise x, then the product of its values and scales (the
 * product's a and a_scales are the quantisation's outputs, and y has x's
 * type).  One launch for a few rows, two otherwise. */
q3s_status q3s_int8_linear(const q3s_quantize_rows_desc* quantize, const q3s_int8_matmul_desc* product, void* stream);

/* sizeof() of the descriptors above as compiled (which: 0 = cache_tables,
 * 1 = cache_append, 2 = prefix_attention, 3 = quantize_rows, 4 = int8_matmul). */
uint32_t q3s_decode_desc_size(int32_t which);

#ifdef __cplusplus
}
#endif

#endif /* Q3S_DECODE_H */
