/* spa.h -- C ABI of the paged key/value cache of softmax differential attention in libtda_hip.so.
 *
 *   spa_append   rows of new positions enter the pages, queries and keys turned by their rotary
 *                positions on the way
 *   spa_attend   softmax differential attention of the new positions over the pages
 *
 * They stand beside the operators of sda.h and share its conventions, element types and error codes
 * (those of tda.h among them): device pointers, all work enqueued on `stream` of the current device,
 * no allocation, no synchronisation, thread-safe; return value 0 or a negative code
 * (spa_error_string).  Every argument is checked before any launch; what lies in device memory (page
 * numbers, lengths, starts, counts) is clamped to its range by the kernels.
 */
#ifndef SPA_H_
#define SPA_H_

#include "sda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SPA_ABI_VERSION 1

/* error codes beyond those of tda.h and sda.h */
#define SPA_ERR_PAGES -30  /* pages, page size or table out of range */
#define SPA_ERR_ROWS  -31  /* sequences, starts or counts do not fit the rows */

/* The pages: k1, k2 (pages, kv_heads, page_size, head_dim) and v (..., v_head_dim), contiguous, 16-byte
 * aligned, of the call's dtype.  page_size is 16, 32, 64, 128 or 256; (head_dim, v_head_dim) is (64, 64),
 * (64, 128), (128, 128) or (128, 256). */
typedef struct spa_cache {
  int64_t pages, kv_heads, page_size, head_dim, v_head_dim;
  void* k1;
  void* k2;
  void* v;
} spa_cache;

/* Whose rows a call has.  Position p of sequence s is row p % page_size of page table[s][p / page_size];
 * an entry that is no page of the cache stands for rows of zeros, and rows appended there are dropped.
 * Sequence s held lengths[s] positions; its new row i stands at lengths[s] + i.  Row tensors have the shape
 * (lead, heads, rows, width): with starts lead is 1 and sequence s has the rows starts[s] .. starts[s + 1] - 1
 * (starts must not decrease), else lead is the number of sequences and s has the first counts[s] rows of
 * entry s (all of them without counts).  Rows of no sequence are read by nothing; they are zero in outputs. */
typedef struct spa_rows {
  int64_t sequences, rows;
  const int32_t* table;     /* (sequences, table_len) */
  int64_t table_stride;     /* elements from one sequence to the next */
  int64_t table_len;
  const int32_t* lengths;   /* (sequences); clamped to +-2^30 */
  const int32_t* starts;    /* optional (sequences + 1): packed rows; clamped to [0, rows] */
  const int32_t* counts;    /* optional (sequences), not with starts; clamped to [0, rows] */
} spa_rows;

typedef struct spa_append_args {
  int32_t abi_version;      /* SPA_ABI_VERSION */
  int32_t dtype;            /* TDA_DTYPE_F32, TDA_DTYPE_BF16 or SDA_DTYPE_F16 */
  spa_cache cache;
  spa_rows at;
  tda_tensor k1, k2, v;     /* (lead, kv_heads, rows, head_dim or v_head_dim) */
  int64_t heads;            /* of the queries; 0: none */
  tda_tensor q1, q2;        /* (lead, heads, rows, head_dim) */
  tda_tensor q1_out, q2_out;/* the same, turned; may be q1, q2 */
  int64_t rot;              /* rotated values of a row: even, 0 .. head_dim; 0: rows enter as they are */
  int32_t axes;             /* 1 .. SDA_MAX_AXES when rot > 0 */
  int32_t sections[SDA_MAX_AXES];   /* pairs of each axis, in order; they add up to rot / 2 */
  int32_t interleaved;      /* pair p: values 2 p and 2 p + 1; else p and p + rot / 2 */
  int32_t position_dtype;   /* bytes of one: 4 or 8 */
  const void* positions;    /* optional (axes, lead, rows) integers; NULL: a row's place on every axis */
  int64_t position_stride[3];
  const float* inv_freq;    /* rot / 2, contiguous */
} spa_append_args;          /* positions outside 0 .. table_len page_size - 1 are dropped */

/* Row i of sequence s sees the positions up to its own that the table has room for; a row that sees none is
 * zero.  Positions behind it may hold anything. */
typedef struct spa_attend_args {
  int32_t abi_version;
  int32_t dtype;
  spa_cache cache;
  spa_rows at;
  int64_t heads;            /* query head h reads key head h / (heads / kv_heads) */
  int64_t most;             /* rows that any one sequence has, at most (what it costs to be wrong is time); 0: rows */
  float   scale;            /* 1e-30 .. 1e30 */
  int32_t lambda_dtype;
  tda_tensor q1, q2;        /* (lead, heads, rows, head_dim) */
  tda_tensor out;           /* (lead, heads, rows, v_head_dim) */
  const void* lambda_param; /* element (lead entry, h, row) at the strides */
  int64_t lambda_stride[3];
  void*   workspace;        /* spa_attend_workspace_bytes(args) bytes, 16-byte aligned */
  size_t  workspace_bytes;
} spa_attend_args;

int32_t     spa_abi_version(void);
const char* spa_error_string(int32_t code);

/* Buffer size (bytes) of a call; 0 when the arguments it depends on are invalid. */
size_t  spa_attend_workspace_bytes(const spa_attend_args* args);

/* Checks alone, without a launch. */
int32_t spa_validate_append(const spa_append_args* args);
int32_t spa_validate_attend(const spa_attend_args* args);

int32_t spa_append(const spa_append_args* args, void* stream);
int32_t spa_attend(const spa_attend_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SPA_H_ */
