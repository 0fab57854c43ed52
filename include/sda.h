/* sda.h -- C ABI of the softmax differential attention operators in libtda_hip.so.
 *
 *   sda_fwd / sda_bwd        O = (softmax(s q1 k1^T + M) - lambda softmax(s q2 k2^T + M)) v
 *   sda_rotary               rotary positions of several axes on up to four tensors
 *   sda_kv4_append / _read / _attend
 *                            a key/value cache held in 4 bits, and the attention over it
 *
 * They stand beside the threshold operators of tda.h and share its tensor type, its error codes
 * and its conventions: device pointers, all work enqueued on `stream` (a hipStream_t) of the
 * current device, no allocation, no synchronisation, thread-safe; return value 0 or a negative
 * code (sda_error_string).  Every argument is checked before any launch; what lies in device
 * memory (lengths, offsets) is clamped to its range by the kernels.
 */
#ifndef SDA_H_
#define SDA_H_

#include "tda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SDA_ABI_VERSION 1

/* element types beyond TDA_DTYPE_F32 / TDA_DTYPE_BF16 */
#define SDA_DTYPE_F16 2

/* error codes beyond those of tda.h */
#define SDA_ERR_HEADS   -20  /* heads not a multiple of kv_heads */
#define SDA_ERR_SCALE   -21  /* scale not in 1e-30 .. 1e30 */
#define SDA_ERR_AXES    -22  /* axes, sections or rotated width out of range */
#define SDA_ERR_CACHE   -23  /* 4-bit cache: capacity, lengths or row count out of range, or start or
                                counts overlapping lengths */

/* Softmax differential attention.  Query row i of sequence b stands at position off_b + i and
 * sees key j when j < len_b and (causal) j <= off_b + i; a row that sees no key is zero.  Keys
 * behind every row's sight may hold anything. */
typedef struct sda_fwd_args {
  int32_t abi_version;      /* SDA_ABI_VERSION */
  int32_t dtype;            /* TDA_DTYPE_F32, TDA_DTYPE_BF16 or SDA_DTYPE_F16: q, k, v, out */
  int32_t causal;           /* 1: keys behind the row's own position are hidden */
  float   scale;            /* s, 1e-30 .. 1e30 */
  int64_t batch, heads, kv_heads;   /* query head h reads key head h / (heads / kv_heads) */
  int64_t seq_len, seq_len_kv;      /* query rows, key rows */
  int64_t head_dim, v_head_dim;     /* (64, 64), (64, 128), (128, 128) or (128, 256) */
  tda_tensor q1, k1, q2, k2, v;     /* (B, H, Nq, d), (B, Hk, Nk, d), ..., (B, Hk, Nk, dv) */
  tda_tensor out;                   /* (B, H, Nq, dv) */
  tda_tensor out2;          /* optional (data may be NULL), f32 rows: softmax(s q2 k2^T + M) v, and */
  tda_tensor out_low;       /* with it but for f32, rows of dtype: what out's rounding left out.  The
                               backward's row sums of the outputs keep 16 bits with them: from the
                               rounded outputs alone they would cost its gradients half again the error
                               that their own rounding has */
  const void* lambda_param; /* element (b, h, i) at b ls[0] + h ls[1] + i ls[2] */
  int64_t lambda_stride[3]; /* 0: the same along that axis */
  int32_t lambda_dtype;     /* as dtype, but of its own */
  int32_t reserved;
  int64_t q_offset;         /* off_b, unless q_offsets is given */
  const int32_t* q_offsets; /* optional (batch): off_b */
  const int32_t* kv_lens;   /* optional (batch): len_b, clamped to [0, Nk]; NULL: Nk */
  float*  lse;              /* optional: 2 B H Nq floats, log2 of each branch's softmax sum (with
                               its maximum), which the backward reads */
  void*   workspace;        /* sda_fwd_workspace_bytes(args) bytes, 16-byte aligned */
  size_t  workspace_bytes;
} sda_fwd_args;

typedef struct sda_bwd_args {
  int32_t abi_version, dtype, causal;
  float   scale;
  int64_t batch, heads, kv_heads, seq_len, seq_len_kv, head_dim, v_head_dim;
  tda_tensor q1, k1, q2, k2, v;     /* the forward's */
  tda_tensor out, out2, out_low, dout;  /* the forward's outputs and the upstream gradient.  Unless seq_len
                               is a multiple of 32, rows of q1, q2 and dout may not overlap
                               (stride[2] >= width) */
  tda_tensor dq1, dk1, dq2, dk2, dv;
  const void* lambda_param;
  int64_t lambda_stride[3];
  int32_t lambda_dtype;
  int32_t reserved;
  int64_t q_offset;
  const int32_t* q_offsets;
  const int32_t* kv_lens;
  const float* lse;
  void*   dlambda;          /* optional: the gradient of lambda_param's distinct elements, in its
                               type, contiguous in (b, h, i) order over the axes whose stride is
                               not 0 */
  void*   workspace;        /* sda_bwd_workspace_bytes(args) bytes, 16-byte aligned */
  size_t  workspace_bytes;
} sda_bwd_args;

/* Rotary positions: pair p of a row at (b, n) turns by angle a = positions[axis(p)][b][n]
 * inv_freq[p]: (x, y) -> (x cos a - y sin a, y cos a + x sin a), its parts at p and p + rot/2, or
 * (interleaved) at 2 p and 2 p + 1; the values from rot on are copied.  inverse turns back,
 * which is the gradient. */
#define SDA_MAX_AXES 4
#define SDA_MAX_ROTARY 4
typedef struct sda_rotary_args {
  int32_t abi_version;
  int32_t dtype;            /* TDA_DTYPE_F32, TDA_DTYPE_BF16 or SDA_DTYPE_F16 */
  int32_t interleaved, inverse;
  int64_t batch, seq_len, head_dim;
  int64_t rot;              /* rotated values of a row: even, at most head_dim */
  int32_t axes;             /* 1 .. SDA_MAX_AXES */
  int32_t sections[SDA_MAX_AXES];   /* pairs of each axis, in order; they add up to rot / 2 */
  int32_t count;            /* tensors: 1 .. SDA_MAX_ROTARY */
  int64_t heads[SDA_MAX_ROTARY];
  tda_tensor x[SDA_MAX_ROTARY], y[SDA_MAX_ROTARY];  /* (B, heads, N, d); y may be x */
  const void* positions;    /* (axes, B, N) integers */
  int64_t position_stride[3];
  int32_t position_dtype;   /* bytes of one: 4 or 8 */
  int32_t reserved;
  const float* inv_freq;    /* rot / 2, contiguous */
} sda_rotary_args;

/* The 4-bit cache.  Each row of k1, k2 (d values) and v (dv values) is held in groups of 64
 * values x: m = bf16(min x), s = bf16((max x - m) / 15) in 32 bits, code =
 * min(max(rint((x - m) / s), 0), 15) (ties to even, 0 when s < 2^-100), value m + s code; a group with a NaN or an infinity, or whose
 * s is not finite, reads as NaN.  Three buffers of
 * sda_kv4_bytes() bytes each: for (b, head) the codes of capacity rows (rounded up to four; d / 2
 * bytes a row), then behind all codes the groups' (m, s); their order within is the kernels' own.
 * capacity is at most 2^24. */
typedef struct sda_kv4 {
  int64_t batch, kv_heads, capacity, head_dim, v_head_dim;
  void*    k1;
  void*    k2;
  void*    v;
  int32_t* lengths;         /* (batch) rows held */
} sda_kv4;

typedef struct sda_kv4_append_args {
  int32_t abi_version;
  int32_t dtype;            /* of the rows: F32, BF16 or F16 */
  sda_kv4 cache;
  int64_t rows;             /* n */
  tda_tensor k1, k2, v;     /* (B, Hk, n, d), (B, Hk, n, d), (B, Hk, n, dv) */
  const int32_t* start;     /* optional (batch): first row written; NULL: lengths */
  const int32_t* counts;    /* optional (batch): rows of each sequence that count (clamped to
                               [0, n]); NULL: n */
} sda_kv4_append_args;      /* rows at start + i < capacity are written; lengths becomes
                               min(start + count, capacity).  start and counts may be lengths, but no
                               other array that overlaps it */

typedef struct sda_kv4_read_args {
  int32_t abi_version;
  int32_t dtype;
  sda_kv4 cache;
  int64_t rows;             /* n <= capacity: rows 0 .. n - 1; rows past a length read as zeros, in F16
                               values past +-65504 as +-65504 */
  tda_tensor k1, k2, v;     /* outputs */
} sda_kv4_read_args;

typedef struct sda_kv4_attend_args {
  int32_t abi_version;
  int32_t dtype;            /* of q1, q2, out: F32, BF16 or F16 */
  sda_kv4 cache;
  int64_t heads, seq_len;   /* the queries are the last seq_len positions of each sequence */
  float   scale;
  int32_t lambda_dtype;
  tda_tensor q1, q2, out;
  const void* lambda_param;
  int64_t lambda_stride[3];
  void*   workspace;        /* sda_kv4_attend_workspace_bytes(args) */
  size_t  workspace_bytes;
} sda_kv4_attend_args;

int32_t     sda_abi_version(void);
const char* sda_error_string(int32_t code);

/* Buffer sizes (bytes) of a call; 0 when the arguments they depend on are invalid. */
size_t  sda_fwd_workspace_bytes(const sda_fwd_args* args);
size_t  sda_bwd_workspace_bytes(const sda_bwd_args* args);
size_t  sda_kv4_attend_workspace_bytes(const sda_kv4_attend_args* args);
size_t  sda_kv4_bytes(int64_t batch, int64_t kv_heads, int64_t capacity, int64_t width);

/* Checks alone, without a launch. */
int32_t sda_validate_fwd(const sda_fwd_args* args);
int32_t sda_validate_bwd(const sda_bwd_args* args);
int32_t sda_validate_rotary(const sda_rotary_args* args);
int32_t sda_validate_kv4_append(const sda_kv4_append_args* args);
int32_t sda_validate_kv4_read(const sda_kv4_read_args* args);
int32_t sda_validate_kv4_attend(const sda_kv4_attend_args* args);

int32_t sda_fwd(const sda_fwd_args* args, void* stream);
int32_t sda_bwd(const sda_bwd_args* args, void* stream);
int32_t sda_rotary(const sda_rotary_args* args, void* stream);
int32_t sda_kv4_append(const sda_kv4_append_args* args, void* stream);
int32_t sda_kv4_read(const sda_kv4_read_args* args, void* stream);
int32_t sda_kv4_attend(const sda_kv4_attend_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SDA_H_ */
