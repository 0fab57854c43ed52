/* sln.h -- C ABI of the layer norm in libtda_hip.so.
 *
 *   sln_fwd   y = (x - mean) rstd w + b over the last axis, rstd = 1 / sqrt(var + eps); without `center` the mean
 *             is left out (RMS norm)
 *   sln_bwd   dx, and the sums over the rows dw = sum dy (x - mean) rstd, db = sum dy
 *
 * Conventions, element types and error codes are those of sda.h (and tda.h): device pointers, all work
 * enqueued on `stream` of the current device, no allocation, no synchronisation, thread-safe; return value 0
 * or a negative code (sln_error_string).
 */
#ifndef SLN_H_
#define SLN_H_

#include "sda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SLN_ABI_VERSION 1
#define SLN_MAX_WIDTH 16384

/* error codes beyond those of tda.h and sda.h */
#define SLN_ERR_WIDTH -40  /* width not in 1 .. SLN_MAX_WIDTH */
#define SLN_ERR_EPS   -41  /* eps negative or not finite */

/* Rows x (batch, heads, rows, width) of any alignment of whole elements, unit last stride, other strides not
 * negative. */
typedef struct sln_fwd_args {
  int32_t abi_version;      /* SLN_ABI_VERSION */
  int32_t dtype;            /* of x, y: TDA_DTYPE_F32, TDA_DTYPE_BF16 or SDA_DTYPE_F16 */
  int64_t batch, heads, rows, width;
  float   eps;
  int32_t center;           /* 1: the mean is taken off */
  int32_t weight_dtype;     /* of weight and bias: dtype or TDA_DTYPE_F32 */
  int32_t weight_heads;     /* 1: weight and bias are (heads, width), else (width); contiguous */
  tda_tensor x, y;
  const void* weight;       /* optional */
  const void* bias;         /* optional */
  float*  stats;            /* optional: (batch, heads, rows, 2) mean and rstd, which the backward reads */
} sln_fwd_args;

typedef struct sln_bwd_args {
  int32_t abi_version;
  int32_t dtype;
  int64_t batch, heads, rows, width;
  int32_t weight_dtype, weight_heads;
  int32_t center;
  int32_t reserved;
  tda_tensor x, dy, dx;     /* dx.data may be NULL: not wanted */
  const void* weight;
  const float* stats;       /* the forward's */
  void*   dweight;          /* optional, like weight */
  void*   dbias;            /* optional, like bias */
  void*   workspace;        /* sln_bwd_workspace_bytes(args) bytes, 16-byte aligned */
  size_t  workspace_bytes;
} sln_bwd_args;

int32_t     sln_abi_version(void);
const char* sln_error_string(int32_t code);

/* Buffer size (bytes) of a call; 0 when the arguments it depends on are invalid. */
size_t  sln_bwd_workspace_bytes(const sln_bwd_args* args);

/* Checks alone, without a launch. */
int32_t sln_validate_fwd(const sln_fwd_args* args);
int32_t sln_validate_bwd(const sln_bwd_args* args);

int32_t sln_fwd(const sln_fwd_args* args, void* stream);
int32_t sln_bwd(const sln_bwd_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SLN_H_ */
