/*
 * ttt_ops.h - C ABI of the model-side operators of libttt_attn.so: layer norm
 * and the linear cross entropy (the token loss of hidden * weight^T without the
 * logits in memory), each with its first and its second gradient.
 *
 * Conventions, in addition to those of ttt_attn.h (status codes, streams, the
 * error word `err`, no allocation, no host synchronization):
 *  - Matrices are row-major with unit column stride; `*_stride` is the row
 *    stride in elements. Inputs may have any row stride >= 0 that the comment
 *    on the field allows; outputs are contiguous unless a stride is given.
 *  - `work` is a caller-owned device buffer of at least the bytes that the
 *    operator's *_work_bytes function returns, 256-byte aligned. It holds
 *    nothing between calls.
 *  - Results do not depend on the run: every sum has a fixed order.
 */
#ifndef TTT_OPS_H_
#define TTT_OPS_H_

#include "ttt_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types, continuing enum ttt_dtype. */
#define TTT_F32 2

/* ------------------------------------------------------------ layer norm */
/* y = (x - mean) * rstd * w + b over rows of dim elements,
 * rstd = (var + eps)^-1/2 with the biased variance. */
#define TTT_NORM_MAX_DIM 16384
typedef struct {
  int64_t rows;    /* 0 .. 2^31 - 1 */
  int32_t dim;     /* 1 .. TTT_NORM_MAX_DIM */
  int32_t dtype;   /* of x, y and their gradients: TTT_F16, TTT_BF16 or TTT_F32 */
  int32_t p_dtype; /* of w, b and their gradients: dtype or TTT_F32 */
  float eps;
} ttt_norm_problem;

typedef struct {
  ttt_norm_problem pb;
  const void* x;
  int64_t x_stride;
  const void* w; /* NULL: ones */
  const void* b; /* NULL: zeros */
  void* y;
  float* mean; /* [rows], may be NULL together with rstd (no gradient wanted) */
  float* rstd;
} ttt_norm_fwd_args;
int ttt_norm_fwd(const ttt_norm_fwd_args* a, void* stream);

/* dx = rstd P(dy w), dw = sum dy xh, db = sum dy, with xh = (x - mean) rstd and
 * P(u) = u - m(u) - xh m(u xh), m = the row mean. */
typedef struct {
  ttt_norm_problem pb;
  const void* x;
  const void* dy;
  int64_t x_stride, dy_stride;
  const void* w; /* NULL: ones */
  const float* mean;
  const float* rstd;
  void* dx; /* NULL: not wanted */
  void* dw; /* NULL: not wanted */
  void* db; /* NULL: not wanted */
  void* work;
  int64_t work_bytes;
} ttt_norm_bwd_args;
int ttt_norm_bwd(const ttt_norm_bwd_args* a, void* stream);

/* Gradients of <dx, ux> + <dw, uw> + <db, ub> with respect to x, w and dy. */
typedef struct {
  ttt_norm_problem pb;
  const void* x;
  const void* dy;
  const void* ux; /* NULL: zeros */
  int64_t x_stride, dy_stride, ux_stride;
  const void* w;  /* NULL: ones */
  const void* uw; /* NULL: zeros */
  const void* ub; /* NULL: zeros */
  const float* mean;
  const float* rstd;
  void* gx;
  void* gw; /* NULL: not wanted */
  void* gdy;
  void* work;
  int64_t work_bytes;
} ttt_norm_bwd2_args;
int ttt_norm_bwd2(const ttt_norm_bwd2_args* a, void* stream);

/* Bytes of work space of ttt_norm_bwd and ttt_norm_bwd2 (the per-block sums of
 * the parameter gradients); depends on the current device's SM count. */
int64_t ttt_norm_work_bytes(const ttt_norm_problem* pb);

#ifdef __cplusplus
}
#endif

#endif /* TTT_OPS_H_ */
