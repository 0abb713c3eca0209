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

/* ---------------------------------------------------- linear cross entropy */
/* Token losses of z = h w^T (h [n, dim], w [vocab, dim], 16-bit), never stored:
 *   ce_i = log sum_j exp(z_ij) - z_{i t_i},   l_i = m_i ce_i
 *   loss = l (TTT_LCE_NONE), sum_i l_i (TTT_LCE_SUM), or
 *          sum_i l_i / N (TTT_LCE_MEAN) with N = max(1, sum_i m_i), and N = n without
 *          a mask; rows with an ignored target count in N (the rule of the meta step's token loss).
 * A row takes part if m_i != 0 and t_i != ignore_index. The others are not read:
 * their loss and gradients are exactly 0 whatever h holds there. A target of a
 * participating row outside [0, vocab) is reported through `err`
 * (TTT_ERR_WORD_TARGET) and the row is left out; with `err` set, later launches
 * that get the word return at once, as for a wait that ran out. */
#define TTT_ERR_WORD_TARGET 0x10000000
enum ttt_lce_reduction { TTT_LCE_NONE = 0, TTT_LCE_MEAN = 1, TTT_LCE_SUM = 2 };
enum ttt_lce_mask { TTT_LCE_MASK_NONE = 0, TTT_LCE_MASK_F32 = 1, TTT_LCE_MASK_U8 = 2 /* bool */ };

typedef struct {
  int64_t n;       /* rows, 0 .. 2^24 */
  int64_t vocab;   /* 1 .. 2^24 */
  int32_t dim;     /* 1 .. 65536 */
  int32_t dtype;   /* TTT_F16 or TTT_BF16, of h, w and their gradients */
  int32_t reduction;
  int32_t mask_kind;
  int64_t ignore_index;
} ttt_lce_problem;

/* `state`: what the forward keeps for the gradients (row list, row statistics;
 * ttt_lce_state_bytes, 256-byte aligned), read-only afterwards. */
typedef struct {
  ttt_lce_problem pb;
  const void* h;
  int64_t h_stride; /* any */
  const void* w;    /* 16-byte aligned */
  int64_t w_stride; /* >= dim, a multiple of 8 */
  const int64_t* targets; /* [n] */
  const void* mask;       /* [n] of mask_kind, or NULL */
  float* loss;            /* [n] or [1] */
  void* state;
  int32_t need_state; /* 0: no gradient will be asked for; state is then only scratch (a few rows take a
                         shorter path), 1 otherwise */
  int32_t* err;
  void* work;
  int64_t work_bytes;
} ttt_lce_fwd_args;
int ttt_lce_fwd(const ttt_lce_fwd_args* a, void* stream);

/* With c_i = dloss m_i / N (dloss_i m_i for TTT_LCE_NONE): G = c (P - onehot(t)),
 * dh = G w, dw = G^T h. h itself is not asked for: `state` holds its participating rows. */
typedef struct {
  ttt_lce_problem pb;
  const void* w;
  int64_t w_stride;
  const void* state;
  const float* dloss; /* [n] or [1] */
  void* dh;           /* [n, dim], NULL: not wanted */
  void* dw;           /* [vocab, dim], NULL: not wanted */
  int32_t* err;
  void* work;
  int64_t work_bytes;
} ttt_lce_bwd_args;
int ttt_lce_bwd(const ttt_lce_bwd_args* a, void* stream);

/* Gradients of <dh, uh> + <dw, uw> with respect to h, w and dloss: with
 * A = uh w^T + h uw^T, rho_i = sum_j P_ij A_ij and D = c P (A - rho):
 * gh = D w + G uw, gw = D^T h + G^T uh, d/dc_i = rho_i - A_{i t_i}. */
typedef struct {
  ttt_lce_problem pb;
  const void* w;
  int64_t w_stride;
  const void* uh; /* [n, dim], any row stride; NULL: zeros */
  int64_t uh_stride;
  const void* uw; /* [vocab, dim], like w; NULL: zeros */
  int64_t uw_stride;
  const void* state;
  const float* dloss;
  void* gh;      /* NULL: not wanted */
  void* gw;      /* NULL: not wanted */
  float* gdloss; /* [n] or [1]; NULL: not wanted */
  int32_t* err;
  void* work;
  int64_t work_bytes;
} ttt_lce_bwd2_args;
int ttt_lce_bwd2(const ttt_lce_bwd2_args* a, void* stream);

/* Copies a [vocab, dim] 16-bit matrix with any row stride into rows that the entry
 * points above accept: dst_stride >= dim, a multiple of 8, dst 16-byte aligned. */
int ttt_lce_pad_weight(const void* src, int64_t src_stride, void* dst, int64_t dst_stride, int64_t vocab, int32_t dim,
                       void* stream);

int64_t ttt_lce_state_bytes(const ttt_lce_problem* pb);
/* pass: 0 forward, 1 gradient, 2 second gradient. The gradients keep the
 * derivative of the logits of one piece of the vocabulary at a time in 16 bits
 * (up to 512 MB, more only when 2048 columns need it). Depends on the current
 * device's SM count. */
int64_t ttt_lce_work_bytes(const ttt_lce_problem* pb, int pass);

#ifdef __cplusplus
}
#endif

#endif /* TTT_OPS_H_ */
