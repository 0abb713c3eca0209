// Interface between the C entry points of the linear cross entropy (lce.cu) and
// its tensor-core kernels (lce_gemm.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ttt {

// Head of the state buffer, written by the forward.
struct LceHead {
  int n_active;     // participating rows, listed first
  float denom;      // N of the mean, 1 otherwise
  float mw_max;     // largest |mask weight| of the participating rows
  unsigned ticket;  // blocks of the forward's last kernel that are done
};

// The row coefficients c of a gradient. One upstream value for all rows (mean, sum)
// multiplies the outputs in fp32, and the stored derivatives carry the mask weights
// only: with weights of 1 the entry of a target is then p - 1, which 16 bits hold far
// better than a multiple of 1 / N (1 / 6144 alone is off by 0.2 % in bf16). Per-row
// upstream values are part of what is stored.
struct LceCoef {
  const LceHead* head;
  const float* dloss;        // the one upstream value, or null
  const float* mw;           // mask weights by slot
  const float* coef;         // stored coefficients by slot, or null: the mask weights
  const unsigned* max_bits;  // bits of the largest magnitude to store, or null: the largest weight

  __device__ __forceinline__ float row(int slot) const { return coef != nullptr ? coef[slot] : mw[slot]; }
  // Power of two that brings the largest magnitude to store near 2^13 (1 for 0, inf and NaN).
  __device__ __forceinline__ float scale() const {
    const float big = max_bits != nullptr ? __uint_as_float(*max_bits) : head->mw_max;
    if (!(big > 0.f && big < INFINITY)) return 1.f;
    int e;
    frexpf(big, &e);  // big < 2^e
    return ldexpf(1.f, max(-100, min(100, 13 - e)));
  }
  // What the sums over stored derivatives are multiplied by.
  __device__ __forceinline__ float out() const { return (dloss != nullptr ? *dloss / head->denom : 1.f) / scale(); }
};

// A tile is formed by a pair of CTAs: 256 rows, 128 in each CTA. Rows are tokens
// or, for the weight gradient, vocabulary entries. The fp32 accumulators of a tile
// fill half of each CTA's tensor memory, so that one tile is formed while the
// previous one is read out.
constexpr int kLceBM = 256;
constexpr int kLceBN = 256;      // single-product tiles
constexpr int kLceBNDual = 128;  // two accumulators side by side
constexpr int kLcePanel = 64;    // columns of an operand box (128 bytes, the swizzle's width)
constexpr int kLceBK = 128;      // contraction of a stage (64 in the dual kinds)

enum LceKind : int {
  kLceStats = 0,      // z -> per-row (max, sum) of the half tile, z at the target
  kLceGrad = 1,       // z -> G
  kLceDualStats = 2,  // z, A -> per-row sum P A of the half tile, its largest |P A|, A at the target
  kLceDualGrad = 3,   // z, A -> G, D
  kLceProd = 4,       // G w (+ D w + G uw) as fp32 partial rows, and G^T h (+ D^T h + G^T uh) as 16-bit rows
};

struct LceGemm {
  // Logit kinds: a = {h, uh}, b = {w, uw}, K-major operands.
  CUtensorMap a[2], b[2];
  CUtensorMap out[2];  // logit gradient kinds: stores of G and D
  // kLceProd, per product: the stored derivative as K-major (gk) and MN-major (gm)
  // operand, and what it meets, MN-major: w or uw (bw), h or uh (bh).
  CUtensorMap gk[2], gm[2], bw[2], bh[2];
  CUtensorMap dw_out;  // kLceProd: stores of the weight gradient's rows (when dim % 8 == 0)
  const LceHead* head;
  LceCoef coef;
  // rows of the state / work arrays, indexed by row slot
  const int* tgt;
  const float *top2, *inv_l;
  const float* rho;
  float2* part;      // statistics kinds: [2 * n_tiles][n_pad]
  float* ztgt;       // statistics kinds: value at the target
  float* acc;        // kLceProd: [splits][n_pad][dim_pad], or null (no hidden gradient)
  uint16_t* dw;      // kLceProd: row 0 of the piece, [cols][dim], or null (no weight gradient)
  unsigned* ticket;  // next tile of the following kLceProd launch (zeroed by the gradient kinds)
  int n_pad;         // row slots (multiple of 256)
  int dim, dim_pad;
  int col0, cols;    // the vocabulary piece
  int seg_w, seg_h;  // kLceProd: products in use (bits) of the hidden and of the weight gradient;
                     // dual kinds: seg_w bit 0 uh given, bit 1 uw given
  int splits;        // kLceProd: shares of the piece's columns in the hidden gradient
  int accumulate;    // kLceProd: add to acc instead of overwriting it
  int* err;
  int* err_host;
};

cudaError_t launch_lce_gemm(const LceGemm& p, int kind, bool bf16, int sms, cudaStream_t stream);

}  // namespace ttt
