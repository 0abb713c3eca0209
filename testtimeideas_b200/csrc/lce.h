// Interface between the C entry points of the linear cross entropy (lce.cu) and
// its tensor-core kernels (lce_gemm.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ttt {

// Head of the state buffer, written by the forward.
struct LceHead {
  int n_active;  // participating rows, listed first
  float denom;   // N of the mean, 1 otherwise
};
// Head of the work space of a gradient.
struct LceScale {
  float scale;        // power of two that the stored derivatives carry
  float inv;          // 1 / scale
  unsigned max_bits;  // second gradient: bits of the largest |stored value| / scale
};

// Tile sides. Rows of a tile are tokens (or, for the weight gradient, vocabulary
// entries); the fp32 accumulators of a tile fill half of tensor memory, so that
// one tile is formed while the previous one is read out.
constexpr int kLceBM = 128;
constexpr int kLceBN = 256;     // single-product tiles
constexpr int kLceBNDual = 128; // two accumulators side by side
constexpr int kLceBK = 64;

enum LceKind : int {
  kLceStats = 0,      // z -> per-row (max, sum) of the tile, z at the target
  kLceGrad = 1,       // z -> G
  kLceDualStats = 2,  // z, A -> per-row sum P A of the tile, its largest |P A|, A at the target
  kLceDualGrad = 3,   // z, A -> G, D
  kLceDH = 4,         // G w (+ D w + G uw): fp32 partial rows
  kLceDW = 5,         // G^T h (+ D^T h + G^T uh): 16-bit rows of the weight gradient
};

struct LceGemm {
  // Operand maps. Logit kinds: a = {h, uh}, b = {w, uw}, K-major. kLceDH: per
  // segment a = stored derivative (K-major), b = w or uw (MN-major). kLceDW: per
  // segment a = stored derivative (MN-major), b = h or uh (MN-major).
  CUtensorMap a[2], b[2];
  CUtensorMap out[2];  // logit gradient kinds: stores of G and D
  const LceHead* head;
  const LceScale* scale;
  // rows of the state / work arrays, indexed by row slot
  const int* tgt;
  const float* lse2;
  const float* coef;
  const float* rho;
  float2* part;  // statistics kinds: [2 * n_tiles][n_pad]
  float* ztgt;   // statistics kinds: value at the target
  float* acc;    // kLceDH: [splits][n_pad][dim_pad]
  uint16_t* dw;  // kLceDW: row 0 of the piece, [cols][dim]
  int n_pad;     // row slots (multiple of 128)
  int dim, dim_pad;
  int col0, cols;  // the vocabulary piece
  int seg_mask;    // segments (products) in use: bit 0, bit 1
  int splits;      // kLceDH: shares of the piece's columns
  int accumulate;  // kLceDH: add to acc instead of overwriting it
  int* err;
  int* err_host;
};

cudaError_t launch_lce_gemm(const LceGemm& p, int kind, bool bf16, int sms, cudaStream_t stream);

}  // namespace ttt
