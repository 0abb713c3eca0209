// Linear cross entropy: C entry points (include/ttt_ops.h), the launch sequence
// of each pass and its row kernels. The tensor-core work is in lce_gemm.cu.
//
// The participating rows are listed first (slots), and h is gathered into a
// compact copy that the state keeps, so masked rows cost no products and whatever
// they hold stays out of every sum. Then
//   forward   statistics of z, combined per row into maximum and sum of exponentials
//   gradient  per piece of the vocabulary: G in 16 bits; then in one launch G w,
//             added to fp32 partial rows, and G^T h, rounded into the piece's rows
//             of dw; at the end the partial rows are added in order and scattered
//   second    statistics of (z, A) combined into rho; then as the gradient with
//             (G, D) and two products per output
// The stored derivatives carry a power of two that puts their largest possible
// magnitude near 2^13: exact in both types, and in fp16 it keeps small
// probabilities (1e-7 and less) out of the subnormals. Rounding G and D to the
// inputs' type is the one rounding before the outputs'; it costs as much as
// rounding an output does, spread over the terms of a sum.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>

#include "host_ctx.h"
#include "lce.h"
#include "prof.h"
#include "tc100.cuh"
#include "ttt_ops.h"

namespace ttt {
// The current context's host mirror of the error word (capi.cu), or null.
int32_t* registered_error_mirror();
// Tensor map encoder of the driver (capi.cu): 2-D, 16-bit, 128-byte swizzle.
bool encode_2d(CUtensorMap* m, bool bf16, const void* base, int64_t cols, int64_t rows, int64_t stride, int box_cols,
               int box_rows);
}  // namespace ttt

namespace {

using ttt::LceCoef;
using ttt::LceHead;

constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- state and work layouts
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Arena {  // hands out 256-byte aligned parts of a buffer (or only counts them)
  char* base;
  int64_t used = 0;
  explicit Arena(void* b) : base(static_cast<char*>(b)) {}
  template <class T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += up(count * static_cast<int64_t>(sizeof(T)), 256);
    return p;
  }
};

struct State {
  LceHead* head;
  int* idx;      // [n_pad] source row of a slot, -1 past the last
  int* tgt;      // [n_pad] target of a slot, -1 past the last
  float* mw;     // [n_pad] mask weight of a slot, 0 past the last
  // The row's log-sum-exp in two parts, p = exp2(z log2 e - top2) / l: one rounded number of the
  // logits' size would leave its ulps in p - 1.
  float* top2;   // [n_pad] base-2 maximum of a slot, +inf past the last
  float* inv_l;  // [n_pad] 1 / l, the sum of exponentials below it, 0 past the last
  uint16_t* hc;  // [n_pad][dim_pad] rows of h by slot, zeros past the last
  int* slot;     // [n] slot of a source row, -1 if it takes no part
};
// The size ends with the last of `slot`, so that a state of one row count does not pass for another's.
int64_t state_layout(const ttt_lce_problem& pb, void* base, State* s) {
  Arena a(base);
  const int64_t n_pad = up(pb.n, ttt::kLceBM);
  State t;
  t.head = a.take<LceHead>(1);
  t.idx = a.take<int>(n_pad);
  t.tgt = a.take<int>(n_pad);
  t.mw = a.take<float>(n_pad);
  t.top2 = a.take<float>(n_pad);
  t.inv_l = a.take<float>(n_pad);
  t.hc = a.take<uint16_t>(n_pad * up(pb.dim, 8));
  const int64_t slots_at = a.used;
  t.slot = a.take<int>(pb.n);
  if (s != nullptr) *s = t;
  return slots_at + pb.n * static_cast<int64_t>(sizeof(int));
}

int device_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
  return n < 1 ? 1 : n;
}

struct Plan {
  int64_t n, n_pad, vocab;
  int dim, dim_pad;
  int64_t piece;  // vocabulary columns per piece
  int splits;     // shares of a piece's columns in the dh product
};
// Time (in 64-wide steps of a pair of CTAs) until `pairs` pairs that take the next tile
// when free have formed n_long tiles of `len` steps and then n_short of `slen`.
int64_t makespan(int64_t pairs, int64_t n_long, int64_t len, int64_t n_short, int64_t slen) {
  const int64_t k = n_long / pairs, r = n_long % pairs;  // r pairs hold one long tile more
  const int64_t full = (k + (r > 0 ? 1 : 0)) * len;
  auto room = [&](int64_t x) {  // short tiles that fit before time x
    const int64_t a = x > full ? (x - full) / slen : 0, b = x > k * len ? (x - k * len) / slen : 0;
    return r > 0 ? r * a + (pairs - r) * b : pairs * b;
  };
  // between a perfect fill and one short tile more
  int64_t lo = std::max(full, (n_short * slen + r * full + (pairs - r) * k * len + pairs - 1) / pairs);
  int64_t hi = lo + slen;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (room(mid) >= n_short)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// The shares into which the hidden gradient's contraction over a piece is cut: more of
// them let the pairs end together and fill the GPU with few tokens, but each costs a
// pass over fp32 partial rows. The count with the least time is taken, with a step at
// 0.3 us (512 cycles), a tile's start and end at eight steps, and the partial rows
// written and read at 6.5 TB/s. The model counts 64-wide steps; the kernel cuts the shares at
// its 128-wide stages, so a modelled length is off by up to one of those. At 8192 x 768 x 32000
// the second gradient's pieces (96 tiles of 512 steps against 189 of 264) take 1552 steps uncut
// and 1408 in three shares.
int plan_splits(const Plan& q, int segs, int64_t pairs) {
  const int64_t cols = std::min(q.piece, q.vocab);
  const int64_t dt = up(q.dim, ttt::kLceBN) / ttt::kLceBN, kt = up(cols, 64) / 64;
  const int64_t n_dh = q.n_pad / ttt::kLceBM * dt, n_dw = up(cols, ttt::kLceBM) / ttt::kLceBM * dt;
  const int64_t dw_len = q.n_pad / 64 * segs + 8;
  int best = 1;
  double best_time = 0;
  for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (s > 1 && kt / s < 8) break;  // of the first piece; the last one may leave shares without columns
    const int64_t dh_len = (kt + s - 1) / s * segs + 8;
    const int64_t steps = dh_len > dw_len ? makespan(pairs, n_dh * s, dh_len, n_dw, dw_len)
                                          : makespan(pairs, n_dw, dw_len, n_dh * s, dh_len);
    const double bytes = 8.0 * s * static_cast<double>(q.n_pad) * q.dim_pad;
    const double time = static_cast<double>(steps) + bytes / (6.5e6 * 0.3);
    if (s == 1 || time < best_time) best = s, best_time = time;
  }
  return best;
}

Plan make_plan(const ttt_lce_problem& pb, int pass, int sms) {
  Plan q;
  q.n = pb.n;
  q.n_pad = up(pb.n, ttt::kLceBM);
  q.vocab = pb.vocab;
  q.dim = pb.dim;
  q.dim_pad = static_cast<int>(up(pb.dim, 8));
  // The stored derivatives (one array, two in the second gradient) of a piece stay
  // within 512 MB, but a piece has at least 2048 columns; equal pieces of whole tiles.
  // Smaller pieces would stay in L2 but end more often: at 8192 x 768 x 32000 160 MB take
  // 1.12 ms for loss and gradient and 80 MB 1.21, against 0.98.
  const int64_t budget = static_cast<int64_t>(512) << 20;
  const int64_t per_col = q.n_pad * 2 * (pass == 2 ? 2 : 1);
  const int64_t most = std::max<int64_t>(2048, budget / std::max<int64_t>(per_col, 1));
  const int64_t pieces = (q.vocab + most - 1) / most;
  q.piece = up((q.vocab + pieces - 1) / pieces, 256);
  q.splits = pass == 0 ? 1 : plan_splits(q, pass, std::max(1, sms / 2));
  return q;
}

// Parts of the statistics: half tiles, or up to two blocks per SM of lce_score_kernel.
int64_t score_parts(int64_t vocab) { return std::max<int64_t>(2 * ((vocab + ttt::kLceBN - 1) / ttt::kLceBN), 512); }

struct Work {
  float2* part;        // statistics of half tiles, [2 * tiles][n_pad]
  float* ztgt;         // [n_pad]
  float* sums;         // [n_pad / 32] sums of the row losses (or derivatives by c) by block
  unsigned* counters;  // [0] ticket of the products, [1] max_bits, [2] ticket of the row sums
  uint16_t* uc;        // gathered uh, [n_pad][dim_pad]
  float* coef;         // [n_pad]
  float* rho;          // [n_pad]
  uint16_t *g, *d;     // stored derivatives, [n_pad][piece]
  float* acc;          // [splits][n_pad][dim_pad]
};
int64_t work_layout(const Plan& q, int pass, void* base, Work* w) {
  Arena a(base);
  Work t{};
  const int64_t rows = q.n_pad, mat = rows * q.dim_pad;
  t.counters = a.take<unsigned>(3);
  if (pass != 1) {
    const int64_t parts = pass == 0 ? score_parts(q.vocab) : 2 * ((q.vocab + ttt::kLceBNDual - 1) / ttt::kLceBNDual);
    t.part = a.take<float2>(parts * rows);
    t.ztgt = a.take<float>(rows);
    t.sums = a.take<float>(rows / 32);
  }
  if (pass != 0) {
    t.coef = a.take<float>(rows);
    if (pass == 2) t.rho = a.take<float>(rows);
    if (pass == 2) t.uc = a.take<uint16_t>(mat);
    t.g = a.take<uint16_t>(rows * q.piece);
    if (pass == 2) t.d = a.take<uint16_t>(rows * q.piece);
    t.acc = a.take<float>(static_cast<int64_t>(q.splits) * mat);
  }
  if (w != nullptr) *w = t;
  return a.used;
}

// ---------------------------------------------------------------- row kernels
// Fixed-order sum over the block (256 threads), returned to every thread.
__device__ __forceinline__ float block_sum(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s += buf[i];
  return s;
}

__device__ __forceinline__ float block_max(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s = fmaxf(s, buf[i]);
  return s;
}

struct RowArgs {
  int64_t n, vocab, ignore_index;
  int n_pad, dim, dim_pad, mask_kind, reduction, list_rows;
  const int64_t* targets;
  const void* mask;
  const uint16_t* src;  // h (forward) or uh
  int64_t src_stride;
  uint16_t* dst;  // its compact copy
  int wide;       // rows can be copied in 16-byte pieces
  State st;
  float* loss;
  const float* dloss;
  float* coef;
  unsigned* counters;
  int* err;
  int* err_host;
};

__device__ __forceinline__ float mask_weight(const RowArgs& a, int64_t i) {
  if (a.mask_kind == TTT_LCE_MASK_F32) return static_cast<const float*>(a.mask)[i];
  if (a.mask_kind == TTT_LCE_MASK_U8) return static_cast<const uint8_t*>(a.mask)[i] ? 1.f : 0.f;
  return 1.f;
}
// 1: takes part, 0: left out, -1: left out and its target is invalid.
__device__ __forceinline__ int row_kind(const RowArgs& a, int64_t i, float m) {
  const int64_t t = a.targets[i];
  if (m == 0.f || t == a.ignore_index) return 0;
  return t >= 0 && t < a.vocab ? 1 : -1;
}

// Copies up to R source rows (row < 0: zeros) into slots (slot < 0: none), the rows'
// loads in flight together; by `count` threads, of which this is number `me`.
template <int R>
__device__ __forceinline__ void copy_rows(const RowArgs& a, const int64_t (&row)[R], const int64_t (&slot)[R], int me,
                                          int count) {
  if (a.src == nullptr) return;
  if (a.wide) {
#pragma unroll 2
    for (int c = me * 8; c < a.dim; c += count * 8) {
      uint4 v[R];
#pragma unroll
      for (int i = 0; i < R; ++i)
        v[i] = slot[i] < 0 || row[i] < 0 ? make_uint4(0, 0, 0, 0)
                                         : *reinterpret_cast<const uint4*>(a.src + row[i] * a.src_stride + c);
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (slot[i] >= 0) *reinterpret_cast<uint4*>(a.dst + slot[i] * a.dim_pad + c) = v[i];
    }
  } else {
#pragma unroll 4
    for (int c = me; c < a.dim; c += count) {
      uint16_t v[R];
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = slot[i] < 0 || row[i] < 0 ? 0 : a.src[row[i] * a.src_stride + c];
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (slot[i] >= 0) a.dst[slot[i] * a.dim_pad + c] = v[i];
    }
  }
}

// Clears row slot `s`; one warp.
__device__ __forceinline__ void clear_slot(const RowArgs& a, int64_t s, int lane) {
  for (int c = lane * 8; c < a.dim_pad; c += 256)
    *reinterpret_cast<uint4*>(a.dst + s * a.dim_pad + c) = make_uint4(0, 0, 0, 0);
  if (lane == 0) {
    a.st.idx[s] = -1, a.st.tgt[s] = -1, a.st.mw[s] = 0.f;
    a.st.top2[s] = INFINITY, a.st.inv_l[s] = 0.f;
  }
}

// Lists the participating rows and gathers h. Block b owns a range of a.list_rows rows,
// 32 at a time; it counts the participating rows before the range itself (n / 2 reads of
// 8 to 12 bytes on average, from L2, by at most 512 blocks), so that one launch does
// without a scan across blocks. The last of them also knows the totals and clears the
// slots up to the next whole tile; the slots past the last row, which no row can take,
// have blocks of their own.
__global__ void __launch_bounds__(256) lce_list_kernel(const RowArgs a) {
  __shared__ float buf[8];
  __shared__ int cnt[8];
  __shared__ int slots[32];
  __shared__ int total;
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * a.list_rows;
  if (first >= a.n) {
    const int64_t s0 = a.n + (blockIdx.x - (a.n + a.list_rows - 1) / a.list_rows) * 32;
    for (int64_t s = s0 + warp; s < s0 + 32 && s < a.n_pad; s += 8) clear_slot(a, s, lane);
    return;
  }
  const int64_t past = min(first + a.list_rows, a.n);
  // participating rows before the range, and the mask's sum and largest magnitude over them
  int before = 0;
  float msum = 0.f, mmax = 0.f;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < first; i += 256) {
    const float m = mask_weight(a, i);
    const bool in = row_kind(a, i, m) > 0;
    before += in;
    msum += m;
    mmax = in ? fmaxf(mmax, fabsf(m)) : mmax;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) cnt[warp] = before;
  __syncthreads();
  int base = 0;
  for (int i = 0; i < 8; ++i) base += cnt[i];
  for (int64_t row0 = first; row0 < past; row0 += 32) {
    if (warp == 0) {
      const int64_t i = row0 + lane;
      float m = 0.f;
      int kind = 0;
      if (i < past) {
        m = mask_weight(a, i);
        kind = row_kind(a, i, m);
        if (kind < 0) ttt::report_error(a.err, a.err_host, TTT_ERR_WORD_TARGET | (static_cast<int>(i) & 0xffffff));
        msum += m;
        mmax = kind > 0 ? fmaxf(mmax, fabsf(m)) : mmax;
      }
      const unsigned bits = __ballot_sync(0xffffffffu, kind > 0);
      const int s = kind > 0 ? base + __popc(bits & ((1u << lane) - 1)) : -1;
      base += __popc(bits);
      slots[lane] = s;
      if (i < past) {
        a.st.slot[i] = s;
        if (s >= 0) {
          a.st.idx[s] = static_cast<int>(i);
          a.st.tgt[s] = static_cast<int>(a.targets[i]);
          a.st.mw[s] = m;
        } else if (a.reduction == TTT_LCE_NONE) {
          a.loss[i] = 0.f;
        }
      }
      if (lane == 0) total = base;
    }
    __syncthreads();
    // aligned rows four to a warp, others (one element a load) four to the block
    for (int j = a.wide ? warp : 0; j < (a.wide ? warp + 1 : 8); ++j) {
      int64_t from[4], to[4];
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = a.wide ? j + 8 * i : j * 4 + i;
        from[i] = row0 + at;
        to[i] = slots[at];
        any = any || to[i] >= 0;
      }
      if (any) copy_rows<4>(a, from, to, a.wide ? lane : threadIdx.x, a.wide ? 32 : 256);
    }
    __syncthreads();
  }
  if (past < a.n) return;
  const int n_active = total;
  const int64_t end = min(static_cast<int64_t>((n_active + ttt::kLceBM - 1) / ttt::kLceBM * ttt::kLceBM), a.n);
  for (int64_t s = n_active + warp; s < end; s += 8) clear_slot(a, s, lane);
  msum = block_sum(msum, buf);
  mmax = block_max(mmax, buf);
  if (threadIdx.x == 0) {
    a.st.head->n_active = n_active;
    float denom = 1.f;
    if (a.reduction == TTT_LCE_MEAN)
      denom = a.mask_kind == TTT_LCE_MASK_NONE ? static_cast<float>(a.n) : fmaxf(msum, 1.f);
    a.st.head->denom = denom;
    a.st.head->mw_max = mmax;
    a.st.head->ticket = 0;
  }
}

// Lists the row coefficients and gathers uh into slots; block 0 also finds the
// largest magnitude (the second gradient raises it in lce_rho_kernel).
__global__ void __launch_bounds__(256) lce_coef_kernel(const RowArgs a) {
  __shared__ float buf[8];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_active = a.st.head->n_active;
  const int end = min((n_active + ttt::kLceBM - 1) / ttt::kLceBM * ttt::kLceBM, a.n_pad);
  auto coef = [&](int s) {
    return a.reduction == TTT_LCE_NONE ? a.dloss[a.st.idx[s]] * a.st.mw[s] : a.st.mw[s];
  };
  for (int s = (blockIdx.x * 8 + warp) * 2; s < end; s += gridDim.x * 16) {  // end is even
    const int64_t from[2] = {s < n_active ? a.st.idx[s] : -1, s + 1 < n_active ? a.st.idx[s + 1] : -1};
    const int64_t to[2] = {s, s + 1};
    copy_rows<2>(a, from, to, lane, 32);
    if (lane < 2) a.coef[s + lane] = s + lane < n_active ? coef(s + lane) : 0.f;
  }
  if (blockIdx.x != 0) return;
  float big = 0.f;
#pragma unroll 4
  for (int s = threadIdx.x; s < n_active; s += 256) big = fmaxf(big, fabsf(coef(s)));
  big = block_max(big, buf);
  if (threadIdx.x == 0) {
    a.counters[1] = __float_as_uint(big);
    a.counters[2] = 0;
  }
}

// Adds v over the 32 lanes of the block's first warp and, in the last block to finish,
// the blocks' sums: out = total / denom. The order is fixed whichever block is last.
__device__ __forceinline__ void total_rows(float v, float* sums, unsigned* ticket, float denom, float* out) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  unsigned done = 0;
  if (threadIdx.x == 0) {
    sums[blockIdx.x] = v;
    __threadfence();
    done = atomicAdd(ticket, 1u);
  }
  done = __shfl_sync(0xffffffffu, done, 0);
  if (done != gridDim.x - 1) return;
  __threadfence();
  float t = 0.f;
#pragma unroll 4
  for (unsigned i = threadIdx.x; i < gridDim.x; i += 32) t += __ldcg(sums + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (threadIdx.x == 0) *out = t / denom;
}

// Merges the half tiles' (max, sum) of a row: 32 rows and 32 shares of the tiles per
// block, shares in order. Writes top2, inv_l and the row's weighted loss.
constexpr int kShares = 32;
__global__ void __launch_bounds__(32 * kShares) lce_lse_kernel(const State st, const float2* part, const float* ztgt,
                                                               int parts, int n_pad, int reduction, float* sums,
                                                               float* loss) {
  __shared__ float2 sh[kShares][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, share = threadIdx.x >> 5;
  const int s = blockIdx.x * 32 + lane, n_active = st.head->n_active;
  float m = -INFINITY, l = 0.f;
  if (s < n_active) {
    constexpr int U = 8;
    for (int i0 = share; i0 < parts; i0 += U * kShares) {
      float2 o[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        o[u] = i0 + u * kShares < parts ? part[static_cast<int64_t>(i0 + u * kShares) * n_pad + s]
                                        : make_float2(-INFINITY, 0.f);
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, o[u].x);
      const float sub = top == -INFINITY ? 0.f : top;
      l *= exp2f(m - sub);
#pragma unroll
      for (int u = 0; u < U; ++u) l += o[u].y * exp2f(o[u].x - sub);
      m = top;
    }
  }
  sh[share][lane] = make_float2(m, l);
  __syncthreads();
  if (share != 0) return;
  float v = 0.f;
  if (s < n_active) {
    for (int i = 1; i < kShares; ++i) m = fmaxf(m, sh[i][lane].x);
    const float sub = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < kShares; ++i) l += sh[i][lane].y * exp2f(sh[i][lane].x - sub);
    st.top2[s] = m;
    st.inv_l[s] = 1.f / l;
    // The large terms first, in one rounding: log-sum-exp and logit, each rounded, would leave ulps of
    // the logit in a loss near 0. m carries the rounding of its own product with log2 e, and so do the
    // exponentials in l.
    const float ce = kLn2 * (fmaf(-ztgt[s], kLog2e, m) + log2f(l));
    v = st.mw[s] * (ce < 0.f ? 0.f : ce);  // NaN stays
    if (reduction == TTT_LCE_NONE) loss[st.idx[s]] = v;
  }
  if (reduction != TTT_LCE_NONE) total_rows(v, sums, &st.head->ticket, st.head->denom, loss);
}

// Adds the half tiles' sums P A of a row into rho, raises the bound of what is stored
// to the largest |c| (max |P A| + |rho|), which bounds |D|, and forms the derivative by c.
__global__ void __launch_bounds__(32 * kShares) lce_rho_kernel(const State st, const float2* part, const float* ztgt,
                                                               const float* coef, int parts, int n_pad, int reduction,
                                                               float* rho, unsigned* counters, float* sums,
                                                               float* gdloss) {
  __shared__ float2 sh[kShares][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, share = threadIdx.x >> 5;
  const int s = blockIdx.x * 32 + lane, n_active = st.head->n_active;
  float sum = 0.f, big = 0.f;
  if (s < n_active) {
#pragma unroll 8
    for (int i = share; i < parts; i += kShares) {
      const float2 o = part[static_cast<int64_t>(i) * n_pad + s];
      sum += o.x;
      big = fmaxf(big, o.y);
    }
  }
  sh[share][lane] = make_float2(sum, big);
  __syncthreads();
  if (share != 0) return;
  float dc = 0.f;
  if (s < n_active) {
    for (int i = 1; i < kShares; ++i) {
      sum += sh[i][lane].x;
      big = fmaxf(big, sh[i][lane].y);
    }
    rho[s] = sum;
    dc = st.mw[s] * (sum - ztgt[s]);
    if (gdloss != nullptr && reduction == TTT_LCE_NONE) gdloss[st.idx[s]] = dc;
    big = fabsf(coef[s]) * (big + fabsf(sum));
  } else if (s < n_pad) {
    rho[s] = 0.f;
  }
  if (s >= n_active || !(big < INFINITY)) big = 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  if (lane == 0) atomicMax(counters + 1, __float_as_uint(big));  // non-negative: ordered like its bits
  if (gdloss != nullptr && reduction != TTT_LCE_NONE) total_rows(dc, sums, counters + 2, st.head->denom, gdloss);
}

// Losses of a few rows without gradients (the score of a token): a product with so
// few rows is bound by reading w once, so CUDA cores form it. Every warp has an equal
// range of the vocabulary, takes four rows at a time (their loads in flight together),
// adds up its lanes' products with the rows of h held in shared memory, and keeps a
// running (max, sum) per row; blocks write theirs as one part each, which
// lce_lse_kernel merges. Block 0 lists the rows. At 1 x 768 x 32000 bf16: 15 us and 6 for
// the merge, each on its own, and 18 a call back to back; the tensor-core path (list,
// 256-row tiles, merge) takes 26 us of kernels and a launch more, 34 a call.
constexpr int kScoreRows = 4, kScoreWarps = 16, kScoreMaxDim = 8192;
template <bool BF16, int NR>
__global__ void __launch_bounds__(32 * kScoreWarps) lce_score_kernel(const RowArgs a, const uint16_t* w, int64_t w_stride,
                                                                     float2* part, float* ztgt) {
  extern __shared__ __align__(16) uint16_t hs[];  // [NR][dim]
  __shared__ float2 sh[kScoreWarps][NR];
  __shared__ int rows[NR], tgts[NR], count;
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this warp's vocabulary rows, on their way into L2 while the block lists the tokens
  const int64_t wid = static_cast<int64_t>(blockIdx.x) * kScoreWarps + warp, warps = gridDim.x * kScoreWarps;
  const int v_begin = static_cast<int>(a.vocab * wid / warps), v_end = static_cast<int>(a.vocab * (wid + 1) / warps);
  for (int v = v_begin; v < v_end; ++v)
    for (int c = lane * 64; c < a.dim; c += 2048)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(w + v * w_stride + c));
  if (warp == 0) {
    float m = 0.f;
    int kind = 0;
    if (lane < a.n) {
      m = mask_weight(a, lane);
      kind = row_kind(a, lane, m);
      if (kind < 0 && blockIdx.x == 0) ttt::report_error(a.err, a.err_host, TTT_ERR_WORD_TARGET | lane);
    }
    const unsigned bits = __ballot_sync(0xffffffffu, kind > 0);
    const int s = __popc(bits & ((1u << lane) - 1));
    if (kind > 0) {
      rows[s] = lane;
      tgts[s] = static_cast<int>(a.targets[lane]);
    }
    if (lane == 0) count = __popc(bits);
    if (blockIdx.x == 0) {
      if (kind > 0) {
        a.st.idx[s] = lane;
        a.st.mw[s] = m;
      } else if (lane < a.n && a.reduction == TTT_LCE_NONE) {
        a.loss[lane] = 0.f;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane == 0) {
        a.st.head->n_active = __popc(bits);
        a.st.head->ticket = 0;
        a.st.head->denom = a.reduction != TTT_LCE_MEAN              ? 1.f
                           : a.mask_kind == TTT_LCE_MASK_NONE ? static_cast<float>(a.n)
                                                              : fmaxf(m, 1.f);
      }
    }
  }
  __syncthreads();
  const int nr = count;
  for (int r = 0; r < NR; ++r)
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x)
      hs[r * a.dim + c] = r < nr ? a.src[rows[r] * a.src_stride + c] : 0;
  __syncthreads();
  float mx[NR], sum[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) mx[r] = -INFINITY, sum[r] = 0.f;
  constexpr int U = 4;
  for (int v0 = v_begin; v0 < v_end; v0 += U) {
    float z[NR][U];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) z[r][u] = 0.f;
#pragma unroll 2
    for (int c = lane * 8; c < a.dim; c += 256) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        q[u] = v0 + u < v_end ? __ldcs(reinterpret_cast<const uint4*>(w + (v0 + u) * w_stride + c))
                              : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const uint4 hq = *reinterpret_cast<const uint4*>(hs + r * a.dim + c);
        const uint32_t hw[4] = {hq.x, hq.y, hq.z, hq.w};
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t ww[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[r][u] = fmaf(ttt::to_f32<BF16>(static_cast<uint16_t>(ww[e])),
                           ttt::to_f32<BF16>(static_cast<uint16_t>(hw[e])), z[r][u]);
            z[r][u] = fmaf(ttt::to_f32<BF16>(static_cast<uint16_t>(ww[e] >> 16)),
                           ttt::to_f32<BF16>(static_cast<uint16_t>(hw[e] >> 16)), z[r][u]);
          }
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) z[r][u] += __shfl_xor_sync(0xffffffffu, z[r][u], o);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (lane == 0 && r < nr && tgts[r] >= v0 && tgts[r] < min(v0 + U, v_end)) {
        float zt = z[r][0];
#pragma unroll
        for (int u = 1; u < U; ++u) zt = tgts[r] == v0 + u ? z[r][u] : zt;
        ztgt[r] = zt;
      }
      float top = mx[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        z[r][u] = v0 + u < v_end ? z[r][u] : -INFINITY;
        top = fmaxf(top, z[r][u]);
      }
      // the maximum's product with log2 e is rounded alike wherever it is used
      const float sub = top == -INFINITY ? 0.f : __fmul_rn(top, kLog2e);
      sum[r] *= exp2f(__fmul_rn(mx[r], kLog2e) - sub);
#pragma unroll
      for (int u = 0; u < U; ++u) sum[r] += exp2f(fmaf(z[r][u], kLog2e, -sub));
      mx[r] = top;
    }
  }
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < NR; ++r) sh[warp][r] = make_float2(__fmul_rn(mx[r], kLog2e), sum[r]);
  }
  __syncthreads();
  if (threadIdx.x < nr) {
    const int r = threadIdx.x;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < kScoreWarps; ++i) m = fmaxf(m, sh[i][r].x);
    const float sub = m == -INFINITY ? 0.f : m;
    for (int i = 0; i < kScoreWarps; ++i) l += sh[i][r].y * exp2f(sh[i][r].x - sub);
    part[static_cast<int64_t>(blockIdx.x) * a.n_pad + r] = make_float2(m, l);
  }
}

__global__ void lce_zero_rows_kernel(const int* slot, int64_t n, float* out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i < n && slot[i] < 0) out[i] = 0.f;
}

// dh[i] = sum over the splits (in order) of acc[split][slot_i] times the outputs' factor, 0 for rows left
// out. Four columns a thread at a time, `width` threads a row.
template <bool BF16>
__global__ void __launch_bounds__(256) lce_scatter_kernel(const int* slot, const LceCoef coef, const float* acc,
                                                          int splits, int64_t n, int n_pad, int dim, int dim_pad,
                                                          int width, uint16_t* dh) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per = 256 / width;  // rows of a block
  const int64_t i = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / width;
  if (i >= n) return;
  const int s = slot[i];
  const float mul = s >= 0 ? coef.out() : 0.f;  // an infinite one leaves the other rows' zeros alone
  uint16_t* dst = dh + i * dim;
#pragma unroll 4
  for (int c = (threadIdx.x % width) * 4; c < dim; c += width * 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s >= 0) {
      const float* src = acc + static_cast<int64_t>(s) * dim_pad + c;
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        const float4 o = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(k) * n_pad * dim_pad);
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
    }
    const uint32_t lo = ttt::pack2<BF16>(v.x * mul, v.y * mul), hi = ttt::pack2<BF16>(v.z * mul, v.w * mul);
    if ((dim & 3) == 0) {
      *reinterpret_cast<uint2*>(dst + c) = make_uint2(lo, hi);
    } else {
      const uint16_t e[4] = {static_cast<uint16_t>(lo), static_cast<uint16_t>(lo >> 16), static_cast<uint16_t>(hi),
                             static_cast<uint16_t>(hi >> 16)};
      for (int j = 0; j < 4; ++j)
        if (c + j < dim) dst[c + j] = e[j];
    }
  }
}

// Rows of unaligned 16-bit elements into aligned rows; a warp per row, consecutive lanes on
// consecutive elements, so that both sides move whole sectors.
__global__ void __launch_bounds__(256) lce_pad_kernel(const uint16_t* src, int64_t src_stride, uint16_t* dst,
                                                      int64_t dst_stride, int64_t rows, int dim) {
  const int lane = threadIdx.x & 31;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < rows; r += step) {
    const uint16_t* from = src + r * src_stride;
    uint16_t* to = dst + r * dst_stride;
    for (int c0 = lane; c0 < dim; c0 += 256) {
      uint16_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = c0 + u * 32 < dim ? from[c0 + u * 32] : 0;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c0 + u * 32 < dim) to[c0 + u * 32] = v[u];
    }
  }
}

// ---------------------------------------------------------------- host side
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_lce(const ttt_lce_problem& pb) {
  if (pb.dtype != TTT_F16 && pb.dtype != TTT_BF16) return TTT_ERR_DTYPE;
  if (pb.n < 0 || pb.n > (1 << 24) || pb.vocab < 1 || pb.vocab > (1 << 24)) return TTT_ERR_SHAPE;
  if (pb.dim < 1 || pb.dim > 65536) return TTT_ERR_SHAPE;
  if (pb.reduction < TTT_LCE_NONE || pb.reduction > TTT_LCE_SUM) return TTT_ERR_UNSUPPORTED;
  if (pb.mask_kind < TTT_LCE_MASK_NONE || pb.mask_kind > TTT_LCE_MASK_U8) return TTT_ERR_UNSUPPORTED;
  return TTT_OK;
}
int check_weight(const void* w, int64_t stride, const ttt_lce_problem& pb) {
  if (w == nullptr) return TTT_ERR_NULL;
  if (!aligned(w, 16)) return TTT_ERR_ALIGN;
  if (pb.vocab > 1 && (stride < pb.dim || stride % 8 != 0)) return TTT_ERR_STRIDE;
  return TTT_OK;
}

#define TTT_TRY(expr)            \
  do {                           \
    const int _s = (expr);       \
    if (_s != TTT_OK) return _s; \
  } while (0)

int launched() { return cudaGetLastError() == cudaSuccess ? TTT_OK : TTT_ERR_LAUNCH; }
int launched(cudaError_t e) { return e == cudaSuccess ? TTT_OK : TTT_ERR_LAUNCH; }

// A weight-like [vocab, dim] matrix; a single row may come with any stride.
struct Weight {
  const uint16_t* p;
  int64_t stride;
  Weight(const void* w, int64_t s, const ttt_lce_problem& pb)
      : p(static_cast<const uint16_t*>(w)), stride(pb.vocab > 1 ? s : up(pb.dim, 8)) {}
  const uint16_t* row(int64_t r) const { return p + r * stride; }
};

// A launch whose start may overlap the previous kernel's end; the kernel waits for it itself.
template <class... K, class... A>
int launch_early(void (*kern)(K...), int64_t grid, int threads, cudaStream_t s, A... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return launched(cudaLaunchKernelEx(&cfg, kern, static_cast<K>(args)...));
}

struct Pass {
  const ttt_lce_problem& pb;
  Plan q;
  State st;
  Work w;
  LceCoef coef;
  const float* upstream;
  int64_t work_need;
  int sms;
  bool bf16;
  int* err;
  int* err_host;
  cudaStream_t s;

  Pass(const ttt_lce_problem& p, int pass, const void* state, void* work, const float* dloss, int32_t* e,
       void* stream)
      : pb(p), sms(device_sms()), bf16(p.dtype == TTT_BF16), err(e),
        err_host(e != nullptr ? ttt::registered_error_mirror() : nullptr), s(static_cast<cudaStream_t>(stream)) {
    q = make_plan(p, pass, sms);
    state_layout(p, const_cast<void*>(state), &st);
    work_need = work_layout(q, pass, work, &w);
    const bool listed = pass == 2 || (pass == 1 && p.reduction == TTT_LCE_NONE);
    coef = {st.head, p.reduction == TTT_LCE_NONE ? nullptr : dloss, st.mw, listed ? w.coef : nullptr,
            listed ? w.counters + 1 : nullptr};
    upstream = dloss;
  }
  // Row kernels; src is gathered into dst when given.
  RowArgs row_args(const void* src, int64_t stride, uint16_t* dst) const {
    RowArgs a;
    std::memset(&a, 0, sizeof(a));
    a.n = pb.n, a.vocab = pb.vocab, a.ignore_index = pb.ignore_index;
    a.n_pad = static_cast<int>(q.n_pad), a.dim = q.dim, a.dim_pad = q.dim_pad;
    a.mask_kind = pb.mask_kind, a.reduction = pb.reduction;
    a.src = static_cast<const uint16_t*>(src), a.src_stride = stride, a.dst = dst;
    a.wide = q.dim % 8 == 0 && aligned(src, 16) && stride % 8 == 0;
    a.st = st;
    a.dloss = upstream, a.coef = w.coef, a.counters = w.counters;
    a.err = err, a.err_host = err_host;
    return a;
  }
  int list_coef(const void* uh, int64_t stride) const {
    const int64_t blocks = uh != nullptr ? std::min<int64_t>(q.n_pad / 8, sms * 8) : 1 + q.n_pad / 2048;
    lce_coef_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(row_args(uh, stride, w.uc));
    return launched();
  }
  ttt::LceGemm gemm(int64_t col0, int64_t cols) const {
    ttt::LceGemm g;
    std::memset(&g, 0, sizeof(g));
    g.head = st.head, g.coef = coef;
    g.tgt = st.tgt, g.top2 = st.top2, g.inv_l = st.inv_l, g.rho = w.rho;
    g.part = w.part, g.ztgt = w.ztgt, g.ticket = w.counters;
    g.n_pad = static_cast<int>(q.n_pad), g.dim = q.dim, g.dim_pad = q.dim_pad;
    g.col0 = static_cast<int>(col0), g.cols = static_cast<int>(cols);
    g.splits = 1;
    g.err = err, g.err_host = err_host;
    return g;
  }
  int run(const ttt::LceGemm& g, int kind) const { return launched(ttt::launch_lce_gemm(g, kind, bf16, sms, s)); }
  bool map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t stride, int bc, int br) const {
    return ttt::encode_2d(m, bf16, base, cols, rows, stride, bc, br);
  }
  // Operands of the logit kinds: rows of hc or uc (128 a CTA), rows of a piece of w or uw (bn / 2 a CTA).
  bool map_rows(CUtensorMap* m, const uint16_t* x) const {
    return map(m, x, q.dim, q.n_pad, q.dim_pad, ttt::kLcePanel, ttt::kLceBM / 2);
  }
  bool map_weight(CUtensorMap* m, const Weight& w, const ttt::LceGemm& g, int bn) const {
    return map(m, w.row(g.col0), q.dim, g.cols, w.stride, ttt::kLcePanel, bn / 2);
  }
};

// The gradients of a piece-wise pass: outh [n, dim] and outw [vocab, dim] (either may
// be null). Per product i with stored derivative S_i, weight-like W_i and rows R_i:
//   outh = sum_i S_i W_i, outw = sum_i S_i^T R_i
// gradient: (G, w, h); second gradient: (D, w, h) and (G, uw, uh).
int run_pieces(const Pass& p, const Weight& w, const Weight* uw, bool second, bool has_uh, uint16_t* outh,
               uint16_t* outw) {
  const Plan& q = p.q;
  if (outh == nullptr && outw == nullptr) return TTT_OK;
  const int bn = second ? ttt::kLceBNDual : ttt::kLceBN;
  constexpr int panel = ttt::kLcePanel, bk = ttt::kLceBK;
  for (int64_t col0 = 0; col0 < q.vocab; col0 += q.piece) {
    const int64_t cols = std::min(q.piece, q.vocab - col0);
    // z (and A) -> G (and D)
    ttt::LceGemm g = p.gemm(col0, cols);
    bool ok = p.map_rows(&g.a[0], p.st.hc) && p.map_weight(&g.b[0], w, g, bn) &&
              p.map(&g.out[0], p.w.g, cols, q.n_pad, q.piece, 64, 32);
    if (second) {
      g.seg_w = (has_uh ? 1 : 0) | (uw != nullptr ? 2 : 0);
      ok = ok && p.map_rows(&g.a[1], p.w.uc) && p.map_weight(&g.b[1], uw != nullptr ? *uw : w, g, bn) &&
           p.map(&g.out[1], p.w.d, cols, q.n_pad, q.piece, 64, 32);
    }
    if (!ok) return TTT_ERR_TENSOR_MAP;
    TTT_TRY(p.run(g, second ? ttt::kLceDualGrad : ttt::kLceGrad));
    // both products in one launch
    ttt::LceGemm t = p.gemm(col0, cols);
    t.acc = outh != nullptr ? p.w.acc : nullptr;
    t.dw = outw != nullptr ? outw + col0 * q.dim : nullptr;
    t.seg_w = outh != nullptr ? (second && uw != nullptr ? 3 : 1) : 0;
    t.seg_h = outw != nullptr ? (second && has_uh ? 3 : 1) : 0;
    t.splits = q.splits;
    t.accumulate = col0 > 0;
    for (int i = 0; i < (second ? 2 : 1); ++i) {
      const uint16_t* stored = second && i == 0 ? p.w.d : p.w.g;
      const Weight& wi = i == 0 || uw == nullptr ? w : *uw;
      const uint16_t* ri = i == 0 || !has_uh ? p.st.hc : p.w.uc;
      ok = p.map(&t.gk[i], stored, cols, q.n_pad, q.piece, panel, ttt::kLceBM / 2) &&
           p.map(&t.gm[i], stored, cols, q.n_pad, q.piece, panel, bk) &&
           p.map(&t.bw[i], wi.row(col0), q.dim, cols, wi.stride, panel, bk) &&
           p.map(&t.bh[i], ri, q.dim, q.n_pad, q.dim_pad, panel, bk);
      if (!ok) return TTT_ERR_TENSOR_MAP;
    }
    if (t.dw != nullptr && q.dim % 8 == 0 && !p.map(&t.dw_out, t.dw, q.dim, cols, q.dim, 64, 32))
      return TTT_ERR_TENSOR_MAP;
    TTT_TRY(p.run(t, ttt::kLceProd));
  }
  if (outh != nullptr) {
    int width = 8;  // threads of a row: with few rows a whole block
    while (width < (q.n < 512 ? 256 : 64) && width * 4 < q.dim) width *= 2;
    TTT_TRY(launch_early(p.bf16 ? lce_scatter_kernel<true> : lce_scatter_kernel<false>,
                         (q.n + 256 / width - 1) / (256 / width), 256, p.s, p.st.slot, p.coef, p.w.acc, q.splits, q.n,
                         static_cast<int>(q.n_pad), q.dim, q.dim_pad, width, outh));
  }
  return TTT_OK;
}

int zero(void* p, int64_t bytes, cudaStream_t s) { return launched(cudaMemsetAsync(p, 0, bytes, s)); }

}  // namespace

extern "C" {

int ttt_lce_pad_weight(const void* src, int64_t src_stride, void* dst, int64_t dst_stride, int64_t vocab, int32_t dim,
                       void* stream) {
  if (src == nullptr || dst == nullptr) return TTT_ERR_NULL;
  if (vocab < 1 || vocab > (1 << 24) || dim < 1 || dim > 65536) return TTT_ERR_SHAPE;
  if (src_stride < 0 || dst_stride < dim || dst_stride % 8 != 0) return TTT_ERR_STRIDE;
  if (!aligned(dst, 16)) return TTT_ERR_ALIGN;
  const int64_t grid = std::min<int64_t>((vocab + 7) / 8, static_cast<int64_t>(device_sms()) * 8);
  lce_pad_kernel<<<static_cast<unsigned>(grid), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint16_t*>(src), src_stride, static_cast<uint16_t*>(dst), dst_stride, vocab, dim);
  return launched();
}

int64_t ttt_lce_state_bytes(const ttt_lce_problem* pb) {
  if (pb == nullptr || check_lce(*pb) != TTT_OK) return 0;
  return state_layout(*pb, nullptr, nullptr);
}

int64_t ttt_lce_work_bytes(const ttt_lce_problem* pb, int pass) {
  if (pb == nullptr || check_lce(*pb) != TTT_OK || pass < 0 || pass > 2) return 0;
  return work_layout(make_plan(*pb, pass, device_sms()), pass, nullptr, nullptr);
}

int ttt_lce_fwd(const ttt_lce_fwd_args* a, void* stream) {
  if (a == nullptr || a->loss == nullptr || a->state == nullptr) return TTT_ERR_NULL;
  const ttt_lce_problem& pb = a->pb;
  TTT_TRY(check_lce(pb));
  TTT_TRY(check_weight(a->w, a->w_stride, pb));
  if (a->need_state != 0 && a->need_state != 1) return TTT_ERR_UNSUPPORTED;
  if (pb.n == 0)
    return pb.reduction == TTT_LCE_NONE ? TTT_OK : zero(a->loss, 4, static_cast<cudaStream_t>(stream));
  if (a->h == nullptr || a->targets == nullptr) return TTT_ERR_NULL;
  if ((a->mask == nullptr) != (pb.mask_kind == TTT_LCE_MASK_NONE)) return TTT_ERR_NULL;
  if (a->work == nullptr) return TTT_ERR_SCRATCH;
  if (!aligned(a->work, 256) || !aligned(a->state, 256)) return TTT_ERR_ALIGN;
  Pass p(pb, 0, a->state, a->work, nullptr, a->err, stream);
  if (a->work_bytes < p.work_need) return TTT_ERR_SCRATCH;
  ttt::ProfSpan prof(TTT_K_LOSS, stream);
  RowArgs r = p.row_args(a->h, a->h_stride, p.st.hc);
  r.targets = a->targets, r.mask = a->mask, r.loss = a->loss;
  const Weight w(a->w, a->w_stride, pb);
  if (a->need_state == 0 && pb.n <= kScoreRows && pb.dim % 8 == 0 && pb.dim <= kScoreMaxDim) {
    // two blocks fit on an SM with one row of h, one with more; no warp has less than two vocabulary rows
    const int64_t fit = std::min<int64_t>(p.sms * (pb.n == 1 ? 2 : 1), score_parts(pb.vocab));
    const int blocks = static_cast<int>(std::min((pb.vocab + 2 * kScoreWarps - 1) / (2 * kScoreWarps), fit));
    auto kern = p.bf16 ? (pb.n == 1 ? lce_score_kernel<true, 1> : lce_score_kernel<true, kScoreRows>)
                       : (pb.n == 1 ? lce_score_kernel<false, 1> : lce_score_kernel<false, kScoreRows>);
    const int smem = (pb.n == 1 ? 1 : kScoreRows) * pb.dim * 2;
    if (smem > 32 * 1024) TTT_TRY(launched(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)));
    kern<<<blocks, 32 * kScoreWarps, smem, p.s>>>(r, w.p, w.stride, p.w.part, p.w.ztgt);
    TTT_TRY(launched());
    return launch_early(lce_lse_kernel, 1, 32 * kShares, p.s, p.st, p.w.part, p.w.ztgt, blocks, static_cast<int>(p.q.n_pad),
                        pb.reduction, p.w.sums, a->loss);
  }
  r.list_rows = static_cast<int>(std::max<int64_t>(32, up((pb.n + 511) / 512, 32)));
  const int64_t row_blocks = (pb.n + r.list_rows - 1) / r.list_rows;
  const int64_t pad_blocks = (p.q.n_pad - pb.n + 31) / 32;
  lce_list_kernel<<<static_cast<unsigned>(row_blocks + pad_blocks), 256, 0, p.s>>>(r);
  TTT_TRY(launched());
  ttt::LceGemm g = p.gemm(0, pb.vocab);
  if (!p.map_rows(&g.a[0], p.st.hc) || !p.map_weight(&g.b[0], w, g, ttt::kLceBN)) return TTT_ERR_TENSOR_MAP;
  TTT_TRY(p.run(g, ttt::kLceStats));
  const int parts = 2 * static_cast<int>((pb.vocab + ttt::kLceBN - 1) / ttt::kLceBN);
  return launch_early(lce_lse_kernel, (pb.n + 31) / 32, 32 * kShares, p.s, p.st, p.w.part, p.w.ztgt, parts, g.n_pad,
                      pb.reduction, p.w.sums, a->loss);
}

int ttt_lce_bwd(const ttt_lce_bwd_args* a, void* stream) {
  if (a == nullptr || a->state == nullptr || a->dloss == nullptr) return TTT_ERR_NULL;
  const ttt_lce_problem& pb = a->pb;
  TTT_TRY(check_lce(pb));
  TTT_TRY(check_weight(a->w, a->w_stride, pb));
  if (a->dw != nullptr && !aligned(a->dw, 16)) return TTT_ERR_ALIGN;
  if (a->dh != nullptr && !aligned(a->dh, 16)) return TTT_ERR_ALIGN;
  if (pb.n == 0)
    return a->dw != nullptr ? zero(a->dw, pb.vocab * pb.dim * 2, static_cast<cudaStream_t>(stream)) : TTT_OK;
  if (a->work == nullptr) return TTT_ERR_SCRATCH;
  if (!aligned(a->work, 256) || !aligned(a->state, 256)) return TTT_ERR_ALIGN;
  Pass p(pb, 1, a->state, a->work, a->dloss, a->err, stream);
  if (a->work_bytes < p.work_need) return TTT_ERR_SCRATCH;
  ttt::ProfSpan prof(TTT_K_LOSS, stream);
  if (p.coef.coef != nullptr) TTT_TRY(p.list_coef(nullptr, 0));
  return run_pieces(p, Weight(a->w, a->w_stride, pb), nullptr, false, false, static_cast<uint16_t*>(a->dh),
                    static_cast<uint16_t*>(a->dw));
}

int ttt_lce_bwd2(const ttt_lce_bwd2_args* a, void* stream) {
  if (a == nullptr || a->state == nullptr || a->dloss == nullptr) return TTT_ERR_NULL;
  const ttt_lce_problem& pb = a->pb;
  TTT_TRY(check_lce(pb));
  TTT_TRY(check_weight(a->w, a->w_stride, pb));
  if (a->uw != nullptr) TTT_TRY(check_weight(a->uw, a->uw_stride, pb));
  if (a->gw != nullptr && !aligned(a->gw, 16)) return TTT_ERR_ALIGN;
  if (a->gh != nullptr && !aligned(a->gh, 16)) return TTT_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t gd = pb.reduction == TTT_LCE_NONE ? pb.n : 1;
  if (pb.n == 0 || (a->uh == nullptr && a->uw == nullptr)) {  // every gradient is zero
    if (a->gh != nullptr && pb.n > 0) TTT_TRY(zero(a->gh, pb.n * pb.dim * 2, s));
    if (a->gw != nullptr) TTT_TRY(zero(a->gw, pb.vocab * pb.dim * 2, s));
    if (a->gdloss != nullptr && gd > 0) TTT_TRY(zero(a->gdloss, gd * 4, s));
    return TTT_OK;
  }
  if (a->work == nullptr) return TTT_ERR_SCRATCH;
  if (!aligned(a->work, 256) || !aligned(a->state, 256)) return TTT_ERR_ALIGN;
  Pass p(pb, 2, a->state, a->work, a->dloss, a->err, stream);
  if (a->work_bytes < p.work_need) return TTT_ERR_SCRATCH;
  ttt::ProfSpan prof(TTT_K_LOSS, stream);
  TTT_TRY(p.list_coef(a->uh, a->uh_stride));
  const Weight w(a->w, a->w_stride, pb);
  const Weight uw = a->uw != nullptr ? Weight(a->uw, a->uw_stride, pb) : w;
  ttt::LceGemm g = p.gemm(0, pb.vocab);
  g.seg_w = (a->uh != nullptr ? 1 : 0) | (a->uw != nullptr ? 2 : 0);
  if (!p.map_rows(&g.a[0], p.st.hc) || !p.map_rows(&g.a[1], p.w.uc) ||
      !p.map_weight(&g.b[0], w, g, ttt::kLceBNDual) || !p.map_weight(&g.b[1], uw, g, ttt::kLceBNDual))
    return TTT_ERR_TENSOR_MAP;
  TTT_TRY(p.run(g, ttt::kLceDualStats));
  const int parts = 2 * static_cast<int>((pb.vocab + ttt::kLceBNDual - 1) / ttt::kLceBNDual);
  TTT_TRY(launch_early(lce_rho_kernel, p.q.n_pad / 32, 32 * kShares, s, p.st, p.w.part, p.w.ztgt, p.w.coef, parts,
                       g.n_pad, pb.reduction, p.w.rho, p.w.counters, p.w.sums, a->gdloss));
  if (a->gdloss != nullptr && pb.reduction == TTT_LCE_NONE) {
    lce_zero_rows_kernel<<<static_cast<unsigned>((pb.n + 255) / 256), 256, 0, s>>>(p.st.slot, pb.n, a->gdloss);
    TTT_TRY(launched());
  }
  return run_pieces(p, w, a->uw != nullptr ? &uw : nullptr, true, a->uh != nullptr, static_cast<uint16_t*>(a->gh),
                    static_cast<uint16_t*>(a->gw));
}

}  // extern "C"
