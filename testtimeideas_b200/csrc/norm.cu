// Layer norm over rows of D elements with its first and second gradient, and
// their C entry points (include/ttt_ops.h).
//
// With m() the mean over a row, xh = (x - m(x)) r, r = (var + eps)^-1/2 and the
// projection P(u) = u - m(u) - xh m(u xh):
//   forward   y  = xh w + b
//   gradient  dx = r P(g), g = dy w;   dw = sum_rows dy xh;   db = sum_rows dy
//   second    with the upstream gradients ux, uw, ub of dx, dw, db, and
//             a = m(g xh), c = m(ux xh), s = m(g P(ux)), h = dy uw:
//             gdy = w r P(ux) + xh uw + ub
//             gw  = sum_rows dy r P(ux)
//             gx  = r P(h - r (c g + a ux)) - r^2 s xh
// (the last term and the sign of the one before it come from dr/dx = -r^2 xh / D).
//
// All three are bound by memory: 2, 3 and 5 passes over [rows, D]. A row is read
// once and stays, packed as it came, in the registers of the NT threads that own
// it: eight elements each up to 2048 (16 to 32 above), so that a thread needs few
// registers (32 elements a thread took 170 and ran at a quarter of the bandwidth), and
// about as many threads as the row needs (8 lanes for 64 columns, three warps for 768).
// Rows come through shared memory up to three ahead of their turn (cp.async), which is
// what covers the memory's latency.
// Mean and variance are two sums over registers, and no statistic is a difference
// of large sums. The threads of a row own fixed columns, so the parameter gradients
// are summed in registers (wide rows: in shared memory, see Row) over all rows that a
// block meets; the blocks' sums (fp32) are added in block order by a second small kernel, launched ahead of the first
// one's end. Everything is computed in fp32 and rounded once on the way out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "prof.h"
#include "ttt_ops.h"

namespace {

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// EPT elements of a row as they lie in memory, two 16-bit elements to a register.
template <class T, int EPT>
struct Pack {
  uint32_t w[EPT / 2];
  __device__ __forceinline__ float at(int i) const {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
    } else {
      return __half2float(__ushort_as_half(static_cast<unsigned short>((i & 1) ? w[i >> 1] >> 16 : w[i >> 1])));
    }
  }
  // Elements i (even) and i + 1.
  __device__ __forceinline__ void set2(int i, float lo, float hi) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
      w[i >> 1] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(lo, hi);
      w[i >> 1] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  __device__ __forceinline__ void set_bits(int i, uint32_t bits) {
    w[i >> 1] = (i & 1) ? (w[i >> 1] & 0xffffu) | (bits << 16) : bits;
  }
  __device__ __forceinline__ uint32_t bits(int i) const { return (i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu; }
};
template <int EPT>
struct Pack<float, EPT> {
  uint32_t w[EPT];
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
  __device__ __forceinline__ void set2(int i, float lo, float hi) {
    w[i] = __float_as_uint(lo);
    w[i + 1] = __float_as_uint(hi);
  }
  __device__ __forceinline__ void set_bits(int i, uint32_t bits) { w[i] = bits; }
  __device__ __forceinline__ uint32_t bits(int i) const { return w[i]; }
};

// Keeps a row packed across a reduction: without it the compiler carries the
// unpacked (and centred) values over, at two to three times the registers.
template <class T, int EPT>
__device__ __forceinline__ void stay_packed(Pack<T, EPT>& v) {
  for (auto& w : v.w) asm volatile("" : "+r"(w));
}

// Threads that an SM holds, which leaves 65536 / threads registers to each: as many as hide
// the memory's latency without registers spilled inside the loop over the rows.
// Forward: 1024, but 512 where a thread has 32 elements (6710x10000 in fp32: 92 us against
// 231 with 1024) and 768 where it has 16 that it loads in small pieces (22362x3001 in bf16:
// 92 us against 118); with 8 elements fewer threads are slower (66974x1002: 62 against 67).
constexpr int fwd_threads(int ept, int piece_bytes) {
  return ept == 32 ? 512 : ept == 16 && piece_bytes < 16 ? 768 : 1024;
}
// Gradient: 512, but 768 where a thread has eight 16-bit elements, two sums a column among
// its registers all the same. Times of a forward and gradient, 768 against 512 threads:
// 43690x1536 143 and 173 us, 262144x256 136 and 151. Three layouts spill at 768: 128 threads
// a row (65536x1024: 170 and 147), 96 (87381x768: 172, 186, and 165 with 576) and rows loaded
// element by element (133949x501: 303 and 217; but 43662x1537, 256 threads: 240 and 266).
constexpr int grad_threads(int ept, int elem_bytes, int vec, int nt) {
  if (ept > 8 || elem_bytes > 2 || nt == 128 || (vec == 1 && nt < 256)) return 512;
  return nt == 96 ? 576 : 768;
}

// The layout of a row: NT threads (part of a warp, or whole warps), each with K pieces of
// VEC elements; piece k of thread t starts at column (k * NT + t) * VEC. VEC is 16 bytes
// of X, or 4 bytes, or one element, as the rows are aligned. A block holds GROUPS rows at
// a time. NT is a constant: with a number of threads known only at run time the kernels
// issue enough more instructions to lose a third of their speed.
template <class X, int NT_, int EPT_, int VEC_>
struct Row {
  static constexpr int NT = NT_, EPT = EPT_, VEC = VEC_, K = EPT / VEC;
  static constexpr int PIECE = VEC * static_cast<int>(sizeof(X));  // bytes
  static constexpr int GROUPS = NT > 256 ? 1 : 256 / NT, THREADS = GROUPS * NT;
  // Blocks that an SM holds.
  static constexpr int FWD_PER_SM = fwd_threads(EPT, PIECE) / THREADS;
  static constexpr int BWD_PER_SM = grad_threads(EPT, sizeof(X), VEC, NT) / THREADS;
  static constexpr int BWD2_PER_SM = 512 / THREADS;

  // Column sums in shared memory, each thread its own, where the loop over the rows spills with
  // them in registers. Forward and gradient: 8184x8200 in fp32 720 -> 302 us, 4096x16384 in bf16
  // 225 -> 173. Forward and both gradients, all in bf16: 16384x4096 374 -> 311, 8192x8192
  // 422 -> 366, 4096x16384 893 -> 440.
  static constexpr bool SHARED_SUMS = EPT == 32;
  static constexpr int SUM_BYTES = SHARED_SUMS ? 2 * EPT * THREADS * static_cast<int>(sizeof(float)) : 0;
  static constexpr bool SHARED_SUMS2 = EPT >= 16;
  static constexpr int SUM2_BYTES = SHARED_SUMS2 ? EPT * THREADS * static_cast<int>(sizeof(float)) : 0;

  static __device__ __forceinline__ int column(int k, int t) { return (k * NT + t) * VEC; }
  static __device__ __forceinline__ bool inside(int i, int t, int D) { return column(i / VEC, t) < D; }

  // Elements outside the row (or a null row) are `fill`.
  template <class T>
  static __device__ __forceinline__ void load(const T* row, int t, int D, Pack<T, EPT>& v, float fill = 0.f) {
    constexpr int WORDS = VEC * static_cast<int>(sizeof(T)) / 4;  // of a piece; T may be wider than X
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = column(k, t);
      const bool in = row != nullptr && c < D;
      if constexpr (VEC == 1) {
        T e = from_f<T>(fill);
        if (in) e = row[c];
        if constexpr (sizeof(T) == 4)
          v.set_bits(k, *reinterpret_cast<const uint32_t*>(&e));
        else
          v.set_bits(k, *reinterpret_cast<const uint16_t*>(&e));
      } else if constexpr (PIECE == 4) {
        static_assert(VEC == 2 && sizeof(X) == 2, "pairs of 16-bit elements");
        v.set2(k * 2, fill, fill);
        if (in) {
          if constexpr (sizeof(T) == 2) {
            v.w[k] = *reinterpret_cast<const uint32_t*>(row + c);
          } else {
            v.w[2 * k] = __float_as_uint(row[c]);
            v.w[2 * k + 1] = __float_as_uint(row[c + 1]);
          }
        }
      } else if (in) {
#pragma unroll
        for (int q = 0; q < WORDS / 4; ++q) {
          const uint4 u = reinterpret_cast<const uint4*>(row + c)[q];
          uint32_t* w = v.w + k * WORDS + q * 4;
          w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) v.set2(k * VEC + j, fill, fill);
      }
    }
  }
  template <class T>
  static __device__ __forceinline__ void store(T* row, int t, int D, const Pack<T, EPT>& v) {
    constexpr int WORDS = VEC * static_cast<int>(sizeof(T)) / 4;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = column(k, t);
      if (c >= D) continue;
      if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 4)
          reinterpret_cast<uint32_t*>(row)[c] = v.bits(k);
        else
          reinterpret_cast<uint16_t*>(row)[c] = static_cast<uint16_t>(v.bits(k));
      } else if constexpr (PIECE == 4) {
        *reinterpret_cast<uint32_t*>(row + c) = v.w[k];
      } else {
#pragma unroll
        for (int q = 0; q < WORDS / 4; ++q) {
          const uint32_t* w = v.w + k * WORDS + q * 4;
          reinterpret_cast<uint4*>(row + c)[q] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
};

// Sums of N values over the NT threads of a row, returned to all of them. Rows of
// several warps go through shared memory and a barrier of their own; `phase`
// alternates between two halves of the buffer so that one barrier is enough.
constexpr int kMaxSums = 6;
// The block's row of this thread's first lane: where several rows share a warp, the warp
// goes on together for as long as its first row exists.
template <class R>
__device__ __forceinline__ int lead_row() {
  return R::NT < 32 ? static_cast<int>(threadIdx.x & ~31u) / R::NT : static_cast<int>(threadIdx.x) / R::NT;
}
template <class R>
struct Sums {
  static constexpr int W = R::NT > 32 ? R::NT / 32 : 1, ROWS = R::NT > 32 ? R::GROUPS : 1;
  float red[ROWS][2][kMaxSums][W];
};
template <class R, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], Sums<R>& sums, int& phase) {
#pragma unroll
  for (int o = (R::NT < 32 ? R::NT : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if constexpr (R::NT > 32) {
    constexpr int W = R::NT / 32;
    const int grp = threadIdx.x / R::NT, warp = (threadIdx.x % R::NT) >> 5;
    auto& buf = sums.red[grp][phase];
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[i][warp] = v[i];
    }
    if constexpr (R::GROUPS == 1)
      __syncthreads();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(grp + 1), "n"(R::NT) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += buf[i][w];
      v[i] = s;
    }
  }
}

// Rows on their way through shared memory: T tensors, S rows ahead of the one being
// summed (cp.async, 16 bytes a thread and piece). A thread reads back only what it
// copied itself, so no barrier is needed. Rows that are not 16-byte aligned, or so wide
// that fewer than two fit, are loaded into registers one row ahead instead (S = 0).
template <class X, class R, int T, int PER_SM, int TAKEN = 0>
struct Ring {
  static constexpr int ROW = R::K * R::THREADS * 16;  // bytes of one tensor's rows of a block
  static constexpr int FIT = ((200 << 10) - PER_SM * TAKEN) / (PER_SM * T * ROW);
  static constexpr int S = R::PIECE < 16 || FIT < 2 ? 0 : (FIT < 4 ? FIT : 4);
  static constexpr int BYTES = S * T * ROW;
  const X* src[T];
  int64_t stride[T];
  uint32_t base;
  int t, D;

  // Starts the copies of row `at` (none past the end) into stage `st`.
  __device__ __forceinline__ void fetch(int64_t at, int64_t rows, int st) const {
    if (at < rows) {
#pragma unroll
      for (int i = 0; i < T; ++i) {
        if (src[i] == nullptr) continue;
        const X* row = src[i] + at * stride[i];
#pragma unroll
        for (int k = 0; k < R::K; ++k) {
          const int c = R::column(k, t);
          if (c < D)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             base + (st * T + i) * ROW + k * R::THREADS * 16),
                         "l"(row + c)
                         : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The oldest row's copies have landed (S - 1 newer rows may be on their way).
  __device__ __forceinline__ void wait() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(S > 0 ? S - 1 : 0) : "memory");
  }
  // Tensor i of the row in stage `st`; zeros outside it, and where there is no such row.
  __device__ __forceinline__ void read(int st, int i, bool exists, Pack<X, R::EPT>& v) const {
    constexpr int WORDS = 4;
#pragma unroll
    for (int k = 0; k < R::K; ++k) {
      uint32_t* w = v.w + k * WORDS;
      if (exists && src[i] != nullptr && R::column(k, t) < D) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(base + (st * T + i) * ROW + k * R::THREADS * 16)
                     : "memory");
      } else {
        w[0] = w[1] = w[2] = w[3] = 0;
      }
    }
  }
};
template <class G>
__device__ __forceinline__ G make_ring(uint8_t* smem, int t, int D) {
  G g;
  g.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16;
  g.t = t;
  g.D = D;
  return g;
}
template <class X, class R>
using FwdRing = Ring<X, R, 1, R::FWD_PER_SM>;
template <class X, class R>
using BwdRing = Ring<X, R, 2, R::BWD_PER_SM, R::SUM_BYTES>;
template <class X, class R>
using Bwd2Ring = Ring<X, R, 3, R::BWD2_PER_SM, R::SUM2_BYTES>;

template <class X, class P>
struct NormArgs {
  const X *x, *dy, *ux;
  int64_t x_stride, dy_stride, ux_stride;
  const P *w, *b, *uw, *ub;
  float *mean, *rstd;
  X *y, *dx, *gx, *gdy;
  float* part;  // [blocks][2][D] sums of the parameter gradients
  int want_dw, want_db;
  int64_t rows;
  int D;
  float eps;
};

template <class X, class P, class R>
__global__ void __launch_bounds__(R::THREADS, R::FWD_PER_SM) norm_fwd_kernel(const NormArgs<X, P> a) {
  constexpr int EPT = R::EPT;
  using G = FwdRing<X, R>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Sums<R> sums;
  int phase = 0;
  const int t = threadIdx.x % R::NT;
  const float inv = 1.f / static_cast<float>(a.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * R::GROUPS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * R::GROUPS + threadIdx.x / R::NT;
  int64_t lead = static_cast<int64_t>(blockIdx.x) * R::GROUPS + lead_row<R>();
  G g = make_ring<G>(smem, t, a.D);
  g.src[0] = a.x;
  g.stride[0] = a.x_stride;
  Pack<X, EPT> xn;  // S = 0: the next row
  if constexpr (G::S > 0) {
#pragma unroll
    for (int i = 0; i < G::S - 1; ++i) g.fetch(row + i * step, a.rows, i);
  } else {
    R::load(row < a.rows ? a.x + row * a.x_stride : nullptr, t, a.D, xn);
  }
  Pack<P, EPT> w, b;
  R::load(a.w, t, a.D, w, 1.f);
  R::load(a.b, t, a.D, b, 0.f);
  for (int st = 0; (R::NT < 32 ? lead : row) < a.rows; row += step, lead += step) {
    const bool exists = R::NT >= 32 || row < a.rows;
    Pack<X, EPT> x;
    if constexpr (G::S > 0) {
      g.fetch(row + (G::S - 1) * step, a.rows, (st + G::S - 1) % G::S);
      g.wait();
      g.read(st, 0, exists, x);
      st = (st + 1) % G::S;
    } else {
      x = xn;
      R::load(row + step < a.rows ? a.x + (row + step) * a.x_stride : nullptr, t, a.D, xn);
    }
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < EPT; ++i) s[0] += x.at(i);
    row_sum<R, 1>(s, sums, phase);
    const float mu = s[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float c = x.at(i) - mu;
      q[0] += R::inside(i, t, a.D) ? c * c : 0.f;
    }
    row_sum<R, 1>(q, sums, phase);
    const float r = rsqrtf(q[0] * inv + a.eps);
#pragma unroll
    for (int i = 0; i < EPT; i += 2)
      x.set2(i, (x.at(i) - mu) * r * w.at(i) + b.at(i), (x.at(i + 1) - mu) * r * w.at(i + 1) + b.at(i + 1));
    if (exists) {
      R::store(a.y + row * a.D, t, a.D, x);
      if (t == 0 && a.mean != nullptr) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
    }
  }
}

// Adds the row groups' column sums of a block and writes them to
// part[block][which]; acc holds this thread's columns.
template <class R>
__device__ __forceinline__ void write_part(float* part, int which, int D, const float (&acc)[R::EPT], float* cols) {
  const int t = threadIdx.x % R::NT;
  float* dst = part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * D;
  if constexpr (R::GROUPS == 1) {
#pragma unroll
    for (int i = 0; i < R::EPT; ++i) {
      const int c = R::column(i / R::VEC, t) + i % R::VEC;
      if (c < D) dst[c] = acc[i];
    }
  } else {
    const int grp = threadIdx.x / R::NT;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R::EPT; ++i) {
      const int c = R::column(i / R::VEC, t) + i % R::VEC;
      if (c < D) cols[grp * D + c] = acc[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += R::THREADS) {
      float s = 0.f;
#pragma unroll 8
      for (int gi = 0; gi < R::GROUPS; ++gi) s += cols[gi * D + c];
      dst[c] = s;
    }
  }
}

template <class X, class P, class R>
__global__ void __launch_bounds__(R::THREADS, R::BWD_PER_SM) norm_bwd_kernel(const NormArgs<X, P> a) {
  constexpr int EPT = R::EPT;
  using G = BwdRing<X, R>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* cols = reinterpret_cast<float*>(smem + G::BYTES);
  __shared__ Sums<R> sums;
  int phase = 0;
  asm volatile("griddepcontrol.launch_dependents;");  // the parameter sums wait for this grid's end
  const int t = threadIdx.x % R::NT;
  const float inv = 1.f / static_cast<float>(a.D);
  float aw[EPT], ab[EPT];
  float* own = cols + threadIdx.x;  // SHARED_SUMS: element i of aw at own[i * THREADS], then ab's
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    aw[i] = ab[i] = 0.f;
    if constexpr (R::SHARED_SUMS) own[i * R::THREADS] = own[(EPT + i) * R::THREADS] = 0.f;
  }
  Pack<P, EPT> w;
  R::load(a.w, t, a.D, w, 1.f);
  const int64_t step = static_cast<int64_t>(gridDim.x) * R::GROUPS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * R::GROUPS + threadIdx.x / R::NT;
  int64_t lead = static_cast<int64_t>(blockIdx.x) * R::GROUPS + lead_row<R>();
  G ring = make_ring<G>(smem, t, a.D);
  ring.src[0] = a.x, ring.stride[0] = a.x_stride;
  ring.src[1] = a.dy, ring.stride[1] = a.dy_stride;
  // S = 0: the next row, where there are registers for it (rows of 32 elements: 16-bit ones in
  // wide pieces; 7455x9001 in bf16 531 us with it, 348 without)
  Pack<X, EPT> xn, dn;
  constexpr bool AHEAD = EPT < 32 || R::PIECE * sizeof(X) == 32;
  float mun[2] = {0.f, 0.f}, rn[2] = {0.f, 0.f};  // statistics of the next two rows
  auto fetch_stats = [&](int64_t at, int i) {
    if (at < a.rows) mun[i] = a.mean[at], rn[i] = a.rstd[at];
  };
  auto fetch_rows = [&](int64_t at) {
    R::load(at < a.rows ? a.x + at * a.x_stride : nullptr, t, a.D, xn);
    R::load(at < a.rows ? a.dy + at * a.dy_stride : nullptr, t, a.D, dn);
  };
  fetch_stats(row, 0);
  fetch_stats(row + step, 1);
  if constexpr (G::S > 0) {
#pragma unroll
    for (int i = 0; i < G::S - 1; ++i) ring.fetch(row + i * step, a.rows, i);
  } else if constexpr (AHEAD) {
    fetch_rows(row);
  }
  for (int st = 0; (R::NT < 32 ? lead : row) < a.rows; row += step, lead += step) {
    const bool exists = R::NT >= 32 || row < a.rows;
    Pack<X, EPT> x, dy;
    const float mu = mun[0], r = rn[0];
    mun[0] = mun[1], rn[0] = rn[1];
    fetch_stats(row + 2 * step, 1);
    if constexpr (G::S > 0) {
      ring.fetch(row + (G::S - 1) * step, a.rows, (st + G::S - 1) % G::S);
      ring.wait();
      ring.read(st, 0, exists, x);
      ring.read(st, 1, exists, dy);
      st = (st + 1) % G::S;
    } else {
      if constexpr (!AHEAD) fetch_rows(row);
      x = xn, dy = dn;
      if constexpr (AHEAD) fetch_rows(row + step);
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      // dy is zero outside the row (and past the last row), so nothing else has to be
      const float xh = (x.at(i) - mu) * r, d = dy.at(i), g = d * w.at(i);
      if constexpr (R::SHARED_SUMS) {
        own[i * R::THREADS] += d * xh;
        own[(EPT + i) * R::THREADS] += d;
      } else {
        aw[i] += d * xh;
        ab[i] += d;
      }
      s[0] += g;
      s[1] += g * xh;
    }
    row_sum<R, 2>(s, sums, phase);
    stay_packed(x);
    stay_packed(dy);
    stay_packed(w);
    if (a.dx != nullptr && exists) {
      const float mg = s[0] * inv, ma = s[1] * inv;
#pragma unroll
      for (int i = 0; i < EPT; i += 2)
        x.set2(i, r * (dy.at(i) * w.at(i) - mg - (x.at(i) - mu) * r * ma),
               r * (dy.at(i + 1) * w.at(i + 1) - mg - (x.at(i + 1) - mu) * r * ma));
      R::store(a.dx + row * a.D, t, a.D, x);
    }
  }
  if constexpr (R::SHARED_SUMS) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) aw[i] = own[i * R::THREADS], ab[i] = own[(EPT + i) * R::THREADS];
  }
  if (a.want_dw) write_part<R>(a.part, 0, a.D, aw, cols);
  if (a.want_db) write_part<R>(a.part, 1, a.D, ab, cols);
}

template <class X, class P, class R>
__global__ void __launch_bounds__(R::THREADS, R::BWD2_PER_SM) norm_bwd2_kernel(const NormArgs<X, P> a) {
  constexpr int EPT = R::EPT;
  using G = Bwd2Ring<X, R>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* cols = reinterpret_cast<float*>(smem + G::BYTES);
  __shared__ Sums<R> sums;
  int phase = 0;
  asm volatile("griddepcontrol.launch_dependents;");
  const int t = threadIdx.x % R::NT;
  const float inv = 1.f / static_cast<float>(a.D);
  float agw[EPT];
  float* own = cols + threadIdx.x;  // SHARED_SUMS2: element i of agw at own[i * THREADS]
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    agw[i] = 0.f;
    if constexpr (R::SHARED_SUMS2) own[i * R::THREADS] = 0.f;
  }
  Pack<P, EPT> w, uw, ub;
  constexpr bool RELOAD = EPT == 32;  // the parameters, for each pass over the row: no registers to keep them
  if constexpr (!RELOAD) {
    R::load(a.w, t, a.D, w, 1.f);
    R::load(a.uw, t, a.D, uw);
    R::load(a.ub, t, a.D, ub);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * R::GROUPS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * R::GROUPS + threadIdx.x / R::NT;
  int64_t lead = static_cast<int64_t>(blockIdx.x) * R::GROUPS + lead_row<R>();
  G ring = make_ring<G>(smem, t, a.D);
  ring.src[0] = a.x, ring.stride[0] = a.x_stride;
  ring.src[1] = a.dy, ring.stride[1] = a.dy_stride;
  ring.src[2] = a.ux, ring.stride[2] = a.ux_stride;
  float mun = 0.f, rn = 0.f;
  if (row < a.rows) mun = a.mean[row], rn = a.rstd[row];
  if constexpr (G::S > 0) {
#pragma unroll
    for (int i = 0; i < G::S - 1; ++i) ring.fetch(row + i * step, a.rows, i);
  }
  for (int st = 0; (R::NT < 32 ? lead : row) < a.rows; row += step, lead += step) {
    const bool exists = R::NT >= 32 || row < a.rows;
    const float mu = mun, r = rn;
    if (row + step < a.rows) mun = a.mean[row + step], rn = a.rstd[row + step];
    Pack<X, EPT> x, dy, u;
    if constexpr (G::S > 0) {
      ring.fetch(row + (G::S - 1) * step, a.rows, (st + G::S - 1) % G::S);
      ring.wait();
      ring.read(st, 0, exists, x);
      ring.read(st, 1, exists, dy);
      ring.read(st, 2, exists, u);
      st = (st + 1) % G::S;
    } else {
      R::load(exists ? a.x + row * a.x_stride : nullptr, t, a.D, x);
      R::load(exists ? a.dy + row * a.dy_stride : nullptr, t, a.D, dy);
      R::load(exists && a.ux != nullptr ? a.ux + row * a.ux_stride : nullptr, t, a.D, u);
    }
    if constexpr (RELOAD) {
      R::load(a.w, t, a.D, w, 1.f);
      R::load(a.uw, t, a.D, uw);
    }
    float s[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // g, u, g xh, u xh, h, h xh
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      // dy and u are zero outside the row
      const float xh = (x.at(i) - mu) * r, d = dy.at(i);
      const float g = d * w.at(i), h = d * uw.at(i);
      s[0] += g;
      s[1] += u.at(i);
      s[2] += g * xh;
      s[3] += u.at(i) * xh;
      s[4] += h;
      s[5] += h * xh;
    }
    row_sum<R, 6>(s, sums, phase);
    stay_packed(x);
    stay_packed(dy);
    stay_packed(u);
    stay_packed(w);
    stay_packed(uw);
    const float mg = s[0] * inv, mu_u = s[1] * inv, ma = s[2] * inv, mc = s[3] * inv;
    float q[1] = {0.f};
    if constexpr (RELOAD) R::load(a.w, t, a.D, w, 1.f);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float xh = (x.at(i) - mu) * r;
      q[0] += dy.at(i) * w.at(i) * (u.at(i) - mu_u - xh * mc);  // dy again
    }
    row_sum<R, 1>(q, sums, phase);
    stay_packed(x);
    stay_packed(dy);
    stay_packed(u);
    stay_packed(w);
    const float ms = q[0] * inv;
    if constexpr (RELOAD) {
      R::load(a.w, t, a.D, w, 1.f);
      R::load(a.uw, t, a.D, uw);
      R::load(a.ub, t, a.D, ub);
    }
    // v = h - r (c g + a u): its mean and its mean against xh
    const float mv = s[4] * inv - r * (mc * mg + ma * mu_u);
    const float mvx = s[5] * inv - 2.f * r * ma * mc;
#pragma unroll
    for (int i = 0; i < EPT; i += 2) {
      float gd[2], gx[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float xh = (x.at(i + j) - mu) * r, d = dy.at(i + j);
        const float pu = r * (u.at(i + j) - mu_u - xh * mc);
        const float v = d * uw.at(i + j) - r * (mc * d * w.at(i + j) + ma * u.at(i + j));
        if constexpr (R::SHARED_SUMS2)
          own[(i + j) * R::THREADS] += d * pu;
        else
          agw[i + j] += d * pu;
        gd[j] = w.at(i + j) * pu + xh * uw.at(i + j) + ub.at(i + j);
        gx[j] = r * (v - mv - xh * mvx) - r * r * ms * xh;
      }
      dy.set2(i, gd[0], gd[1]);
      x.set2(i, gx[0], gx[1]);
    }
    if (exists) {
      R::store(a.gdy + row * a.D, t, a.D, dy);
      R::store(a.gx + row * a.D, t, a.D, x);
    }
  }
  if constexpr (R::SHARED_SUMS2) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) agw[i] = own[i * R::THREADS];
  }
  if (a.want_dw) write_part<R>(a.part, 0, a.D, agw, cols);
}

// out[c] = sum over blocks of part[block][which][c]: 32 interleaved shares, each in
// block order, then the shares in order. One block: 32 columns of one array.
template <class P>
__global__ void __launch_bounds__(1024) norm_param_reduce_kernel(const float* part, int blocks, int D, P* dw, P* db) {
  __shared__ float s[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the blocks' sums are complete
  const int which = blockIdx.y;
  P* out = which == 0 ? dw : db;
  if (out == nullptr) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float acc = 0.f;
  if (c < D) {
#pragma unroll 4
    for (int p = ty; p < blocks; p += 32) acc += part[(static_cast<int64_t>(p) * 2 + which) * D + c];
  }
  s[ty][tx] = acc;
  __syncthreads();
  if (ty == 0 && c < D) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += s[i][tx];
    out[c] = from_f<P>(v);
  }
}

// ---------------------------------------------------------------- host side
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
  return n < 1 ? 1 : n;
}

// Threads of a row: eight elements each up to 2048 columns, then 16 and 32. Aligned rows
// have 8 to 256 threads with steps of a half between 64 and 256, others powers of two
// from a warp up (which keeps the number of kernels down).
int row_threads(int D, bool wide) {
  if (D > 4096) return 512;
  if (D > 2048) return 256;
  if (wide)
    for (const int nt : {8, 16, 32, 64, 96, 128, 192})
      if (nt * 8 >= D) return nt;
  int nt = 32;
  while (nt * 8 < D) nt *= 2;
  return nt;
}

// Blocks of the gradient kernels: all that fit on the SMs at once, or as many as there are rows for.
int grad_blocks(const ttt_norm_problem& pb, bool second, int vec, int sms) {
  const int elem = pb.dtype == TTT_F32 ? 4 : 2;
  const int nt = row_threads(pb.dim, vec * elem == 16), groups = nt > 256 ? 1 : 256 / nt, threads = groups * nt;
  const int64_t fit = second ? 512 : grad_threads(pb.dim <= 2048 ? 8 : 16, elem, vec, nt);
  return static_cast<int>(
      std::min<int64_t>(std::max<int64_t>((pb.rows + groups - 1) / groups, 1), sms * (fit / threads)));
}

int check_norm(const ttt_norm_problem& pb) {
  if (pb.dtype != TTT_F16 && pb.dtype != TTT_BF16 && pb.dtype != TTT_F32) return TTT_ERR_DTYPE;
  if (pb.p_dtype != pb.dtype && pb.p_dtype != TTT_F32) return TTT_ERR_DTYPE;
  if (pb.rows < 0 || pb.rows > 0x7fffffff || pb.dim < 1 || pb.dim > TTT_NORM_MAX_DIM) return TTT_ERR_SHAPE;
  return TTT_OK;
}

enum Pass { kFwd, kBwd, kBwd2 };

template <class X, class P, class R>
cudaError_t launch_rows(const NormArgs<X, P>& a, Pass pass, int blocks, int sms, cudaStream_t s) {
  auto launch = [&](auto kern, int64_t grid, int smem) {
    if (smem > 32 * 1024) {  // 48 KB, the kernels' static shared memory included, need no permission
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
    }
    kern<<<static_cast<unsigned>(grid), R::THREADS, smem, s>>>(a);
    return cudaGetLastError();
  };
  if (pass == kFwd) {
    const int64_t need = (a.rows + R::GROUPS - 1) / R::GROUPS, fit = static_cast<int64_t>(sms) * R::FWD_PER_SM;
    return launch(norm_fwd_kernel<X, P, R>, std::min(need, fit), FwdRing<X, R>::BYTES);
  }
  // several rows a block: their column sums, at most 8 KB (D <= 8 NT, 256 threads)
  const int cols = R::GROUPS > 1 ? static_cast<int>(sizeof(float)) * R::GROUPS * a.D : 0;
  if (pass == kBwd) return launch(norm_bwd_kernel<X, P, R>, blocks, BwdRing<X, R>::BYTES + R::SUM_BYTES + cols);
  return launch(norm_bwd2_kernel<X, P, R>, blocks, Bwd2Ring<X, R>::BYTES + R::SUM2_BYTES + cols);
}

template <class X, class P, int VEC>
cudaError_t launch_width(const NormArgs<X, P>& a, Pass pass, int blocks, int sms, cudaStream_t s) {
  constexpr bool WIDE = VEC * sizeof(X) == 16;
  if (a.D > 8192) return launch_rows<X, P, Row<X, 512, 32, VEC>>(a, pass, blocks, sms, s);
  if (a.D > 4096) return launch_rows<X, P, Row<X, 512, 16, VEC>>(a, pass, blocks, sms, s);
  if (a.D > 2048) return launch_rows<X, P, Row<X, 256, 16, VEC>>(a, pass, blocks, sms, s);
  switch (row_threads(a.D, WIDE)) {
    case 8:
      if constexpr (WIDE) return launch_rows<X, P, Row<X, 8, 8, VEC>>(a, pass, blocks, sms, s);
      break;
    case 16:
      if constexpr (WIDE) return launch_rows<X, P, Row<X, 16, 8, VEC>>(a, pass, blocks, sms, s);
      break;
    case 96:
      if constexpr (WIDE) return launch_rows<X, P, Row<X, 96, 8, VEC>>(a, pass, blocks, sms, s);
      break;
    case 192:
      if constexpr (WIDE) return launch_rows<X, P, Row<X, 192, 8, VEC>>(a, pass, blocks, sms, s);
      break;
    case 32: return launch_rows<X, P, Row<X, 32, 8, VEC>>(a, pass, blocks, sms, s);
    case 64: return launch_rows<X, P, Row<X, 64, 8, VEC>>(a, pass, blocks, sms, s);
    case 128: return launch_rows<X, P, Row<X, 128, 8, VEC>>(a, pass, blocks, sms, s);
    default: return launch_rows<X, P, Row<X, 256, 8, VEC>>(a, pass, blocks, sms, s);
  }
  return cudaErrorInvalidValue;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class X, class P>
int run_norm(NormArgs<X, P> a, const ttt_norm_problem& pb, Pass pass, void* dw, void* db, void* work,
             int64_t work_bytes, cudaStream_t s) {
  a.rows = pb.rows;
  a.D = pb.dim;
  a.eps = pb.eps;
  a.want_dw = dw != nullptr;
  a.want_db = db != nullptr;
  const int sms = sm_count();
  // 16-byte pieces need every row and every parameter vector on a 16-byte boundary, 4-byte
  // pieces (two 16-bit elements) the rows and 16-bit parameters on a 4-byte one
  constexpr int V = 16 / static_cast<int>(sizeof(X)), H = 4 / static_cast<int>(sizeof(X));
  const void* rows_at[] = {a.x, a.dy, a.ux, a.y, a.dx, a.gx, a.gdy};
  const void* params_at[] = {a.w, a.b, a.uw, a.ub};
  uintptr_t row_bits = 0, param_bits = 0;
  for (const void* p : rows_at) row_bits |= reinterpret_cast<uintptr_t>(p);
  for (const void* p : params_at) param_bits |= reinterpret_cast<uintptr_t>(p);
  const int64_t steps = pb.dim | a.x_stride | a.dy_stride | a.ux_stride;
  const int vec = ((row_bits | param_bits) & 15) == 0 && steps % V == 0  ? V
                  : ((row_bits | param_bits) & 3) == 0 && steps % H == 0 ? H
                                                                         : 1;
  const int blocks = pass == kFwd ? 0 : grad_blocks(pb, pass == kBwd2, vec, sms);
  if (a.want_dw || a.want_db) {
    if (work == nullptr || !aligned16(work) || work_bytes < static_cast<int64_t>(blocks) * 2 * pb.dim * 4)
      return TTT_ERR_SCRATCH;
    a.part = static_cast<float*>(work);
  }
  if (pb.rows > 0 || pass != kFwd) {
    cudaError_t e;
    if (vec == V)
      e = launch_width<X, P, V>(a, pass, blocks, sms, s);
    else if (vec == H && H == 2)
      e = launch_width<X, P, H>(a, pass, blocks, sms, s);
    else
      e = launch_width<X, P, 1>(a, pass, blocks, sms, s);
    if (e != cudaSuccess) return TTT_ERR_LAUNCH;
  }
  if (a.want_dw || a.want_db) {
    const dim3 grid((pb.dim + 31) / 32, a.want_db ? 2 : 1);
    cudaLaunchAttribute early;  // may start before the gradient kernel's end, for which it waits itself
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, norm_param_reduce_kernel<P>, static_cast<const float*>(a.part), blocks, pb.dim,
                           static_cast<P*>(dw), static_cast<P*>(db)) != cudaSuccess)
      return TTT_ERR_LAUNCH;
  }
  return TTT_OK;
}

// Calls f(X{}, P{}) for the problem's element types.
template <class F>
int with_types(const ttt_norm_problem& pb, F f) {
  const bool p32 = pb.p_dtype == TTT_F32;
  if (pb.dtype == TTT_F32) return f(float{}, float{});
  if (pb.dtype == TTT_F16) return p32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return p32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

}  // namespace

extern "C" {

int64_t ttt_norm_work_bytes(const ttt_norm_problem* pb) {
  if (pb == nullptr || check_norm(*pb) != TTT_OK) return 0;
  const int sms = sm_count();
  int blocks = 0;  // the gradient's, in whichever layout has most of them
  for (const int vec : {1, 2, 4, 8})
    for (const bool second : {false, true}) blocks = std::max(blocks, grad_blocks(*pb, second, vec, sms));
  return static_cast<int64_t>(blocks) * 2 * pb->dim * 4;
}

int ttt_norm_fwd(const ttt_norm_fwd_args* g, void* stream) {
  if (g == nullptr) return TTT_ERR_NULL;
  if (const int st = check_norm(g->pb)) return st;
  if (g->pb.rows > 0 && (g->x == nullptr || g->y == nullptr)) return TTT_ERR_NULL;
  if ((g->mean == nullptr) != (g->rstd == nullptr)) return TTT_ERR_NULL;
  if (g->x_stride < 0) return TTT_ERR_STRIDE;
  ttt::ProfSpan prof(TTT_K_NORM, stream);
  return with_types(g->pb, [&](auto xt, auto pt) {
    using X = decltype(xt);
    using P = decltype(pt);
    NormArgs<X, P> a{};
    a.x = static_cast<const X*>(g->x);
    a.x_stride = g->x_stride;
    a.w = static_cast<const P*>(g->w);
    a.b = static_cast<const P*>(g->b);
    a.y = static_cast<X*>(g->y);
    a.mean = g->mean;
    a.rstd = g->rstd;
    return run_norm<X, P>(a, g->pb, kFwd, nullptr, nullptr, nullptr, 0, static_cast<cudaStream_t>(stream));
  });
}

int ttt_norm_bwd(const ttt_norm_bwd_args* g, void* stream) {
  if (g == nullptr) return TTT_ERR_NULL;
  if (const int st = check_norm(g->pb)) return st;
  if (g->pb.rows > 0 && (g->x == nullptr || g->dy == nullptr || g->mean == nullptr || g->rstd == nullptr))
    return TTT_ERR_NULL;
  if (g->x_stride < 0 || g->dy_stride < 0) return TTT_ERR_STRIDE;
  ttt::ProfSpan prof(TTT_K_NORM, stream);
  return with_types(g->pb, [&](auto xt, auto pt) {
    using X = decltype(xt);
    using P = decltype(pt);
    NormArgs<X, P> a{};
    a.x = static_cast<const X*>(g->x);
    a.dy = static_cast<const X*>(g->dy);
    a.x_stride = g->x_stride;
    a.dy_stride = g->dy_stride;
    a.w = static_cast<const P*>(g->w);
    a.mean = const_cast<float*>(g->mean);
    a.rstd = const_cast<float*>(g->rstd);
    a.dx = static_cast<X*>(g->dx);
    return run_norm<X, P>(a, g->pb, kBwd, g->dw, g->db, g->work, g->work_bytes, static_cast<cudaStream_t>(stream));
  });
}

int ttt_norm_bwd2(const ttt_norm_bwd2_args* g, void* stream) {
  if (g == nullptr) return TTT_ERR_NULL;
  if (const int st = check_norm(g->pb)) return st;
  if (g->pb.rows > 0 && (g->x == nullptr || g->dy == nullptr || g->mean == nullptr || g->rstd == nullptr ||
                         g->gx == nullptr || g->gdy == nullptr))
    return TTT_ERR_NULL;
  if (g->x_stride < 0 || g->dy_stride < 0 || g->ux_stride < 0) return TTT_ERR_STRIDE;
  ttt::ProfSpan prof(TTT_K_NORM, stream);
  return with_types(g->pb, [&](auto xt, auto pt) {
    using X = decltype(xt);
    using P = decltype(pt);
    NormArgs<X, P> a{};
    a.x = static_cast<const X*>(g->x);
    a.dy = static_cast<const X*>(g->dy);
    a.ux = static_cast<const X*>(g->ux);
    a.x_stride = g->x_stride;
    a.dy_stride = g->dy_stride;
    a.ux_stride = g->ux_stride;
    a.w = static_cast<const P*>(g->w);
    a.uw = static_cast<const P*>(g->uw);
    a.ub = static_cast<const P*>(g->ub);
    a.mean = const_cast<float*>(g->mean);
    a.rstd = const_cast<float*>(g->rstd);
    a.gx = static_cast<X*>(g->gx);
    a.gdy = static_cast<X*>(g->gdy);
    return run_norm<X, P>(a, g->pb, kBwd2, g->gw, nullptr, g->work, g->work_bytes,
                          static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
