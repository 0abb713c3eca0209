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
// once and stays in the registers of the NT threads that own it (a warp up to
// 1024 elements, a block of 128 or 512 threads above), so mean and variance are
// two sums over registers, and no statistic is a difference of large sums. The
// threads of a row own fixed columns, so the parameter gradients are summed in
// registers over all rows that a block meets; the blocks' sums (fp32) are added
// in block order by a second small kernel. Everything is computed in fp32 and
// rounded once on the way out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ttt_ops.h"

namespace {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
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

// N consecutive elements starting at p; N * sizeof(T) is 16 bytes or a multiple
// of it (then p is 16-byte aligned), or N is 1.
template <class T, int N>
__device__ __forceinline__ void load_n(const T* p, float* v) {
  if constexpr (N == 1) {
    v[0] = to_f(*p);
  } else {
    constexpr int PER = 16 / sizeof(T);
    static_assert(N % PER == 0, "whole 16-byte pieces");
#pragma unroll
    for (int q = 0; q < N / PER; ++q) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + q * PER);
      T e[PER];
      *reinterpret_cast<uint4*>(e) = u;
#pragma unroll
      for (int j = 0; j < PER; ++j) v[q * PER + j] = to_f(e[j]);
    }
  }
}
template <class T, int N>
__device__ __forceinline__ void store_n(T* p, const float* v) {
  if constexpr (N == 1) {
    *p = from_f<T>(v[0]);
  } else {
    constexpr int PER = 16 / sizeof(T);
    static_assert(N % PER == 0, "whole 16-byte pieces");
#pragma unroll
    for (int q = 0; q < N / PER; ++q) {
      __align__(16) T e[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) e[j] = from_f<T>(v[q * PER + j]);
      *reinterpret_cast<uint4*>(p + q * PER) = *reinterpret_cast<const uint4*>(e);
    }
  }
}

// The layout of a row: NT threads, each with K pieces of VEC elements; piece k
// of thread t starts at column (k * NT + t) * VEC. VEC is 16 bytes of X, or 1
// for rows that are not 16-byte aligned.
template <class X, int NT_, int EPT_, bool WIDE>
struct Row {
  static constexpr int NT = NT_, EPT = EPT_;
  static constexpr int VEC = WIDE ? 16 / static_cast<int>(sizeof(X)) : 1;
  static constexpr int K = EPT / VEC;
  // Threads of a block: eight rows (warps) per block for warp rows, else one row.
  static constexpr int GROUPS = NT == 32 ? 8 : 1;
  static constexpr int THREADS = NT * GROUPS;

  template <class T>
  static __device__ __forceinline__ void load(const T* row, int t, int D, float (&v)[EPT], float fill = 0.f) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + t) * VEC;
      if (row != nullptr && c < D) {
        load_n<T, VEC>(row + c, v + k * VEC);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k * VEC + j] = fill;
      }
    }
  }
  template <class T>
  static __device__ __forceinline__ void store(T* row, int t, int D, const float (&v)[EPT]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + t) * VEC;
      if (c < D) store_n<T, VEC>(row + c, v + k * VEC);
    }
  }
  static __device__ __forceinline__ bool inside(int i, int t, int D) { return ((i / VEC) * NT + t) * VEC < D; }
};

// Sums of N values over the NT threads of a row, returned to all of them. Block
// rows go through shared memory; `red` holds 2 * N * NT/32 floats, and `phase`
// alternates its halves so that one barrier per reduction is enough.
template <int NT, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& phase) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if constexpr (NT > 32) {
    constexpr int W = NT / 32;
    float* buf = red + phase * 8 * W;
    phase ^= 1;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[i * W + warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += buf[i * W + w];
      v[i] = s;
    }
  }
}

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
__global__ void __launch_bounds__(R::THREADS) norm_fwd_kernel(const NormArgs<X, P> a) {
  constexpr int EPT = R::EPT;
  __shared__ float red[R::NT > 32 ? 16 * (R::NT / 32) : 1];
  int phase = 0;
  const int t = threadIdx.x % R::NT;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * R::GROUPS + threadIdx.x / R::NT;
  if (row >= a.rows) return;  // whole warps (warp rows) or no thread at all (block rows)
  const float inv = 1.f / static_cast<float>(a.D);
  float x[EPT];
  R::load(a.x + row * a.x_stride, t, a.D, x);
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < EPT; ++i) s[0] += x[i];
  row_sum<R::NT, 1>(s, red, phase);
  const float mu = s[0] * inv;
  float q[1] = {0.f};
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    x[i] -= mu;
    q[0] += R::inside(i, t, a.D) ? x[i] * x[i] : 0.f;
  }
  row_sum<R::NT, 1>(q, red, phase);
  const float r = rsqrtf(q[0] * inv + a.eps);
  float w[EPT], b[EPT];
  R::load(a.w, t, a.D, w, 1.f);
  R::load(a.b, t, a.D, b, 0.f);
#pragma unroll
  for (int i = 0; i < EPT; ++i) x[i] = x[i] * r * w[i] + b[i];
  R::store(a.y + row * a.D, t, a.D, x);
  if (t == 0 && a.mean != nullptr) {
    a.mean[row] = mu;
    a.rstd[row] = r;
  }
}

// Adds the row groups' column sums of a block and writes them to
// part[block][which]; acc holds this thread's columns.
template <class R>
__device__ __forceinline__ void write_part(float* part, int which, int D, const float (&acc)[R::EPT], float* sums) {
  const int t = threadIdx.x % R::NT;
  float* dst = part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * D;
  if constexpr (R::GROUPS == 1) {
    R::store(dst, t, D, acc);
  } else {
    const int grp = threadIdx.x / R::NT;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R::EPT; ++i) {
      const int c = ((i / R::VEC) * R::NT + t) * R::VEC + i % R::VEC;
      if (c < D) sums[grp * D + c] = acc[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += R::THREADS) {
      float s = 0.f;
#pragma unroll
      for (int gi = 0; gi < R::GROUPS; ++gi) s += sums[gi * D + c];
      dst[c] = s;
    }
  }
}

template <class X, class P, class R>
__global__ void __launch_bounds__(R::THREADS) norm_bwd_kernel(const NormArgs<X, P> a) {
  constexpr int EPT = R::EPT;
  extern __shared__ float sums[];
  __shared__ float red[R::NT > 32 ? 16 * (R::NT / 32) : 1];
  int phase = 0;
  const int t = threadIdx.x % R::NT;
  const float inv = 1.f / static_cast<float>(a.D);
  float aw[EPT], ab[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) aw[i] = ab[i] = 0.f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * R::GROUPS;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * R::GROUPS + threadIdx.x / R::NT; row < a.rows; row += step) {
    const float mu = a.mean[row], r = a.rstd[row];
    float x[EPT], dy[EPT], w[EPT];
    R::load(a.x + row * a.x_stride, t, a.D, x);
    R::load(a.dy + row * a.dy_stride, t, a.D, dy);
    R::load(a.w, t, a.D, w, 1.f);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      x[i] = (x[i] - mu) * r;
      aw[i] += dy[i] * x[i];
      ab[i] += dy[i];
      w[i] *= dy[i];  // g; zero outside the row, as dy is
      s[0] += w[i];
      s[1] += w[i] * x[i];
    }
    row_sum<R::NT, 2>(s, red, phase);
    if (a.dx != nullptr) {
      const float mg = s[0] * inv, ma = s[1] * inv;
#pragma unroll
      for (int i = 0; i < EPT; ++i) x[i] = r * (w[i] - mg - x[i] * ma);
      R::store(a.dx + row * a.D, t, a.D, x);
    }
  }
  if (a.want_dw) write_part<R>(a.part, 0, a.D, aw, sums);
  if (a.want_db) write_part<R>(a.part, 1, a.D, ab, sums);
}

template <class X, class P, class R>
__global__ void __launch_bounds__(R::THREADS) norm_bwd2_kernel(const NormArgs<X, P> a) {
  constexpr int EPT = R::EPT;
  extern __shared__ float sums[];
  __shared__ float red[R::NT > 32 ? 16 * (R::NT / 32) : 1];
  int phase = 0;
  const int t = threadIdx.x % R::NT;
  const float inv = 1.f / static_cast<float>(a.D);
  float agw[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) agw[i] = 0.f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * R::GROUPS;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * R::GROUPS + threadIdx.x / R::NT; row < a.rows; row += step) {
    const float mu = a.mean[row], r = a.rstd[row];
    float x[EPT], dy[EPT], u[EPT];
    R::load(a.x + row * a.x_stride, t, a.D, x, mu);  // xh is zero outside the row
    R::load(a.dy + row * a.dy_stride, t, a.D, dy);
    R::load(a.ux == nullptr ? nullptr : a.ux + row * a.ux_stride, t, a.D, u);
    float s[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // g, u, g xh, u xh, h, h xh
    {
      float w[EPT], uw[EPT];
      R::load(a.w, t, a.D, w, 1.f);
      R::load(a.uw, t, a.D, uw);
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        x[i] = (x[i] - mu) * r;
        const float g = dy[i] * w[i], h = dy[i] * uw[i];
        s[0] += g;
        s[1] += u[i];
        s[2] += g * x[i];
        s[3] += u[i] * x[i];
        s[4] += h;
        s[5] += h * x[i];
      }
    }
    row_sum<R::NT, 6>(s, red, phase);
    const float mg = s[0] * inv, mu_u = s[1] * inv, ma = s[2] * inv, mc = s[3] * inv;
    float q[1] = {0.f};
    float w[EPT];
    R::load(a.w, t, a.D, w, 1.f);
#pragma unroll
    for (int i = 0; i < EPT; ++i) q[0] += dy[i] * w[i] * (u[i] - mu_u - x[i] * mc);
    row_sum<R::NT, 1>(q, red, phase);
    const float ms = q[0] * inv;
    // v = h - r (c g + a u): its mean and its mean against xh
    const float mv = s[4] * inv - r * (mc * mg + ma * mu_u);
    const float mvx = s[5] * inv - 2.f * r * ma * mc;
    float uw[EPT], ub[EPT], gx[EPT], gdy[EPT];
    R::load(a.uw, t, a.D, uw);
    R::load(a.ub, t, a.D, ub);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float pu = r * (u[i] - mu_u - x[i] * mc);
      const float v = dy[i] * uw[i] - r * (mc * dy[i] * w[i] + ma * u[i]);
      agw[i] += dy[i] * pu;
      gdy[i] = w[i] * pu + x[i] * uw[i] + ub[i];
      gx[i] = r * (v - mv - x[i] * mvx) - r * r * ms * x[i];
    }
    R::store(a.gdy + row * a.D, t, a.D, gdy);
    R::store(a.gx + row * a.D, t, a.D, gx);
  }
  if (a.want_dw) write_part<R>(a.part, 0, a.D, agw, sums);
}

// out[c] = sum over blocks (in order within each of 16 interleaved shares, then
// share by share) of part[block][which][c]. One block: 32 columns of one array.
template <class P>
__global__ void __launch_bounds__(512) norm_param_reduce_kernel(const float* part, int blocks, int D, P* dw, P* db) {
  __shared__ float s[16][33];
  const int which = blockIdx.y;
  P* out = which == 0 ? dw : db;
  if (out == nullptr) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float acc = 0.f;
  if (c < D) {
    for (int p = ty; p < blocks; p += 16) acc += part[(static_cast<int64_t>(p) * 2 + which) * D + c];
  }
  s[ty][tx] = acc;
  __syncthreads();
  if (ty == 0 && c < D) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += s[i][tx];
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

int row_threads(int D) { return D <= 1024 ? 32 : (D <= 4096 ? 128 : 512); }

// Blocks of the gradient kernels: enough row groups to fill the SMs, few enough
// that the blocks' parameter sums stay small beside the rows.
int grad_blocks(int64_t rows, int D, int sms) {
  const int nt = row_threads(D);
  const int64_t groups = nt == 32 ? 8 : 1;
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t cap = static_cast<int64_t>(sms) * (nt == 512 ? 1 : (nt == 128 ? 4 : 2));
  return static_cast<int>(need < cap ? (need < 1 ? 1 : need) : cap);
}

int check_norm(const ttt_norm_problem& pb) {
  if (pb.dtype != TTT_F16 && pb.dtype != TTT_BF16 && pb.dtype != TTT_F32) return TTT_ERR_DTYPE;
  if (pb.p_dtype != pb.dtype && pb.p_dtype != TTT_F32) return TTT_ERR_DTYPE;
  if (pb.rows < 0 || pb.rows > 0x7fffffff || pb.dim < 1 || pb.dim > TTT_NORM_MAX_DIM) return TTT_ERR_SHAPE;
  return TTT_OK;
}

enum Pass { kFwd, kBwd, kBwd2 };

template <class X, class P, class R>
cudaError_t launch_rows(const NormArgs<X, P>& a, Pass pass, int blocks, cudaStream_t s) {
  if (pass == kFwd) {
    const int64_t grid = (a.rows + R::GROUPS - 1) / R::GROUPS;
    norm_fwd_kernel<X, P, R><<<static_cast<unsigned>(grid), R::THREADS, 0, s>>>(a);
    return cudaGetLastError();
  }
  const size_t smem = R::GROUPS > 1 ? sizeof(float) * R::GROUPS * a.D : 0;
  if (pass == kBwd)
    norm_bwd_kernel<X, P, R><<<blocks, R::THREADS, smem, s>>>(a);
  else
    norm_bwd2_kernel<X, P, R><<<blocks, R::THREADS, smem, s>>>(a);
  return cudaGetLastError();
}

// Elements per thread: the row rounded up to NT * {8, 16, 32}.
template <class X, class P, bool WIDE>
cudaError_t launch_width(const NormArgs<X, P>& a, Pass pass, int blocks, cudaStream_t s) {
  const int D = a.D;
  if (D <= 256) return launch_rows<X, P, Row<X, 32, 8, WIDE>>(a, pass, blocks, s);
  if (D <= 512) return launch_rows<X, P, Row<X, 32, 16, WIDE>>(a, pass, blocks, s);
  if (D <= 1024) return launch_rows<X, P, Row<X, 32, 32, WIDE>>(a, pass, blocks, s);
  if (D <= 2048) return launch_rows<X, P, Row<X, 128, 16, WIDE>>(a, pass, blocks, s);
  if (D <= 4096) return launch_rows<X, P, Row<X, 128, 32, WIDE>>(a, pass, blocks, s);
  if (D <= 8192) return launch_rows<X, P, Row<X, 512, 16, WIDE>>(a, pass, blocks, s);
  return launch_rows<X, P, Row<X, 512, 32, WIDE>>(a, pass, blocks, s);
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
  const int blocks = pass == kFwd ? 0 : grad_blocks(pb.rows, pb.dim, sm_count());
  if (a.want_dw || a.want_db) {
    if (work == nullptr || !aligned16(work) || work_bytes < static_cast<int64_t>(blocks) * 2 * pb.dim * 4)
      return TTT_ERR_SCRATCH;
    a.part = static_cast<float*>(work);
  }
  if (pb.rows > 0 || pass != kFwd) {
    // 16-byte pieces need every row and every parameter vector on a 16-byte boundary
    constexpr int V = 16 / static_cast<int>(sizeof(X));
    bool wide = pb.dim % V == 0;
    const void* rows_at[] = {a.x, a.dy, a.ux, a.w, a.b, a.uw, a.ub, a.y, a.dx, a.gx, a.gdy};
    for (const void* p : rows_at) wide = wide && aligned16(p);
    wide = wide && a.x_stride % V == 0 && a.dy_stride % V == 0 && a.ux_stride % V == 0;
    const cudaError_t e = wide ? launch_width<X, P, true>(a, pass, blocks, s)
                               : launch_width<X, P, false>(a, pass, blocks, s);
    if (e != cudaSuccess) return TTT_ERR_LAUNCH;
  }
  if (a.want_dw || a.want_db) {
    const dim3 grid((pb.dim + 31) / 32, a.want_db ? 2 : 1);
    norm_param_reduce_kernel<P><<<grid, 512, 0, s>>>(a.part, blocks, pb.dim, static_cast<P*>(dw), static_cast<P*>(db));
    if (cudaGetLastError() != cudaSuccess) return TTT_ERR_LAUNCH;
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
  return static_cast<int64_t>(grad_blocks(pb->rows, pb->dim, sm_count())) * 2 * pb->dim * 4;
}

int ttt_norm_fwd(const ttt_norm_fwd_args* g, void* stream) {
  if (g == nullptr) return TTT_ERR_NULL;
  if (const int st = check_norm(g->pb)) return st;
  if (g->pb.rows > 0 && (g->x == nullptr || g->y == nullptr)) return TTT_ERR_NULL;
  if ((g->mean == nullptr) != (g->rstd == nullptr)) return TTT_ERR_NULL;
  if (g->x_stride < 0) return TTT_ERR_STRIDE;
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
