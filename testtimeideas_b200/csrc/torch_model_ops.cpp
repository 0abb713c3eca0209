// PyTorch operators over include/ttt_ops.h: ttt::layer_norm* (forward, gradient
// and gradient of the gradient). Like torch_ops.cpp: argument checks, output
// and work space allocation (PyTorch's caching allocator, on the current device
// and stream) and the call into the C ABI.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "torch_common.h"
#include "ttt_ops.h"

namespace {

using ttt_torch::check;
using ttt_torch::error_word_for;
using ttt_torch::raise_if_pending;
using OptTensor = std::optional<at::Tensor>;

int type_code(at::ScalarType t) {
  return t == at::kFloat ? TTT_F32 : (t == at::kBFloat16 ? TTT_BF16 : TTT_F16);
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// x as [rows, dim] with unit column stride: a view where the layout allows one, else a copy.
at::Tensor as_rows(const at::Tensor& x, int64_t dim) {
  at::Tensor r = x.reshape({-1, dim});
  return (r.size(0) == 0 || dim == 1 || r.stride(1) == 1) && (r.size(0) < 2 || r.stride(0) >= 0) ? r : r.contiguous();
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor scratch(int64_t bytes, const at::Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

// ---------------------------------------------------------------- layer norm
ttt_norm_problem norm_problem(const at::Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  TORCH_CHECK(x.is_cuda(), "ttt layer norm needs CUDA tensors");
  const auto xt = x.scalar_type();
  TORCH_CHECK(xt == at::kHalf || xt == at::kBFloat16 || xt == at::kFloat,
              "ttt layer norm takes fp16, bf16 or fp32 tensors, got ", xt);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "layer norm needs a last dimension of at least 1, got ", x.sizes());
  TORCH_CHECK(x.size(-1) <= TTT_NORM_MAX_DIM, "layer norm takes rows of at most ", TTT_NORM_MAX_DIM, " elements, got ",
              x.size(-1));
  auto pt = xt;
  for (const OptTensor* p : {&w, &b}) {
    if (!p->has_value()) continue;
    const at::Tensor& v = **p;
    TORCH_CHECK(v.device() == x.device(), "layer norm: weight and bias must be on x's device");
    TORCH_CHECK(v.dim() == 1 && v.size(0) == x.size(-1), "layer norm: weight and bias must be [", x.size(-1), "], got ",
                v.sizes());
    TORCH_CHECK(v.scalar_type() == xt || v.scalar_type() == at::kFloat,
                "layer norm: weight and bias must have x's dtype or fp32, got ", v.scalar_type());
    pt = v.scalar_type();
  }
  TORCH_CHECK(!w.has_value() || !b.has_value() || w->scalar_type() == b->scalar_type(),
              "layer norm: weight and bias must share one dtype");
  ttt_norm_problem pb;
  pb.dim = static_cast<int32_t>(x.size(-1));
  pb.rows = x.numel() / pb.dim;
  pb.dtype = type_code(xt);
  pb.p_dtype = type_code(pt);
  pb.eps = static_cast<float>(eps);
  return pb;
}

at::Tensor vec(const OptTensor& p) { return p.has_value() ? p->contiguous() : at::Tensor(); }

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_layer_norm(const at::Tensor& x_, const OptTensor& w_,
                                                             const OptTensor& b_, double eps, bool need_stats) {
  const ttt_norm_problem pb = norm_problem(x_, w_, b_, eps);
  c10::cuda::CUDAGuard guard(x_.device());
  at::Tensor word = error_word_for(x_.get_device());
  raise_if_pending(x_.get_device(), word);
  const at::Tensor x = as_rows(x_, pb.dim), w = vec(w_), b = vec(b_);
  at::Tensor y = at::empty(x_.sizes(), x_.options());
  at::Tensor stats = at::empty({2, need_stats ? pb.rows : 0}, x_.options().dtype(at::kFloat));
  at::Tensor mean = stats.select(0, 0), rstd = stats.select(0, 1);
  ttt_norm_fwd_args a{};
  a.pb = pb;
  a.x = ptr(x);
  a.x_stride = x.stride(0);
  a.w = ptr(w);
  a.b = ptr(b);
  a.y = y.data_ptr();
  if (need_stats) {
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
    if (pb.rows == 0) a.mean = a.rstd = nullptr;
  }
  check(ttt_norm_fwd(&a, stream()), "ttt::layer_norm");
  return {y, mean, rstd};
}

// The gradient inputs of both gradients: dy, ux as rows of x's dtype.
at::Tensor grad_rows(const at::Tensor& g, const at::Tensor& x, int64_t dim, const char* what) {
  TORCH_CHECK(g.sizes() == x.sizes(), "layer norm: ", what, " must have x's shape");
  TORCH_CHECK(g.device() == x.device(), "layer norm: ", what, " must be on x's device");
  return as_rows(g.to(x.scalar_type()), dim);
}

void check_stats(const at::Tensor& mean, const at::Tensor& rstd, int64_t rows) {
  for (const at::Tensor* s : {&mean, &rstd})
    TORCH_CHECK(s->is_cuda() && s->scalar_type() == at::kFloat && s->numel() == rows && s->is_contiguous(),
                "layer norm: mean and rstd must be the forward's fp32 [rows]");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_layer_norm_bwd(const at::Tensor& dy_, const at::Tensor& x_,
                                                                 const OptTensor& w_, const at::Tensor& mean,
                                                                 const at::Tensor& rstd, bool need_dx, bool need_dw,
                                                                 bool need_db, at::ScalarType p_type) {
  ttt_norm_problem pb = norm_problem(x_, w_, std::nullopt, 0.0);
  pb.p_dtype = type_code(p_type);
  c10::cuda::CUDAGuard guard(x_.device());
  at::Tensor word = error_word_for(x_.get_device());
  raise_if_pending(x_.get_device(), word);
  check_stats(mean, rstd, pb.rows);
  const at::Tensor x = as_rows(x_, pb.dim), dy = grad_rows(dy_, x_, pb.dim, "dy"), w = vec(w_);
  const auto po = x_.options().dtype(p_type);
  at::Tensor dx = need_dx ? at::empty(x_.sizes(), x_.options()) : at::empty({0}, x_.options());
  at::Tensor dw = at::empty({need_dw ? pb.dim : 0}, po), db = at::empty({need_db ? pb.dim : 0}, po);
  at::Tensor work = need_dw || need_db ? scratch(ttt_norm_work_bytes(&pb), x_) : at::Tensor();
  ttt_norm_bwd_args a{};
  a.pb = pb;
  a.x = ptr(x);
  a.dy = ptr(dy);
  a.x_stride = x.stride(0);
  a.dy_stride = dy.stride(0);
  a.w = ptr(w);
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.dx = need_dx ? dx.data_ptr() : nullptr;
  a.dw = need_dw ? dw.data_ptr() : nullptr;
  a.db = need_db ? db.data_ptr() : nullptr;
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_norm_bwd(&a, stream()), "ttt::layer_norm_bwd");
  return {dx, dw, db};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_layer_norm_bwd2(const at::Tensor& dy_, const at::Tensor& x_,
                                                                  const OptTensor& w_, const at::Tensor& mean,
                                                                  const at::Tensor& rstd, const OptTensor& ux_,
                                                                  const OptTensor& uw_, const OptTensor& ub_) {
  const ttt_norm_problem pb = norm_problem(x_, w_, std::nullopt, 0.0);
  c10::cuda::CUDAGuard guard(x_.device());
  at::Tensor word = error_word_for(x_.get_device());
  raise_if_pending(x_.get_device(), word);
  check_stats(mean, rstd, pb.rows);
  const auto pt = w_.has_value() ? w_->scalar_type() : x_.scalar_type();
  const at::Tensor x = as_rows(x_, pb.dim), dy = grad_rows(dy_, x_, pb.dim, "dy"), w = vec(w_);
  const at::Tensor ux = ux_.has_value() ? grad_rows(*ux_, x_, pb.dim, "ux") : at::Tensor();
  at::Tensor up[2];
  for (int i = 0; i < 2; ++i) {
    const OptTensor& u = i == 0 ? uw_ : ub_;
    if (!u.has_value()) continue;
    TORCH_CHECK(u->dim() == 1 && u->size(0) == pb.dim && u->device() == x_.device(),
                "layer norm: uw and ub must be [dim] on x's device");
    up[i] = u->to(pt).contiguous();
  }
  at::Tensor gx = at::empty(x_.sizes(), x_.options()), gdy = at::empty(x_.sizes(), x_.options());
  at::Tensor gw = at::empty({w_.has_value() ? pb.dim : 0}, x_.options().dtype(pt));
  at::Tensor work = w_.has_value() ? scratch(ttt_norm_work_bytes(&pb), x_) : at::Tensor();
  ttt_norm_bwd2_args a{};
  a.pb = pb;
  a.x = ptr(x);
  a.dy = ptr(dy);
  a.ux = ptr(ux);
  a.x_stride = x.stride(0);
  a.dy_stride = dy.stride(0);
  a.ux_stride = ux.defined() ? ux.stride(0) : 0;
  a.w = ptr(w);
  a.uw = ptr(up[0]);
  a.ub = ptr(up[1]);
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.gx = gx.data_ptr();
  a.gw = w_.has_value() ? gw.data_ptr() : nullptr;
  a.gdy = gdy.data_ptr();
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_norm_bwd2(&a, stream()), "ttt::layer_norm_bwd2");
  return {gdy, gx, gw};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(ttt, m) {
  // mean and rstd (fp32 [rows]) are empty unless need_stats.
  m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, bool need_stats) -> (Tensor y, Tensor mean, "
        "Tensor rstd)");
  // An output that is not needed is empty; dw and db have dtype p_type.
  m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor? w, Tensor mean, Tensor rstd, bool need_dx, bool need_dw, "
        "bool need_db, ScalarType p_type) -> (Tensor dx, Tensor dw, Tensor db)");
  m.def("layer_norm_bwd2(Tensor dy, Tensor x, Tensor? w, Tensor mean, Tensor rstd, Tensor? ux, Tensor? uw, "
        "Tensor? ub) -> (Tensor gdy, Tensor gx, Tensor gw)");
}

TORCH_LIBRARY_IMPL(ttt, CUDA, m) {
  m.impl("layer_norm", &op_layer_norm);
  m.impl("layer_norm_bwd", &op_layer_norm_bwd);
  m.impl("layer_norm_bwd2", &op_layer_norm_bwd2);
}
