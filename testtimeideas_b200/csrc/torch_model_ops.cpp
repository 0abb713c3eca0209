// PyTorch operators over include/ttt_ops.h: ttt::layer_norm* and ttt::linear_ce*
// (forward, gradient and gradient of the gradient). Like torch_ops.cpp: argument checks, output
// and work space allocation (PyTorch's caching allocator, on the current device
// and stream) and the call into the C ABI.
//
// ttt::layer_norm_ad and ttt::linear_ce_ad are what the public functions call:
// autograd Functions over those operators, in C++ because the norms' kernels take
// a few microseconds and Python Functions cost about 30 us a node. The backward of
// each is itself a Function with a closed-form backward, as the attention's is,
// and computes only the gradients that the running backward asks for.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
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

// A tensor's last dimension as rows of unit column stride: the tensor itself where its
// layout is one row stride over all leading dimensions, else a contiguous copy.
struct Rows {
  at::Tensor keep;
  void* p = nullptr;
  int64_t stride = 0;
  Rows() = default;
  Rows(const at::Tensor& x, int64_t dim) : keep(x), stride(dim) {
    bool ok = dim == 1 || x.stride(-1) == 1;
    if (ok && !x.is_contiguous()) {
      int64_t inner = -1;  // row stride; every outer dimension must step over whole inner ones
      int64_t span = 1;
      for (int64_t d = x.dim() - 2; d >= 0 && ok; --d) {
        if (x.size(d) == 1) continue;
        if (inner < 0) inner = x.stride(d);
        ok = x.stride(d) == inner * span && inner >= 0;
        span *= x.size(d);
      }
      if (inner >= 0) stride = inner;
    }
    if (!ok) {
      keep = x.contiguous();
      stride = dim;
    }
    if (keep.numel() > 0) p = keep.data_ptr();
  }
};

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

std::tuple<at::Tensor, at::Tensor> op_layer_norm(const at::Tensor& x_, const OptTensor& w_, const OptTensor& b_,
                                                 double eps, bool need_stats) {
  const ttt_norm_problem pb = norm_problem(x_, w_, b_, eps);
  c10::cuda::CUDAGuard guard(x_.device());
  at::Tensor word = error_word_for(x_.get_device());
  raise_if_pending(x_.get_device(), word);
  const Rows x(x_, pb.dim);
  const at::Tensor w = vec(w_), b = vec(b_);
  at::Tensor y = at::empty(x_.sizes(), x_.options());
  at::Tensor stats = at::empty({2, need_stats ? pb.rows : 0}, x_.options().dtype(at::kFloat));
  ttt_norm_fwd_args a{};
  a.pb = pb;
  a.x = x.p;
  a.x_stride = x.stride;
  a.w = ptr(w);
  a.b = ptr(b);
  a.y = y.data_ptr();
  if (need_stats && pb.rows > 0) {
    a.mean = stats.data_ptr<float>();
    a.rstd = a.mean + pb.rows;
  }
  check(ttt_norm_fwd(&a, stream()), "ttt::layer_norm");
  return {y, stats};
}

// The gradient inputs of both gradients: dy, ux as rows of x's dtype.
Rows grad_rows(const at::Tensor& g, const at::Tensor& x, int64_t dim, const char* what) {
  TORCH_CHECK(g.sizes() == x.sizes(), "layer norm: ", what, " must have x's shape");
  TORCH_CHECK(g.device() == x.device(), "layer norm: ", what, " must be on x's device");
  return Rows(g.scalar_type() == x.scalar_type() ? g : g.to(x.scalar_type()), dim);
}

void check_stats(const at::Tensor& stats, const at::Tensor& x, int64_t rows) {
  TORCH_CHECK(stats.device() == x.device() && stats.scalar_type() == at::kFloat && stats.numel() == 2 * rows &&
                  stats.is_contiguous(),
              "layer norm: stats must be the forward's fp32 [2, rows] on x's device");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_layer_norm_bwd(const at::Tensor& dy_, const at::Tensor& x_,
                                                                 const OptTensor& w_, const at::Tensor& stats,
                                                                 bool need_dx, bool need_dw, bool need_db,
                                                                 at::ScalarType p_type) {
  ttt_norm_problem pb = norm_problem(x_, w_, std::nullopt, 0.0);
  pb.p_dtype = type_code(p_type);
  c10::cuda::CUDAGuard guard(x_.device());
  at::Tensor word = error_word_for(x_.get_device());
  raise_if_pending(x_.get_device(), word);
  check_stats(stats, x_, pb.rows);
  const Rows x(x_, pb.dim), dy = grad_rows(dy_, x_, pb.dim, "dy");
  const at::Tensor w = vec(w_);
  const auto po = x_.options().dtype(p_type);
  at::Tensor dx = need_dx ? at::empty(x_.sizes(), x_.options()) : at::empty({0}, x_.options());
  at::Tensor dw = at::empty({need_dw ? pb.dim : 0}, po), db = at::empty({need_db ? pb.dim : 0}, po);
  at::Tensor work = need_dw || need_db ? scratch(ttt_norm_work_bytes(&pb), x_) : at::Tensor();
  ttt_norm_bwd_args a{};
  a.pb = pb;
  a.x = x.p;
  a.dy = dy.p;
  a.x_stride = x.stride;
  a.dy_stride = dy.stride;
  a.w = ptr(w);
  a.mean = stats.data_ptr<float>();
  a.rstd = a.mean + pb.rows;
  a.dx = need_dx ? dx.data_ptr() : nullptr;
  a.dw = need_dw ? dw.data_ptr() : nullptr;
  a.db = need_db ? db.data_ptr() : nullptr;
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_norm_bwd(&a, stream()), "ttt::layer_norm_bwd");
  return {dx, dw, db};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_layer_norm_bwd2(const at::Tensor& dy_, const at::Tensor& x_,
                                                                  const OptTensor& w_, const at::Tensor& stats,
                                                                  const OptTensor& ux_, const OptTensor& uw_,
                                                                  const OptTensor& ub_) {
  ttt_norm_problem pb = norm_problem(x_, w_, std::nullopt, 0.0);
  c10::cuda::CUDAGuard guard(x_.device());
  at::Tensor word = error_word_for(x_.get_device());
  raise_if_pending(x_.get_device(), word);
  check_stats(stats, x_, pb.rows);
  // without a weight the parameters' type is that of what comes for the bias
  auto pt = w_.has_value() ? w_->scalar_type() : x_.scalar_type();
  for (const OptTensor* u : {&uw_, &ub_})
    if (!w_.has_value() && u->has_value() && (*u)->scalar_type() == at::kFloat) pt = at::kFloat;
  pb.p_dtype = type_code(pt);
  const Rows x(x_, pb.dim), dy = grad_rows(dy_, x_, pb.dim, "dy");
  const at::Tensor w = vec(w_);
  const Rows ux = ux_.has_value() ? grad_rows(*ux_, x_, pb.dim, "ux") : Rows();
  at::Tensor up[2];
  for (int i = 0; i < 2; ++i) {
    const OptTensor& u = i == 0 ? uw_ : ub_;
    if (!u.has_value()) continue;
    TORCH_CHECK(u->dim() == 1 && u->size(0) == pb.dim && u->device() == x_.device(),
                "layer norm: uw and ub must be [dim] on x's device");
    up[i] = u->to(pt).contiguous();
  }
  at::Tensor gx = at::empty(x_.sizes(), x_.options()), gdy = at::empty(x_.sizes(), x_.options());
  at::Tensor gw = at::empty({w_.has_value() ? pb.dim : 0}, x_.options().dtype(w_.has_value() ? pt : x_.scalar_type()));
  at::Tensor work = w_.has_value() ? scratch(ttt_norm_work_bytes(&pb), x_) : at::Tensor();
  ttt_norm_bwd2_args a{};
  a.pb = pb;
  a.x = x.p;
  a.dy = dy.p;
  a.ux = ux.p;
  a.x_stride = x.stride;
  a.dy_stride = dy.stride;
  a.ux_stride = ux.stride;
  a.w = ptr(w);
  a.uw = ptr(up[0]);
  a.ub = ptr(up[1]);
  a.mean = stats.data_ptr<float>();
  a.rstd = a.mean + pb.rows;
  a.gx = gx.data_ptr();
  a.gw = w_.has_value() ? gw.data_ptr() : nullptr;
  a.gdy = gdy.data_ptr();
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_norm_bwd2(&a, stream()), "ttt::layer_norm_bwd2");
  return {gdy, gx, gw};
}

// ---------------------------------------------------------------- linear cross entropy
// w as the kernels read it: unit column stride, a row stride that is a multiple of
// 8 elements, 16-byte aligned; else a copy with padded rows.
at::Tensor weight_rows(const at::Tensor& w) {
  const bool ok = w.stride(1) == 1 && (reinterpret_cast<uintptr_t>(w.data_ptr()) & 15u) == 0 &&
                  (w.size(0) == 1 || (w.stride(0) >= w.size(1) && w.stride(0) % 8 == 0)) &&
                  (w.size(0) > 1 || w.size(1) % 8 == 0);  // one row: any stride, but whole 16-byte pieces
  if (ok) return w;
  at::Tensor buf = at::empty({w.size(0), (w.size(1) + 7) / 8 * 8}, w.options());
  at::Tensor r = buf.narrow(1, 0, w.size(1));
  if (w.size(1) > 1 && w.stride(1) != 1) {
    r.copy_(w);
  } else {
    check(ttt_lce_pad_weight(w.data_ptr(), w.stride(0), buf.data_ptr(), buf.stride(0), w.size(0),
                             static_cast<int32_t>(w.size(1)), stream()),
          "ttt::linear_ce");
  }
  return r;
}

ttt_lce_problem lce_problem(const at::Tensor& h, const at::Tensor& w, int64_t reduction, int64_t ignore_index) {
  TORCH_CHECK(h.is_cuda() && w.is_cuda(), "ttt linear cross entropy needs CUDA tensors");
  const auto t = h.scalar_type();
  TORCH_CHECK(t == at::kHalf || t == at::kBFloat16, "ttt linear cross entropy takes fp16 or bf16 tensors, got ", t);
  TORCH_CHECK(w.scalar_type() == t, "linear cross entropy: hidden and weight must share one dtype, got ", t, " and ",
              w.scalar_type());
  TORCH_CHECK(w.device() == h.device(), "linear cross entropy: hidden and weight must be on one device");
  TORCH_CHECK(h.dim() >= 1 && w.dim() == 2 && h.size(-1) == w.size(1) && w.size(0) >= 1 && w.size(1) >= 1,
              "linear cross entropy: expected hidden [..., dim] and weight [vocab, dim], got ", h.sizes(), " and ",
              w.sizes());
  ttt_lce_problem pb{};
  pb.n = h.numel() / w.size(1);
  pb.vocab = w.size(0);
  TORCH_CHECK(w.size(1) <= 65536 && pb.n <= (1 << 24) && pb.vocab <= (1 << 24),
              "linear cross entropy takes at most 2^24 rows, 2^24 vocabulary entries and 65536 columns");
  pb.dim = static_cast<int32_t>(w.size(1));
  pb.dtype = type_code(t);
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "linear cross entropy: unknown reduction ", reduction);
  pb.reduction = static_cast<int32_t>(reduction);
  pb.ignore_index = ignore_index;
  return pb;
}

at::Tensor lce_work(const ttt_lce_problem& pb, int pass, const at::Tensor& like) {
  return scratch(ttt_lce_work_bytes(&pb, pass), like);
}

std::tuple<at::Tensor, at::Tensor> op_linear_ce(const at::Tensor& h_, const at::Tensor& w_, const at::Tensor& targets_,
                                                const OptTensor& mask_, int64_t reduction, int64_t ignore_index,
                                                bool need_state) {
  ttt_lce_problem pb = lce_problem(h_, w_, reduction, ignore_index);
  TORCH_CHECK(targets_.device() == h_.device() && at::isIntegralType(targets_.scalar_type(), false),
              "linear cross entropy: targets must be integers on hidden's device");
  TORCH_CHECK(targets_.sizes() == h_.sizes().slice(0, h_.dim() - 1),
              "linear cross entropy: targets must have hidden's leading shape ", h_.sizes().slice(0, h_.dim() - 1),
              ", got ", targets_.sizes());
  c10::cuda::CUDAGuard guard(h_.device());
  at::Tensor word = error_word_for(h_.get_device());
  raise_if_pending(h_.get_device(), word);
  at::Tensor mask;
  if (mask_.has_value()) {
    TORCH_CHECK(mask_->device() == h_.device() && mask_->sizes() == targets_.sizes(),
                "linear cross entropy: mask must have the targets' shape and device, got ", mask_->sizes());
    const bool u8 = mask_->scalar_type() == at::kBool;
    mask = (u8 ? *mask_ : mask_->to(at::kFloat)).contiguous();
    pb.mask_kind = u8 ? TTT_LCE_MASK_U8 : TTT_LCE_MASK_F32;
  }
  const Rows h(h_, pb.dim);
  const at::Tensor w = weight_rows(w_);
  const at::Tensor targets = targets_.to(at::kLong).contiguous();
  const auto f32 = h_.options().dtype(at::kFloat);
  at::Tensor loss = reduction == TTT_LCE_NONE ? at::empty(targets_.sizes(), f32) : at::empty({}, f32);
  at::Tensor state = at::empty({ttt_lce_state_bytes(&pb)}, h_.options().dtype(at::kByte));
  at::Tensor work = lce_work(pb, 0, h_);
  ttt_lce_fwd_args a{};
  a.pb = pb;
  a.h = h.p;
  a.h_stride = h.stride;
  a.w = w.data_ptr();
  a.w_stride = w.stride(0);
  a.targets = pb.n > 0 ? targets.data_ptr<int64_t>() : nullptr;
  a.mask = mask.defined() ? mask.data_ptr() : nullptr;
  // an empty loss has no storage; the entry point wants an address
  a.loss = loss.numel() > 0 ? loss.data_ptr<float>() : reinterpret_cast<float*>(word.data_ptr());
  a.state = state.numel() > 0 ? state.data_ptr() : nullptr;
  a.need_state = need_state ? 1 : 0;
  a.err = word.data_ptr<int32_t>();
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_lce_fwd(&a, stream()), "ttt::linear_ce");
  // without need_state the buffer was scratch, which no gradient may read
  if (!need_state) state = at::empty({0}, state.options());
  return {loss, state};
}

// dloss as the entry points read it: fp32, one value or one per row.
at::Tensor lce_upstream(const at::Tensor& dloss, const at::Tensor& h, const ttt_lce_problem& pb) {
  TORCH_CHECK(dloss.device() == h.device() && dloss.numel() == (pb.reduction == TTT_LCE_NONE ? pb.n : 1),
              "linear cross entropy: dloss must have the loss's shape, got ", dloss.sizes());
  return dloss.to(at::kFloat).contiguous();
}
void check_state(const at::Tensor& state, const at::Tensor& h, const ttt_lce_problem& pb) {
  TORCH_CHECK(state.device() == h.device() && state.scalar_type() == at::kByte && state.is_contiguous() &&
                  state.numel() == ttt_lce_state_bytes(&pb),
              "linear cross entropy: state must be that of a forward with need_state, on hidden's device");
}

std::tuple<at::Tensor, at::Tensor> op_linear_ce_bwd(const at::Tensor& dloss_, const at::Tensor& h_,
                                                    const at::Tensor& w_, const at::Tensor& state, int64_t reduction,
                                                    bool need_dh, bool need_dw) {
  const ttt_lce_problem pb = lce_problem(h_, w_, reduction, 0);
  c10::cuda::CUDAGuard guard(h_.device());
  at::Tensor word = error_word_for(h_.get_device());
  raise_if_pending(h_.get_device(), word);
  check_state(state, h_, pb);
  const at::Tensor w = weight_rows(w_), dloss = lce_upstream(dloss_, h_, pb);
  at::Tensor dh = need_dh ? at::empty(h_.sizes(), h_.options()) : at::empty({0}, h_.options());
  at::Tensor dw = need_dw ? at::empty(w_.sizes(), w_.options()) : at::empty({0}, w_.options());
  at::Tensor work = lce_work(pb, 1, h_);
  ttt_lce_bwd_args a{};
  a.pb = pb;
  a.w = w.data_ptr();
  a.w_stride = w.stride(0);
  a.state = state.data_ptr();
  a.dloss = pb.n > 0 || reduction != TTT_LCE_NONE ? dloss.data_ptr<float>() : reinterpret_cast<float*>(word.data_ptr());
  a.dh = need_dh && pb.n > 0 ? dh.data_ptr() : nullptr;
  a.dw = need_dw ? dw.data_ptr() : nullptr;
  a.err = word.data_ptr<int32_t>();
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_lce_bwd(&a, stream()), "ttt::linear_ce_bwd");
  return {dh, dw};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_linear_ce_bwd2(const at::Tensor& dloss_, const at::Tensor& h_,
                                                                 const at::Tensor& w_, const at::Tensor& state,
                                                                 int64_t reduction, const OptTensor& uh_,
                                                                 const OptTensor& uw_, bool need_gdloss, bool need_gh,
                                                                 bool need_gw) {
  const ttt_lce_problem pb = lce_problem(h_, w_, reduction, 0);
  c10::cuda::CUDAGuard guard(h_.device());
  at::Tensor word = error_word_for(h_.get_device());
  raise_if_pending(h_.get_device(), word);
  check_state(state, h_, pb);
  const at::Tensor w = weight_rows(w_), dloss = lce_upstream(dloss_, h_, pb);
  Rows uh;
  at::Tensor uw;
  if (uh_.has_value()) {
    TORCH_CHECK(uh_->sizes() == h_.sizes() && uh_->device() == h_.device(),
                "linear cross entropy: uh must have hidden's shape and device");
    uh = Rows(uh_->to(h_.scalar_type()), pb.dim);
  }
  if (uw_.has_value()) {
    TORCH_CHECK(uw_->sizes() == w_.sizes() && uw_->device() == h_.device(),
                "linear cross entropy: uw must have the weight's shape and device");
    uw = weight_rows(uw_->to(w_.scalar_type()));
  }
  at::Tensor gd = need_gdloss ? at::empty(dloss_.sizes(), dloss.options()) : at::empty({0}, dloss.options());
  at::Tensor gh = need_gh ? at::empty(h_.sizes(), h_.options()) : at::empty({0}, h_.options());
  at::Tensor gw = need_gw ? at::empty(w_.sizes(), w_.options()) : at::empty({0}, w_.options());
  at::Tensor work = lce_work(pb, 2, h_);
  ttt_lce_bwd2_args a{};
  a.pb = pb;
  a.w = w.data_ptr();
  a.w_stride = w.stride(0);
  a.uh = uh.p;
  a.uh_stride = uh.stride;
  a.uw = uw.defined() ? uw.data_ptr() : nullptr;
  a.uw_stride = uw.defined() ? uw.stride(0) : 0;
  a.state = state.data_ptr();
  a.dloss = pb.n > 0 || reduction != TTT_LCE_NONE ? dloss.data_ptr<float>() : reinterpret_cast<float*>(word.data_ptr());
  a.gh = need_gh && pb.n > 0 ? gh.data_ptr() : nullptr;
  a.gw = need_gw ? gw.data_ptr() : nullptr;
  a.gdloss = need_gdloss && gd.numel() > 0 ? gd.data_ptr<float>() : nullptr;
  a.err = word.data_ptr<int32_t>();
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(ttt_lce_bwd2(&a, stream()), "ttt::linear_ce_bwd2");
  return {gd, gh, gw};
}

// ---------------------------------------------------------------- autograd
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The operators run below the autograd keys, where a forward-mode tangent would be lost: refused instead.
void refuse_tangents(const char* op, std::initializer_list<const at::Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op, " has no forward-mode derivative");
}
constexpr const char *kNormOp = "layer norm", *kLceOp = "linear cross entropy";

at::Tensor defined_or(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

template <class Sig>
auto raw_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}
auto& raw_layer_norm() {
  static auto op = raw_op<decltype(op_layer_norm)>("ttt::layer_norm");
  return op;
}
auto& raw_layer_norm_bwd() {
  static auto op = raw_op<decltype(op_layer_norm_bwd)>("ttt::layer_norm_bwd");
  return op;
}
auto& raw_layer_norm_bwd2() {
  static auto op = raw_op<decltype(op_layer_norm_bwd2)>("ttt::layer_norm_bwd2");
  return op;
}
auto& raw_linear_ce() {
  static auto op = raw_op<decltype(op_linear_ce)>("ttt::linear_ce");
  return op;
}
auto& raw_linear_ce_bwd() {
  static auto op = raw_op<decltype(op_linear_ce_bwd)>("ttt::linear_ce_bwd");
  return op;
}
auto& raw_linear_ce_bwd2() {
  static auto op = raw_op<decltype(op_linear_ce_bwd2)>("ttt::linear_ce_bwd2");
  return op;
}

// An output of a second gradient, tied to the tensors it was computed from by a
// backward that raises, so that a third derivative is refused rather than wrong.
struct LastFn : torch::autograd::Function<LastFn> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& out, const OptTensor&, const OptTensor&,
                            const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&) {
    return out.view_as(out);
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "the second gradient of this op is not differentiable (a third derivative was requested)");
  }
};
// Marks the defined ones of `outs`, in place; up to six inputs, any of them undefined.
void mark_last(variable_list& outs, variable_list inputs) {
  if (!at::GradMode::is_enabled()) return;
  inputs.resize(6);
  for (at::Tensor& o : outs)
    if (o.defined())
      o = LastFn::apply(o, opt(inputs[0]), opt(inputs[1]), opt(inputs[2]), opt(inputs[3]), opt(inputs[4]),
                        opt(inputs[5]));
}

// (dy, x, w) -> (dx, dw, db); `need` has a bit per output.
struct LayerNormBwdFn : torch::autograd::Function<LayerNormBwdFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& dy, const at::Tensor& x, const OptTensor& w,
                               const at::Tensor& stats, int64_t need, int64_t p_type) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({dy, x, defined_or(w), stats});
    ctx->set_materialize_grads(false);
    auto [dx, dw, db] = raw_layer_norm_bwd().call(dy, x, w, stats, (need & 1) != 0, (need & 2) != 0, (need & 4) != 0,
                                                  static_cast<at::ScalarType>(p_type));
    return {dx, dw, db};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& up) {
    const variable_list v = ctx->get_saved_variables();
    variable_list g(6);
    if (!up[0].defined() && !up[1].defined() && !up[2].defined()) return g;
    refuse_tangents(kNormOp, {&up[0], &up[1], &up[2]});
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(g[0], g[1], g[2]) =
          raw_layer_norm_bwd2().call(v[0], v[1], opt(v[2]), v[3], opt(up[0]), opt(up[1]), opt(up[2]));
      g[0] = g[0].to(v[0].scalar_type());
      if (!v[2].defined()) g[2] = at::Tensor();
    }
    mark_last(g, {v[0], v[1], v[2], up[0], up[1], up[2]});
    return g;
  }
};

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& w, const OptTensor& b,
                            double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, stats] = raw_layer_norm().call(x, w, b, eps, true);
    ctx->save_for_backward({x, defined_or(w), stats});
    ctx->set_materialize_grads(false);
    ctx->saved_data["p_type"] = static_cast<int64_t>((w.has_value() ? *w : (b.has_value() ? *b : x)).scalar_type());
    ctx->saved_data["has_b"] = b.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& up) {
    variable_list g(4);
    if (!up[0].defined()) return g;
    refuse_tangents(kNormOp, {&up[0]});
    const variable_list v = ctx->get_saved_variables();
    const int64_t p_type = ctx->saved_data["p_type"].toInt();
    // needs_input_grad counts the tensors that were given: x, then w and b where present
    const bool has_w = v[1].defined(), has_b = ctx->saved_data["has_b"].toBool();
    int64_t need = ctx->needs_input_grad(0) ? 1 : 0;
    if (has_w && ctx->needs_input_grad(1)) need |= 2;
    if (has_b && ctx->needs_input_grad(has_w ? 2 : 1)) need |= 4;
    variable_list out;
    if (at::GradMode::is_enabled()) {
      out = LayerNormBwdFn::apply(up[0], v[0], opt(v[1]), v[2], need, p_type);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dx, dw, db] = raw_layer_norm_bwd().call(up[0], v[0], opt(v[1]), v[2], (need & 1) != 0, (need & 2) != 0,
                                                    (need & 4) != 0, static_cast<at::ScalarType>(p_type));
      out = {dx, dw, db};
    }
    for (int i = 0; i < 3; ++i)
      if (need & (1 << i)) g[i] = out[i];
    return g;
  }
};

bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

at::Tensor op_layer_norm_ad(const at::Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps) {
  const at::Tensor w = defined_or(w_), b = defined_or(b_);
  refuse_tangents(kNormOp, {&x, &w, &b});
  if (wants_grad({&x, &w, &b})) return LayerNormFn::apply(x, w_, b_, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(raw_layer_norm().call(x, w_, b_, eps, false));
}

// Weights that the kernels cannot read in place (odd widths) are copied once, in the
// forward, and the copy (`rows`, else undefined) is kept for both gradients. The copy moves
// 16-bit elements, so what the operator refuses is refused before it.
at::Tensor kept_rows(const at::Tensor& h, const at::Tensor& w) {
  if (!h.is_cuda() || !w.is_cuda() || h.key_set().has(c10::DispatchKey::Python) ||
      w.key_set().has(c10::DispatchKey::Python))
    return at::Tensor();  // refused by the operator, or being traced
  lce_problem(h, w, TTT_LCE_NONE, 0);
  c10::cuda::CUDAGuard guard(w.device());
  const at::Tensor r = weight_rows(w);
  return r.is_same(w) ? at::Tensor() : r;
}
const at::Tensor& rows_or(const at::Tensor& rows, const at::Tensor& w) { return rows.defined() ? rows : w; }

// (dloss, h, w) -> (dh, dw); `need` has a bit per output.
struct LinearCEBwdFn : torch::autograd::Function<LinearCEBwdFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& dloss, const at::Tensor& h, const at::Tensor& w,
                               const at::Tensor& state, const OptTensor& rows, int64_t reduction, int64_t need) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({dloss, h, w, state, defined_or(rows)});
    ctx->set_materialize_grads(false);
    ctx->saved_data["reduction"] = reduction;
    auto [dh, dw] = raw_linear_ce_bwd().call(dloss, h, rows_or(defined_or(rows), w), state, reduction,
                                             (need & 1) != 0, (need & 2) != 0);
    return {dh, dw};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& up) {
    const variable_list v = ctx->get_saved_variables();
    variable_list g(7);
    if (!up[0].defined() && !up[1].defined()) return g;
    refuse_tangents(kLceOp, {&up[0], &up[1]});
    bool need[3];
    for (int i = 0; i < 3; ++i) need[i] = ctx->needs_input_grad(i);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(g[0], g[1], g[2]) = raw_linear_ce_bwd2().call(v[0], v[1], rows_or(v[4], v[2]), v[3],
                                                             ctx->saved_data["reduction"].toInt(), opt(up[0]),
                                                             opt(up[1]), need[0], need[1], need[2]);
      for (int i = 0; i < 3; ++i)
        if (!need[i]) g[i] = at::Tensor();
    }
    mark_last(g, {v[0], v[1], v[2], up[0], up[1]});
    return g;
  }
};

struct LinearCEFn : torch::autograd::Function<LinearCEFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& targets,
                            const OptTensor& mask, int64_t reduction, int64_t ignore_index) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor rows = kept_rows(h, w);
    auto [loss, state] = raw_linear_ce().call(h, rows_or(rows, w), targets, mask, reduction, ignore_index, true);
    ctx->save_for_backward({h, w, state, rows});
    ctx->set_materialize_grads(false);
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& up) {
    variable_list g(6);
    if (!up[0].defined()) return g;
    refuse_tangents(kLceOp, {&up[0]});
    const variable_list v = ctx->get_saved_variables();
    const int64_t reduction = ctx->saved_data["reduction"].toInt();
    const int64_t need = (ctx->needs_input_grad(0) ? 1 : 0) | (ctx->needs_input_grad(1) ? 2 : 0);
    variable_list out;
    if (at::GradMode::is_enabled()) {
      out = LinearCEBwdFn::apply(up[0], v[0], v[1], v[2], opt(v[3]), reduction, need);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dh, dw] = raw_linear_ce_bwd().call(up[0], v[0], rows_or(v[3], v[1]), v[2], reduction, (need & 1) != 0,
                                               (need & 2) != 0);
      out = {dh, dw};
    }
    for (int i = 0; i < 2; ++i)
      if (need & (1 << i)) g[i] = out[i];
    return g;
  }
};

at::Tensor op_linear_ce_ad(const at::Tensor& h, const at::Tensor& w, const at::Tensor& targets, const OptTensor& mask,
                           int64_t reduction, int64_t ignore_index) {
  const at::Tensor weights = defined_or(mask);
  refuse_tangents(kLceOp, {&h, &w, &weights});
  TORCH_CHECK(!wants_grad({&weights}), "linear cross entropy forms no gradient by the mask: detach it");
  if (wants_grad({&h, &w})) return LinearCEFn::apply(h, w, targets, mask, reduction, ignore_index);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(raw_linear_ce().call(h, w, targets, mask, reduction, ignore_index, false));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(ttt, m) {
  // stats: fp32 [2, rows], mean and 1/std of each row; [2, 0] unless need_stats.
  m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, bool need_stats) -> (Tensor y, Tensor stats)");
  // An output that is not needed is empty; dw and db have dtype p_type.
  m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor? w, Tensor stats, bool need_dx, bool need_dw, "
        "bool need_db, ScalarType p_type) -> (Tensor dx, Tensor dw, Tensor db)");
  m.def("layer_norm_bwd2(Tensor dy, Tensor x, Tensor? w, Tensor stats, Tensor? ux, Tensor? uw, Tensor? ub) "
        " -> (Tensor gdy, Tensor gx, Tensor gw)");
  // reduction: 0 none, 1 mean, 2 sum; state (bytes) is what the gradients need of the forward
  // (empty without need_state); of h itself they take the shape and the type.
  m.def("linear_ce(Tensor h, Tensor w, Tensor targets, Tensor? mask, int reduction, int ignore_index, bool "
        "need_state) -> (Tensor loss, Tensor state)");
  m.def("linear_ce_bwd(Tensor dloss, Tensor h, Tensor w, Tensor state, int reduction, bool need_dh, bool need_dw) -> "
        "(Tensor dh, Tensor dw)");
  m.def("linear_ce_bwd2(Tensor dloss, Tensor h, Tensor w, Tensor state, int reduction, Tensor? uh, Tensor? uw, "
        "bool need_gdloss, bool need_gh, bool need_gw) -> (Tensor gdloss, Tensor gh, Tensor gw)");
}

TORCH_LIBRARY_FRAGMENT(ttt, m) {
  // Differentiable (twice) forms of layer_norm and linear_ce.
  m.def("layer_norm_ad(Tensor x, Tensor? w, Tensor? b, float eps) -> Tensor");
  m.def("linear_ce_ad(Tensor h, Tensor w, Tensor targets, Tensor? mask, int reduction, int ignore_index) -> Tensor");
}

TORCH_LIBRARY_IMPL(ttt, CompositeImplicitAutograd, m) {
  m.impl("layer_norm_ad", &op_layer_norm_ad);
  m.impl("linear_ce_ad", &op_linear_ce_ad);
}

TORCH_LIBRARY_IMPL(ttt, CUDA, m) {
  m.impl("layer_norm", &op_layer_norm);
  m.impl("layer_norm_bwd", &op_layer_norm_bwd);
  m.impl("layer_norm_bwd2", &op_layer_norm_bwd2);
  m.impl("linear_ce", &op_linear_ce);
  m.impl("linear_ce_bwd", &op_linear_ce_bwd);
  m.impl("linear_ce_bwd2", &op_linear_ce_bwd2);
}
