#include "ops/norm.h"

#include <torch/csrc/autograd/custom_function.h>

#include <array>
#include <cmath>

#include "kernels/norm_api.h"
#include "ops/block_common.h"

namespace mccl {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr const char* kWhat = "layer_norm";

kern::NormRows norm_rows(const at::Tensor& t) { return {t.const_data_ptr(), row_stride(t), elem_of(t, kWhat)}; }
const void* data_of(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

struct Affine {
  at::Tensor weight, bias;
  // What a gradient of either is kept like.
  const at::Tensor& any() const { return weight.defined() ? weight : bias; }
};

kern::NormShape shape_of(const at::Tensor& rows, const Affine& p, double eps) {
  kern::NormShape s{};
  s.rows = rows.size(0);
  s.cols = static_cast<int>(rows.size(1));
  s.eps = static_cast<float>(eps);
  s.weight = data_of(p.weight);
  s.bias = data_of(p.bias);
  if (p.any().defined()) s.weight_type = elem_of(p.any(), kWhat);
  return s;
}

void check_call(const at::Tensor& x, const Affine& p, double eps, const at::Tensor& residual, at::ScalarType dtype) {
  check_block_tensor(x, kWhat);
  elem_of(x, kWhat);
  MCCL_CHECK_T(TensorError, x.dim() >= 1 && x.size(-1) > 0, kWhat << ": rows of at least one number expected, got " << x.sizes());
  // (32 bits count a row's numbers, up to a block's step behind the last)
  MCCL_CHECK_T(TensorError, x.size(-1) <= kern::kNormMostCols && x.numel() / x.size(-1) <= 0x7FFFFFFF,
               kWhat << ": at most " << kern::kNormMostCols << " numbers a row and 2^31 - 1 rows, got " << x.sizes());
  for (const at::Tensor* t : {&p.weight, &p.bias}) {
    if (!t->defined()) continue;
    check_block_tensor(*t, kWhat);
    MCCL_CHECK_T(TensorError, t->dim() == 1 && t->size(0) == x.size(-1) && t->is_contiguous() && t->device() == x.device() &&
                                  (t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type()) && t->scalar_type() == p.any().scalar_type(),
                 kWhat << ": weight and bias are " << x.size(-1) << " numbers of float32 or of x's type, on its device, both alike");
  }
  if (residual.defined()) {
    check_block_tensor(residual, kWhat);
    MCCL_CHECK_T(TensorError, residual.sizes() == x.sizes() && residual.device() == x.device() &&
                                  (residual.scalar_type() == at::kFloat || residual.scalar_type() == x.scalar_type()),
                 kWhat << ": a residual of x's shape, of float32 or of its type, on its device expected");
  }
  MCCL_CHECK_T(TensorError, dtype == at::kFloat || dtype == at::kHalf || dtype == at::kBFloat16, kWhat << ": dtype is float32, float16 or bfloat16");
  MCCL_CHECK_T(TensorError, eps > 0 && std::isfinite(eps), kWhat << ": eps must be positive");
}

// y and, with a residual, the sum, of x's shape; mean and rstd where they are asked for, and the rows that were normed.
std::vector<at::Tensor> forward_of(const at::Tensor& x_in, const Affine& p, double eps, const at::Tensor& residual_in, at::ScalarType dtype, at::Tensor* stats,
                                   at::Tensor* normed) {
  const at::Tensor x = normed != nullptr ? rows_kept(x_in) : rows_of(x_in), residual = residual_in.defined() ? rows_of(residual_in) : residual_in;
  c10::cuda::CUDAGuard guard(x.device());
  kern::NormForward a{};
  a.shape = shape_of(x, p, eps);
  a.x = norm_rows(x);
  at::Tensor sum, y = at::empty(x_in.sizes(), x.options().dtype(dtype));
  if (residual.defined()) {
    a.residual = norm_rows(residual);
    sum = at::empty(x_in.sizes(), residual.options());
    a.sum = sum.data_ptr();
  }
  a.y = y.data_ptr();
  a.y_type = elem_of(y, kWhat);
  if (stats != nullptr) {
    *stats = at::empty({2, x.size(0)}, x.options().dtype(at::kFloat));
    a.mean = stats->data_ptr<float>();
    a.rstd = a.mean + x.size(0);
  }
  if (normed != nullptr) *normed = sum.defined() ? sum : x;
  OPS_CK(kern::launch_norm_forward(a, at::cuda::getCurrentCUDAStream()));
  if (sum.defined()) return {y, sum};
  return {y};
}

// Takes and gives tensors of the caller's shape.  As views of them rows would each have a gradient of their own over one memory, and leaves keep
// as theirs what nothing else seems to hold: x and the residual, whose gradients are the same numbers, would add up the next pass's in one place.
struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias,
                               const c10::optional<at::Tensor>& residual, double eps, int64_t dtype) {
    const Affine p{weight.value_or(at::Tensor()), bias.value_or(at::Tensor())};
    const bool with = residual.has_value();
    at::Tensor stats, normed;
    auto out = forward_of(x, p, eps, residual.value_or(at::Tensor()), static_cast<at::ScalarType>(dtype), &stats, &normed);
    ctx->save_for_backward({normed, p.weight, p.bias, stats});
    ctx->set_materialize_grads(false);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["dtype"] = dtype;
    ctx->saved_data["with"] = with;
    ctx->saved_data["x_type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->saved_data["sum_type"] = static_cast<int64_t>(with ? out[1].scalar_type() : x.scalar_type());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    MCCL_CHECK_T(TensorError, !at::GradMode::is_enabled(), kWhat << ": the backward pass is not differentiable (create_graph)");
    check_not_traced(kWhat);
    const bool with = ctx->saved_data["with"].toBool();
    at::Tensor dy = grads[0], ds = with ? grads[1] : at::Tensor();
    if (!dy.defined() && !ds.defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const auto x_type = static_cast<at::ScalarType>(ctx->saved_data["x_type"].toInt()), sum_type = static_cast<at::ScalarType>(ctx->saved_data["sum_type"].toInt()),
               dtype = static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt());
    const at::Device device = (dy.defined() ? dy : ds).device();
    const int64_t cols = sizes.back(), rows = (dy.defined() ? dy : ds).numel() / cols;
    const std::array<int64_t, 2> flat{rows, cols};
    check_saved(saved[0], with ? at::IntArrayRef(sizes) : at::IntArrayRef(flat), sum_type, device, kWhat);
    const at::Tensor s = rows_of(saved[0]);
    check_saved(saved[3], {2, rows}, at::kFloat, device, kWhat);
    Affine p{saved[1], saved[2]};
    for (at::Tensor* t : {&p.weight, &p.bias}) {
      if (!t->defined()) continue;
      check_saved(*t, {cols}, p.any().scalar_type(), device, kWhat);
      *t = t->contiguous();
    }
    c10::cuda::CUDAGuard guard(device);
    const at::Tensor stats = saved[3].contiguous();
    for (const auto& [g, type] : {std::pair<const at::Tensor&, at::ScalarType>(dy, dtype), std::pair<const at::Tensor&, at::ScalarType>(ds, sum_type)}) {
      if (!g.defined()) continue;
      check_saved(g, sizes, type, device, kWhat);
    }
    size_t input = 0;  // tensors that there are not are not counted
    auto needed = [&](bool there) { return there && ctx->needs_input_grad(input++); };
    const bool need_x = needed(true), need_weight = needed(p.weight.defined()), need_bias = needed(p.bias.defined()), need_residual = needed(with);
    if (!dy.defined())  // the sum's alone: it is x's and the residual's
      return {need_x ? ds.to(x_type) : at::Tensor(), need_weight ? at::zeros_like(p.weight) : at::Tensor(), need_bias ? at::zeros_like(p.bias) : at::Tensor(),
              need_residual ? ds : at::Tensor(), {}, {}};
    kern::NormBackward a{};
    a.shape = shape_of(s, p, ctx->saved_data["eps"].toDouble());
    a.s = norm_rows(s);
    const at::Tensor dy_rows = rows_of(dy), ds_rows = ds.defined() ? rows_of(ds) : at::Tensor();
    a.dy = norm_rows(dy_rows);
    if (ds.defined()) a.ds = norm_rows(ds_rows);
    a.mean = stats.const_data_ptr<float>();
    a.rstd = a.mean + rows;
    at::Tensor dx, dresidual, dweight, dbias, partial;
    if (need_x) dx = at::empty(sizes, s.options().dtype(x_type));
    if (need_residual) dresidual = need_x && x_type == sum_type ? dx : at::empty(sizes, s.options());
    a.dx = need_x ? dx.data_ptr() : nullptr;
    a.dx_type = x_type == at::kFloat ? kern::Elem::kF32 : x_type == at::kHalf ? kern::Elem::kF16 : kern::Elem::kBF16;
    a.dresidual = need_residual && !dresidual.is_same(dx) ? dresidual.data_ptr() : nullptr;
    if (need_weight || need_bias) {
      // without rows nothing is launched, and the sums over none are zeros
      if (need_weight) dweight = rows == 0 ? at::zeros_like(p.weight) : at::empty_like(p.weight);
      if (need_bias) dbias = rows == 0 ? at::zeros_like(p.bias) : at::empty_like(p.bias);
      a.dweight = need_weight ? dweight.data_ptr() : nullptr;
      a.dbias = need_bias ? dbias.data_ptr() : nullptr;
      partial = at::empty({std::max<int64_t>(1, kern::norm_partial_bytes(a.shape) / 4)}, stats.options());
      a.partial = partial.data_ptr<float>();
    }
    OPS_CK(kern::launch_norm_backward(a, at::cuda::getCurrentCUDAStream()));
    return {dx, dweight, dbias, dresidual, {}, {}};
  }
};

}  // namespace

std::vector<at::Tensor> layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias, double eps,
                                   const std::optional<at::Tensor>& residual, std::optional<at::ScalarType> dtype) {
  const Affine p{weight.value_or(at::Tensor()), bias.value_or(at::Tensor())};
  const at::Tensor r = residual.value_or(at::Tensor());
  const at::ScalarType y_type = dtype.value_or(x.scalar_type());
  check_call(x, p, eps, r, y_type);
  bool grad = false;
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&x, &p.weight, &p.bias, &r}) grad = grad || (t->defined() && t->requires_grad());
  if (!grad || !at::GradMode::is_enabled()) return forward_of(x, p, eps, r, y_type, nullptr, nullptr);
  auto given = [](const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; };
  return LayerNormFn::apply(x, given(p.weight), given(p.bias), given(r), eps, static_cast<int64_t>(y_type));
}

}  // namespace mccl
