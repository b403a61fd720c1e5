#include "ops/fused_linear.h"

#include <torch/csrc/autograd/custom_function.h>

#include "ops/linear.h"
#include "ops/products.h"

namespace mccl {

namespace {

using kern::GatedProduct;
using kern::LayerActivation;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr const char* kWhat = "fused_linear";

LayerActivation activation_of(const std::string& name) {
  if (name == "none") return LayerActivation::kNone;
  if (name == "relu") return LayerActivation::kRelu;
  if (name == "silu") return LayerActivation::kSilu;
  if (name == "gelu") return LayerActivation::kGelu;
  MCCL_CHECK_T(TensorError, name == "gelu_tanh", kWhat << ": activation is none, \"relu\", \"silu\", \"gelu\" or \"gelu_tanh\", got \"" << name << "\"");
  return LayerActivation::kGeluTanh;
}

void check_call(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& residual) {
  for (const at::Tensor* t : {&x, &w, &bias}) {
    if (t == &bias && !bias.defined()) continue;
    check_block_tensor(*t, kWhat);
    MCCL_CHECK_T(TensorError, t->scalar_type() == x.scalar_type() && t->device() == x.device(), kWhat << ": tensors differ in type or device");
  }
  elem_of(x, kWhat);
  MCCL_CHECK_T(TensorError, x.dim() >= 1 && w.dim() == 2 && w.numel() > 0 && w.size(1) == x.size(-1) && (!bias.defined() || (bias.dim() == 1 && bias.size(0) == w.size(0))),
               kWhat << ": x [..., in], weight [out, in] and bias [out] expected, got " << x.sizes() << ", " << w.sizes() << " and "
                     << (bias.defined() ? bias.sizes() : at::IntArrayRef{}));
  if (!residual.defined()) return;
  check_block_tensor(residual, kWhat);
  auto sizes = x.sizes().vec();
  sizes.back() = w.size(0);
  MCCL_CHECK_T(TensorError, residual.sizes() == sizes && residual.device() == x.device() &&
                                (residual.scalar_type() == at::kFloat || residual.scalar_type() == x.scalar_type()),
               kWhat << ": a residual of the result's shape, of float32 or of x's type, on its device expected, got " << residual.scalar_type() << " " << residual.sizes());
}

kern::LayerRows layer_rows(const at::Tensor& t) {
  if (!t.defined()) return {nullptr, 0, kern::Elem::kF32};
  return {t.const_data_ptr(), row_stride(t), elem_of(t, kWhat)};
}

// The products' shape: `width` is what comes out.
kern::GatedShape shape_of(const at::Tensor& x, const at::Tensor& w) {
  return {x.size(0), w.size(0), w.size(1), x.scalar_type() == at::kBFloat16, kern::GatedActivation::kSilu, kern::GatedKeep::kNone};
}

// y of 16-bit rows, of the shape `sizes`; x w^T + bias to `z` where there is one to keep.
at::Tensor forward16(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias_in, LayerActivation act, const at::Tensor& residual, at::IntArrayRef sizes,
                     at::Tensor* z, int64_t wait_limit = -1) {
  check_waits(x);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t tokens = x.size(0), out = w.size(0);
  const auto type = residual.defined() ? residual.scalar_type() : x.scalar_type();
  at::Tensor y = at::empty(sizes, x.options().dtype(type));
  if (z != nullptr) *z = at::empty({tokens, kern::gated_row(out)}, x.options());
  if (tokens == 0) return y;
  const at::Tensor bias = bias_in.defined() ? bias_in.contiguous() : bias_in;
  const kern::LayerRows r = layer_rows(residual);
  const kern::LayerFinish finish{act, bias.defined() ? bias.const_data_ptr() : nullptr, r.data, r.ld, type == at::kFloat};
  const kern::GatedShape s = shape_of(x, w);
  Operands m;
  const int ox = m.add(x), ow = m.add(w);
  if (z == nullptr && wait_limit < 0 && kern::layer_is_few(tokens, out, !m.any())) {
    const at::Tensor xs = few_rows(x), ws = few_rows(w);
    const kern::LayerFew few{tokens, w.size(1), out, s.bf16, {xs.const_data_ptr(), row_stride(xs)}, {ws.const_data_ptr(), row_stride(ws)}, finish, y.data_ptr()};
    OPS_CK(kern::launch_layer_few(few, at::cuda::getCurrentCUDAStream()));
    return y;
  }
  m.copy(x);
  if (kern::layer_tile(tokens, w.size(1), out) > 0) {
    const kern::LayerTiles tiles{tokens, w.size(1), out, s.bf16, m[ox], m[ow], finish, y.data_ptr(), z != nullptr ? z->data_ptr() : nullptr, wait_status(x), wait_limit};
    OPS_CK(kern::launch_layer_tiles(tiles, at::cuda::getCurrentCUDAStream()));
    return y;
  }
  Products run(s, x, wait_limit);
  run.r.layer = &finish;
  const kern::GatedArgs g{GatedProduct::kLayer, m[ox], {}, m[ow], {}, y.data_ptr(), z != nullptr ? z->data_ptr() : nullptr, nullptr, out};
  run.launch(&g, 1, x);
  return y;
}

struct Needs {
  bool x, w, bias;
};
struct Gradients {
  at::Tensor x, w, bias;
};

// The pass before the products: dz where it is not dy itself, and the bias's gradient.
at::Tensor derive(const at::Tensor& dy, const at::Tensor& z, int64_t out, LayerActivation act, const at::TensorOptions& like, const Needs& need, Gradients& r) {
  const int64_t tokens = dy.size(0);
  const auto type = like.dtype().toScalarType();
  const bool own = (act != LayerActivation::kNone || dy.scalar_type() != type) && (need.x || need.w);
  at::Tensor dz, partial;
  if (own) dz = at::empty({tokens, type == at::kFloat ? out : kern::gated_row(out)}, like);
  if (need.bias) r.bias = tokens == 0 ? at::zeros({out}, like) : at::empty({out}, like);
  if (tokens > 0 && (own || need.bias)) {
    kern::LayerDerive g{};
    g.rows = tokens;
    g.cols = out;
    g.dy = layer_rows(dy);
    if (act != LayerActivation::kNone) g.z = layer_rows(z);
    g.activation = act;
    g.dz_type = type == at::kFloat ? kern::Elem::kF32 : type == at::kHalf ? kern::Elem::kF16 : kern::Elem::kBF16;
    if (own) {
      g.dz = dz.data_ptr();
      g.dz_ld = dz.size(1);
    }
    if (need.bias) {
      partial = at::empty({kern::layer_partial_bytes(tokens, out) / 4}, like.dtype(at::kFloat));
      g.partial = partial.data_ptr<float>();
      g.bias = r.bias.data_ptr();
      g.bias_type = g.dz_type;
    }
    OPS_CK(kern::launch_layer_derive(g, at::cuda::getCurrentCUDAStream()));
  }
  return own ? dz.narrow(1, 0, out) : dy;
}

Gradients backward16(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const at::Tensor& z, LayerActivation act, const Needs& need) {
  check_waits(x);
  c10::cuda::CUDAGuard guard(x.device());
  Gradients r;
  const at::Tensor dz = derive(dy, z, w.size(0), act, x.options(), need, r);
  if (need.x) r.x = at::empty(x.sizes(), x.options());
  if (need.w) r.w = x.size(0) == 0 ? at::zeros(w.sizes(), w.options()) : at::empty(w.sizes(), w.options());
  if ((!need.x && !need.w) || x.size(0) == 0) return r;
  const kern::GatedShape s = shape_of(x, w);
  Operands m;
  const int odz = m.add(dz), ow = need.x ? m.add(w) : 0, ox = need.w ? m.add(x) : 0;
  m.copy(x);
  Products run(s, x, -1);
  kern::GatedArgs g[2];
  int n = 0;
  if (need.x) g[n++] = {GatedProduct::kBack, m[odz], {}, m[ow], {}, r.x.data_ptr(), nullptr, nullptr, s.hidden};
  if (need.w) g[n++] = {GatedProduct::kWeightDown, m[odz], {}, m[ox], {}, r.w.data_ptr(), nullptr, nullptr, s.hidden};
  run.launch(g, n, x);
  return r;
}

// ---- fp32: the linear layer's products, and a pass behind or before them; small ones whole ------------------------------
// (what the linear layer has on the tensor cores stays there)
bool rows_ok(const at::Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1; }
bool goes_small(const at::Tensor& x, const at::Tensor& w, bool small) { return small && x.size(0) > 0 && rows_ok(x) && rows_ok(w) && !linear_native(x, w, c10::nullopt); }
at::Tensor forward32(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias_in, LayerActivation act, const at::Tensor& residual, at::IntArrayRef sizes,
                     at::Tensor* z_out) {
  c10::cuda::CUDAGuard guard(x.device());
  if (goes_small(x, w, kern::layer_is_small(x.size(0), w.size(1), w.size(0)))) {
    const at::Tensor bias = bias_in.defined() ? bias_in.contiguous() : bias_in;
    at::Tensor y = at::empty(sizes, x.options());
    if (z_out != nullptr) *z_out = at::empty({x.size(0), w.size(0)}, x.options());
    const kern::LayerRows r = layer_rows(residual);
    const kern::LayerSmall g{x.size(0), w.size(1), w.size(0), x.const_data_ptr<float>(), w.const_data_ptr<float>(), bias.defined() ? bias.const_data_ptr<float>() : nullptr,
                             static_cast<const float*>(r.data), row_stride(x), row_stride(w), r.ld, act, y.data_ptr<float>(), z_out != nullptr ? z_out->data_ptr<float>() : nullptr};
    OPS_CK(kern::launch_layer_small(g, at::cuda::getCurrentCUDAStream()));
    return y;
  }
  const at::Tensor& bias = bias_in;
  const at::Tensor z = mccl::linear(x, w, bias.defined() ? c10::optional<at::Tensor>(bias) : c10::nullopt).contiguous();
  if (z_out != nullptr) *z_out = z;
  if (act == LayerActivation::kNone && !residual.defined()) return sizes.size() == 2 ? z : at::_unsafe_view(z, sizes);
  at::Tensor y = at::empty(sizes, z.options());
  OPS_CK(kern::launch_layer_finish(z.const_data_ptr<float>(), layer_rows(residual), y.data_ptr<float>(), z.size(0), z.size(1), act, at::cuda::getCurrentCUDAStream()));
  return y;
}
Gradients backward32(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const at::Tensor& z, LayerActivation act, const Needs& need) {
  c10::cuda::CUDAGuard guard(x.device());
  Gradients r;
  if (goes_small(x, w, kern::layer_is_small_backward(x.size(0), w.size(1), w.size(0)))) {
    const at::Tensor dz = derive(dy, z, w.size(0), act, x.options(), {true, true, false}, r);
    if (need.x) r.x = at::empty(x.sizes(), x.options());
    if (need.w) r.w = at::empty(w.sizes(), w.options());
    if (need.bias) r.bias = at::empty({w.size(0)}, w.options());
    auto to = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    const kern::LayerSmallBackward g{x.size(0), w.size(1), w.size(0), dz.const_data_ptr<float>(), x.const_data_ptr<float>(), w.const_data_ptr<float>(),
                                     row_stride(dz), row_stride(x), row_stride(w), to(r.x), to(r.w), to(r.bias)};
    OPS_CK(kern::launch_layer_small_backward(g, at::cuda::getCurrentCUDAStream()));
    return r;
  }
  const at::Tensor dz = derive(dy, z, w.size(0), act, x.options(), need, r);
  if (need.x || need.w) std::tie(r.x, r.w) = linear_gradients(dz, x, w, need.x, need.w);
  return r;
}

at::DimVector sizes_of(const at::Tensor& x, const at::Tensor& w) {
  at::DimVector sizes(x.sizes());
  sizes.back() = w.size(0);
  return sizes;
}
at::Tensor forward_of(const at::Tensor& rows, const at::Tensor& w, const at::Tensor& bias, LayerActivation act, const at::Tensor& residual_in, at::IntArrayRef sizes,
                      at::Tensor* z) {
  const at::Tensor residual = residual_in.defined() ? rows_of(residual_in) : residual_in;
  return rows.scalar_type() == at::kFloat ? forward32(rows, w, bias, act, residual, sizes, z) : forward16(rows, w, bias, act, residual, sizes, z);
}

// Takes and gives tensors of the caller's shape: the residual's gradient is the result's itself, and as a view of it, which nothing else seems to hold, a
// leaf would keep the caller's memory as its own.
struct FusedLinearFn : torch::autograd::Function<FusedLinearFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x_in, const at::Tensor& w, const c10::optional<at::Tensor>& bias,
                            const c10::optional<at::Tensor>& residual, int64_t act) {
    const auto activation = static_cast<LayerActivation>(act);
    const at::Tensor x = rows_kept(x_in);
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor b = bias.value_or(at::Tensor()), r = residual.value_or(at::Tensor());
    at::Tensor z;  // where one but the residual wants a gradient
    at::Tensor* const keep =
        activation == LayerActivation::kNone || !(x_in.requires_grad() || w.requires_grad() || (b.defined() && b.requires_grad())) ? nullptr : &z;
    const at::Tensor y = forward_of(x, w, b, activation, r, sizes_of(x_in, w), keep);
    ctx->save_for_backward({x, w, z});
    ctx->set_materialize_grads(false);
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = b.defined();
    ctx->saved_data["residual"] = r.defined();
    ctx->saved_data["type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["y_type"] = static_cast<int64_t>(y.scalar_type());
    ctx->saved_data["out"] = w.size(0);
    ctx->saved_data["sizes"] = x_in.sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    MCCL_CHECK_T(TensorError, !at::GradMode::is_enabled(), kWhat << ": the backward pass is not differentiable (create_graph)");
    const at::Tensor& dy_in = grads[0];
    if (!dy_in.defined()) return variable_list(5);
    check_not_traced(kWhat);
    // products that are torch's are of the tensors' types, also where this is called inside of an autocast region
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
    const auto saved = ctx->get_saved_variables();
    const auto act = static_cast<LayerActivation>(ctx->saved_data["act"].toInt());
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), y_type = static_cast<at::ScalarType>(ctx->saved_data["y_type"].toInt());
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t in = sizes.back(), out = ctx->saved_data["out"].toInt();
    at::DimVector y_sizes(sizes.begin(), sizes.end());
    y_sizes.back() = out;
    const at::Device device = dy_in.device();
    check_saved(dy_in, y_sizes, y_type, device, kWhat);
    const int64_t rows = dy_in.numel() / out;
    check_saved(saved[0], {rows, in}, type, device, kWhat);
    check_saved(saved[1], {out, in}, type, device, kWhat);
    c10::cuda::CUDAGuard guard(device);
    size_t input = 0;  // tensors that there are not are not counted
    auto needed = [&](bool there) { return there && ctx->needs_input_grad(input++); };
    const bool need_x = needed(true), need_w = needed(true), need_bias = needed(ctx->saved_data["bias"].toBool()),
               need_residual = needed(ctx->saved_data["residual"].toBool());
    if (!need_x && !need_w && !need_bias) return {{}, {}, {}, need_residual ? dy_in : at::Tensor(), {}};
    const Needs need{need_x, need_w, need_bias};
    if (act != LayerActivation::kNone) check_saved(saved[2], {rows, type == at::kFloat ? out : kern::gated_row(out)}, type, device, kWhat);
    const at::Tensor dy = rows_of(dy_in), z = act != LayerActivation::kNone ? rows_of(saved[2]) : at::Tensor();
    const Gradients r = type == at::kFloat ? backward32(dy, saved[0], saved[1], z, act, need) : backward16(dy, saved[0], saved[1], z, act, need);
    return {need_x && sizes.size() != 2 ? r.x.view(sizes) : r.x, r.w, r.bias, need_residual ? dy_in : at::Tensor(), {}};
  }
};

}  // namespace

at::Tensor fused_linear(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, const std::string& activation,
                        const std::optional<at::Tensor>& residual) {
  const LayerActivation act = activation_of(activation);
  const at::Tensor b = bias.value_or(at::Tensor()), r = residual.value_or(at::Tensor());
  check_call(x, w, b, r);
  bool grad = false;
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&x, &w, &b, &r}) grad = grad || (t->defined() && t->requires_grad());
  if (!grad || !at::GradMode::is_enabled()) return forward_of(rows_of(x), w, b, act, r, sizes_of(x, w), nullptr);
  auto given = [](const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; };
  return FusedLinearFn::apply(x, w, given(b), given(r), static_cast<int64_t>(act));
}

at::Tensor fused_linear_with_limit(const at::Tensor& x, const at::Tensor& w, int64_t wait_limit) {
  check_call(x, w, at::Tensor(), at::Tensor());
  MCCL_CHECK_T(TensorError, wait_limit >= 0 && x.dim() == 2 && x.scalar_type() != at::kFloat, "not a call for the 16-bit kernels");
  return forward16(x, w, at::Tensor(), LayerActivation::kNone, at::Tensor(), {x.size(0), w.size(0)}, nullptr, wait_limit);
}

}  // namespace mccl
