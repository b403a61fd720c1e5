#include "ops/gated.h"

#include <torch/csrc/autograd/custom_function.h>

#include <algorithm>

#include "kernels/gated_api.h"
#include "ops/block_common.h"
#include "ops/checkpoint.h"
#include "ops/linear.h"
#include "ops/products.h"

namespace mccl {

namespace {

using kern::GatedProduct;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr const char* kWhat = "gated_feed_forward";

kern::GatedActivation activation_of(const std::string& name) {
  if (name == "silu") return kern::GatedActivation::kSilu;
  MCCL_CHECK_T(TensorError, name == "gelu_tanh", kWhat << ": activation is \"silu\" or \"gelu_tanh\", got \"" << name << "\"");
  return kern::GatedActivation::kGeluTanh;
}

void check_call(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd) {
  for (const at::Tensor* t : {&x, &wg, &wu, &wd}) {
    check_block_tensor(*t, kWhat);
    MCCL_CHECK_T(TensorError, t->scalar_type() == x.scalar_type() && t->device() == x.device(), kWhat << ": tensors differ in type or device");
  }
  elem_of(x, kWhat);
  MCCL_CHECK_T(TensorError, x.dim() >= 1 && wg.dim() == 2 && wu.dim() == 2 && wd.dim() == 2 && wg.sizes() == wu.sizes() && wg.size(1) == x.size(-1) &&
                                wd.size(0) == wg.size(1) && wd.size(1) == wg.size(0),
               kWhat << ": x [..., width], w_gate and w_up [hidden, width] and w_down [width, hidden] expected, got " << x.sizes() << ", " << wg.sizes()
                     << ", " << wu.sizes() << " and " << wd.sizes());
  MCCL_CHECK_T(TensorError, wg.size(0) > 0 && wg.size(1) > 0, kWhat << ": empty weights");
}

kern::GatedShape shape_of(const at::Tensor& rows, int64_t hidden, kern::GatedActivation act, kern::GatedKeep keep) {
  return {rows.size(0), rows.size(1), hidden, rows.scalar_type() == at::kBFloat16, act, keep};
}

void few(const kern::GatedShape& s, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& y) {
  const at::Tensor rows[4] = {few_rows(x), few_rows(wg), few_rows(wu), few_rows(wd)};
  const bool f32 = x.scalar_type() == at::kFloat;
  const at::Tensor h = at::empty({f32 ? 1 : 2, s.tokens, kern::gated_pitch(s.hidden)}, x.options());
  kern::GatedOperand m[4];
  for (int i = 0; i < 4; ++i) m[i] = {rows[i].const_data_ptr(), row_stride(rows[i])};
  OPS_CK(kern::launch_gated_few({s, m[0], m[1], m[2], m[3], h.data_ptr(), y.data_ptr(), f32}, at::cuda::getCurrentCUDAStream()));
}

// y of 16-bit rows; g and u to `kept` where there is one.
at::Tensor forward16(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, kern::GatedActivation act,
                     kern::GatedKeep keep, at::Tensor* kept, int64_t wait_limit = -1) {
  check_waits(x);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty(x.sizes(), x.options());
  const kern::GatedShape s = shape_of(x, wg.size(0), act, keep);
  if (keep != kern::GatedKeep::kNone) *kept = at::empty({kern::gated_kept_bytes(s)}, x.options().dtype(at::kByte));
  if (x.size(0) == 0) return y;
  if (keep == kern::GatedKeep::kNone && kern::gated_is_few(s) && wait_limit < 0) {
    few(s, x, wg, wu, wd, y);
    return y;
  }
  Operands m;
  const int ox = m.add(x), og = m.add(wg), ou = m.add(wu);
  const bool first = m.any();  // else a copy of w_down has time until the second product
  const int od = m.add(wd);
  if (first) m.copy(x);
  else m.reserve(x);
  const at::Tensor h = at::empty({s.tokens, kern::gated_pitch(s.hidden)}, x.options());
  Products run(s, x, wait_limit);
  run.r.kept = kept ? kept->data_ptr() : nullptr;
  const kern::GatedArgs up{GatedProduct::kUp, m[ox], {}, m[og], m[ou], h.data_ptr(), nullptr, nullptr, 0};
  run.launch(&up, 1, x);
  if (!first) m.copy(x, true);
  const kern::GatedArgs down{GatedProduct::kDown, {h.const_data_ptr(), h.size(1)}, {}, m[od], {}, y.data_ptr(), nullptr, nullptr, s.width};
  run.launch(&down, 1, x);
  return y;
}

struct Needs {
  bool x, gate, up, down;
};
struct Gradients {
  at::Tensor x, gate, up, down;
};

Gradients backward16(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& kept,
                     kern::GatedActivation act, kern::GatedKeep keep, const Needs& need) {
  check_waits(dy);
  c10::cuda::CUDAGuard guard(dy.device());
  const auto like = dy.options();
  const kern::GatedShape s = shape_of(dy, wg.size(0), act, keep);
  Gradients r;
  if (need.x) r.x = at::empty(dy.sizes(), like);
  if (need.gate || need.up) {
    r.gate = at::empty(wg.sizes(), like);
    r.up = at::empty(wu.sizes(), like);
  }
  if (need.down) r.down = at::empty(wd.sizes(), like);
  if (s.tokens == 0) {
    for (at::Tensor* t : {&r.gate, &r.up, &r.down})
      if (t->defined()) t->zero_();
    return r;
  }
  const int64_t pitch = kern::gated_pitch(s.hidden);
  Operands m;
  const int ody = m.add(dy), od = m.add(wd);
  const int og = need.x ? m.add(wg) : 0, ou = need.x ? m.add(wu) : 0, ox = need.gate || need.up ? m.add(x) : 0;
  m.copy(dy);
  const at::Tensor between = at::empty({3, s.tokens, pitch}, like);
  const int64_t each = s.tokens * pitch * 2;
  char *const h = static_cast<char*>(between.data_ptr()), *const dg = h + each, *const du = dg + each;
  const kern::GatedOperand mh{h, pitch}, mg{dg, pitch}, mu{du, pitch};
  Products run(s, dy, -1);
  run.r.kept = kept.data_ptr();
  const kern::GatedArgs gate{GatedProduct::kGate, m[ody], {}, m[od], {}, h, dg, du, 0};
  run.launch(&gate, 1, dy);
  kern::GatedArgs rest[3];
  int n = 0;
  if (need.x) rest[n++] = {GatedProduct::kInput, mg, mu, m[og], m[ou], r.x.data_ptr(), nullptr, nullptr, s.width};
  if (need.gate || need.up) rest[n++] = {GatedProduct::kWeightUp, mg, mu, m[ox], {}, r.gate.data_ptr(), r.up.data_ptr(), nullptr, s.width};
  if (need.down) rest[n++] = {GatedProduct::kWeightDown, m[ody], {}, mh, {}, r.down.data_ptr(), nullptr, nullptr, s.hidden};
  if (n > 0) run.launch(rest, n, dy);
  return r;
}

// ---- fp32: the products of the linear layer -----------------------------------------------------------------------
// With gradients both projections are one product of the two weights one behind the other: two thirds of the products of three
// weights, and one sum for the gradient of x.  (Putting them together costs their size twice in traffic; 256 x 1024 x 2816, forward and
// backward: 215 us without, 193 so.)  A forward pass alone leaves them where they are; of few tokens it has kernels of its own.
at::Tensor joined(const at::Tensor& wg, const at::Tensor& wu) { return at::cat({wg, wu}, 0); }

at::Tensor gate32(const at::Tensor& g, const at::Tensor& u, kern::GatedActivation act) {
  at::Tensor h = at::empty(g.sizes(), g.options());
  OPS_CK(kern::launch_gate_f32(g.const_data_ptr<float>(), u.const_data_ptr<float>(), g.stride(0), h.data_ptr<float>(), h.size(0), h.size(1), act,
                               at::cuda::getCurrentCUDAStream()));
  return h;
}
at::Tensor gate32(const at::Tensor& gu, kern::GatedActivation act) {
  const int64_t hidden = gu.size(1) / 2;
  return gate32(gu.narrow(1, 0, hidden), gu.narrow(1, hidden, hidden), act);
}
at::Tensor forward32(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, kern::GatedActivation act, at::Tensor* kept) {
  c10::cuda::CUDAGuard guard(x.device());
  if (kept) {
    *kept = mccl::linear(x, joined(wg, wu), c10::nullopt);
    return mccl::linear(gate32(*kept, act), wd, c10::nullopt);
  }
  const kern::GatedShape s = shape_of(x, wg.size(0), act, kern::GatedKeep::kNone);
  if (x.size(0) > 0 && kern::gated_is_few_f32(s)) {
    const at::Tensor y = at::empty(x.sizes(), x.options());
    few(s, x, wg, wu, wd, y);
    return y;
  }
  return mccl::linear(gate32(mccl::linear(x, wg, c10::nullopt), mccl::linear(x, wu, c10::nullopt), act), wd, c10::nullopt);
}
Gradients backward32(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& gu,
                     kern::GatedActivation act, const Needs& need) {
  Gradients r;
  const int64_t hidden = wg.size(0);
  const bool up = need.gate || need.up;
  at::Tensor dh;
  // (without a gradient of w_down the other operand counts for its shape alone)
  std::tie(dh, r.down) = linear_gradients(dy, need.down ? gate32(gu, act) : gu.narrow(1, 0, hidden), wd, need.x || up, need.down);
  if (!need.x && !up) return r;
  at::Tensor dgu = at::empty(gu.sizes(), gu.options()), both;
  OPS_CK(kern::launch_gate_f32_backward(gu.const_data_ptr<float>(), dh.const_data_ptr<float>(), dgu.data_ptr<float>(), gu.size(0), hidden, act,
                                        at::cuda::getCurrentCUDAStream()));
  // (without a gradient of x the weights count for their shape alone)
  std::tie(r.x, both) = linear_gradients(dgu, x, need.x ? joined(wg, wu) : at::empty({2 * hidden, wg.size(1)}, wg.options()), need.x, up);
  if (up) {
    r.gate = both.narrow(0, 0, hidden);
    r.up = both.narrow(0, hidden, hidden);
  }
  return r;
}

// ---- autograd -----------------------------------------------------------------------------------------------------
// What is packed, to rows of a matrix.
void unpack_to(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales) {
  const kern::Packed8Rows p{const_cast<int8_t*>(codes.const_data_ptr<int8_t>()), const_cast<float*>(scales.const_data_ptr<float>()), x.size(0), x.size(1),
                            kern::pack8_pitch(x.size(1))};
  OPS_CK(kern::launch_unpack8(p, x.data_ptr(), elem_of(x, kWhat), x.stride(0), at::cuda::getCurrentCUDAStream()));
}

struct GatedFn : torch::autograd::Function<GatedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act,
                            bool eight) {
    const auto activation = static_cast<kern::GatedActivation>(act);
    c10::cuda::CUDAGuard guard(x.device());
    ctx->saved_data["act"] = act;
    ctx->saved_data["eight"] = eight;
    ctx->saved_data["rows"] = x.size(0);
    ctx->saved_data["width"] = wg.size(1);
    ctx->saved_data["hidden"] = wg.size(0);
    std::vector<at::Tensor> saved{wg, wu, wd};
    at::Tensor y;
    if (x.scalar_type() == at::kFloat) {
      at::Tensor gu;
      y = forward32(x, wg, wu, wd, activation, &gu);
      if (eight) {
        const int64_t hidden = wg.size(0);
        for (const at::Tensor& t : {x, gu.narrow(1, 0, hidden), gu.narrow(1, hidden, hidden)}) {
          const auto [codes, scales] = pack8(t);
          saved.insert(saved.end(), {codes, scales});
        }
      } else {
        saved.insert(saved.end(), {x, gu});
      }
    } else {
      at::Tensor kept;
      y = forward16(x, wg, wu, wd, activation, eight ? kern::GatedKeep::kEight : kern::GatedKeep::kWide, &kept);
      if (eight) {
        const auto [codes, scales] = pack8(x);
        saved.insert(saved.end(), {codes, scales, kept});
      } else {
        saved.insert(saved.end(), {x, kept});
      }
    }
    ctx->save_for_backward(saved);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    MCCL_CHECK_T(TensorError, !at::GradMode::is_enabled(), kWhat << ": the backward pass is not differentiable (create_graph)");
    at::Tensor dy = grads[0];
    if (!dy.defined()) return variable_list(6);
    check_not_traced(kWhat);
    // products that are torch's are of the tensors' types, also where this is called inside of an autocast region
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &wg = saved[0], &wu = saved[1], &wd = saved[2];
    const auto act = static_cast<kern::GatedActivation>(ctx->saved_data["act"].toInt());
    const bool eight = ctx->saved_data["eight"].toBool();
    const int64_t rows = ctx->saved_data["rows"].toInt(), width = ctx->saved_data["width"].toInt(), hidden = ctx->saved_data["hidden"].toInt();
    check_block_tensor(dy, kWhat);
    MCCL_CHECK_T(TensorError, dy.dim() == 2 && dy.size(0) == rows && dy.size(1) == width, kWhat << ": not a gradient of its result");
    const auto type = dy.scalar_type();
    auto back = [&](const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType of) -> const at::Tensor& {
      check_saved(t, sizes, of, dy.device(), kWhat);
      return t;
    };
    back(wg, {hidden, width}, type);
    back(wu, {hidden, width}, type);
    back(wd, {width, hidden}, type);
    c10::cuda::CUDAGuard guard(dy.device());
    // codes and scales of `cols` columns from saved[i] on, to rows of x
    auto unpack = [&](const at::Tensor& x, size_t i) {
      unpack_to(x, packed_again(back(saved[i], {rows, kern::pack8_pitch(x.size(1))}, at::kChar)),
                packed_again(back(saved[i + 1], {rows, kern::pack8_groups(x.size(1))}, at::kFloat)));
    };
    // Values of codes are rounded to the type here, as unpack8 rounds them: of the gradients of w_gate and w_up a third rounding, beside
    // dg's or du's and their own (2.8e-3 against 64 bits in bf16, 2.3e-3 without it, where the codes themselves are 6e-3 of x off).
    // Multiplied with what it loses, too, they take 482 us for 379 of 8192 tokens of 1024 x 2816, forward and backward.
    auto kept_x = [&] {
      if (!eight) return back(saved[3], {rows, width}, type);
      const at::Tensor x = at::empty({rows, kern::gated_row(width)}, dy.options()).narrow(1, 0, width);
      unpack(x, 3);
      return x;
    };
    const Needs need{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    const bool need_up = need.gate || need.up;
    Gradients r;
    if (type == at::kFloat) {
      dy = dy.contiguous();
      at::Tensor gu;
      if (eight) {
        gu = at::empty({rows, 2 * hidden}, dy.options());
        unpack(gu.narrow(1, 0, hidden), 5);
        unpack(gu.narrow(1, hidden, hidden), 7);
      } else {
        gu = back(saved[4], {rows, 2 * hidden}, type).contiguous();
      }
      r = backward32(dy, need_up ? kept_x() : at::empty({rows, width}, dy.options()), wg, wu, wd, gu, act, need);
    } else {
      const auto keep = eight ? kern::GatedKeep::kEight : kern::GatedKeep::kWide;
      const at::Tensor kept = packed_again(back(saved.back(), {kern::gated_kept_bytes(shape_of(dy, hidden, act, keep))}, at::kByte));
      r = backward16(dy, need_up && rows > 0 ? kept_x() : at::Tensor(), wg, wu, wd, kept, act, keep, need);
    }
    return {r.x, need.gate ? r.gate : at::Tensor(), need.up ? r.up : at::Tensor(), r.down, {}, {}};
  }
};

}  // namespace

at::Tensor gated_feed_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const std::string& activation,
                              bool eight_bits) {
  const auto act = activation_of(activation);
  check_call(x, wg, wu, wd);
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad());
  const at::Tensor rows = rows_of(x);
  at::Tensor y;
  if (grad) {
    y = GatedFn::apply(rows, wg, wu, wd, static_cast<int64_t>(act), eight_bits);
  } else if (x.scalar_type() == at::kFloat) {
    y = forward32(rows, wg, wu, wd, act, nullptr);
  } else {
    y = forward16(rows, wg, wu, wd, act, kern::GatedKeep::kNone, nullptr);
  }
  return x.dim() == 2 ? y : y.view(x.sizes());
}

at::Tensor gated_with_limit(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t wait_limit) {
  check_call(x, wg, wu, wd);
  MCCL_CHECK_T(TensorError, wait_limit >= 0 && x.dim() == 2 && x.scalar_type() != at::kFloat, "not a call for the 16-bit kernels");
  return forward16(x, wg, wu, wd, kern::GatedActivation::kSilu, kern::GatedKeep::kNone, nullptr, wait_limit);
}

}  // namespace mccl
