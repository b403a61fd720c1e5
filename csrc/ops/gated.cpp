#include "ops/gated.h"

#include <torch/csrc/autograd/custom_function.h>

#include <algorithm>

#include "kernels/gated_api.h"
#include "ops/block_common.h"
#include "ops/checkpoint.h"
#include "ops/linear.h"

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

// Matrices as the products read them: rows of 16-byte multiples.  Those that are not laid out so are copied, all in one launch.
class Operands {
 public:
  // Which of them it is.
  int add(const at::Tensor& t) {
    const int64_t rows = t.size(0), cols = t.size(1), ld = rows <= 1 ? kern::gated_row(cols) : t.stride(0);
    if ((cols <= 1 || t.stride(1) == 1) && ld % 8 == 0 && ld >= cols && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0) {
      m_[n_] = {t.const_data_ptr(), ld};
    } else {
      m_[n_] = {nullptr, kern::gated_row(cols)};
      copies_[copied_] = {t.const_data_ptr(), t.stride(0), t.stride(1), rows, cols, nullptr, kern::gated_row(cols)};
      of_[copied_++] = n_;
      bytes_ += (rows * kern::gated_row(cols) * 2 + 255) / 256 * 256;
    }
    return n_++;
  }
  void copy(const at::Tensor& like) {
    if (copied_ == 0) return;
    held_ = at::empty({bytes_}, like.options().dtype(at::kByte));
    char* at = static_cast<char*>(held_.data_ptr());
    for (int i = 0; i < copied_; ++i) {
      copies_[i].to = at;
      m_[of_[i]].data = at;
      at += (copies_[i].rows * copies_[i].ld * 2 + 255) / 256 * 256;
    }
    OPS_CK(kern::launch_gated_copies(copies_, copied_, at::cuda::getCurrentCUDAStream()));
  }
  const kern::GatedOperand& operator[](int i) const { return m_[i]; }

 private:
  int n_ = 0, copied_ = 0, of_[kern::kGatedCopies] = {};
  int64_t bytes_ = 0;
  kern::GatedOperand m_[kern::kGatedCopies] = {};
  kern::GatedCopy copies_[kern::kGatedCopies] = {};
  at::Tensor held_;
};

// Partial sums of the products of one pass, which follow each other on a stream.
at::Tensor partial_for(std::initializer_list<GatedProduct> ps, const kern::GatedShape& s, const at::TensorOptions& like) {
  int64_t bytes = 0;
  for (const auto p : ps) bytes = std::max(bytes, kern::gated_partial_bytes(p, s));
  return bytes > 0 ? at::empty({bytes / 4}, like.dtype(at::kFloat)) : at::Tensor();
}
void launch(kern::GatedArgs& a, const at::Tensor& partial, const at::Tensor& like, int64_t wait_limit = -1) {
  a.partial = partial.defined() ? partial.data_ptr<float>() : nullptr;
  a.failed = wait_status(like);
  a.wait_limit = wait_limit;
  OPS_CK(kern::launch_gated(a, at::cuda::getCurrentCUDAStream()));
}

at::Tensor few_rows(const at::Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

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
    const at::Tensor rows[4] = {few_rows(x), few_rows(wg), few_rows(wu), few_rows(wd)};
    const at::Tensor h = at::empty({2, s.tokens, kern::gated_pitch(s.hidden)}, x.options());
    kern::GatedOperand m[4];
    for (int i = 0; i < 4; ++i) m[i] = {rows[i].const_data_ptr(), row_stride(rows[i])};
    OPS_CK(kern::launch_gated_few({s, m[0], m[1], m[2], m[3], h.data_ptr(), y.data_ptr()}, at::cuda::getCurrentCUDAStream()));
    return y;
  }
  Operands m;
  const int ox = m.add(x), og = m.add(wg), ou = m.add(wu), od = m.add(wd);
  m.copy(x);
  const at::Tensor h = at::empty({s.tokens, kern::gated_pitch(s.hidden)}, x.options());
  const at::Tensor partial = partial_for({GatedProduct::kUp, GatedProduct::kDown}, s, x.options());
  kern::GatedArgs a{};
  a.product = GatedProduct::kUp;
  a.shape = s;
  a.a0 = m[ox];
  a.b0 = m[og];
  a.b1 = m[ou];
  a.out0 = h.data_ptr();
  a.kept = kept ? kept->data_ptr() : nullptr;
  launch(a, partial, x, wait_limit);
  a = {};
  a.product = GatedProduct::kDown;
  a.shape = s;
  a.a0 = {h.const_data_ptr(), h.size(1)};
  a.b0 = m[od];
  a.out0 = y.data_ptr();
  a.ldo = s.width;
  launch(a, partial, x, wait_limit);
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
  const at::Tensor partial = partial_for({GatedProduct::kGate, GatedProduct::kInput, GatedProduct::kWeightUp, GatedProduct::kWeightDown}, s, like);
  const kern::GatedOperand mh{h, pitch}, mg{dg, pitch}, mu{du, pitch};
  kern::GatedArgs a{};
  a.product = GatedProduct::kGate;
  a.shape = s;
  a.a0 = m[ody];
  a.b0 = m[od];
  a.out0 = h;
  a.out1 = dg;
  a.out2 = du;
  a.kept = kept.data_ptr();
  launch(a, partial, dy);
  if (need.x) {
    a = {};
    a.product = GatedProduct::kInput;
    a.shape = s;
    a.a0 = mg;
    a.a1 = mu;
    a.b0 = m[og];
    a.b1 = m[ou];
    a.out0 = r.x.data_ptr();
    a.ldo = s.width;
    launch(a, partial, dy);
  }
  if (need.gate || need.up) {
    a = {};
    a.product = GatedProduct::kWeightUp;
    a.shape = s;
    a.a0 = mg;
    a.a1 = mu;
    a.b0 = m[ox];
    a.out0 = r.gate.data_ptr();
    a.out1 = r.up.data_ptr();
    a.ldo = s.width;
    launch(a, partial, dy);
  }
  if (need.down) {
    a = {};
    a.product = GatedProduct::kWeightDown;
    a.shape = s;
    a.a0 = m[ody];
    a.b0 = mh;
    a.out0 = r.down.data_ptr();
    a.ldo = s.hidden;
    launch(a, partial, dy);
  }
  return r;
}

// ---- fp32: the products of the linear layer -----------------------------------------------------------------------
at::Tensor gate32(const at::Tensor& g, const at::Tensor& u, kern::GatedActivation act) {
  c10::cuda::CUDAGuard guard(g.device());
  at::Tensor h = at::empty(g.sizes(), g.options());
  OPS_CK(kern::launch_gate_f32(g.const_data_ptr<float>(), u.const_data_ptr<float>(), h.data_ptr<float>(), g.numel(), act, at::cuda::getCurrentCUDAStream()));
  return h;
}
Gradients backward32(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& g,
                     const at::Tensor& u, kern::GatedActivation act, const Needs& need) {
  c10::cuda::CUDAGuard guard(dy.device());
  Gradients r;
  const at::Tensor h = need.down ? gate32(g, u, act) : g;  // (else for its shape alone)
  const bool inner = need.x || need.gate || need.up;
  at::Tensor dh;
  std::tie(dh, r.down) = linear_gradients(dy, h, wd, inner, need.down);
  if (!inner) return r;
  at::Tensor dg = at::empty(g.sizes(), g.options()), du = at::empty(g.sizes(), g.options());
  OPS_CK(kern::launch_gate_f32_backward(g.const_data_ptr<float>(), u.const_data_ptr<float>(), dh.const_data_ptr<float>(), dg.data_ptr<float>(),
                                        du.data_ptr<float>(), g.numel(), act, at::cuda::getCurrentCUDAStream()));
  at::Tensor second;
  std::tie(r.x, r.gate) = linear_gradients(dg, x, wg, need.x, need.gate);
  std::tie(second, r.up) = linear_gradients(du, x, wu, need.x, need.up);
  if (need.x) r.x.add_(second);
  return r;
}

// ---- autograd -----------------------------------------------------------------------------------------------------
// Packed rows as an operand of 16-bit products, or as they were.
at::Tensor unpacked(const at::Tensor& codes, const at::Tensor& scales, int64_t rows, int64_t cols, const at::TensorOptions& like) {
  const int64_t ld = (cols + 7) / 8 * 8;
  at::Tensor x = at::empty({rows, ld}, like);
  const kern::Packed8Rows p{const_cast<int8_t*>(codes.const_data_ptr<int8_t>()), const_cast<float*>(scales.const_data_ptr<float>()), rows, cols,
                            kern::pack8_pitch(cols)};
  OPS_CK(kern::launch_unpack8(p, x.data_ptr(), elem_of(x, kWhat), ld, at::cuda::getCurrentCUDAStream()));
  return x.narrow(1, 0, cols);
}

struct GatedFn : torch::autograd::Function<GatedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act,
                            bool eight) {
    const auto activation = static_cast<kern::GatedActivation>(act);
    c10::cuda::CUDAGuard guard(x.device());
    ctx->saved_data["act"] = act;
    ctx->saved_data["eight"] = eight;
    ctx->saved_data["rows"] = x.size(0);
    std::vector<at::Tensor> saved{wg, wu, wd};
    at::Tensor y;
    if (x.scalar_type() == at::kFloat) {
      const at::Tensor g = mccl::linear(x, wg, c10::nullopt), u = mccl::linear(x, wu, c10::nullopt);
      y = mccl::linear(gate32(g, u, activation), wd, c10::nullopt);
      for (const at::Tensor* t : {&x, &g, &u}) {
        if (eight) {
          const auto [codes, scales] = pack8(*t);
          saved.insert(saved.end(), {codes, scales});
        } else {
          saved.push_back(*t);
        }
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
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &wg = saved[0], &wu = saved[1], &wd = saved[2];
    const auto act = static_cast<kern::GatedActivation>(ctx->saved_data["act"].toInt());
    const bool eight = ctx->saved_data["eight"].toBool();
    const int64_t rows = ctx->saved_data["rows"].toInt(), width = wg.size(1), hidden = wg.size(0);
    check_block_tensor(dy, kWhat);
    MCCL_CHECK_T(TensorError, dy.dim() == 2 && dy.size(0) == rows && dy.size(1) == width && dy.scalar_type() == wg.scalar_type() && dy.device() == wg.device(),
                 kWhat << ": not a gradient of its result");
    c10::cuda::CUDAGuard guard(dy.device());
    const Needs need{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    const bool need_up = need.gate || need.up;
    Gradients r;
    if (wg.scalar_type() == at::kFloat) {
      dy = dy.contiguous();
      at::Tensor x, g, u;
      if (eight) {
        x = need_up ? unpacked(saved[3], saved[4], rows, width, wg.options()) : at::empty({rows, width}, wg.options());
        g = unpacked(saved[5], saved[6], rows, hidden, wg.options()).contiguous();
        u = unpacked(saved[7], saved[8], rows, hidden, wg.options()).contiguous();
      } else {
        x = saved[3];
        g = saved[4];
        u = saved[5];
      }
      r = backward32(dy, x, wg, wu, wd, g, u, act, need);
    } else {
      const at::Tensor x = !need_up || rows == 0 ? at::Tensor() : eight ? unpacked(saved[3], saved[4], rows, width, wg.options()) : saved[3];
      r = backward16(dy, x, wg, wu, wd, saved.back(), act, eight ? kern::GatedKeep::kEight : kern::GatedKeep::kWide, need);
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
    const at::Tensor g = mccl::linear(rows, wg, c10::nullopt), u = mccl::linear(rows, wu, c10::nullopt);
    y = mccl::linear(gate32(g, u, act), wd, c10::nullopt);
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
