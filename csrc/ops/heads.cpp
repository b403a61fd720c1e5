#include "ops/heads.h"

#include <torch/csrc/autograd/custom_function.h>

#include <cmath>

#include "kernels/heads_api.h"
#include "ops/block_common.h"

namespace mccl {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

kern::HeadRows head_rows(const at::Tensor& t) { return {t.const_data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }
// [batch, tokens, heads, dim] with its numbers side by side.
at::Tensor side_by_side(const at::Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

kern::HeadsShape shape_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight, const at::Tensor& k_weight, const at::Tensor& table,
                          const at::Tensor& positions, double eps, bool interleaved) {
  constexpr const char* what = "norm_rotate";
  check_block_tensor(q, what);
  check_block_tensor(k, what);
  MCCL_CHECK_T(TensorError, q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
               what << ": queries [batch, tokens, heads, dim] and keys [batch, tokens, kv heads, dim] expected, got " << q.sizes() << " and " << k.sizes());
  const int64_t dim = q.size(3);
  MCCL_CHECK_T(TensorError, q.scalar_type() == k.scalar_type() && q.device() == k.device(), what << ": queries and keys differ in type or device");
  MCCL_CHECK_T(TensorError, q.size(2) > 0 && k.size(2) > 0 && q.size(2) <= 65536 && k.size(2) <= 65536, what << ": 1 to 65536 heads expected");
  MCCL_CHECK_T(TensorError, dim > 0 && dim <= kern::kMaxHeadDim, what << ": head sizes up to " << kern::kMaxHeadDim << ", got " << dim);
  kern::HeadsShape s{};
  s.type = elem_of(q, what);
  for (const at::Tensor* w : {&q_weight, &k_weight}) {
    check_block_tensor(*w, what);
    MCCL_CHECK_T(TensorError, w->dim() == 1 && w->size(0) == dim && w->is_contiguous() && w->device() == q.device() &&
                                  (w->scalar_type() == at::kFloat || w->scalar_type() == q.scalar_type()) && w->scalar_type() == q_weight.scalar_type(),
                 what << ": weights are " << dim << " numbers of float32 or of the queries' type, on their device, both alike");
  }
  check_block_tensor(table, what);
  MCCL_CHECK_T(TensorError, table.dim() == 3 && table.size(1) == 2 && table.scalar_type() == at::kFloat && table.is_contiguous() && table.device() == q.device() &&
                                !table.requires_grad() && 2 * table.size(2) <= dim,
               what << ": a contiguous float32 table [positions, 2, rotary / 2] without gradient expected, rotary at most " << dim);
  MCCL_CHECK_T(TensorError, eps > 0 && std::isfinite(eps), what << ": eps must be positive");
  s.batches = q.size(0);
  s.tokens = q.size(1);
  s.heads = static_cast<int>(q.size(2));
  s.kv_heads = static_cast<int>(k.size(2));
  s.dim = static_cast<int>(dim);
  s.rotary = static_cast<int>(2 * table.size(2));
  s.interleaved = interleaved;
  s.eps = static_cast<float>(eps);
  s.q_weight = q_weight.const_data_ptr();
  s.k_weight = k_weight.const_data_ptr();
  s.weights_f32 = q_weight.scalar_type() == at::kFloat;
  s.table = table.const_data_ptr<float>();
  s.table_rows = table.size(0);
  if (positions.defined()) {
    check_block_tensor(positions, what);
    MCCL_CHECK_T(TensorError,
                 (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt) && positions.device() == q.device() &&
                     ((positions.dim() == 1 && positions.size(0) == s.tokens) ||
                      (positions.dim() == 2 && (positions.size(0) == s.batches || positions.size(0) == 1) && positions.size(1) == s.tokens)),
                 what << ": positions are int64 or int32, [tokens] or [batch, tokens]");
    s.positions = positions.const_data_ptr();
    s.positions_32 = positions.scalar_type() == at::kInt;
    s.pos_batch = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    s.pos_token = positions.stride(-1);
  }
  return s;
}

at::Tensor out_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options()); }

std::tuple<at::Tensor, at::Tensor> forward_of(const kern::HeadsShape& s, const at::Tensor& q, const at::Tensor& k) {
  c10::cuda::CUDAGuard guard(q.device());
  kern::HeadsForward a{};
  a.shape = s;
  const at::Tensor qs = side_by_side(q), ks = side_by_side(k);
  a.q = head_rows(qs);
  a.k = head_rows(ks);
  at::Tensor qo = out_like(q), ko = out_like(k);
  a.q_out = qo.data_ptr();
  a.k_out = ko.data_ptr();
  OPS_CK(kern::launch_heads_forward(a, at::cuda::getCurrentCUDAStream()));
  return {qo, ko};
}

// A gradient as the kernels read it; none is zeros.
at::Tensor grad_for(const at::Tensor& g, const at::Tensor& like, at::IntArrayRef sizes) {
  if (!g.defined()) return at::zeros(sizes, like.options());
  MCCL_CHECK_T(TensorError, ordinary(g) && g.scalar_type() == like.scalar_type() && g.sizes() == sizes, "norm_rotate: not a gradient of its results");
  return side_by_side(g);
}

// qkv views: queries, keys, values
std::array<at::Tensor, 3> parts_of(const at::Tensor& qkv, int64_t heads, int64_t kv_heads) {
  const int64_t all = heads + 2 * kv_heads, dim = qkv.size(2) / all;
  const at::Tensor rows = qkv.view({qkv.size(0), qkv.size(1), all, dim});
  return {rows.narrow(2, 0, heads), rows.narrow(2, heads, kv_heads), rows.narrow(2, heads + kv_heads, kv_heads)};
}

struct Kept {
  at::Tensor q_weight, k_weight, table, positions;
};

variable_list backward_of(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const Kept& kept, const at::Tensor& dq, const at::Tensor& dk,
                          const at::Tensor& dv, at::Tensor& dq_out, at::Tensor& dk_out, at::Tensor dv_out, bool need_qw, bool need_kw) {
  c10::cuda::CUDAGuard guard(q.device());
  kern::HeadsBackward a{};
  a.shape = shape_of(q, k, kept.q_weight, kept.k_weight, kept.table, kept.positions, ctx->saved_data["eps"].toDouble(),
                     ctx->saved_data["interleaved"].toBool());
  a.q = head_rows(q);
  a.k = head_rows(k);
  a.dq = head_rows(dq);
  a.dk = head_rows(dk);
  a.dq_out = dq_out.data_ptr();
  a.dk_out = dk_out.data_ptr();
  a.dq_token = dq_out.stride(1);
  a.dk_token = dk_out.stride(1);
  if (dv_out.defined()) {
    a.dv = head_rows(dv);
    a.dv_out = dv_out.data_ptr();
    a.dv_token = dv_out.stride(1);
  }
  at::Tensor partial, qw, kw;
  if (need_qw || need_kw) {
    // no token: nothing is launched, and the sums over none are zeros
    const bool none = a.shape.batches * a.shape.tokens == 0;
    partial = at::empty({kern::heads_partials(), a.shape.dim}, q.options().dtype(at::kFloat));
    a.partial = partial.data_ptr<float>();
    if (need_qw) qw = none ? at::zeros_like(kept.q_weight) : at::empty_like(kept.q_weight);
    if (need_kw) kw = none ? at::zeros_like(kept.k_weight) : at::empty_like(kept.k_weight);
    a.dq_weight = need_qw ? qw.data_ptr() : nullptr;
    a.dk_weight = need_kw ? kw.data_ptr() : nullptr;
  }
  OPS_CK(kern::launch_heads_backward(a, at::cuda::getCurrentCUDAStream()));
  return {qw, kw};
}

void no_second(const char* what) {
  MCCL_CHECK_T(TensorError, !at::GradMode::is_enabled(), what << ": the backward pass is not differentiable (create_graph)");
}

struct NormRotate : torch::autograd::Function<NormRotate> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
                               const at::Tensor& table, const c10::optional<at::Tensor>& positions, double eps, bool interleaved) {
    const at::Tensor pos = positions ? *positions : at::Tensor();
    const auto [qo, ko] = forward_of(shape_of(q, k, qw, kw, table, pos, eps, interleaved), q, k);
    ctx->save_for_backward({q, k, qw, kw, table, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second("norm_rotate");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor q = side_by_side(saved[0]), k = side_by_side(saved[1]);
    const at::Tensor dq = grad_for(g[0], q, q.sizes()), dk = grad_for(g[1], k, k.sizes());
    at::Tensor dqo = out_like(q), dko = out_like(k);
    const auto w = backward_of(ctx, q, k, {saved[2], saved[3], saved[4], saved[5]}, dq, dk, {}, dqo, dko, {}, ctx->needs_input_grad(2),
                               ctx->needs_input_grad(3));
    return {dqo, dko, w[0], w[1], {}, {}, {}, {}};
  }
};

struct NormRotatePacked : torch::autograd::Function<NormRotatePacked> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& qkv, const at::Tensor& qw, const at::Tensor& kw, const at::Tensor& table,
                               const c10::optional<at::Tensor>& positions, int64_t heads, int64_t kv_heads, double eps, bool interleaved) {
    const at::Tensor pos = positions ? *positions : at::Tensor();
    const auto parts = parts_of(qkv, heads, kv_heads);
    const auto [qo, ko] = forward_of(shape_of(parts[0], parts[1], qw, kw, table, pos, eps, interleaved), parts[0], parts[1]);
    ctx->save_for_backward({qkv, qw, kw, table, pos});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["kv_heads"] = kv_heads;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {qo, ko, parts[2]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second("norm_rotate_packed");
    const auto saved = ctx->get_saved_variables();
    const int64_t heads = ctx->saved_data["heads"].toInt(), kv_heads = ctx->saved_data["kv_heads"].toInt();
    const auto parts = parts_of(saved[0], heads, kv_heads);
    at::Tensor out = at::empty(saved[0].sizes(), saved[0].options());
    auto outs = parts_of(out, heads, kv_heads);
    at::Tensor d[3];
    for (int i = 0; i < 3; ++i) d[i] = grad_for(g[i], parts[i], parts[i].sizes());
    const auto w = backward_of(ctx, parts[0], parts[1], {saved[1], saved[2], saved[3], saved[4]}, d[0], d[1], d[2], outs[0], outs[1], outs[2],
                               ctx->needs_input_grad(1), ctx->needs_input_grad(2));
    return {out, w[0], w[1], {}, {}, {}, {}, {}, {}};
  }
};

bool differentiates(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> norm_rotate(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                               const at::Tensor& table, const c10::optional<at::Tensor>& positions, double eps, bool interleaved) {
  if (!differentiates({&q, &k, &q_weight, &k_weight}))
    return forward_of(shape_of(q, k, q_weight, k_weight, table, positions ? *positions : at::Tensor(), eps, interleaved), q, k);
  const auto r = NormRotate::apply(q, k, q_weight, k_weight, table, positions, eps, interleaved);
  return {r[0], r[1]};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_rotate_packed(const at::Tensor& qkv_in, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                                                  const at::Tensor& table, const c10::optional<at::Tensor>& positions,
                                                                  int64_t heads, int64_t kv_heads, double eps, bool interleaved) {
  check_block_tensor(qkv_in, "norm_rotate_packed");
  MCCL_CHECK_T(TensorError, heads > 0 && kv_heads > 0 && heads <= 65536 && kv_heads <= 65536, "norm_rotate_packed: 1 to 65536 heads expected");
  MCCL_CHECK_T(TensorError, qkv_in.dim() == 3 && qkv_in.size(2) > 0 && qkv_in.size(2) % (heads + 2 * kv_heads) == 0,
               "norm_rotate_packed: [batch, tokens, (heads + 2 kv_heads) dim] expected, got " << qkv_in.sizes());
  const at::Tensor qkv = qkv_in.size(2) == 1 || qkv_in.stride(2) == 1 ? qkv_in : qkv_in.contiguous();
  if (!differentiates({&qkv, &q_weight, &k_weight})) {
    const auto parts = parts_of(qkv, heads, kv_heads);
    const auto [q, k] = forward_of(
        shape_of(parts[0], parts[1], q_weight, k_weight, table, positions ? *positions : at::Tensor(), eps, interleaved), parts[0], parts[1]);
    return {q, k, parts[2]};
  }
  const auto r = NormRotatePacked::apply(qkv, q_weight, k_weight, table, positions, heads, kv_heads, eps, interleaved);
  return {r[0], r[1], r[2]};
}

}  // namespace mccl
