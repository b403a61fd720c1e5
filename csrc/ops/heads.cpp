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

constexpr const char* kWhat = "norm_rotate";

// What the queries and keys have in common, and everything else that both directions are told.
struct Heads {
  int64_t batches, tokens, heads, kv_heads, dim;
};
kern::HeadsShape shape_of(const Heads& h, const at::Tensor& q, const at::Tensor& q_weight, const at::Tensor& k_weight, const at::Tensor& table,
                          const at::Tensor& positions, double eps, bool interleaved) {
  MCCL_CHECK_T(TensorError, h.heads > 0 && h.kv_heads > 0 && h.heads <= 65536 && h.kv_heads <= 65536, kWhat << ": 1 to 65536 heads expected");
  MCCL_CHECK_T(TensorError, h.dim > 0 && h.dim <= kern::kMaxHeadDim, kWhat << ": head sizes up to " << kern::kMaxHeadDim << ", got " << h.dim);
  kern::HeadsShape s{};
  s.type = elem_of(q, kWhat);
  for (const at::Tensor* w : {&q_weight, &k_weight}) {
    check_block_tensor(*w, kWhat);
    MCCL_CHECK_T(TensorError, w->dim() == 1 && w->size(0) == h.dim && w->is_contiguous() && w->device() == q.device() &&
                                  (w->scalar_type() == at::kFloat || w->scalar_type() == q.scalar_type()) && w->scalar_type() == q_weight.scalar_type(),
                 kWhat << ": weights are " << h.dim << " numbers of float32 or of the queries' type, on their device, both alike");
  }
  check_block_tensor(table, kWhat);
  MCCL_CHECK_T(TensorError, table.dim() == 3 && table.size(1) == 2 && table.scalar_type() == at::kFloat && table.is_contiguous() && table.device() == q.device() &&
                                !table.requires_grad() && 2 * table.size(2) <= h.dim,
               kWhat << ": a contiguous float32 table [positions, 2, rotary / 2] without gradient expected, rotary at most " << h.dim);
  MCCL_CHECK_T(TensorError, eps > 0 && std::isfinite(eps), kWhat << ": eps must be positive");
  s.batches = h.batches;
  s.tokens = h.tokens;
  s.heads = static_cast<int>(h.heads);
  s.kv_heads = static_cast<int>(h.kv_heads);
  s.dim = static_cast<int>(h.dim);
  s.rotary = static_cast<int>(2 * table.size(2));
  s.interleaved = interleaved;
  s.eps = static_cast<float>(eps);
  s.q_weight = q_weight.const_data_ptr();
  s.k_weight = k_weight.const_data_ptr();
  s.weights_f32 = q_weight.scalar_type() == at::kFloat;
  s.table = table.const_data_ptr<float>();
  s.table_rows = table.size(0);
  if (positions.defined()) {
    check_block_tensor(positions, kWhat);
    MCCL_CHECK_T(TensorError,
                 (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt) && positions.device() == q.device() &&
                     ((positions.dim() == 1 && positions.size(0) == s.tokens) ||
                      (positions.dim() == 2 && (positions.size(0) == s.batches || positions.size(0) == 1) && positions.size(1) == s.tokens)),
                 kWhat << ": positions are int64 or int32, [tokens] or [batch, tokens]");
    s.positions = positions.const_data_ptr();
    s.positions_32 = positions.scalar_type() == at::kInt;
    s.pos_batch = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    s.pos_token = positions.stride(-1);
  }
  return s;
}
Heads heads_of(const at::Tensor& q, const at::Tensor& k) {
  check_block_tensor(q, kWhat);
  check_block_tensor(k, kWhat);
  MCCL_CHECK_T(TensorError, q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
               kWhat << ": queries [batch, tokens, heads, dim] and keys [batch, tokens, kv heads, dim] expected, got " << q.sizes() << " and " << k.sizes());
  MCCL_CHECK_T(TensorError, q.scalar_type() == k.scalar_type() && q.device() == k.device(), kWhat << ": queries and keys differ in type or device");
  return {q.size(0), q.size(1), q.size(2), k.size(2), q.size(3)};
}

at::Tensor out_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options()); }

std::tuple<at::Tensor, at::Tensor> forward_of(const kern::HeadsShape& s, const kern::HeadRows& q, const kern::HeadRows& k, const at::Tensor& like) {
  kern::HeadsForward a{};
  a.shape = s;
  a.q = q;
  a.k = k;
  at::Tensor qo = at::empty({s.batches, s.tokens, s.heads, s.dim}, like.options()), ko = at::empty({s.batches, s.tokens, s.kv_heads, s.dim}, like.options());
  a.q_out = qo.data_ptr();
  a.k_out = ko.data_ptr();
  OPS_CK(kern::launch_heads_forward(a, at::cuda::getCurrentCUDAStream()));
  return {qo, ko};
}

// A gradient as the kernels read it; none is zeros.
at::Tensor grad_for(const at::Tensor& g, const at::Tensor& like, at::IntArrayRef sizes) {
  if (!g.defined()) return at::zeros(sizes, like.options());
  MCCL_CHECK_T(TensorError, ordinary(g) && g.scalar_type() == like.scalar_type() && g.device() == like.device() && g.sizes() == sizes, "norm_rotate: not a gradient of its results");
  return side_by_side(g);
}

// The rows of a projection [batch, tokens, (heads + 2 kv_heads) dim]: queries, keys, values.
struct Packed {
  Heads h;
  kern::HeadRows rows[3];
};
Packed packed_of(const at::Tensor& qkv, int64_t heads, int64_t kv_heads) {
  const int64_t dim = qkv.size(2) / (heads + 2 * kv_heads), size = qkv.element_size();
  Packed p{{qkv.size(0), qkv.size(1), heads, kv_heads, dim}, {}};
  const char* base = static_cast<const char*>(qkv.const_data_ptr());
  const int64_t first[3] = {0, heads, heads + kv_heads};
  for (int i = 0; i < 3; ++i) p.rows[i] = {base + first[i] * dim * size, qkv.stride(0), qkv.stride(1), dim};
  return p;
}
at::Tensor values_of(const at::Tensor& qkv, const Heads& h) {
  return qkv.as_strided({h.batches, h.tokens, h.kv_heads, h.dim}, {qkv.stride(0), qkv.stride(1), h.dim, 1}, qkv.storage_offset() + (h.heads + h.kv_heads) * h.dim);
}

struct Kept {
  at::Tensor q_weight, k_weight, table, positions;
};

// Launches with everything but the weights' gradients set, and returns these.
variable_list backward_of(kern::HeadsBackward& a, const at::Tensor& like, const Kept& kept, bool need_qw, bool need_kw) {
  at::Tensor partial, qw, kw;
  if (need_qw || need_kw) {
    // no token: nothing is launched, and the sums over none are zeros
    const bool none = a.shape.batches * a.shape.tokens == 0;
    partial = at::empty({kern::heads_partials(), a.shape.dim}, like.options().dtype(at::kFloat));
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
  check_not_traced(what);
}

std::tuple<at::Tensor, at::Tensor> plain_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw, const at::Tensor& table,
                                                 const at::Tensor& positions, double eps, bool interleaved) {
  const kern::HeadsShape s = shape_of(heads_of(q, k), q, qw, kw, table, positions, eps, interleaved);
  c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor qs = side_by_side(q), ks = side_by_side(k);
  return forward_of(s, head_rows(qs), head_rows(ks), q);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_forward(const at::Tensor& qkv, const at::Tensor& qw, const at::Tensor& kw, const at::Tensor& table,
                                                              const at::Tensor& positions, int64_t heads, int64_t kv_heads, double eps, bool interleaved) {
  const Packed p = packed_of(qkv, heads, kv_heads);
  const kern::HeadsShape s = shape_of(p.h, qkv, qw, kw, table, positions, eps, interleaved);
  c10::cuda::CUDAGuard guard(qkv.device());
  auto [q, k] = forward_of(s, p.rows[0], p.rows[1], qkv);
  return {q, k, values_of(qkv, p.h)};
}

struct NormRotate : torch::autograd::Function<NormRotate> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
                               const at::Tensor& table, const c10::optional<at::Tensor>& positions, double eps, bool interleaved) {
    const at::Tensor pos = positions ? *positions : at::Tensor();
    const auto [qo, ko] = plain_forward(q, k, qw, kw, table, pos, eps, interleaved);
    ctx->save_for_backward({q, k, qw, kw, table, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second("norm_rotate");
    const auto saved = ctx->get_saved_variables();
    heads_of(saved[0], saved[1]);
    c10::cuda::CUDAGuard guard(saved[0].device());
    const at::Tensor q = side_by_side(saved[0]), k = side_by_side(saved[1]);
    const Kept kept{saved[2].contiguous(), saved[3].contiguous(), saved[4].contiguous(), saved[5]};
    const at::Tensor dq = grad_for(g[0], q, q.sizes()), dk = grad_for(g[1], k, k.sizes());
    at::Tensor dqo = out_like(q), dko = out_like(k);
    kern::HeadsBackward a{};
    a.shape = shape_of(heads_of(q, k), q, kept.q_weight, kept.k_weight, kept.table, kept.positions, ctx->saved_data["eps"].toDouble(),
                       ctx->saved_data["interleaved"].toBool());
    a.q = head_rows(q);
    a.k = head_rows(k);
    a.dq = head_rows(dq);
    a.dk = head_rows(dk);
    a.dq_out = dqo.data_ptr();
    a.dk_out = dko.data_ptr();
    a.dq_token = dqo.stride(1);
    a.dk_token = dko.stride(1);
    const auto w = backward_of(a, q, kept, ctx->needs_input_grad(2), ctx->needs_input_grad(3));
    return {dqo, dko, w[0], w[1], {}, {}, {}, {}};
  }
};

struct NormRotatePacked : torch::autograd::Function<NormRotatePacked> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& qkv, const at::Tensor& qw, const at::Tensor& kw, const at::Tensor& table,
                               const c10::optional<at::Tensor>& positions, int64_t heads, int64_t kv_heads, double eps, bool interleaved) {
    const at::Tensor pos = positions ? *positions : at::Tensor();
    const auto [qo, ko, v] = packed_forward(qkv, qw, kw, table, pos, heads, kv_heads, eps, interleaved);
    ctx->save_for_backward({qkv, qw, kw, table, pos});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["kv_heads"] = kv_heads;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {qo, ko, v};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second("norm_rotate_packed");
    const auto saved = ctx->get_saved_variables();
    check_block_tensor(saved[0], kWhat);
    const int64_t kinds = ctx->saved_data["heads"].toInt() + 2 * ctx->saved_data["kv_heads"].toInt();
    MCCL_CHECK_T(TensorError, saved[0].dim() == 3 && saved[0].size(2) > 0 && saved[0].size(2) % kinds == 0,
                 "norm_rotate_packed: a tensor saved for the backward pass came back as " << saved[0].sizes());
    const at::Tensor qkv = saved[0].size(2) == 1 || saved[0].stride(2) == 1 ? saved[0] : saved[0].contiguous();
    const Kept kept{saved[1].contiguous(), saved[2].contiguous(), saved[3].contiguous(), saved[4]};
    c10::cuda::CUDAGuard guard(qkv.device());
    const Packed p = packed_of(qkv, ctx->saved_data["heads"].toInt(), ctx->saved_data["kv_heads"].toInt());
    at::Tensor out = at::empty(qkv.sizes(), qkv.options());
    at::Tensor d[3];
    for (int i = 0; i < 3; ++i) d[i] = grad_for(g[i], qkv, {p.h.batches, p.h.tokens, i == 0 ? p.h.heads : p.h.kv_heads, p.h.dim});
    kern::HeadsBackward a{};
    a.shape = shape_of(p.h, qkv, kept.q_weight, kept.k_weight, kept.table, kept.positions, ctx->saved_data["eps"].toDouble(),
                       ctx->saved_data["interleaved"].toBool());
    a.q = p.rows[0];
    a.k = p.rows[1];
    a.dq = head_rows(d[0]);
    a.dk = head_rows(d[1]);
    a.dv = head_rows(d[2]);
    char* to = static_cast<char*>(out.data_ptr());
    const int64_t row = p.h.dim * out.element_size();
    a.dq_out = to;
    a.dk_out = to + p.h.heads * row;
    a.dv_out = to + (p.h.heads + p.h.kv_heads) * row;
    a.dq_token = a.dk_token = a.dv_token = out.size(2);
    const auto w = backward_of(a, qkv, kept, ctx->needs_input_grad(1), ctx->needs_input_grad(2));
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
  if (!differentiates({&q, &k, &q_weight, &k_weight})) return plain_forward(q, k, q_weight, k_weight, table, positions ? *positions : at::Tensor(), eps, interleaved);
  const auto r = NormRotate::apply(q, k, q_weight, k_weight, table, positions, eps, interleaved);
  return {r[0], r[1]};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_rotate_packed(const at::Tensor& qkv_in, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                                                  const at::Tensor& table, const c10::optional<at::Tensor>& positions,
                                                                  int64_t heads, int64_t kv_heads, double eps, bool interleaved) {
  check_block_tensor(qkv_in, kWhat);
  MCCL_CHECK_T(TensorError, heads > 0 && kv_heads > 0 && heads <= 65536 && kv_heads <= 65536, "norm_rotate_packed: 1 to 65536 heads expected");
  MCCL_CHECK_T(TensorError, qkv_in.dim() == 3 && qkv_in.size(2) > 0 && qkv_in.size(2) % (heads + 2 * kv_heads) == 0,
               "norm_rotate_packed: [batch, tokens, (heads + 2 kv_heads) dim] expected, got " << qkv_in.sizes());
  const at::Tensor qkv = qkv_in.size(2) == 1 || qkv_in.stride(2) == 1 ? qkv_in : qkv_in.contiguous();
  if (!differentiates({&qkv, &q_weight, &k_weight}))
    return packed_forward(qkv, q_weight, k_weight, table, positions ? *positions : at::Tensor(), heads, kv_heads, eps, interleaved);
  const auto r = NormRotatePacked::apply(qkv, q_weight, k_weight, table, positions, heads, kv_heads, eps, interleaved);
  return {r[0], r[1], r[2]};
}

}  // namespace mccl
