// What the operators made of the 16-bit products (kernels/gated.cu) share: operands laid out for them, and the launches of one pass.
#pragma once

#include "kernels/gated_api.h"
#include "ops/block_common.h"

namespace mccl {

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
  bool any() const { return copied_ > 0; }
  // The copies' memory.  What was freed before had its last use on this stream before now.
  void reserve(const at::Tensor& like) {
    if (copied_ > 0 && !held_.defined()) held_ = at::empty({bytes_}, like.options().dtype(at::kByte));
  }
  // Before what reads them.  `beside`: while the products launched since reserve() run, none of which reads them; the copies don't wait
  // for these, nor for what another thread has launched on this stream since then, so no memory that was in use since may be theirs.
  void copy(const at::Tensor& like, bool beside = false) {
    if (copied_ == 0) return;
    reserve(like);
    char* at = static_cast<char*>(held_.data_ptr());
    for (int i = 0; i < copied_; ++i) {
      copies_[i].to = at;
      m_[of_[i]].data = at;
      at += (copies_[i].rows * copies_[i].ld * 2 + 255) / 256 * 256;
    }
    OPS_CK(kern::launch_gated_copies(copies_, copied_, beside, at::cuda::getCurrentCUDAStream()));
  }
  const kern::GatedOperand& operator[](int i) const { return m_[i]; }

 private:
  int n_ = 0, copied_ = 0, of_[kern::kGatedCopies] = {};
  int64_t bytes_ = 0;
  kern::GatedOperand m_[kern::kGatedCopies] = {};
  kern::GatedCopy copies_[kern::kGatedCopies] = {};
  at::Tensor held_;
};

// Products of one pass, which follow each other on a stream and share the scratch for their partial sums.
struct Products {
  kern::GatedLaunch r;
  at::Tensor partial;
  Products(const kern::GatedShape& s, const at::Tensor& like, int64_t wait_limit) {
    r.shape = s;
    r.layer = nullptr;
    r.kept = nullptr;
    r.failed = wait_status(like);
    r.wait_limit = wait_limit;
    r.partial = nullptr;
  }
  void launch(const kern::GatedArgs* g, int n, const at::Tensor& like) {
    kern::GatedProduct p[3];
    for (int i = 0; i < n; ++i) p[i] = g[i].product;
    const int64_t bytes = kern::gated_partial_bytes(p, n, r.shape);
    if (bytes > (partial.defined() ? partial.numel() * 4 : 0)) {
      partial = at::empty({bytes / 4}, like.options().dtype(at::kFloat));
      r.partial = partial.data_ptr<float>();
    }
    OPS_CK(kern::launch_gated(g, n, r, at::cuda::getCurrentCUDAStream()));
  }
};

// Rows for kernels that read any alignment, but numbers side by side.
inline at::Tensor few_rows(const at::Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

}  // namespace mccl
