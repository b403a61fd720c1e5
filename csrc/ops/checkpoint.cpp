#include "ops/checkpoint.h"

#include "ops/block_common.h"

namespace mccl {

std::tuple<at::Tensor, at::Tensor> pack8(const at::Tensor& x) {
  check_block_tensor(x, "pack8");
  const kern::Elem type = elem_of(x, "pack8");
  c10::cuda::CUDAGuard guard(x.device());
  at::AutoDispatchBelowADInplaceOrView no_graph;
  const at::Tensor r = rows_of(x);
  const int64_t rows = r.size(0), cols = r.size(1), pitch = kern::pack8_pitch(cols);
  at::Tensor codes = at::empty({rows, pitch}, x.options().dtype(at::kChar));
  at::Tensor scales = at::empty({rows, kern::pack8_groups(cols)}, x.options().dtype(at::kFloat));
  const kern::Packed8Rows p{codes.data_ptr<int8_t>(), scales.data_ptr<float>(), rows, cols, pitch};
  OPS_CK(kern::launch_pack8(r.const_data_ptr(), type, row_stride(r), p, at::cuda::getCurrentCUDAStream()));
  return {codes, scales};
}

at::Tensor unpack8(const at::Tensor& codes_in, const at::Tensor& scales_in, at::IntArrayRef shape, at::ScalarType type) {
  check_block_tensor(codes_in, "unpack8");
  check_block_tensor(scales_in, "unpack8");
  int64_t rows = 1;
  for (size_t d = 0; d < shape.size(); ++d) {
    MCCL_CHECK_T(TensorError, shape[d] >= 0, "unpack8: negative size");
    if (d + 1 < shape.size()) rows *= shape[d];
  }
  const int64_t cols = shape.empty() ? 1 : shape.back();
  MCCL_CHECK_T(TensorError,
               codes_in.scalar_type() == at::kChar && scales_in.scalar_type() == at::kFloat && codes_in.dim() == 2 && scales_in.dim() == 2 &&
                   codes_in.size(0) == rows && scales_in.size(0) == rows && codes_in.size(1) == kern::pack8_pitch(cols) &&
                   scales_in.size(1) == kern::pack8_groups(cols) && codes_in.device() == scales_in.device(),
               "unpack8: codes and scales are not those of pack8 for this shape");
  c10::cuda::CUDAGuard guard(codes_in.device());
  const at::Tensor codes = packed_again(codes_in), scales = packed_again(scales_in);
  at::Tensor x = at::empty(shape, codes.options().dtype(type));
  const kern::Packed8Rows p{const_cast<int8_t*>(codes.const_data_ptr<int8_t>()), const_cast<float*>(scales.const_data_ptr<float>()), rows, cols,
                            kern::pack8_pitch(cols)};
  OPS_CK(kern::launch_unpack8(p, x.data_ptr(), elem_of(x, "unpack8"), cols, at::cuda::getCurrentCUDAStream()));
  return x;
}

}  // namespace mccl
