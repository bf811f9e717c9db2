// Residual norm kernels of f32 residual streams and f16 blocks.
#include "residual_norm_backward.cuh"
#include "residual_norm_forward.cuh"

namespace opus {

int residual_norm_f32_f16(const opus_residual_norm_args& a, bool vec, cudaStream_t st) {
  return forward_by_alignment<float, __half>(a, vec, st);
}
int residual_norm_grad_f32_f16(const opus_residual_norm_args& a, bool vec, int wanted, const ColumnOutputs& out, uint8_t* ws,
                           cudaStream_t st) {
  return backward_by_alignment<float, __half>(a, vec, wanted, out, ws, st);
}

}  // namespace opus
