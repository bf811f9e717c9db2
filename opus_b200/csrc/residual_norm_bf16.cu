// Residual norm kernels of bf16.
#include "residual_norm_backward.cuh"
#include "residual_norm_forward.cuh"

namespace opus {

int residual_norm_bf16(const opus_residual_norm_args& a, bool vec, cudaStream_t st) {
  return forward_by_alignment<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
}
int residual_norm_grad_bf16(const opus_residual_norm_args& a, bool vec, int wanted, const ColumnOutputs& out, uint8_t* ws,
                           cudaStream_t st) {
  return backward_by_alignment<__nv_bfloat16, __nv_bfloat16>(a, vec, wanted, out, ws, st);
}

}  // namespace opus
