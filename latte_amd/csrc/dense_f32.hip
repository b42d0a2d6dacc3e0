// The tiled products of the dense operators for f32 (kernels and reasons: dense_gemm.h).
#include "dense_gemm.h"

template <>
int lt_gemm_launch<float>(const LtGemm& g, const LtPlan& p, float* part, hipStream_t stream) {
  return lt_gemm_launch_impl<float>(g, p, part, stream);
}
