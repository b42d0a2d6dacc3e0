// The tiled products of the dense operators for f32 (kernels and reasons: dense_gemm.h).
#include "dense_plan.h"

template <>
int lt_gemm_launch<float>(const LtGemm& g, const LtPlan& p, float* part, hipStream_t stream) {
  return lt_gemm_launch_impl<float>(g, p, part, stream);
}

template <>
int lt_rows_bwd_launch<float>(const LtRowsBwdArgs& a, const LtRowsBwdPlan& p, hipStream_t stream) {
  return lt_rows_bwd_impl<float>(a, p, stream);
}
