// The tiled products of the dense operators for bf16 (kernels and reasons: dense_gemm.h).
#include "dense_plan.h"

template <>
int lt_gemm_launch<lt_bf16>(const LtGemm& g, const LtPlan& p, float* part, hipStream_t stream) {
  return lt_gemm_launch_impl<lt_bf16>(g, p, part, stream);
}

template <>
int lt_rows_bwd_launch<lt_bf16>(const LtRowsBwdArgs& a, const LtRowsBwdPlan& p, hipStream_t stream) {
  return lt_rows_bwd_impl<lt_bf16>(a, p, stream);
}
