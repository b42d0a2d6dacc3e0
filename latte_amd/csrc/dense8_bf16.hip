// The mx8 products with bf16 results (kernels and reasons: dense8.h).
#include "dense8.h"

template <>
int lt_gemm8_launch<lt_bf16>(const LtTile8Args& b, const LtPlan& p, int act, hipStream_t stream) {
  return lt_gemm8_launch_impl<lt_bf16>(b, p, act, stream);
}
