// The mx8 products with f16 results (kernels and reasons: dense8.h).
#include "dense8.h"

template <>
int lt_gemm8_launch<lt_f16>(const LtTile8Args& b, const LtPlan& p, int act, hipStream_t stream) {
  return lt_gemm8_launch_impl<lt_f16>(b, p, act, stream);
}
