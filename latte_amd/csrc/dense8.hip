// lt_linear_mx8_fwd: both operands in mx8 (kernels and reasons: dense8.h).
#include "dense8.h"

template <> int lt_gemm8_launch<lt_bf16>(const LtTile8Args&, const LtPlan&, int, hipStream_t);
template <> int lt_gemm8_launch<lt_f16>(const LtTile8Args&, const LtPlan&, int, hipStream_t);

// Both sides of each rule, us.  Up to 32 rows, this way and on tiles: 4096 -> 4096 6.1 and 8.6 for one row, 11.1 and 10.7 for 32; 1024 ->
// 1024 4.7 and 7.6 for 32.  256 x 256 tiles and 128 x 128: x 4096 -> 4096 with 128 of the larger 57 and 39, 160 of them 57.8 and 60.2,
// 192 of them 58.7 and 61.6, 256 of them 62 and 73 (320: 115 and 94, a second turn).  128 x 128 and 64 x 64: x 4096 -> 2048 with 128 of the
// larger 28 and 23, 256 of them 30 and 30; x 1024 -> 2048 with 128 of them 20.3 and 8.5 (split in two), 256 of them 11.9 and 11.8.  Split
// and whole: 64 x 4096 -> 4096 13.1 and 16.2, 256 x 8192 -> 512 13.4 and 28.5, 300 x 1024 -> 1024 8.7 and 6.5.
static LtPlan plan8(int64_t M, int K, int N, bool direct) {
  LtPlan p = {};
  p.direct = direct;
  p.splits = 1;
  p.slice = K;
  p.few = M <= 32;
  if (p.few) return p;
  auto tiles = [&](int b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
  int b = 64;
  p.tile = LT_TILE_64x64;
  if (direct && N >= 192 && tiles(256) >= 192) p.tile = LT_TILE_256x256, b = 256;
  else if (direct && tiles(128) >= 128) p.tile = LT_TILE_128x128, b = 128;
  p.tr = (int)((M + b - 1) / b);
  p.tc = (N + b - 1) / b;
  const int64_t t = (int64_t)p.tr * p.tc, steps = (K + 127) / 128;
  if (b != 256 && t < 256) {   // fewer tiles than the chip runs at once: split k, at least four steps each
    int64_t s = (512 + t - 1) / t;
    if (s > steps / 4) s = steps / 4;
    if (s > 1) {
      const int64_t per = (steps + s - 1) / s;
      p.slice = per * 128;
      p.splits = (int)((steps + per - 1) / per);
    }
  }
  return p;
}
static int64_t part8(const LtPlan& p, int64_t M, int N) { return p.splits > 1 ? p.splits * M * N * 4 : 0; }

static int check8(const char* who, int64_t M, int32_t K, int32_t N) {
  LT_REQUIRE(M >= 0 && K >= 1 && N >= 1 && K <= INT32_MAX - 1024 && N <= INT32_MAX - 1024, LT_ERR_ARG,
             "%s: bad sizes M=%lld K=%d N=%d", who, (long long)M, K, N);
  const int64_t most = (int64_t)1 << 42;   // elements: more than any memory holds, and byte counts stay within 64 bits
  LT_REQUIRE(M <= most / (K > N ? K : N) && K <= most / N, LT_ERR_RANGE, "%s: M=%lld K=%d N=%d is too large", who, (long long)M, K, N);
  return LT_OK;
}

// Rows whose length is no multiple of 16 bytes go through registers at 610 TFLOP/s, whole pieces straight into LDS at 1800: a
// large product is worth a copy of its values with the rows filled up by zeros (the scales stay: a block of 32 ends behind
// them).  8192 x 4095 -> 4096: 450 us as it is, 159 with the copies; 65536 x 511 -> 511: 103 and 69.
static bool pad8(int64_t M, int K, int N) {
  const double gain = 2e-6 * (double)M * N * K * (1 / 610. - 1 / 1800.);   // us
  return K % 16 != 0 && gain > 10 + 2e6 * (double)(M + N) * K / 3.5e12;     // two launches, a read and a write
}
static int64_t pad8_bytes(int64_t M, int K, int N) {
  return pad8(M, K, N) ? lt_align_up((M + N) * (((int64_t)K + 15) / 16 * 16), 256) : 0;
}

__global__ __launch_bounds__(256) void k_pad8(const uint8_t* __restrict__ x, int64_t M, int K, uint8_t* __restrict__ out) {
  const int L = (K + 15) >> 4;
  const int64_t total = M * L, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += stride) {
    int64_t row;
    int l;
    lt_divmod(i, L, row, l);
    const uint8_t* p = x + row * K + l * 16;
    const int n = K - l * 16;
    uint8_t v[16];
    if (n >= 16) __builtin_memcpy(v, p, 16);
    else {
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = t < n ? p[t] : 0;
    }
    __builtin_memcpy(out + i * 16, v, 16);
  }
}

extern "C" int64_t lt_linear_mx8_workspace_bytes(int64_t M, int32_t K, int32_t N) {
  if (check8("lt_linear_mx8_workspace_bytes", M, K, N)) return -1;
  if (M == 0) return 0;
  const int64_t a = part8(plan8(M, K, N, true), M, N), b = part8(plan8(M, K, N, false), M, N);
  return pad8_bytes(M, K, N) + (a > b ? a : b);
}

extern "C" int lt_linear_mx8_fwd(const void* x, const void* x_scales, const void* w, const void* w_scales, const void* bias,
                                 const void* res, int64_t ldres, int32_t act, int64_t M, int32_t K, int32_t N, int32_t dt, void* y,
                                 void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check8("lt_linear_mx8_fwd", M, K, N);
  if (rc) return rc;
  LT_REQUIRE(dt == LT_DT_BF16 || dt == LT_DT_F16, LT_ERR_ARG, "lt_linear_mx8_fwd: type %d: results are bfloat16 or float16", dt);
  LT_REQUIRE(act >= LT_ACT_NONE && act <= LT_ACT_SILU, LT_ERR_ARG, "lt_linear_mx8_fwd: act=%d is none of LT_ACT_*", act);
  if (M == 0) return LT_OK;
  LT_REQUIRE(x && x_scales && w && w_scales && y, LT_ERR_ARG, "lt_linear_mx8_fwd: null pointer");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  int64_t ld = K;
  const int64_t pad = pad8_bytes(M, K, N);
  ws_bytes = ws ? ws_bytes : 0;
  if (pad > 0) {
    LT_REQUIRE(pad <= ws_bytes, LT_ERR_WORKSPACE, "lt_linear_mx8_fwd: workspace too small");
    ld = ((int64_t)K + 15) / 16 * 16;
    uint8_t *w16 = (uint8_t*)ws, *x16 = w16 + N * ld;
    hipLaunchKernelGGL(k_pad8, dim3(lt_grid(N * ld / 16, 256)), dim3(256), 0, stream, (const uint8_t*)w, (int64_t)N, K, w16);
    LT_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_pad8, dim3(lt_grid(M * ld / 16, 256)), dim3(256), 0, stream, (const uint8_t*)x, M, K, x16);
    LT_LAUNCH_CHECK();
    w = w16;
    x = x16;
    ws = (char*)ws + pad;
    ws_bytes -= pad;
  }
  const bool direct = ld % 16 == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0 && ld * 256 < (int64_t)1 << 31;
  const LtPlan p = plan8(M, K, N, direct);
  LT_REQUIRE(part8(p, M, N) <= ws_bytes, LT_ERR_WORKSPACE, "lt_linear_mx8_fwd: workspace too small");
  LT_REQUIRE((int64_t)p.tr * p.tc * p.splits < (int64_t)1 << 22, LT_ERR_RANGE, "lt_linear_mx8_fwd: too many tiles");
  LtTile8Args b = {};
  b.t.P = (const char*)w;
  b.t.Q = (const char*)x;
  b.t.ldp = b.t.ldq = ld;
  b.t.rows = M;
  b.t.cols = N;
  b.t.depth = K;
  b.t.tr = p.tr;
  b.t.tc = p.tc;
  b.t.splits = p.splits;
  b.t.slice = p.slice;
  b.t.part = (float*)ws;
  b.t.ps = (const uint8_t*)w_scales;
  b.t.epi = LtEpi{bias, res, ldres, y, N, nullptr, LT_DERIV_NONE, M, N};
  b.qs = (const uint8_t*)x_scales;
  b.nb = (K + 31) / 32;
  return dt == LT_DT_BF16 ? lt_gemm8_launch<lt_bf16>(b, p, act, stream) : lt_gemm8_launch<lt_f16>(b, p, act, stream);
}
