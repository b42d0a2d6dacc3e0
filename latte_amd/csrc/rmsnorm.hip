// rms_norm: h = x + r;  n = h / sqrt(mean_c h^2 + eps);  y = n w, in the operands' type or in mx8; and its backward
//   g = dy w;  dx = dr = rstd (g - n mean_c(g n)) + dh;  dw = sum_rows dy n.
// A norm over the row alone: no batch statistics, so a batch of one scan (or one row) is normalised like any other, and
// nothing is exchanged between ranks -- beside the BatchNorm of latte/models/basic_blocks.py:22-75, which needs both.
//
// HBM-bound, one pass: LANES lanes hold a row in registers (8 neighbours a lane and turn), so the sum of squares, the
// normalised row and its 8-bit form need no second read; workgroups stride over the rows with w in registers.  h is summed
// in fp32 and enters the norm unrounded; the backward pass reads h from fp32 or mx8, or adds x and r again beside 16-bit types
// (the rounded h would add as much variance to dw as dw's own rounding does; one more read of five).
#include "dense.h"

struct LtRmsArgs {
  const void* x;
  const void* res;
  const void* w;
  int64_t ldx, ldres, M;
  int C;
  float eps;
  void* h;            // [M][C] or NULL
  void* y;            // [M][C] or NULL
  uint8_t *y8, *y8s;  // y in mx8, or NULL
  uint8_t *h8, *h8s;  // h in mx8, or NULL
  float* rstd;        // [M] or NULL
};

// sum over the LANES lanes of a row, the same bits in each of them
template <int LANES, class F>
__device__ __forceinline__ F row_sum(F v, F* s_red) {
#pragma unroll
  for (int o = 1; o < (LANES < 64 ? LANES : 64); o <<= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LANES == 256) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
  }
  return v;
}

// y + c (|c| of a few last places of y) to fp32 with the last bit set where anything is left out: rounding that once more to 4
// bits is rounding y + c itself.  NaN and infinite parts change nothing.
__device__ __forceinline__ float round_odd(float y, float c) {
#pragma clang fp contract(off)   // y is a product and c the rest of it: fused with one another they would count twice
  const float f = y + c, e = c - (f - y);
  unsigned b = __float_as_uint(f);
  const unsigned by = (e > 0.f) == !(b >> 31) ? 1u : ~0u;
  b += (e > 0.f || e < 0.f) && !(b & 1u) ? by : 0u;
  return __uint_as_float(b);
}

template <class T, int LANES, int ITEMS>
__global__ __launch_bounds__(256) void k_rms_fwd(LtRmsArgs a) {
  __shared__ float s_red[4];
  __shared__ double s_redd[4];
  constexpr int RPB = 256 / LANES;
  const int l = threadIdx.x % LANES, nb = (a.C + 31) >> 5;
  float w[ITEMS][8];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int col = (it * LANES + l) * 8;
    lt_ldv<T, 8>((const T*)a.w + col, a.C - col, w[it]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.M; r0 += (int64_t)gridDim.x * RPB) {   // uniform: all lanes of a row sum
    const int64_t row = r0 + threadIdx.x / LANES;
    const bool live = row < a.M;
    float h[ITEMS][8], ss = 0.f;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * LANES + l) * 8;
      lt_ldv<T, 8>((const T*)a.x + row * a.ldx + col, live ? a.C - col : 0, h[it]);
      if (a.res) {
        float r[8];
        lt_ldv<T, 8>((const T*)a.res + row * a.ldres + col, live ? a.C - col : 0, r);
#pragma unroll
        for (int t = 0; t < 8; ++t) h[it][t] += r[t];
      }
    }
    // y that is held in 8 bits comes from a 64-bit sum and from products with their rounding errors carried along: the last
    // bit of an fp32 y would decide between two neighbours some 2^-4 apart once in a million elements (8192 x 4096 bf16: 48 us
    // in plain fp32, 49 us this way)
    float rstd, rhi = 0.f, rlo = 0.f;
    if (a.y8) {
      double s8 = 0.0;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
#pragma unroll
        for (int t = 0; t < 8; ++t) s8 = fma((double)h[it][t], (double)h[it][t], s8);
      const double r8 = 1.0 / sqrt(row_sum<LANES, double>(s8, s_redd) / (double)a.C + (double)a.eps);
      rstd = rhi = (float)r8;
      rlo = (float)(r8 - (double)rhi);
    } else {
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
#pragma unroll
        for (int t = 0; t < 8; ++t) ss = __fmaf_rn(h[it][t], h[it][t], ss);
      ss = row_sum<LANES, float>(ss, s_red);
      rstd = 1.f / sqrtf(ss / (float)a.C + a.eps);
    }
    if (a.rstd && l == 0 && live) a.rstd[row] = rstd;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * LANES + l) * 8, n = live ? a.C - col : 0;
      const int64_t at = row * a.C + col;
      if (a.h) lt_stv<T, 8>((T*)a.h + at, n, h[it]);
      if (a.h8) lt_mx8_put8(h[it], n, 127, a.h8 + at, a.h8s + row * nb + (col >> 5));   // read back in 32 bits
      float y[8];
      if (a.y) {
#pragma unroll
        for (int t = 0; t < 8; ++t) y[t] = h[it][t] * rstd * w[it][t];
        lt_stv<T, 8>((T*)a.y + at, n, y);
      }
      if (a.y8) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float n1 = h[it][t] * rhi, n2 = __fmaf_rn(h[it][t], rlo, __fmaf_rn(h[it][t], rhi, -n1));
          const float y1 = n1 * w[it][t];
          y[t] = round_odd(y1, __fmaf_rn(n2, w[it][t], __fmaf_rn(n1, w[it][t], -y1)));
        }
        lt_mx8_put8(y, n, LtType<T>::kMaxExp, a.y8 + at, a.y8s + row * nb + (col >> 5));
      }
    }
  }
}

struct LtRmsBwdArgs {
  const void* dy;
  const void* dh;            // or NULL
  const void* h;             // [M][ldh], or NULL when h8 is there
  const void* h2;            // or NULL: the second summand, h + h2 is the row that was normalised
  const uint8_t *h8, *h8s;
  const void* w;
  const float* rstd;
  int64_t lddy, lddh, ldh, ldh2, M;
  int C;
  void* dx;                  // or NULL
  float* part;               // [grid][C] column sums of dy n, or NULL
};

template <class T, int LANES, int ITEMS>
__global__ __launch_bounds__(256) void k_rms_bwd(LtRmsBwdArgs a) {
  constexpr int RPB = 256 / LANES;
  __shared__ float s_red[4];
  __shared__ float s_dw[RPB > 1 ? RPB * LANES * ITEMS * 8 : 1];
  const int l = threadIdx.x % LANES, nb = (a.C + 31) >> 5;
  float w[ITEMS][8], dw[ITEMS][8];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int col = (it * LANES + l) * 8;
    lt_ldv<T, 8>((const T*)a.w + col, a.C - col, w[it]);
#pragma unroll
    for (int t = 0; t < 8; ++t) dw[it][t] = 0.f;
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.M; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / LANES;
    const bool live = row < a.M;
    const float rstd = live ? a.rstd[row] : 0.f;
    float g[ITEMS][8], n[ITEMS][8], dot = 0.f;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * LANES + l) * 8, m = live ? a.C - col : 0;
      lt_ldv<T, 8>((const T*)a.dy + row * a.lddy + col, m, g[it]);
      if (a.h8) {
        if (m > 0) lt_mx8_get8(a.h8 + row * a.C + col, m, a.h8s[row * nb + (col >> 5)], n[it]);
        else
#pragma unroll
          for (int t = 0; t < 8; ++t) n[it][t] = 0.f;
      } else {
        lt_ldv<T, 8>((const T*)a.h + row * a.ldh + col, m, n[it]);
        if (a.h2) {
          float v[8];
          lt_ldv<T, 8>((const T*)a.h2 + row * a.ldh2 + col, m, v);
#pragma unroll
          for (int t = 0; t < 8; ++t) n[it][t] += v[t];
        }
      }
    }
#pragma unroll
    for (int it = 0; it < ITEMS; ++it)
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        n[it][t] *= rstd;
        dw[it][t] = __fmaf_rn(g[it][t], n[it][t], dw[it][t]);
        g[it][t] *= w[it][t];
        dot = __fmaf_rn(g[it][t], n[it][t], dot);
      }
    dot = row_sum<LANES, float>(dot, s_red) / (float)a.C;
    if (!a.dx) continue;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * LANES + l) * 8, m = live ? a.C - col : 0;
      float o[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) o[t] = rstd * (g[it][t] - n[it][t] * dot);
      if (a.dh) {
        float d[8];
        lt_ldv<T, 8>((const T*)a.dh + row * a.lddh + col, m, d);
#pragma unroll
        for (int t = 0; t < 8; ++t) o[t] += d[t];
      }
      lt_stv<T, 8>((T*)a.dx + row * a.C + col, m, o);
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * a.C;
  if constexpr (RPB > 1) {   // the rows' lanes add up in row order
#pragma unroll
    for (int it = 0; it < ITEMS; ++it)
#pragma unroll
      for (int t = 0; t < 8; ++t) s_dw[(threadIdx.x / LANES) * (LANES * ITEMS * 8) + (it * LANES + l) * 8 + t] = dw[it][t];
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += 256) {
      float s = 0.f;
#pragma unroll 8
      for (int r = 0; r < RPB; ++r) s += s_dw[r * (LANES * ITEMS * 8) + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * LANES + l) * 8;
      lt_stv<float, 8>(out + col, a.C - col, dw[it]);
    }
  }
}

// ------------------------------------------------------------------ host
// lanes per row: the row fits 8 neighbours a lane as far as it can, a wave from 264 columns on, a workgroup from 2056 on (forward
// with a residual, bf16, 8192 rows, a wave and a workgroup a row, us: 1024 columns 15.5 and 16.3, 2048 columns 30.7 and 21.9)
static int rms_lanes(int C) {
  if (C > 2048) return 256;
  int l = 4;
  while (l < 64 && l * 8 < C) l <<= 1;
  return l;
}
static int rms_bwd_grid(int64_t M, int C) {
  const int64_t rpb = 256 / rms_lanes(C);
  int64_t g = (M + rpb * 4 - 1) / (rpb * 4);   // four rows a lane group at least, so that the column sums stay few
  // trained with at most 256, 512, 1024, 2048, 4096 workgroups, us: 8192 x 4096 bf16 174, 129, 112, 126, 127; 34816 x 256 fp32 48, 47,
  // 47, 50, 50.  Rows a lane group at least, 1, 4 and 16: 2000 x 256 fp32 12, 13 and 21; 8192 x 4096 bf16 112, 115 and 130
  if (g > 1024) g = 1024;
  return (int)(g < 1 ? 1 : g);
}

template <class T, template <class, int, int> class Launch, class Args>
static void rms_dispatch(int C, const Args& a, int grid, hipStream_t stream) {
  const int l = rms_lanes(C), items = (C + l * 8 - 1) / (l * 8);
  if (l == 4) Launch<T, 4, 1>::go(a, grid, stream);
  else if (l == 8) Launch<T, 8, 1>::go(a, grid, stream);
  else if (l == 16) Launch<T, 16, 1>::go(a, grid, stream);
  else if (l == 32) Launch<T, 32, 1>::go(a, grid, stream);
  else if (l == 64) {
    if (items == 1) Launch<T, 64, 1>::go(a, grid, stream);
    else if (items == 2) Launch<T, 64, 2>::go(a, grid, stream);
    else Launch<T, 64, 4>::go(a, grid, stream);
  } else if (items == 2) Launch<T, 256, 2>::go(a, grid, stream);
  else if (items <= 4) Launch<T, 256, 4>::go(a, grid, stream);
  else Launch<T, 256, 8>::go(a, grid, stream);
}
template <class T, int L, int I> struct RmsFwdLaunch {
  static void go(const LtRmsArgs& a, int grid, hipStream_t s) { hipLaunchKernelGGL((k_rms_fwd<T, L, I>), dim3(grid), dim3(256), 0, s, a); }
};
template <class T, int L, int I> struct RmsBwdLaunch {
  static void go(const LtRmsBwdArgs& a, int grid, hipStream_t s) { hipLaunchKernelGGL((k_rms_bwd<T, L, I>), dim3(grid), dim3(256), 0, s, a); }
};

#define LT_RMS_MAX_C 16384
static int check_rms(const char* who, int64_t M, int32_t C, int32_t dt) {
  LT_REQUIRE(dt == LT_DT_F32 || dt == LT_DT_BF16 || dt == LT_DT_F16, LT_ERR_ARG, "%s: type %d is none of LT_DT_*", who, dt);
  LT_REQUIRE(M >= 0 && M <= (int64_t)1 << 40 && C >= 1, LT_ERR_ARG, "%s: bad sizes M=%lld C=%d", who, (long long)M, C);
  LT_REQUIRE(C <= LT_RMS_MAX_C, LT_ERR_RANGE, "%s: C=%d, at most %d columns", who, C, LT_RMS_MAX_C);
  return LT_OK;
}

extern "C" int lt_rms_norm_fwd(const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w, float eps, int64_t M,
                               int32_t C, int32_t dt, void* h, void* y, void* y8, void* y8_scales, void* h8, void* h8_scales,
                               float* rstd, hipStream_t stream) {
  int rc = check_rms("lt_rms_norm_fwd", M, C, dt);
  if (rc) return rc;
  if (M == 0) return LT_OK;
  LT_REQUIRE(x && w && (y || y8) && (!y8 || y8_scales) && (!h8 || h8_scales), LT_ERR_ARG, "lt_rms_norm_fwd: null pointer");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  const LtRmsArgs a = {x, res, w, ldx, ldres, M, C, eps, h, y, (uint8_t*)y8, (uint8_t*)y8_scales, (uint8_t*)h8, (uint8_t*)h8_scales, rstd};
  const int64_t rpb = 256 / rms_lanes(C);
  int64_t g = (M + rpb - 1) / rpb;
  if (g > 4096) g = 4096;   // 8192 x 4096 bf16 with 512, 1024, 4096, 16384: 56, 43.6, 44.1, 47.2 us
  LT_DENSE_TYPES(dt, rms_dispatch<T, RmsFwdLaunch>(C, a, (int)g, stream));
  LT_LAUNCH_CHECK();
  return LT_OK;
}

extern "C" int64_t lt_rms_norm_bwd_workspace_bytes(int64_t M, int32_t C) {
  if (check_rms("lt_rms_norm_bwd_workspace_bytes", M, C, LT_DT_F32)) return -1;
  return (int64_t)rms_bwd_grid(M, C) * C * 4;
}

extern "C" int lt_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh,
                               const void* h2, int64_t ldh2, const void* h8, const void* h8_scales, const void* w, const float* rstd, int64_t M, int32_t C,
                               int32_t dt, void* dx, void* dw, void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check_rms("lt_rms_norm_bwd", M, C, dt);
  if (rc) return rc;
  const int grid = M > 0 ? rms_bwd_grid(M, C) : 0;
  LT_REQUIRE(!dw || (int64_t)grid * C * 4 <= ws_bytes, LT_ERR_WORKSPACE, "lt_rms_norm_bwd: workspace too small");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  if (M > 0) {
    LT_REQUIRE(dy && w && rstd && (h || (h8 && h8_scales)) && (!dw || ws), LT_ERR_ARG, "lt_rms_norm_bwd: null pointer");
    const LtRmsBwdArgs a = {dy, dh, h, h2, (const uint8_t*)h8, (const uint8_t*)h8_scales, w, rstd, lddy, lddh, ldh, ldh2, M, C, dx,
                            dw ? (float*)ws : nullptr};
    LT_DENSE_TYPES(dt, rms_dispatch<T, RmsBwdLaunch>(C, a, grid, stream));
    LT_LAUNCH_CHECK();
  }
  if (dw) {
    LT_DENSE_TYPES(dt, hipLaunchKernelGGL((k_col_join<T>), dim3((C + 15) / 16), dim3(256), 0, stream, (const float*)ws, grid, C, (T*)dw));
    LT_LAUNCH_CHECK();
  }
  return LT_OK;
}
