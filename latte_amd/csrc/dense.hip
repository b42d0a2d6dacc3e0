// linear: y = act(x W^T + b) + r, its backward, and what the backward pass keeps in 8 bits.
//
//   forward    z = x W^T + b (fp32 sums);  y = act(z) + r;  kept: x (or mx8(x)), W, act'(z)
//   backward   dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum_rows dz;  dr = dy
// act' is kept instead of z: the ReLU's is one bit, the others fit a uniform grid (8 bits with a checkpoint, |error| <=
// 1/384; 16 bits beside 16-bit types, 1e-5), and the backward pass needs no exponential.  dz is rounded to the operands'
// type, as the matrix instructions take it.
//
// An nn.Linear for models built on this framework: the widths are those of the point branches and heads (latte/models/spvcnn.py:
// 95-111, latte/models/xmuda_arch.py:326-335).  Those layers themselves do not call it: a point branch has a BatchNorm behind its
// product, where no epilogue can stand, and the heads are gathered in head.hip.
#include "dense_plan.h"

template <> int lt_gemm_launch<float>(const LtGemm&, const LtPlan&, float*, hipStream_t);
template <> int lt_gemm_launch<lt_bf16>(const LtGemm&, const LtPlan&, float*, hipStream_t);
template <> int lt_gemm_launch<lt_f16>(const LtGemm&, const LtPlan&, float*, hipStream_t);
template <> int lt_rows_bwd_launch<float>(const LtRowsBwdArgs&, const LtRowsBwdPlan&, hipStream_t);
template <> int lt_rows_bwd_launch<lt_bf16>(const LtRowsBwdArgs&, const LtRowsBwdPlan&, hipStream_t);
template <> int lt_rows_bwd_launch<lt_f16>(const LtRowsBwdArgs&, const LtRowsBwdPlan&, hipStream_t);

static int64_t part_bytes(const LtPlan& p, int64_t rows, int cols) {
  return p.splits > 1 ? lt_align_up(p.splits * rows * cols * 4, 256) : 0;
}

// Lines whose length is no multiple of 16 bytes are staged through registers, in 128 x 128 tiles at most.  A large product is
// worth a copy of its operands with their lines filled up by zeros: whole pieces go straight into LDS.  TFLOP/s measured
// without and with (beside the copies): 16 bits forward 480 and 700, backward 240 and 700; fp32 backward 78 and 103, forward alike.
// 9000 x 1001 -> 4001 fp16: forward 150 us as it is, 129 with the copies, a training step 786 and 359; 3000 x
// 1001 -> 1003 fp16: 108 and 86.
static bool pad_pays(double products, double copied, int dt, double as_is, double filled) {
  const double gain = 2e-6 * products * (1 / as_is - 1 / filled);   // us
  return gain > 10 + 1e6 * copied * 2 * lt_dt_size(dt) / 3.5e12;    // two launches, a read and a write of `copied` elements
}
static int64_t up_to_16(int64_t n, int dt) {
  const int64_t ch = 16 / lt_dt_size(dt);
  return (n + ch - 1) / ch * ch;
}
static bool pad_fwd(int64_t M, int K, int N, int dt) {
  return dt != LT_DT_F32 && up_to_16(K, dt) != K && pad_pays((double)M * N * K, (double)(M + N) * K, dt, 480, 700);
}

// the larger of what the two staging paths want: which one runs depends on the operands' alignment
static int64_t gemm_ws_bytes(int64_t rows, int cols, int64_t depth, int dt, bool nn) {
  const int64_t a = part_bytes(lt_gemm_plan(rows, cols, depth, dt, nn, true), rows, cols);
  const int64_t b = part_bytes(lt_gemm_plan(rows, cols, depth, dt, nn, false), rows, cols);
  return a > b ? a : b;
}

// rows of n elements -> rows of ldo >= n, filled up with zeros.  HBM-bound; a thread takes eight neighbours.
template <class T>
__global__ __launch_bounds__(256) void k_pad(const T* __restrict__ x, int64_t ldx, int64_t M, int n, int ldo, T* __restrict__ out) {
  const int L = (ldo + 7) >> 3;
  const int64_t total = M * L, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += stride) {
    int64_t row;
    int l;
    lt_divmod(i, L, row, l);
    float v[8];
    lt_ldv<T, 8>(x + row * ldx + l * 8, n - l * 8, v);
    lt_stv<T, 8>(out + row * ldo + l * 8, ldo - l * 8, v);
  }
}
static int pad_run(const void* x, int64_t ldx, int64_t M, int n, int dt, void* out, hipStream_t stream) {
  const int ldo = (int)up_to_16(n, dt);
  LT_DENSE_TYPES(dt, hipLaunchKernelGGL((k_pad<T>), dim3(lt_grid(M * ((ldo + 7) >> 3), 256)), dim3(256), 0, stream, (const T*)x, ldx, M,
                                        n, ldo, (T*)out));
  LT_LAUNCH_CHECK();
  return LT_OK;
}

static int gemm_run(const LtGemm& g, void* ws, int64_t ws_bytes, hipStream_t stream) {
  const int sz = lt_dt_size(g.dt), ch = 16 / sz;
  auto aligned = [&](const void* p, int64_t ld, int64_t run, bool kmajor) {
    // whole 16-byte chunks along memory, and a tile's offsets within the 31 bits of a buffer descriptor
    return ((uintptr_t)p & 15) == 0 && ld * sz % 16 == 0 && (run % ch == 0 || g.padded) && (kmajor ? 64 : 256) * ld * sz < (int64_t)1 << 31;
  };
  const bool direct = !g.p_scales && aligned(g.P, g.ldp, g.p_kmajor ? g.cols : g.depth, g.p_kmajor) &&
                      aligned(g.Q, g.ldq, g.q_kmajor ? g.rows : g.depth, g.q_kmajor);
  const LtPlan p = lt_gemm_plan(g.rows, g.cols, g.depth, g.dt, !g.p_kmajor && !g.q_kmajor, direct);
  LT_REQUIRE(part_bytes(p, g.rows, g.cols) <= ws_bytes, LT_ERR_WORKSPACE, "linear: workspace too small (%lld bytes)",
             (long long)ws_bytes);
  LT_REQUIRE((int64_t)p.tr * p.tc * p.splits < (int64_t)1 << 22, LT_ERR_RANGE, "linear: too many tiles");
  LT_DENSE_TYPES(g.dt, return lt_gemm_launch<T>(g, p, (float*)ws, stream));
}

// ------------------------------------------------------------------ dz = dy act'(z) and its column sums
// HBM-bound: one pass over dy and act', dz written once (not at all without an activation, where dz is dy).  A thread owns
// four columns, a workgroup a slab of rows; the slabs' sums are joined in a fixed order by k_col_join.
template <class T, int DK>
__global__ __launch_bounds__(256) void k_dz(const T* __restrict__ dy, int64_t lddy, const void* __restrict__ deriv, int64_t M,
                                            int N, int lddz, int tx, int64_t rows_per, T* __restrict__ dz, T* __restrict__ dz2, float* __restrict__ part,
                                            T* __restrict__ db) {
  __shared__ lt_f32x4 s_sum[256];
  const int x = threadIdx.x % tx, yy = threadIdx.x / tx, ty = 256 / tx;
  const int col = (blockIdx.x * tx + x) * 4;
  const int n = N - col, nz = lddz - col;   // lddz > N: zeros behind the columns
  const int64_t r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < M ? r0 + rows_per : M;
  lt_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (nz > 0) {
#pragma unroll 4
    for (int64_t row = r0 + yy; row < r1; row += ty) {
      float g[4], d[4];
      lt_ldv<T, 4>(dy + row * lddy + col, n, g);
      if (n <= 0) {   // padding: g is 0
      } else if constexpr (DK == LT_DERIV_BITS) {
        const unsigned m = ((const uint16_t*)deriv)[row * ((N + 15) >> 4) + (col >> 4)] >> (col & 15);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = (m >> i) & 1 ? g[i] : 0.f;
      } else if constexpr (DK == LT_DERIV_BYTE) {
        const uint8_t* p = (const uint8_t*)deriv + row * N + col;
        uint8_t c[4] = {0, 0, 0, 0};
        if (n >= 4) __builtin_memcpy(c, p, 4);
        else
          for (int i = 0; i < n; ++i) c[i] = p[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] *= lt_deriv_value(c[i]);
      } else if constexpr (DK == LT_DERIV_FULL) {
        if constexpr (sizeof(T) == 4) lt_ldv<float, 4>((const float*)deriv + row * N + col, n, d);
        else {
          const uint16_t* p = (const uint16_t*)deriv + row * N + col;
          uint16_t c[4] = {0, 0, 0, 0};
          if (n >= 4) __builtin_memcpy(c, p, 8);
          else
            for (int i = 0; i < n; ++i) c[i] = p[i];
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = lt_deriv_word_value(c[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] *= d[i];
      }
      if (DK != LT_DERIV_NONE || dz) lt_stv<T, 4>(dz + row * lddz + col, nz, g);
      if constexpr (sizeof(T) == 2 && (DK == LT_DERIV_BYTE || DK == LT_DERIV_FULL)) {
        if (dz2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float t = (float)(T)g[i];
            d[i] = lt_finite_abs(t) == fabsf(t) ? g[i] - t : 0.f;   // an infinity has no rest (it would be NaN)
          }
          lt_stv<T, 4>(dz2 + row * lddz + col, nz, d);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += i < n ? g[i] : 0.f;
    }
  }
  if (!part) return;
  s_sum[threadIdx.x] = sum;
  __syncthreads();
  if (yy == 0 && n > 0) {
    for (int j = 1; j < ty; ++j) sum += s_sum[j * tx + x];
    const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (gridDim.y == 1) lt_stv<T, 4>(db + col, n, v);   // one slab: the sums are db
    else lt_stv<float, 4>(part + (int64_t)blockIdx.y * N + col, n, v);
  }
}

struct DzPlan {
  int tx, gx, slabs;
  int64_t rows_per;
};
static DzPlan dz_plan(int64_t M, int N) {
  DzPlan p;
  const int cg = (N + 3) / 4;
  p.tx = 1;
  while (p.tx < cg && p.tx < 64) p.tx <<= 1;
  p.gx = (cg + p.tx - 1) / p.tx;
  const int ty = 256 / p.tx;
  // 2048 workgroups (a training step with 256, 512, 1024, 2048, 4096 of them, us: 16384 x 1024 -> 4096 bf16 747, 630, 547, 531,
  // 529; 100000 x 300 -> 300 bf16 486, 399, 359, 333, 337)
  int64_t s = (2048 + p.gx - 1) / p.gx, most = (M + ty * 4 - 1) / (ty * 4);   // four rows a thread at least
  if (M <= ty * 16) most = 1;   // one slab is db: no join to launch (64 x 128 -> 128 bf16, a training step: 70.4 -> 66.0 us)
  if (s > most) s = most;
  if (s < 1) s = 1;
  p.rows_per = (M + s - 1) / s;
  if (p.rows_per < 1) p.rows_per = 1;
  p.slabs = (int)((M + p.rows_per - 1) / p.rows_per);
  return p;
}

template <class T>
static int dz_run(const void* dy, int64_t lddy, const void* deriv, int dkind, int64_t M, int N, int lddz, void* dz, void* dz2, float* part, void* db,
                  hipStream_t stream) {
  const DzPlan p = dz_plan(M, lddz);
  if (p.slabs > 0 && (part || dz)) {
    const dim3 grid(p.gx, p.slabs), block(256);
    const T* g = (const T*)dy;
    switch (dkind) {
      case LT_DERIV_BITS: hipLaunchKernelGGL((k_dz<T, LT_DERIV_BITS>), grid, block, 0, stream, g, lddy, deriv, M, N, lddz, p.tx, p.rows_per, (T*)dz, (T*)dz2, part, (T*)db); break;
      case LT_DERIV_BYTE: hipLaunchKernelGGL((k_dz<T, LT_DERIV_BYTE>), grid, block, 0, stream, g, lddy, deriv, M, N, lddz, p.tx, p.rows_per, (T*)dz, (T*)dz2, part, (T*)db); break;
      case LT_DERIV_FULL: hipLaunchKernelGGL((k_dz<T, LT_DERIV_FULL>), grid, block, 0, stream, g, lddy, deriv, M, N, lddz, p.tx, p.rows_per, (T*)dz, (T*)dz2, part, (T*)db); break;
      default: hipLaunchKernelGGL((k_dz<T, LT_DERIV_NONE>), grid, block, 0, stream, g, lddy, deriv, M, N, lddz, p.tx, p.rows_per, (T*)dz, (T*)dz2, part, (T*)db); break;
    }
    LT_LAUNCH_CHECK();
  }
  if (db && p.slabs != 1) {
    hipLaunchKernelGGL((k_col_join<T>), dim3((N + 15) / 16), dim3(256), 0, stream, part, p.slabs, N, (T*)db);
    LT_LAUNCH_CHECK();
  }
  return LT_OK;
}

// ------------------------------------------------------------------ mx8 (layout and rounding: dense.h)
// HBM-bound, one pass: a lane holds 8 neighbours, four lanes a block of 32.
template <class T>
__global__ __launch_bounds__(256) void k_mx8_quantize(const T* __restrict__ x, int64_t ldx, int64_t M, int K,
                                                      uint8_t* __restrict__ q, uint8_t* __restrict__ sc) {
  const int nb = (K + 31) >> 5, L = nb * 4;
  const int64_t n = M * L, stride = (int64_t)gridDim.x * 256;
  for (int64_t b = blockIdx.x * (int64_t)256; b < n; b += stride) {
    const int64_t i = b + threadIdx.x;
    int64_t row = 0;
    int l = 0;
    const bool live = i < n;
    if (live) lt_divmod(i, L, row, l);
    const int col = l * 8;
    float v[8];
    lt_ldv<T, 8>(x + row * ldx + col, live ? K - col : 0, v);
    lt_mx8_put8(v, live ? K - col : 0, LtType<T>::kMaxExp, q + row * K + col, sc + row * nb + (l >> 2));
  }
}

template <class T>
__global__ __launch_bounds__(256) void k_mx8_dequantize(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc, int64_t M,
                                                        int K, int ldo, T* __restrict__ out) {
  const int nb = (K + 31) >> 5, L = nb * 4;
  const int64_t n = M * L, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += stride) {
    int64_t row;
    int l;
    lt_divmod(i, L, row, l);
    const int col = l * 8, m = K - col;
    if (m <= 0) continue;
    float v[8];
    lt_mx8_get8(q + row * K + col, m, sc[row * nb + (l >> 2)], v);
    lt_stv<T, 8>(out + row * ldo + col, ldo - col, v);   // ldo > K: zeros behind the row
  }
}

// ------------------------------------------------------------------ the C entry points
static int check_dense(const char* who, int64_t M, int64_t K, int64_t N, int dt) {
  LT_REQUIRE(dt == LT_DT_F32 || dt == LT_DT_BF16 || dt == LT_DT_F16, LT_ERR_ARG, "%s: type %d is none of LT_DT_*", who, dt);
  LT_REQUIRE(M >= 0 && K >= 1 && N >= 1 && K <= INT32_MAX - 1024 && N <= INT32_MAX - 1024, LT_ERR_ARG,
             "%s: bad sizes M=%lld K=%lld N=%lld", who, (long long)M, (long long)K, (long long)N);
  const int64_t most = (int64_t)1 << 42;   // elements: more than any memory holds, and byte counts stay within 64 bits
  LT_REQUIRE(M <= most / (K > N ? K : N) && K <= most / N, LT_ERR_RANGE, "%s: M=%lld K=%lld N=%lld is too large", who, (long long)M,
             (long long)K, (long long)N);
  return LT_OK;
}

extern "C" int lt_mx8_quantize(const void* x, int64_t ldx, int64_t M, int32_t K, int32_t dt, void* values, void* scales,
                               hipStream_t stream) {
  int rc = check_dense("lt_mx8_quantize", M, K, 1, dt);
  if (rc) return rc;
  if (M == 0) return LT_OK;
  LT_REQUIRE(x && values && scales, LT_ERR_ARG, "lt_mx8_quantize: null pointer");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  const int64_t n = M * (int64_t)((K + 31) / 32 * 4);
  LT_DENSE_TYPES(dt, hipLaunchKernelGGL((k_mx8_quantize<T>), dim3(lt_grid(n, 256)), dim3(256), 0, stream, (const T*)x, ldx, M, K,
                                        (uint8_t*)values, (uint8_t*)scales));
  LT_LAUNCH_CHECK();
  return LT_OK;
}

static int dequantize_run(const void* values, const void* scales, int64_t M, int K, int ldo, int dt, void* out, hipStream_t stream) {
  const int64_t n = M * (int64_t)((K + 31) / 32 * 4);
  LT_DENSE_TYPES(dt, hipLaunchKernelGGL((k_mx8_dequantize<T>), dim3(lt_grid(n, 256)), dim3(256), 0, stream, (const uint8_t*)values,
                                        (const uint8_t*)scales, M, K, ldo, (T*)out));
  LT_LAUNCH_CHECK();
  return LT_OK;
}

extern "C" int lt_mx8_dequantize(const void* values, const void* scales, int64_t M, int32_t K, int32_t dt, void* out,
                                 hipStream_t stream) {
  int rc = check_dense("lt_mx8_dequantize", M, K, 1, dt);
  if (rc) return rc;
  if (M == 0) return LT_OK;
  LT_REQUIRE(out && values && scales, LT_ERR_ARG, "lt_mx8_dequantize: null pointer");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  return dequantize_run(values, scales, M, K, K, dt, out, stream);
}

extern "C" int64_t lt_linear_workspace_bytes(int64_t M, int32_t K, int32_t N, int32_t dt) {
  if (check_dense("lt_linear_workspace_bytes", M, K, N, dt)) return -1;
  const int64_t pad = pad_fwd(M, K, N, dt) ? lt_align_up((M + N) * up_to_16(K, dt) * lt_dt_size(dt), 256) : 0;
  return pad + gemm_ws_bytes(M, N, K, dt, true);
}

extern "C" int lt_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res,
                             int64_t ldres, int32_t act, int64_t M, int32_t K, int32_t N, int32_t dt, void* y, void* deriv,
                             int32_t deriv_kind, void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check_dense("lt_linear_fwd", M, K, N, dt);
  if (rc) return rc;
  LT_REQUIRE(act >= LT_ACT_NONE && act <= LT_ACT_SILU, LT_ERR_ARG, "lt_linear_fwd: act=%d is none of LT_ACT_*", act);
  LT_REQUIRE(deriv_kind == LT_DERIV_NONE || (deriv_kind == LT_DERIV_BITS && act == LT_ACT_RELU) ||
                 ((deriv_kind == LT_DERIV_BYTE || deriv_kind == LT_DERIV_FULL) && act >= LT_ACT_GELU),
             LT_ERR_ARG, "lt_linear_fwd: deriv_kind=%d does not go with act=%d", deriv_kind, act);
  if (M == 0) return LT_OK;
  LT_REQUIRE(x && w && y && (deriv_kind == LT_DERIV_NONE || deriv), LT_ERR_ARG, "lt_linear_fwd: null pointer");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  LtGemm g = {};
  g.P = w;
  g.ldp = ldw;
  g.Q = x;
  g.ldq = ldx;
  g.rows = M;
  g.cols = N;
  g.depth = K;
  g.dt = dt;
  g.act = act;
  g.epi = LtEpi{bias, res, ldres, y, N, deriv, deriv_kind, M, N};
  ws_bytes = ws ? ws_bytes : 0;
  if (pad_fwd(M, K, N, dt)) {
    const int64_t K8 = up_to_16(K, dt), row = K8 * lt_dt_size(dt), pad = lt_align_up((M + N) * row, 256);
    LT_REQUIRE(pad <= ws_bytes, LT_ERR_WORKSPACE, "lt_linear_fwd: workspace too small (%lld bytes)", (long long)ws_bytes);
    if ((rc = pad_run(w, ldw, N, K, dt, ws, stream)) || (rc = pad_run(x, ldx, M, K, dt, (char*)ws + N * row, stream))) return rc;
    g.P = ws;
    g.Q = (char*)ws + N * row;
    g.ldp = g.ldq = K8;
    g.padded = true;
    ws = (char*)ws + pad;
    ws_bytes -= pad;
  }
  return gemm_run(g, ws, ws_bytes, stream);
}

// dW = dz^T x with x in mx8: up to 256 output columns the product widens x while it stages it (x is read once or twice);
// wider layers would do that once per column tile and without direct staging, so x is widened into the workspace first.
// 16384 x 1024 -> 4096, bf16: a training step 1130 us with the widening in the staging, 696 us with it first
static bool widen_first(int64_t M, int K, int N) { return N > 256 && M > 0; }

// dz beside 16-bit types is rounded for the matrix instructions.  Among thousands of elements that adds as much variance
// to a gradient as its own last rounding does; a handful can have bad luck, so a small dz goes in as two terms, itself and
// what its rounding left (the products are launch-bound there).
static bool two_terms(int64_t M, int N, int dt) { return dt != LT_DT_F32 && M * N <= 4096; }

// the backward pass's dz, x and W with their lines filled up (dz comes that way at no cost where there is an act')
static bool pad_bwd(int64_t M, int K, int N, int dt, bool has_act) {
  const bool k = up_to_16(K, dt) != K, n = up_to_16(N, dt) != N;
  return (k || n) && pad_pays(2.0 * M * N * K, (k ? (double)(M + N) * K : 0.0) + (n && !has_act ? (double)M * N : 0.0), dt,
                              dt == LT_DT_F32 ? 78 : 240, dt == LT_DT_F32 ? 103 : 700);
}

struct BwdWs {
  int64_t dz, dz2, part, wide, w, gemm, bytes;
};
// the larger of the two routes: one pass over the rows, or dz and two products
static BwdWs bwd_ws(int64_t M, int K, int N, int dt, bool x8) {
  BwdWs w;
  int64_t off = 0;
  const LtRowsBwdPlan p = lt_rows_bwd_plan(M, K, N, dt);
  const bool pad = !p.ok && pad_bwd(M, K, N, dt, true);   // with an act' more often than without
  const int64_t N8 = p.ok ? (N + 7) / 8 * 8 : pad ? up_to_16(N, dt) : N, K8 = pad ? up_to_16(K, dt) : K;
  w.dz = off;
  off += lt_align_up(M * N8 * lt_dt_size(dt), 256);
  w.dz2 = off;   // the second term has the first one's rows, their filled-up ends among them
  off += two_terms(M, N, dt) ? lt_align_up(M * N8 * lt_dt_size(dt), 256) : 0;
  w.part = off;
  const int64_t s = dz_plan(M, N).slabs, s8 = dz_plan(M, (int)N8).slabs;
  off += lt_align_up((s > s8 ? s : s8) * N * 4, 256);
  w.wide = off;
  if ((x8 && (widen_first(M, K, N) || pad)) || K8 != K) off += lt_align_up(M * K8 * lt_dt_size(dt), 256);
  w.w = off;
  if (K8 != K) off += lt_align_up(N * K8 * lt_dt_size(dt), 256);
  w.gemm = off;
  const int64_t a = gemm_ws_bytes(M, K, N, dt, false), b = gemm_ws_bytes(N, K, M, dt, false);
  off += a > b ? a : b;
  const int64_t rows = p.ok ? w.gemm + lt_align_up((int64_t)p.grid * N * K * 4, 256) + (int64_t)p.grid * N * 4 : 0;
  w.bytes = off > rows ? off : rows;
  return w;
}

extern "C" int64_t lt_linear_bwd_workspace_bytes(int64_t M, int32_t K, int32_t N, int32_t dt, int32_t x_mx8) {
  if (check_dense("lt_linear_bwd_workspace_bytes", M, K, N, dt)) return -1;
  return bwd_ws(M, K, N, dt, x_mx8 != 0).bytes;
}

extern "C" int lt_linear_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* x_scales, const void* w,
                             int64_t ldw, const void* deriv, int32_t deriv_kind, int64_t M, int32_t K, int32_t N, int32_t dt,
                             void* dx, void* dw, void* db, void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check_dense("lt_linear_bwd", M, K, N, dt);
  if (rc) return rc;
  LT_REQUIRE(deriv_kind >= LT_DERIV_NONE && deriv_kind <= LT_DERIV_FULL, LT_ERR_ARG, "lt_linear_bwd: deriv_kind=%d", deriv_kind);
  LT_REQUIRE(!x_scales || ldx == K, LT_ERR_ARG, "lt_linear_bwd: an mx8 x has rows of K values, not ldx=%lld", (long long)ldx);
  const BwdWs o = bwd_ws(M, K, N, dt, x_scales != nullptr);
  LT_REQUIRE(ws_bytes >= o.bytes && (ws || o.bytes == 0), LT_ERR_WORKSPACE, "lt_linear_bwd: workspace too small");
  if (M > 0)
    LT_REQUIRE(dy && (deriv_kind == LT_DERIV_NONE || deriv) && (!dx || w) && (!dw || x), LT_ERR_ARG, "lt_linear_bwd: null pointer");
  LtOnStream on;
  if ((rc = on.enter(stream))) return rc;
  char* wsb = (char*)ws;
  const LtRowsBwdPlan rp = lt_rows_bwd_plan(M, K, N, dt);
  if (rp.ok) {   // whichever gradients are asked for: each has the same bits alone as with the others
    float* part_w = (float*)(wsb + o.gemm);
    float* part_b = (float*)(wsb + o.gemm + lt_align_up((int64_t)rp.grid * N * K * 4, 256));
    LtRowsBwdArgs a = {dy, x, (const uint8_t*)x_scales, w, deriv, lddy, ldx, ldw, deriv_kind, M, N, K, N, dx, dw ? part_w : nullptr,
                       db ? part_b : nullptr};
    if (N % 8) {   // odd widths (class counts): dz and db in a pass of their own, with whole chunks for this one
      const int N8 = (N + 7) / 8 * 8;
      LT_DENSE_TYPES(dt, rc = dz_run<T>(dy, lddy, deriv, deriv_kind, M, N, N8, wsb + o.dz, nullptr, db ? (float*)(wsb + o.part) : nullptr, db, stream));
      if (rc) return rc;
      a.dy = wsb + o.dz;
      a.lddy = a.N = N8;
      a.dkind = LT_DERIV_NONE;
      a.db = nullptr;
      db = nullptr;
      if (!dx && !dw) return LT_OK;
    }
    LT_DENSE_TYPES(dt, rc = lt_rows_bwd_launch<T>(a, rp, stream));
    if (rc) return rc;
    if (dw) {
      const LtEpi e = {nullptr, nullptr, 0, dw, K, nullptr, LT_DERIV_NONE, N, K};
      LT_DENSE_TYPES(dt, rc = lt_launch_join<T, LT_ACT_NONE>(e, part_w, rp.grid, stream));
      if (rc) return rc;
    }
    if (db) {
      LT_DENSE_TYPES(dt, hipLaunchKernelGGL((k_col_join<T>), dim3((N + 15) / 16), dim3(256), 0, stream, part_b, rp.grid, N, (T*)db));
      LT_LAUNCH_CHECK();
    }
    return LT_OK;
  }
  const bool pad = pad_bwd(M, K, N, dt, deriv_kind != LT_DERIV_NONE);
  const int N8 = pad ? (int)up_to_16(N, dt) : N, K8 = pad ? (int)up_to_16(K, dt) : K;
  const void* dz = dy;
  int64_t lddz = lddy;
  const bool own_dz = deriv_kind != LT_DERIV_NONE || N8 != N;
  if (own_dz) {
    dz = wsb + o.dz;
    lddz = N8;
  }
  void* dz2 = two_terms(M, N, dt) && (deriv_kind == LT_DERIV_BYTE || deriv_kind == LT_DERIV_FULL) ? wsb + o.dz2 : nullptr;
  LT_DENSE_TYPES(dt, rc = dz_run<T>(dy, lddy, deriv, deriv_kind, M, N, N8, own_dz ? wsb + o.dz : nullptr, dz2, db ? (float*)(wsb + o.part) : nullptr, db, stream));
  if (rc) return rc;
  LtGemm g = {};
  g.dt = dt;
  g.act = LT_ACT_NONE;
  g.Q2 = dz2;
  g.padded = pad;
  if (dx && M > 0) {
    g.P = w;
    g.ldp = ldw;
    if (K8 != K) {
      if ((rc = pad_run(w, ldw, N, K, dt, wsb + o.w, stream))) return rc;
      g.P = wsb + o.w;
      g.ldp = K8;
    }
    g.p_kmajor = true;
    g.Q = dz;
    g.ldq = lddz;
    g.rows = M;
    g.cols = K;
    g.depth = N;
    g.epi = LtEpi{nullptr, nullptr, 0, dx, K, nullptr, LT_DERIV_NONE, M, K};
    if ((rc = gemm_run(g, wsb + o.gemm, ws_bytes - o.gemm, stream))) return rc;
  }
  if (dw) {
    g.P = x;
    g.ldp = ldx;
    g.p_kmajor = true;
    g.p_scales = (const uint8_t*)x_scales;
    if (x_scales && (widen_first(M, K, N) || pad)) {
      if ((rc = dequantize_run(x, x_scales, M, K, K8, dt, wsb + o.wide, stream))) return rc;
      g.P = wsb + o.wide;
      g.ldp = K8;
      g.p_scales = nullptr;
    } else if (K8 != K) {
      if ((rc = pad_run(x, ldx, M, K, dt, wsb + o.wide, stream))) return rc;
      g.P = wsb + o.wide;
      g.ldp = K8;
    }
    g.Q = dz;
    g.ldq = lddz;
    g.q_kmajor = true;
    g.rows = N;
    g.cols = K;
    g.depth = M;
    g.epi = LtEpi{nullptr, nullptr, 0, dw, K, nullptr, LT_DERIV_NONE, N, K};
    if ((rc = gemm_run(g, wsb + o.gemm, ws_bytes - o.gemm, stream))) return rc;
  }
  return LT_OK;
}
