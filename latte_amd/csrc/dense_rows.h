// Long and narrow layers (a few hundred channels, many rows: layers over all points): forward and backward in one pass over
// the rows.  Tiles would pad 96 columns to 128 and read dz and x once per product; here W stays in LDS for the whole launch,
// in fragment order, and rows stream past it.
#pragma once
#include "dense_gemm.h"

// ------------------------------------------------------------------ forward
// A wave takes strips of 16 rows: its x fragments come straight from memory (a strip ahead), W's from LDS, no barriers.
//   310017 x 128 -> 96 + residual, fp32: 103 us (3.9 TB/s; 145 on tiles); bf16: 38 us (5.2 TB/s)
template <class T, int KC, int FC, int ACT>
__global__ __launch_bounds__(512) void k_rows_fwd(LtTileArgs a) {
  typedef typename LtMma<T>::frag Frag;
  constexpr int CH = 16 / sizeof(T), KF = 4 * CH;
  extern __shared__ __attribute__((aligned(1024))) char s_tile[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (a.cols + 16 * FC - 1) / (16 * FC), NT = groups * FC;
  const int K = (int)a.depth;   // a multiple of CH: a lane's chunk is all there or not at all
  auto get = [&](const T* line, bool ok, int k) -> Frag {   // no branches: what is not there is read elsewhere and cleared
    Frag v;
    ok = ok && k < K;
    __builtin_memcpy(&v, line + (k < K ? k : 0), 16);
    if (!ok) v = Frag{};
    return v;
  };
  for (int f = tid; f < KC * NT * 64; f += 512) {   // fragment (kk, c) of W: lane (r, g) holds row 16 c + r, k = kk KF + g CH ..
    const int l = f & 63, c = (f >> 6) % NT, kk = (f >> 6) / NT, n = 16 * c + (l & 15);
    const bool ok = n < a.cols;
    const Frag v = get((const T*)(a.P + (int64_t)(ok ? n : 0) * a.ldp), ok, kk * KF + (l >> 4) * CH);
    *reinterpret_cast<Frag*>(s_tile + f * 16) = v;
  }
  __syncthreads();
  float* turn = reinterpret_cast<float*>(s_tile + KC * NT * 1024 + wave * LtTurn<FC>::BYTES);
  const int64_t strips = (a.rows + 15) >> 4, step = (int64_t)gridDim.x * 8;
  Frag x[KC], nx[KC];
  auto fetch = [&](int64_t s) {
    const int64_t row = s * 16 + r;
    const bool ok = row < a.rows;
    const T* line = (const T*)(a.Q + (ok ? row : 0) * a.ldq);
#pragma unroll
    for (int kk = 0; kk < KC; ++kk) nx[kk] = get(line, true, kk * KF + g * CH);   // rows past the end are not stored
  };
  int64_t s = (int64_t)blockIdx.x * 8 + wave;
  if (s < strips) fetch(s);
  for (; s < strips; s += step) {
#pragma unroll
    for (int kk = 0; kk < KC; ++kk) x[kk] = nx[kk];
    if (s + step < strips) fetch(s + step);
    for (int cg = 0; cg < groups; ++cg) {
      lt_f32x4 acc[1][FC];
#pragma unroll
      for (int j = 0; j < FC; ++j) acc[0][j] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) {
        Frag p[FC];
#pragma unroll
        for (int j = 0; j < FC; ++j) p[j] = *reinterpret_cast<const Frag*>(s_tile + (kk * NT + cg * FC + j) * 1024 + lane * 16);
        const Frag q[1] = {x[kk]};
        lt_mma_block<T, 1, FC>(p, q, acc);
      }
      lt_tile_store_<T, 1, FC, ACT, true>(a, acc, 0, s * 16, cg * 16 * FC, lane, turn);
    }
  }
}

// ------------------------------------------------------------------ backward
// One pass: a workgroup takes tiles of R rows, forms dz = dy act' on the way into LDS (its column sums stay in registers),
// and from the two tiles dz [R][N] and x [R][K] its waves compute dx = dz W (W in LDS) and add dz^T x to the workgroup's
// own dW, which they hold in registers until the end.  dy, act' and x are read once, dz is never written.
//   310017 x 128 -> 96, fp32: 223 us alone, matrix pipes busy 46 % of the cycles, 37 % of the LDS cycles are conflicts (dz, dx
//   and dW apart: 282 us); bf16: 73 us.
struct LtRowsBwdArgs {
  const void* dy;
  const void* x;
  const uint8_t* xs;      // x is mx8, or NULL
  const void* w;
  const void* deriv;
  int64_t lddy, ldx, ldw; // elements
  int dkind;
  int64_t M;
  int N, K;               // columns of dy (a multiple of 8) and of x
  int n_out;              // rows of W, dW and db: N, or less where dy's last columns are padding
  void* dx;               // [M][K] or NULL
  float* dw;              // [grid][n_out][K] or NULL
  float* db;              // [grid][n_out] or NULL
};

template <class T, int NP, int KP>
struct LtRowsBwd {
  // rows a tile, the k of dW's product: about 16 KB each of dz and x, so that what a tile waits for memory is small beside
  // what it moves (310017 x 64 -> 64 bf16: 84 us in tiles of 32 rows, 42 in tiles of 128)
  static constexpr int R = NP * KP == 64 * 64 ? 256 / sizeof(T) : sizeof(T) == 2 && NP + KP <= 256 ? 64 : 32;
  static constexpr int CH = 16 / sizeof(T), BKB = R * sizeof(T);
  typedef LtTile<T, true, NP, BKB> TZ;
  typedef LtTile<T, true, KP, BKB> TX;
  static constexpr int NT = 1024;   // 16 waves: with 8 the LDS latencies showed (128 -> 96 fp32 took 39 us more)
  static constexpr int NZ = (TZ::BYTES / 16 + NT - 1) / NT, NX = (TX::BYTES / 16 + NT - 1) / NT;
  static constexpr int TN = NP / 64, TK = KP / 64;                  // the waves' 4 x 4 grid over dW: 16 x 16 tiles a wave
  static constexpr int SX = R / 16, GX = 16 / SX;                   // dx: SX strips x GX column groups
  static constexpr int FX = KP / 16 > GX ? KP / 16 / GX : 1;        // of FX tiles
  static constexpr int BUF = TZ::BYTES + TX::BYTES;
  static int lds(int N, int K) {
    const int nf = (N + 4 * CH - 1) / (4 * CH), kt = (K + 15) / 16;
    return 2 * BUF + nf * kt * 1024 + NT / 64 * LtTurn<FX>::BYTES;
  }
};

template <class T, int NP, int KP>
__global__ __launch_bounds__(1024) void k_rows_bwd(LtRowsBwdArgs a) {
  typedef LtRowsBwd<T, NP, KP> S;
  typedef typename S::TZ TZ;
  typedef typename S::TX TX;
  typedef typename LtMma<T>::frag Frag;
  constexpr int CH = S::CH, KF = 4 * CH, KK = S::R / KF;   // fragments along the rows of a tile
  extern __shared__ __attribute__((aligned(1024))) char s_tile[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = a.N, K = a.K, nf = (N + KF - 1) / KF, nt = (N + 15) / 16, kt = (K + 15) / 16;
  char* s_w = s_tile + 2 * S::BUF;
  float* turn = reinterpret_cast<float*>(s_w + nf * kt * 1024 + wave * LtTurn<S::FX>::BYTES);
  // W for dx: fragment (f, c): lane (r, g) holds column 16 c + r of W, rows f KF + g CH ..
  if (a.dx) {
    for (int i = tid; i < nf * kt * 64; i += S::NT) {
      const int l = i & 63, c = (i >> 6) % kt, f = (i >> 6) / kt, k = 16 * c + (l & 15), n0 = f * KF + (l >> 4) * CH;
      Frag v;
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = (n0 + j < a.n_out && k < K) ? ((const T*)a.w)[(int64_t)(n0 + j) * a.ldw + k] : (T)0.f;
      *reinterpret_cast<Frag*>(s_w + i * 16) = v;
    }
  }
  float db[S::NZ][CH];
#pragma unroll
  for (int i = 0; i < S::NZ; ++i)
#pragma unroll
    for (int j = 0; j < CH; ++j) db[i][j] = 0.f;
  lt_f32x4 dw[S::TN][S::TK];
#pragma unroll
  for (int i = 0; i < S::TN; ++i)
#pragma unroll
    for (int j = 0; j < S::TK; ++j) dw[i][j] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};

  // The next tile on its way, as it lies in memory (a thread keeps its columns over all tiles): 16 bytes of dy and x (8 or 4
  // of an mx8 x), and the derivatives that go with them.  Nothing is touched before put(), so nothing is waited for.
  lt_i32x4 gz[S::NZ], gd[S::NZ], gx[S::NX];
  unsigned gs[S::NX];
  auto fetch = [&](int64_t m0) {
#pragma unroll
    for (int i = 0; i < S::NZ; ++i) {
      int line, c;
      TZ::where(tid + i * S::NT, line, c);
      const int64_t row = m0 + line < a.M ? m0 + line : a.M - 1;   // what does not exist is read elsewhere and cleared in put()
      const int col = c * CH < N ? c * CH : 0;
      __builtin_memcpy(&gz[i], (const T*)a.dy + row * a.lddy + col, 16);
      if (a.dkind == LT_DERIV_BITS) gd[i][0] = ((const uint8_t*)a.deriv)[row * (((N + 15) >> 4) * 2) + (col >> 3)];
      else if (a.dkind == LT_DERIV_BYTE) __builtin_memcpy(&gd[i], (const uint8_t*)a.deriv + row * N + col, CH);
      else if (a.dkind == LT_DERIV_FULL) __builtin_memcpy(&gd[i], (const char*)a.deriv + (row * N + col) * sizeof(T), 16);
    }
    if (!a.dw) return;
#pragma unroll
    for (int i = 0; i < S::NX; ++i) {
      int line, c;
      TX::where(tid + i * S::NT, line, c);
      const int64_t row = m0 + line < a.M ? m0 + line : a.M - 1;
      const int col = c * CH < K ? c * CH : 0;
      if (a.xs) {
        __builtin_memcpy(&gx[i], (const uint8_t*)a.x + row * K + col, CH);
        gs[i] = a.xs[row * ((K + 31) >> 5) + (col >> 5)];
      } else {
        __builtin_memcpy(&gx[i], (const T*)a.x + row * a.ldx + col, 16);
      }
    }
  };
  auto put = [&](char* buf, int64_t m0) {
#pragma unroll
    for (int i = 0; i < S::NZ; ++i) {
      int line, c;
      TZ::where(tid + i * S::NT, line, c);
      const bool ok = line < S::R && m0 + line < a.M && c * CH < N;
      T t[CH], y[CH];
      __builtin_memcpy(y, &gz[i], 16);
      float z[CH];
#pragma unroll
      for (int j = 0; j < CH; ++j) z[j] = (float)y[j];
      if (a.dkind == LT_DERIV_BITS) {
        const unsigned m = (unsigned)gd[i][0] >> ((c * CH) & 7);
#pragma unroll
        for (int j = 0; j < CH; ++j) z[j] = (m >> j) & 1 ? z[j] : 0.f;
      } else if (a.dkind == LT_DERIV_BYTE) {
#pragma unroll
        for (int j = 0; j < CH; ++j) z[j] *= lt_deriv_value(((unsigned)gd[i][j >> 2] >> (8 * (j & 3))) & 255u);
      } else if (a.dkind == LT_DERIV_FULL) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          if constexpr (sizeof(T) == 4) z[j] *= __uint_as_float((unsigned)gd[i][j]);
          else z[j] *= lt_deriv_word_value(((unsigned)gd[i][j >> 1] >> (16 * (j & 1))) & 65535u);
        }
      }
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        z[j] = ok ? z[j] : 0.f;
        db[i][j] += z[j];
        t[j] = (T)z[j];
      }
      if (tid + i * S::NT < TZ::BYTES / 16) __builtin_memcpy(buf + (tid + i * S::NT) * 16, t, 16);
    }
    if (!a.dw) return;
#pragma unroll
    for (int i = 0; i < S::NX; ++i) {
      int line, c;
      TX::where(tid + i * S::NT, line, c);
      const bool ok = line < S::R && m0 + line < a.M && c * CH < K;
      lt_i32x4 v = gx[i];
      if (a.xs) {
        const float sc = __uint_as_float(gs[i] << 23);
        float f[8];
        lt_mx8_get2<0>(gx[i][0], sc, f[0], f[1]);
        lt_mx8_get2<1>(gx[i][0], sc, f[2], f[3]);
        if constexpr (CH == 8) {
          lt_mx8_get2<0>(gx[i][1], sc, f[4], f[5]);
          lt_mx8_get2<1>(gx[i][1], sc, f[6], f[7]);
        }
        T t[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) t[j] = (T)f[j];
        __builtin_memcpy(&v, t, 16);
      }
      if (!ok) v = (lt_i32x4){0, 0, 0, 0};
      if (tid + i * S::NT < TX::BYTES / 16) *reinterpret_cast<lt_i32x4*>(buf + TZ::BYTES + (tid + i * S::NT) * 16) = v;
    }
  };

  LtTileArgs e = {};       // dx's store
  e.rows = a.M;
  e.cols = K;
  e.splits = 1;
  e.epi = LtEpi{nullptr, nullptr, 0, a.dx, K, nullptr, LT_DERIV_NONE, a.M, K};
  const int strip = wave % S::SX, xg = wave / S::SX;   // dx: rows 16 strip .., columns 16 FX xg ..
  const int wn = (wave >> 2) * S::TN, wk = (wave & 3) * S::TK;
  const int tiles = (int)((a.M + S::R - 1) / S::R);
  auto do_dx = [&](const char* buf, int64_t m0) {
    if (!a.dx || xg * S::FX >= kt) return;
    lt_f32x4 acc[1][S::FX];
#pragma unroll
    for (int j = 0; j < S::FX; ++j) acc[0][j] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};
    const int m = 16 * strip + r;
#pragma unroll 4
    for (int f = 0; f < nf; ++f) {
      const int c = f * 4 + g;                         // chunk of CH columns n of row m
      const Frag q = *reinterpret_cast<const Frag*>(buf + m * (NP * (int)sizeof(T)) + ((c ^ TZ::kswz(m)) << 4));
#pragma unroll
      for (int j = 0; j < S::FX; ++j)   // (a tile past the last column multiplies whatever lies behind W: it is not stored)
        acc[0][j] = LtMma<T>::mma(*reinterpret_cast<const Frag*>(s_w + (f * kt + xg * S::FX + j) * 1024 + lane * 16), q, acc[0][j]);
    }
    lt_tile_store_<T, 1, S::FX, LT_ACT_NONE, true>(e, acc, 0, m0 + 16 * strip, 16 * S::FX * xg, lane, turn);
  };
  auto do_dw = [&](const char* buf) {
    if (!a.dw || wn >= nt || wk >= kt) return;   // a wave's tiles are all multiplied or none: no branches between the products
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      Frag p[S::TK], q[S::TN];
#pragma unroll
      for (int j = 0; j < S::TK; ++j) p[j] = TX::frag(buf + TZ::BYTES, 16 * (wk + j), kk, lane);
#pragma unroll
      for (int i = 0; i < S::TN; ++i) q[i] = TZ::frag(buf, 16 * (wn + i), kk, lane);
      lt_mma_block<T, S::TN, S::TK>(p, q, dw);
    }
  };
  int t = blockIdx.x;
  if (t < tiles) fetch((int64_t)t * S::R);
  for (int b = 0; t < tiles; t += gridDim.x, b ^= 1) {
    char* buf = s_tile + b * S::BUF;
    const int64_t m0 = (int64_t)t * S::R;
    put(buf, m0);
    __syncthreads();       // (W is in place too); the other buffer's readers are past the barrier before
    if (t + (int)gridDim.x < tiles) fetch((int64_t)(t + gridDim.x) * S::R);
    do_dx(buf, m0);
    do_dw(buf);
  }
  float* out = a.dw ? a.dw + (int64_t)blockIdx.x * a.n_out * K : nullptr;
#pragma unroll
  for (int i = 0; i < S::TN; ++i)
#pragma unroll
    for (int j = 0; j < S::TK; ++j) {
      const int n = 16 * (wn + i) + r, k = 16 * (wk + j) + 4 * g;
      const float v[4] = {dw[i][j][0], dw[i][j][1], dw[i][j][2], dw[i][j][3]};
      if (out && n < a.n_out && k < K) lt_stv<float, 4>(out + (int64_t)n * K + k, K - k, v);
    }
  if (!a.db) return;
  __syncthreads();
  float* s_db = reinterpret_cast<float*>(s_tile);      // [lines][NP]: every thread's sums at its line and columns, then by column
#pragma unroll
  for (int i = 0; i < S::NZ; ++i) {
    int line, c;
    TZ::where(tid + i * S::NT, line, c);
    if (line < S::R)
#pragma unroll
      for (int j = 0; j < CH; ++j) s_db[line * NP + c * CH + j] = db[i][j];
  }
  __syncthreads();
  for (int n = tid; n < a.n_out; n += S::NT) {
    float s = 0.f;
#pragma unroll 8
    for (int l = 0; l < S::R; ++l) s += s_db[l * NP + n];
    a.db[(int64_t)blockIdx.x * a.n_out + n] = s;
  }
}

// ------------------------------------------------------------------ host
// forward: at least 8192 rows, both widths at most 256 and multiples of 8, W and the turned rows within half a CU's LDS (two workgroups a CU).
// This kernel and tiles, us: 64 -> 64 fp32 7.7 and 8.5 at 8192 rows, 9.2 and 10.0 at 32768; 128 -> 96 fp32 14.0 and 7.5 at 8192, 17.2 and
// 17.9 at 32768, 103 and 145 at 310017; 32 -> 256 fp32 17.5 and 7.4, 20.8 and 20.4; 128 -> 96 bf16 6.7 and 4.2, 7.7 and 8.1.  The
// wider layers pay for laying out W in every workgroup up to some 30000 rows.
template <class T>
static int lt_rows_kc(int K) {
  const int kf = 4 * (16 / (int)sizeof(T)), n = (K + kf - 1) / kf;
  return n <= 2 ? n : n <= 4 ? 4 : n <= 6 ? 6 : n <= 8 ? 8 : 16;
}
template <class T> struct LtRowsFC { static constexpr int value = sizeof(T) == 4 ? 2 : 4; };
template <class T>
static int lt_rows_lds(int N, int K) {
  constexpr int FC = LtRowsFC<T>::value;
  return lt_rows_kc<T>(K) * ((N + 16 * FC - 1) / (16 * FC) * FC) * 1024 + 8 * LtTurn<FC>::BYTES;
}
template <class T>
static bool lt_rows_fwd_ok(int64_t M, int N, int K) {
  return M >= 8192 && N <= 256 && K <= 256 && N % 8 == 0 && K % 8 == 0 && lt_rows_lds<T>(N, K) <= 80 * 1024;
}

template <class T, int KC, int ACT>
static int lt_rows_fwd_go(const LtTileArgs& a, hipStream_t stream) {
  constexpr int FC = LtRowsFC<T>::value;
  const int smem = lt_rows_lds<T>(a.cols, (int)a.depth);
  if (smem > 65536)
    LT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_rows_fwd<T, KC, FC, ACT>), hipFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t strips = (a.rows + 15) / 16;
  const int64_t want = (strips + 7) / 8;
  hipLaunchKernelGGL((k_rows_fwd<T, KC, FC, ACT>), dim3((unsigned)(want > 512 ? 512 : want)), dim3(512), smem, stream, a);
  LT_LAUNCH_CHECK();
  return LT_OK;
}
template <class T, int ACT>
static int lt_rows_fwd(const LtTileArgs& a, hipStream_t stream) {
  switch (lt_rows_kc<T>((int)a.depth)) {
    case 1: return lt_rows_fwd_go<T, 1, ACT>(a, stream);
    case 2: return lt_rows_fwd_go<T, 2, ACT>(a, stream);
    case 4: return lt_rows_fwd_go<T, 4, ACT>(a, stream);
    case 6: return lt_rows_fwd_go<T, 6, ACT>(a, stream);
    case 8: return lt_rows_fwd_go<T, 8, ACT>(a, stream);
    default:
      if constexpr (sizeof(T) == 4) return lt_rows_fwd_go<T, 16, ACT>(a, stream);
      return LT_ERR_ARG;
  }
}

// backward: widths that are multiples of 8 and whose dW a workgroup's registers and whose W its LDS hold
struct LtRowsBwdPlan {
  bool ok;
  int np, kp, grid, lds;
};
// at least 256 rows (three launches instead of four to six; a 16-bit dz of up to 4096 elements goes in as two terms: dense.hip),
// widths that are multiples of 8 (N may also be padded: dz is then written out with zeros behind its columns)
static inline LtRowsBwdPlan lt_rows_bwd_plan(int64_t M, int K, int N_, int dt) {
  LtRowsBwdPlan p = {};
  const int N = N_ <= 256 ? (N_ + 7) / 8 * 8 : N_;
  auto pad = [](int v) { return v <= 64 ? 64 : v <= 128 ? 128 : 256; };
  if (N > 256 || K > 256 || K % 8 || M < 256 || (dt != LT_DT_F32 && M * N_ <= 4096) || M > (int64_t)1 << 34) return p;
  p.np = pad(N);
  p.kp = pad(K);
  const int sz = lt_dt_size(dt), kf = 64 / sz;   // as in LtRowsBwd, which checks the two against each other
  const int R = p.np * p.kp == 64 * 64 ? 256 / sz : sz == 2 && p.np + p.kp <= 256 ? 64 : 32;
  const int gx = 16 / (R / 16), fx = p.kp / 16 > gx ? p.kp / 16 / gx : 1;
  const int w = ((N + kf - 1) / kf) * ((K + 15) / 16) * 1024, turn = 16 * 16 * (16 * fx + 4) * 4;
  p.lds = 2 * R * (p.np + p.kp) * sz + w + turn;
  p.ok = p.lds <= 160 * 1024 && p.np * p.kp <= 256 * 128 && (sz == 2 || p.np + p.kp <= 320);   // fp32 tiles of 128 and 256: no room
  const int64_t tiles = (M + R - 1) / R;
  p.grid = (int)(tiles < 256 ? tiles : 256);
  return p;
}
template <class T, int NP, int KP>
static int lt_rows_bwd_go(const LtRowsBwdArgs& a, const LtRowsBwdPlan& p, hipStream_t stream) {
  const int smem = LtRowsBwd<T, NP, KP>::lds(a.N, a.K), grid = p.grid;
  LT_REQUIRE(smem == p.lds, LT_ERR_ARG, "linear: plan and kernel disagree (%d, %d bytes of LDS)", p.lds, smem);
  if (smem > 65536)
    LT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_rows_bwd<T, NP, KP>), hipFuncAttributeMaxDynamicSharedMemorySize, smem));
  hipLaunchKernelGGL((k_rows_bwd<T, NP, KP>), dim3(grid), dim3(1024), smem, stream, a);
  LT_LAUNCH_CHECK();
  return LT_OK;
}
template <class T> int lt_rows_bwd_launch(const LtRowsBwdArgs& a, const LtRowsBwdPlan& p, hipStream_t stream);
template <class T>
static int lt_rows_bwd_impl(const LtRowsBwdArgs& a, const LtRowsBwdPlan& p, hipStream_t stream) {
  switch (p.np * 1000 + p.kp) {
    case 64064: return lt_rows_bwd_go<T, 64, 64>(a, p, stream);
    case 64128: return lt_rows_bwd_go<T, 64, 128>(a, p, stream);
    case 64256: return lt_rows_bwd_go<T, 64, 256>(a, p, stream);
    case 128064: return lt_rows_bwd_go<T, 128, 64>(a, p, stream);
    case 128128: return lt_rows_bwd_go<T, 128, 128>(a, p, stream);
    case 256064: return lt_rows_bwd_go<T, 256, 64>(a, p, stream);
    default:
      if constexpr (sizeof(T) == 2) {
        if (p.kp == 256) return lt_rows_bwd_go<T, 128, 256>(a, p, stream);
        return lt_rows_bwd_go<T, 256, 128>(a, p, stream);
      }
      lt_set_error("linear: no one-pass backward for %d x %d", p.np, p.kp);
      return LT_ERR_ARG;
  }
}
