// Which product kernel runs, with which tile and how many splits, and its launch (kernels: dense_gemm.h, dense_rows.h).
#pragma once
#include "dense_rows.h"

// ---- host: which kernel, which tile, how many splits
// tile shapes (rows x columns of the output)
enum { LT_TILE_256x256, LT_TILE_128x128, LT_TILE_128x64, LT_TILE_256x32, LT_TILE_64x64 };

struct LtPlan {
  int tile, tr, tc, splits;
  int64_t slice;
  bool few, rows, direct;
};

static inline LtPlan lt_gemm_plan(int64_t rows, int cols, int64_t depth, int dt, bool nn, bool direct) {
  LtPlan p = {};
  p.direct = direct;
  p.splits = 1;
  p.slice = depth;
  // up to 32 rows the tile kernels would leave most of a tile idle; both operands must run along k (4096 -> 4096 bf16, this way and
  // on tiles, us: 1 row 9.9 and 11.2, 16 rows 10.2 and 12.1, 32 rows 13.9 and 13.5, 64 rows 22 and 17; 1024 -> 1024, 32 rows: 5.3 and 7.9)
  p.few = nn && rows <= 32;
  if (p.few || rows <= 0 || depth <= 0) return p;
  p.rows = nn && (dt == LT_DT_F32 ? lt_rows_fwd_ok<float>(rows, cols, (int)depth) : lt_rows_fwd_ok<lt_bf16>(rows, cols, (int)depth));
  if (p.rows) return p;
  const int bk = dt == LT_DT_F32 ? 32 : 64;
  auto tiles = [&](int br, int bc) { return ((rows + br - 1) / br) * ((cols + bc - 1) / bc); };
  int br, bc;
  // the widest tile needs the fewest operand bytes a product, and one workgroup a CU: 192 of them, or fewer whose k is long
  // enough to be split into at least 32 steps each (training 16384 x 1024 -> 4096, bf16: its dW on 128 x 128 tiles 618 us a
  // step, on 256 x 256 tiles split four ways 554 us; forward x 1024 -> 4096 bf16 on the widest and on 128 x 128, us: 128 tiles of the
  // widest 42 and 22, 192 of them 36.4 and 36.4, 256 of them 38.9 and 41.7).  256 x 128 tiles, also one a CU, lose to two of 128 x 128 (training
  // 4096 x 2048 -> 2048, bf16: 187 us a step and 146).
  const int64_t t256 = tiles(256, 256);
  const bool wide = direct && dt != LT_DT_F32 && cols >= 192 && rows >= 192;
  if (wide && (t256 >= 192 || (t256 >= 16 && depth >= 64 * 32 * (256 / t256)))) p.tile = LT_TILE_256x256, br = 256, bc = 256;
  else if (cols <= 32 && direct) p.tile = LT_TILE_256x32, br = 256, bc = 32;
  else if (cols <= 64 && direct) p.tile = LT_TILE_128x64, br = 128, bc = 64;
  // 128 x 128 tiles where they nearly fill the chip, else 64 x 64, four of which share a CU (1777 x 1000 -> 1000 bf16: 26 us
  // on 112 of the larger, split four ways, 12 us on 448 of the smaller).  x 1024 -> 2048 bf16 on the larger and the smaller, us: 160
  // of the larger 25 and 13, 224 of them 27 and 16 (split in two), 256 of them 16.6 and 16.2, 320 of them 19.7 and 24.3.  fp32 is bound by the matrix rate alone, so there the
  // smaller tiles cost 6 % (8192 x 1024 -> 1024: 137 and 144 us) and a chip half idle in its last turn costs more (3000 x 1500
  // -> 1500: 191 and 154 us): the larger ones where the turns of two a CU are 93 % full.
  else if (dt == LT_DT_F32 ? (double)rows * cols >= 0.93 * 128 * 128 * 512 * ((tiles(128, 128) + 511) / 512) : tiles(128, 128) >= 224) p.tile = LT_TILE_128x128, br = 128, bc = 128;
  else p.tile = LT_TILE_64x64, br = 64, bc = 64;
  p.tr = (int)((rows + br - 1) / br);
  p.tc = (cols + bc - 1) / bc;
  // Fewer tiles than the chip runs at once: split k, at least four steps each.  The join reads and writes splits + 1 times
  // the output, so where the chip is full once (256 tiles) only a long k is split (1024 x 4096 -> 1024 bf16: 36 us whole,
  // 25 us in four; 1777 x 1000 -> 1000: 12 us whole, 24 us in two).  64 x 64 tiles from 48 steps on: 256 tiles split and whole, us, 32
  // steps 21 and 14, 40 steps 23 and 19, 50 steps 23 and 30, 64 steps 24 and 37; 512 tiles, 40 steps 27 and 26, 50 steps 29 and 31.
  const int64_t t = (int64_t)p.tr * p.tc, steps = (depth + bk - 1) / bk;
  const int64_t full = p.tile == LT_TILE_256x256 ? 256 : steps >= 48 ? 1024 : 512;
  if (t < (p.tile == LT_TILE_256x256 ? 192 : p.tile == LT_TILE_64x64 && steps >= 48 ? 513 : 256)) {
    int64_t s = full / t;
    if (s > steps / 4) s = steps / 4;
    if (s > 256) s = 256;
    if (s > 1) {
      const int64_t per = (steps + s - 1) / s;
      p.slice = per * bk;
      p.splits = (int)((steps + per - 1) / per);
    }
  }
  return p;
}

// the launches for one value type (dense_f32.hip, dense_bf16.hip, dense_f16.hip)
template <class T> int lt_gemm_launch(const LtGemm& g, const LtPlan& p, float* part, hipStream_t stream);

template <class T, bool PKM, bool QKM, int BR, int BC, int WR, int WC, bool DIRECT, bool P8, int ACT>
static int lt_launch_tile(const LtTileArgs& a, hipStream_t stream) {
  // a single step needs one buffer: more workgroups a CU (310017 x 32 -> 256 fp32: 196 -> 178 us)
  const bool one = a.slice <= 128 / (int64_t)sizeof(T) && !a.Q2;
  const int need = WR * WC * LtTurn<BC / WC / 16>::BYTES;
  int smem = (one ? 1 : 2) * (BR + BC) * 128;
  if (smem < need) smem = need;
  if (smem > 65536)
    LT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_dense<T, PKM, QKM, BR, BC, WR, WC, DIRECT, P8, ACT>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, smem));
  hipLaunchKernelGGL((k_dense<T, PKM, QKM, BR, BC, WR, WC, DIRECT, P8, ACT>), dim3((unsigned)a.tr * a.tc * a.splits),
                     dim3(64 * WR * WC), smem, stream, a);
  LT_LAUNCH_CHECK();
  return LT_OK;
}

template <class T, bool PKM, bool QKM, int ACT>
static int lt_launch_shape(const LtPlan& p, const LtTileArgs& a, bool p8, hipStream_t stream) {
  if constexpr (PKM && QKM) {
    if (p8) {
      if (p.tile == LT_TILE_128x128) return lt_launch_tile<T, true, true, 128, 128, 2, 2, false, true, LT_ACT_NONE>(a, stream);
      return lt_launch_tile<T, true, true, 64, 64, 2, 2, false, true, LT_ACT_NONE>(a, stream);
    }
  }
  if (p.direct) {
    switch (p.tile) {
      case LT_TILE_256x256:
        if constexpr (sizeof(T) == 2) return lt_launch_tile<T, PKM, QKM, 256, 256, 2, 4, true, false, ACT>(a, stream);
        break;
      case LT_TILE_128x128: return lt_launch_tile<T, PKM, QKM, 128, 128, 2, 2, true, false, ACT>(a, stream);
      case LT_TILE_128x64: return lt_launch_tile<T, PKM, QKM, 128, 64, 2, 2, true, false, ACT>(a, stream);
      case LT_TILE_256x32: return lt_launch_tile<T, PKM, QKM, 256, 32, 4, 1, true, false, ACT>(a, stream);
      default: return lt_launch_tile<T, PKM, QKM, 64, 64, 2, 2, true, false, ACT>(a, stream);
    }
  }
  if (p.tile == LT_TILE_128x128) return lt_launch_tile<T, PKM, QKM, 128, 128, 2, 2, false, false, ACT>(a, stream);
  return lt_launch_tile<T, PKM, QKM, 64, 64, 2, 2, false, false, ACT>(a, stream);
}

template <class T, int ACT>
static int lt_launch_few(const LtTileArgs& a, hipStream_t stream) {
  const dim3 grid((a.cols + 15) / 16), block(512);
  const int fr = (int)((a.rows + 15) / 16);
  if (fr == 1) hipLaunchKernelGGL((k_dense_few<T, 1, ACT>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((k_dense_few<T, 2, ACT>), grid, block, 0, stream, a);
  LT_LAUNCH_CHECK();
  return LT_OK;
}

template <class T, int ACT>
static int lt_launch_join(const LtEpi& e, const float* part, int splits, hipStream_t stream) {
  const int64_t n = e.rows * (int64_t)((e.cols + 7) >> 3);
  if (splits >= 64) hipLaunchKernelGGL((k_dense_join<T, ACT, 16>), dim3(lt_grid(n, 16)), dim3(256), 0, stream, part, splits, e);
  else if (splits >= 8) hipLaunchKernelGGL((k_dense_join<T, ACT, 4>), dim3(lt_grid(n, 64)), dim3(256), 0, stream, part, splits, e);
  else hipLaunchKernelGGL((k_dense_join<T, ACT, 1>), dim3(lt_grid(n, 256)), dim3(256), 0, stream, part, splits, e);
  LT_LAUNCH_CHECK();
  return LT_OK;
}

template <class T, int ACT>
static int lt_gemm_launch_act(const LtGemm& g, const LtPlan& p, const LtTileArgs& a, float* part, hipStream_t stream) {
  int rc = LT_OK;
  if (g.depth > 0) {
    if (p.few) return lt_launch_few<T, ACT>(a, stream);
    if (p.rows) return lt_rows_fwd<T, ACT>(a, stream);
    if (!g.p_kmajor) rc = lt_launch_shape<T, false, false, ACT>(p, a, false, stream);
    else if constexpr (ACT == LT_ACT_NONE) {
      if (!g.q_kmajor) rc = lt_launch_shape<T, true, false, ACT>(p, a, false, stream);
      else rc = lt_launch_shape<T, true, true, ACT>(p, a, g.p_scales != nullptr, stream);
    }
    if (rc) return rc;
    if (p.splits == 1) return LT_OK;
  }
  return lt_launch_join<T, ACT>(g.epi, part, g.depth > 0 ? p.splits : 0, stream);   // no k at all: the sum is zero
}

template <class T>
static int lt_gemm_launch_impl(const LtGemm& g, const LtPlan& p, float* part, hipStream_t stream) {
  LtTileArgs a = {};
  a.P = (const char*)g.P;
  a.Q = (const char*)g.Q;
  a.Q2 = (const char*)g.Q2;
  a.ldp = g.ldp * (g.p_scales ? 1 : (int64_t)sizeof(T));
  a.ldq = g.ldq * (int64_t)sizeof(T);
  a.rows = g.rows;
  a.depth = g.depth;
  a.cols = g.cols;
  a.tr = p.tr;
  a.tc = p.tc;
  a.splits = p.splits;
  a.slice = p.slice;
  a.part = part;
  a.ps = g.p_scales;
  a.ldps = (g.cols + 31) / 32;
  a.epi = g.epi;
  switch (g.act) {
    case LT_ACT_RELU: return lt_gemm_launch_act<T, LT_ACT_RELU>(g, p, a, part, stream);
    case LT_ACT_GELU: return lt_gemm_launch_act<T, LT_ACT_GELU>(g, p, a, part, stream);
    case LT_ACT_SILU: return lt_gemm_launch_act<T, LT_ACT_SILU>(g, p, a, part, stream);
    default: return lt_gemm_launch_act<T, LT_ACT_NONE>(g, p, a, part, stream);
  }
}
