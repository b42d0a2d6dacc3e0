// The product of two mx8 matrices: y = act(x8 W8^T + b) + r on the scaled matrix instructions.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 128 k of 16 rows an operand and one power-of-two scale per row and 32 k -- the
// mx8 format itself, so nothing is widened on the way.  Lane l = 16 g + r holds k 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g
// + 15 of row r in its 32 bytes, and the scale of row r's 32-block g in its scale register's low byte (measured).  Tiles,
// staging, splits and epilogue are those of dense_gemm.h: a step of 128 bytes is one instruction's k.
//
// Sums: the instruction adds 8 neighbouring products in fixed point, each cut to a multiple of 2^-13 times the power of two
// of the group's largest (measured), and goes on in fp32.  That is the price of the 8-bit rate (twice the 16-bit one); the
// operands were rounded to within 2^-4, and widening them to bf16 instead would keep every product whole at half the rate.
#pragma once
#include "dense_plan.h"

struct LtTile8Args {
  LtTileArgs t;
  const uint8_t* qs;    // scales of Q; those of P are t.ps
  int nb;               // scales a row
};

template <int V> struct LtInt { static constexpr int value = V; };

// scale byte of k-block kb of a row; blocks past the end hold zeros, whose scale must only be finite
__device__ __forceinline__ int lt_scale8(const uint8_t* row, int kb, int nb) { return kb < nb ? row[kb] : 127; }

template <int R>
__device__ __forceinline__ lt_i32x8 lt_frag8(const char* t, int i0, int lane) {
  const int i = i0 + (lane & 15), g = lane >> 4;
  union { lt_i32x4 h[2]; lt_i32x8 f; } u;
  u.h[0] = *reinterpret_cast<const lt_i32x4*>(t + i * 128 + ((g ^ (i & 7)) << 4));
  u.h[1] = *reinterpret_cast<const lt_i32x4*>(t + i * 128 + (((g + 4) ^ (i & 7)) << 4));
  return u.f;
}

template <class T, int BR, int BC, int WR, int WC, bool DIRECT, int ACT>
__global__ __launch_bounds__(64 * WR * WC) void k_dense8(LtTile8Args b) {
  const LtTileArgs& a = b.t;
  typedef LtTile<uint8_t, false, BC, 128> TP;
  typedef LtTile<uint8_t, false, BR, 128> TQ;
  constexpr int NW = WR * WC, NT = 64 * NW, FR = BR / WR / 16, FC = BC / WC / 16;
  constexpr int BUF = TP::BYTES + TQ::BYTES, NBUF = 2;
  extern __shared__ __attribute__((aligned(1024))) char s_tile[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned tiles = (unsigned)a.tr * a.tc;
  const unsigned L = lt_xcd_map(blockIdx.x, tiles * a.splits);
  const unsigned split = L / tiles, t_ = L % tiles;
  const unsigned grp = t_ / (8u * a.tc), in = t_ - grp * 8u * a.tc;
  const unsigned gr = (unsigned)a.tr - grp * 8u < 8u ? (unsigned)a.tr - grp * 8u : 8u;
  const int64_t row0 = (int64_t)(grp * 8u + in % gr) * BR;
  const int col0 = (int)(in / gr) * BC;
  const int64_t k0 = split * a.slice;
  const int64_t kend = k0 + a.slice < a.depth ? k0 + a.slice : a.depth;
  const int nk = (int)((kend - k0 + 127) >> 7);
  const char* pb = a.P + col0 * a.ldp + k0;
  const char* qb = a.Q + row0 * a.ldq + k0;
  const int64_t pn = a.cols - col0, qn = a.rows - row0;
  const int wr = (wave / WC) * (BR / WR), wc = (wave % WC) * (BC / WC);

  // Scales: four steps' worth, 16 bytes a row, go through LDS at a time.  They are turned there so that a lane's four bytes
  // (block g of each of the four steps) are one word, of which the instruction picks byte t & 3 itself.  Loading each
  // fragment's byte from memory instead took more address cycles than the tiles' own loads (8192^3: 956 us, this: 521 us).
  char* s_sc = s_tile + 2 * BUF;                 // [2][BC + BR][16]
  const bool srow_ok = tid < BC ? tid < pn : (tid < BC + BR && tid - BC < qn);
  const uint8_t* srow = tid < BC ? a.ps + (int64_t)(srow_ok ? col0 + tid : 0) * b.nb : b.qs + (srow_ok ? row0 + tid - BC : 0) * (int64_t)b.nb;
  unsigned sw[4];
  auto sc_load = [&](int kb) {                   // blocks past the end hold zeros, whose scale must only be finite
    const int n = srow_ok ? b.nb - kb : 0;
    if (n >= 16) __builtin_memcpy(sw, srow + kb, 16);
    else {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        sw[w] = 0x7F7F7F7Fu;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (4 * w + t < n) sw[w] = (sw[w] & ~(0xFFu << (8 * t))) | ((unsigned)srow[kb + 4 * w + t] << (8 * t));
      }
    }
  };
  auto sc_store = [&](int buf) {
    if (tid < BC + BR) {
      const unsigned l01 = __builtin_amdgcn_perm(sw[1], sw[0], 0x05010400u), h01 = __builtin_amdgcn_perm(sw[1], sw[0], 0x07030602u);
      const unsigned l23 = __builtin_amdgcn_perm(sw[3], sw[2], 0x05010400u), h23 = __builtin_amdgcn_perm(sw[3], sw[2], 0x07030602u);
      lt_i32x4 o;
      o[0] = (int)__builtin_amdgcn_perm(l23, l01, 0x05040100u);   // block 0 of steps 0 .. 3
      o[1] = (int)__builtin_amdgcn_perm(l23, l01, 0x07060302u);
      o[2] = (int)__builtin_amdgcn_perm(h23, h01, 0x05040100u);
      o[3] = (int)__builtin_amdgcn_perm(h23, h01, 0x07060302u);
      *reinterpret_cast<lt_i32x4*>(s_sc + buf * (BC + BR) * 16 + tid * 16) = o;
    }
  };
  lt_f32x4 acc[FR][FC];
#pragma unroll
  for (int i = 0; i < FR; ++i)
#pragma unroll
    for (int j = 0; j < FC; ++j) acc[i][j] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};

  int sp_[FC], sq_[FR];
  auto sc_read = [&](int buf) {
    const char* p = s_sc + buf * (BC + BR) * 16 + 4 * g;
#pragma unroll
    for (int j = 0; j < FC; ++j) sp_[j] = *reinterpret_cast<const int*>(p + (wc + 16 * j + r) * 16);
#pragma unroll
    for (int i = 0; i < FR; ++i) sq_[i] = *reinterpret_cast<const int*>(p + (BC + wr + 16 * i + r) * 16);
  };
  auto mma = [&](const char* buf, auto sel, auto ahead) {
    constexpr int S = decltype(sel)::value;
    lt_i32x8 p[FC];
#pragma unroll
    for (int j = 0; j < FC; ++j) p[j] = lt_frag8<BC>(buf, wc + 16 * j, lane);
    ahead();
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const lt_i32x8 q = lt_frag8<BR>(buf + TP::BYTES, wr + 16 * i, lane);
#pragma unroll
      for (int j = 0; j < FC; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p[j], q, acc[i][j], 0, 0, S, sp_[j], S, sq_[i]);
    }
  };
  const int kb0 = (int)(k0 >> 5);
  const int64_t len = kend - k0;
  sc_load(kb0);
  if constexpr (DIRECT) {
    LtDirect<TP, false, NW> sp;
    LtDirect<TQ, false, NW> sq;
    sp.init(a.ldp, pn, wave, lane);
    sq.init(a.ldq, qn, wave, lane);
    auto issue = [&](int t) {
      char* buf = s_tile + (t & 1) * BUF;
      sp.load(pb + (int64_t)t * 128, buf, len - (int64_t)t * 128, wave, lane);
      sq.load(qb + (int64_t)t * 128, buf + TP::BYTES, len - (int64_t)t * 128, wave, lane);
    };
    auto step = [&](int t, auto sel) {
      constexpr int S = decltype(sel)::value;
      if (t >= nk) return;
      if (S == 0) sc_store((t >> 2) & 1);        // its last readers are two barriers back
      lt_wait_barrier();                         // this step's tiles (and scales) are there, nobody reads the other buffer
      if (S == 0) {
        sc_read((t >> 2) & 1);
        if (t + 4 < nk) sc_load(kb0 + 4 * (t + 4));
      }
      mma(s_tile + (t & 1) * BUF, sel, [&]() {
        if (t + 1 < nk) issue(t + 1);
      });
    };
    issue(0);
    for (int t = 0; t < nk; t += 4) {
      step(t, LtInt<0>());
      step(t + 1, LtInt<1>());
      step(t + 2, LtInt<2>());
      step(t + 3, LtInt<3>());
    }
  } else {
    LtStaged<uint8_t, TP, false, false, NT> sp;
    LtStaged<uint8_t, TQ, false, false, NT> sq;
    auto get = [&](int t) {
      sp.load(pb + (int64_t)t * 128, a.ldp, pn, len - (int64_t)t * 128, nullptr, 0, 0, tid);
      sq.load(qb + (int64_t)t * 128, a.ldq, qn, len - (int64_t)t * 128, nullptr, 0, 0, tid);
    };
    auto step = [&](int t, auto sel) {
      constexpr int S = decltype(sel)::value;
      if (t >= nk) return;
      char* cur = s_tile + (t & 1) * BUF;
      sp.store(cur, tid);
      sq.store(cur + TP::BYTES, tid);
      if (S == 0) sc_store((t >> 2) & 1);
      __syncthreads();
      if (S == 0) {
        sc_read((t >> 2) & 1);
        if (t + 4 < nk) sc_load(kb0 + 4 * (t + 4));
      }
      if (t + 1 < nk) get(t + 1);
      mma(cur, sel, [] {});
    };
    get(0);
    for (int t = 0; t < nk; t += 4) {
      step(t, LtInt<0>());
      step(t + 1, LtInt<1>());
      step(t + 2, LtInt<2>());
      step(t + 3, LtInt<3>());
    }
  }
  static_assert(NW * LtTurn<FC>::BYTES <= NBUF * BUF, "the turned rows do not fit the tiles' LDS");
  __syncthreads();
  lt_tile_store<T, FR, FC, ACT>(a, acc, split, row0 + wr, col0 + wc, lane,
                                reinterpret_cast<float*>(s_tile + wave * LtTurn<FC>::BYTES));
}

// few rows: as k_dense_few, 128 k an instruction straight from memory
template <class T, int FR, int ACT>
__global__ __launch_bounds__(512) void k_dense8_few(LtTile8Args b) {
  const LtTileArgs& a = b.t;
  constexpr int U = 2;
  __shared__ lt_f32x4 s_acc[8][FR][64];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col0 = blockIdx.x * 16;
  const bool pok = col0 + r < a.cols;
  const int64_t prow = pok ? col0 + r : 0;
  lt_f32x4 acc[FR];
#pragma unroll
  for (int f = 0; f < FR; ++f) acc[f] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};
  auto get = [&](const char* line, bool ok, int64_t k) -> lt_i32x8 {   // the lane's 32 bytes of the 128 from k
    union { lt_i32x4 h[2]; lt_i32x8 f; } u;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int64_t at = k + 64 * c + 16 * g, n = ok ? a.depth - at : 0;
      u.h[c] = (lt_i32x4){0, 0, 0, 0};
      if (n >= 16) __builtin_memcpy(&u.h[c], line + at, 16);
      else if (n > 0) {
        uint8_t t[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) t[j] = j < n ? (uint8_t)line[at + j] : 0;
        __builtin_memcpy(&u.h[c], t, 16);
      }
    }
    return u.f;
  };
  for (int64_t k = (int64_t)wave * U * 128; k < a.depth; k += 8 * U * 128) {
    lt_i32x8 p[U], q[FR][U];
    int sp_[U], sq_[FR][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u] = get(a.P + prow * a.ldp, pok, k + 128 * u);
      sp_[u] = lt_scale8(a.ps + prow * b.nb, (int)((k + 128 * u) >> 5) + g, b.nb);
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        const bool ok = f * 16 + r < a.rows;
        const int64_t row = ok ? f * 16 + r : 0;
        q[f][u] = get(a.Q + row * a.ldq, ok, k + 128 * u);
        sq_[f][u] = lt_scale8(b.qs + row * b.nb, (int)((k + 128 * u) >> 5) + g, b.nb);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < FR; ++f)
        acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p[u], q[f][u], acc[f], 0, 0, 0, sp_[u], 0, sq_[f][u]);
  }
  lt_few_store<T, FR, ACT>(a, acc, s_acc, col0, wave, lane);
}

template <class T> int lt_gemm8_launch(const LtTile8Args& b, const LtPlan& p, int act, hipStream_t stream);

template <class T, int BR, int BC, int WR, int WC, bool DIRECT, int ACT>
static int lt_launch_tile8(const LtTile8Args& b, hipStream_t stream) {
  const int smem = 2 * (BR + BC) * 128 + 2 * (BR + BC) * 16;
  if (smem > 65536)
    LT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_dense8<T, BR, BC, WR, WC, DIRECT, ACT>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, smem));
  hipLaunchKernelGGL((k_dense8<T, BR, BC, WR, WC, DIRECT, ACT>), dim3((unsigned)b.t.tr * b.t.tc * b.t.splits), dim3(64 * WR * WC), smem,
                     stream, b);
  LT_LAUNCH_CHECK();
  return LT_OK;
}

template <class T, int ACT>
static int lt_gemm8_launch_act(const LtTile8Args& b, const LtPlan& p, hipStream_t stream) {
  int rc;
  if (p.few) {
    const dim3 grid((b.t.cols + 15) / 16), block(512);
    const int fr = (int)((b.t.rows + 15) / 16);
    if (fr == 1) hipLaunchKernelGGL((k_dense8_few<T, 1, ACT>), grid, block, 0, stream, b);
    else hipLaunchKernelGGL((k_dense8_few<T, 2, ACT>), grid, block, 0, stream, b);
    LT_LAUNCH_CHECK();
    return LT_OK;
  }
  if (!p.direct) rc = lt_launch_tile8<T, 64, 64, 2, 2, false, ACT>(b, stream);
  else if (p.tile == LT_TILE_256x256) rc = lt_launch_tile8<T, 256, 256, 2, 4, true, ACT>(b, stream);
  else if (p.tile == LT_TILE_128x128) rc = lt_launch_tile8<T, 128, 128, 2, 2, true, ACT>(b, stream);
  else rc = lt_launch_tile8<T, 64, 64, 2, 2, true, ACT>(b, stream);
  if (rc || p.splits == 1) return rc;
  return lt_launch_join<T, ACT>(b.t.epi, b.t.part, p.splits, stream);
}

template <class T>
static int lt_gemm8_launch_impl(const LtTile8Args& b, const LtPlan& p, int act, hipStream_t stream) {
  switch (act) {
    case LT_ACT_RELU: return lt_gemm8_launch_act<T, LT_ACT_RELU>(b, p, stream);
    case LT_ACT_GELU: return lt_gemm8_launch_act<T, LT_ACT_GELU>(b, p, stream);
    case LT_ACT_SILU: return lt_gemm8_launch_act<T, LT_ACT_SILU>(b, p, stream);
    default: return lt_gemm8_launch_act<T, LT_ACT_NONE>(b, p, stream);
  }
}
