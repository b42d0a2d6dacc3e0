// The tiled product of the dense operators, and its joins.  out[i][j] = sum_k Q(i,k) P(j,k).
//
// The matrix instructions compute D = A B with A = P (output columns) and B = Q (output rows): a lane then holds four
// neighbouring COLUMNS of one output row.  A workgroup owns a BR x BC tile of the output and walks k.
// k in steps of 128 bytes (64 16-bit or 32 fp32 values) through two LDS buffers, one barrier a step: while the step's
// matrix instructions run, the next step's tiles are on the way.  Tiles go from memory straight into LDS where lines are
// 16-byte aligned, through registers elsewhere (and where mx8 is widened on the way).
//   8192 x 4096 -> 4096, bf16: 210 to 219 us, 1250 to 1310 TFLOP/s (224 us with a residual); steps of 64 bytes through four buffers, three
//   steps ahead: 253 us -- the barriers and the 64-byte requests cost more than the distance gives.
//
// LDS images, 16-byte chunks:
//   operand [i][k]  (k runs along memory)  : tile [R][BKB], chunk c of row i at position c ^ rswz(i)
//   operand [k][i]  (i runs along memory)  : tile [BK][R], chunk c of line k at position c ^ kswz(k); 16-bit fragments are
//                                            read with the transposing LDS read (4 lines x 16 columns)
// Both spread the lanes that are served together over all banks (conflicts: 2 % of the LDS cycles).
#pragma once
#include "dense.h"

struct LtTileArgs {
  const char* P;
  const char* Q;
  const char* Q2;         // or NULL: the sum goes over Q and, once more with the same P, over Q2 (laid out like Q)
  int64_t ldp, ldq;       // bytes
  int64_t rows, depth;
  int cols;
  int tr, tc;             // tiles along rows / columns
  int splits;
  int64_t slice;          // k per split, a multiple of BK
  float* part;            // [splits][rows][cols] when splits > 1
  const uint8_t* ps;      // scales of an mx8 P
  int64_t ldps;
  LtEpi epi;
};

template <class T> struct LtMma;
template <> struct LtMma<lt_bf16> {
  typedef lt_bf16x8 frag;
  static __device__ __forceinline__ lt_f32x4 mma(frag a, frag b, lt_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct LtMma<lt_f16> {
  typedef lt_f16x8 frag;
  static __device__ __forceinline__ lt_f32x4 mma(frag a, frag b, lt_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct LtMma<float> {
  typedef lt_f32x4 frag;   // four k of one row: k = 16 j + 4 g + t goes into instruction t (the same for both operands)
  static __device__ __forceinline__ lt_f32x4 mma(frag a, frag b, lt_f32x4 c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
    return c;
  }
};

// acc[i][j] += P_j Q_i for a block of fragments: fp32 goes round the block four times, so that no
// instruction waits for the one just before it (k_rows_bwd, 310017 x 128 -> 96, fp32: 240.5 -> 237.8 us)
template <class T, int FR, int FC>
__device__ __forceinline__ void lt_mma_block(const typename LtMma<T>::frag (&p)[FC], const typename LtMma<T>::frag (&q)[FR],
                                             lt_f32x4 (&acc)[FR][FC]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[j][t], q[i][t], acc[i][j], 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int j = 0; j < FC; ++j) acc[i][j] = LtMma<T>::mma(p[j], q[i], acc[i][j]);
  }
}

template <> struct LtMma<uint8_t> { typedef lt_i32x8 frag; };   // mx8: dense8.h

template <class T, bool KM, int R, int BKB>   // an operand's tile: R rows (or columns) of the product, BKB bytes' worth of k
struct LtTile {
  static constexpr int SZ = sizeof(T), CH = 16 / SZ, BK = BKB / SZ;
  static constexpr int BYTES = R * BKB, SEGS = BYTES / 1024;
  static constexpr int CPL = KM ? R / CH : BKB / 16;   // chunks per line
  // rows of 128 (64) bytes meet in a bank every 2 (4) rows
  static __device__ __forceinline__ int rswz(int i) { return BKB == 128 ? i & 7 : (i >> 2) & 3; }
  // k-major lines of one fragment read must not meet in a bank: 16-bit reads take 32 bytes of lines k0 + {0..3} per 16
  // lanes, fp32 reads 64 bytes of lines k0 + {0, 4, 8, 12}
  static __device__ __forceinline__ int kswz(int k) {
    if constexpr (SZ == 2) return (((k & 3) | ((k >> 1) & 4)) << 1) & (CPL - 1);
    else return (((k >> 2) & 3) << 2) & (CPL - 1);
  }
  // chunk L (linear position in the image) -> its line and its chunk within the line in memory
  static __device__ __forceinline__ void where(int L, int& line, int& c) {
    line = L / CPL;
    c = (L % CPL) ^ (KM ? kswz(line) : rswz(line));
  }
  // fragment kk of the 16 rows from i0: k = kk * KF + ..., KF = 32 (16-bit) or 16 (fp32)
  static __device__ __forceinline__ typename LtMma<T>::frag frag(const char* t, int i0, int kk, int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!KM) {
      const int i = i0 + r, c = kk * 4 + g;
      return *reinterpret_cast<const typename LtMma<T>::frag*>(t + i * BKB + ((c ^ rswz(i)) << 4));
    } else if constexpr (SZ == 2) {
      const int k = kk * 32 + 8 * g + (r >> 2), col = i0 + 4 * (r & 3);
      const char* p = t + k * (R * 2) + (((col >> 3) ^ kswz(k)) << 4) + (col & 7) * 2;   // kswz(k + 4) == kswz(k)
      union { lt_s16x4 h[2]; typename LtMma<T>::frag f; } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LT_LDS_PTR(lt_s16x4, p));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LT_LDS_PTR(lt_s16x4, p + 4 * (R * 2)));
      return u.f;
    } else {
      const int col = i0 + r;
      typename LtMma<T>::frag f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = kk * 16 + 4 * g + q;
        f[q] = *reinterpret_cast<const float*>(t + k * (R * 4) + (((col >> 2) ^ kswz(k)) << 4) + (col & 3) * 4);
      }
      return f;
    }
  }
};

// 64 lanes x 16 bytes from memory to 1024 consecutive bytes of LDS (device pass only: the host pass knows no 16-byte form)
__device__ __forceinline__ void lt_load_lds16(const char* base, char* lds, unsigned off) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x7FFFFFFF, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LT_LDS_PTR(void, lds), 16, off, 0, 0, 0);
#endif
}

// ---- staging straight into LDS.  Lines or chunks that do not exist get an offset past the descriptor's range, which
// loads zeros.  Needs 16-byte aligned lines, k (or the columns, k-major) in whole chunks, and tiles below 2 GiB.
template <class TL, bool KM, int NW>
struct LtDirect {
  // where there are fewer 1024-byte pieces than waves, several waves load the same piece
  static constexpr int N = TL::SEGS >= NW ? TL::SEGS / NW : 1;
  static_assert(TL::SEGS % NW == 0 || NW % TL::SEGS == 0, "pieces and waves");
  static __device__ __forceinline__ int seg(int wave, int i) { return TL::SEGS >= NW ? wave + i * NW : wave % TL::SEGS; }
  unsigned off[N];
  __device__ __forceinline__ void init(int64_t ld, int64_t n_lines_or_cols, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int line, c;
      TL::where(seg(wave, i) * 64 + lane, line, c);
      const bool ok = KM ? c * TL::CH < n_lines_or_cols : line < n_lines_or_cols;
      off[i] = ok ? (unsigned)(line * ld + c * 16) : 0x80000000u;
    }
  }
  // kleft: how much of k is left from this step on (may exceed BK)
  __device__ __forceinline__ void load(const char* base, char* lds, int64_t kleft, int wave, int lane) const {
    if (kleft >= TL::BK) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        lt_load_lds16(base, lds + seg(wave, i) * 1024, off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int line, c;
        TL::where(seg(wave, i) * 64 + lane, line, c);
        const bool ok = KM ? line < kleft : c * TL::CH < kleft;
        lt_load_lds16(base, lds + seg(wave, i) * 1024, ok ? off[i] : 0x80000000u);
      }
    }
  }
};

// ---- staging through registers: any alignment, any length; an mx8 operand is widened on the way
template <class T, class TL, bool KM, bool MX8, int NT>
struct LtStaged {
  static constexpr int N = TL::BYTES / 16 / NT;
  lt_i32x4 v[N];
  __device__ __forceinline__ void load(const char* base, int64_t ld, int64_t n_lines_or_cols, int64_t kleft, const uint8_t* sc,
                                       int64_t ldsc, int col0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int line, c;
      TL::where(tid + i * NT, line, c);
      const bool line_ok = KM ? line < kleft : line < n_lines_or_cols;
      const int64_t n = line_ok ? (KM ? n_lines_or_cols : kleft) - c * TL::CH : 0;
      lt_i32x4 w = {0, 0, 0, 0};
      if constexpr (MX8) {
        if (n > 0) {
          const char* p = base + line * ld + c * TL::CH;
          const float s = __uint_as_float((unsigned)sc[line * ldsc + ((col0 + c * TL::CH) >> 5)] << 23);
          int q[2] = {0, 0};
          if (n >= TL::CH) __builtin_memcpy(q, p, TL::CH);
          else {
            unsigned long long b = 0;
            for (int j = 0; j < n; ++j) b |= (unsigned long long)(uint8_t)p[j] << (8 * j);
            q[0] = (int)b;
            q[1] = (int)(b >> 32);
          }
          if constexpr (sizeof(T) == 4) {
            float a[4];
            lt_mx8_get2<0>(q[0], s, a[0], a[1]);
            lt_mx8_get2<1>(q[0], s, a[2], a[3]);
            __builtin_memcpy(&w, a, 16);
          } else {
            T a[8];   // e4m3 times a power of two has 4 bits: exact in either 16-bit type
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float f[4];
              lt_mx8_get2<0>(q[j], s, f[0], f[1]);
              lt_mx8_get2<1>(q[j], s, f[2], f[3]);
#pragma unroll
              for (int t = 0; t < 4; ++t) a[4 * j + t] = (T)f[t];
            }
            __builtin_memcpy(&w, a, 16);
          }
        }
      } else {
        const char* p = base + line * ld + c * 16;
        if (n >= TL::CH) __builtin_memcpy(&w, p, 16);
        else if (n > 0) {
          T a[TL::CH];
#pragma unroll
          for (int j = 0; j < TL::CH; ++j) a[j] = j < n ? reinterpret_cast<const T*>(p)[j] : (T)0.f;
          __builtin_memcpy(&w, a, 16);
        }
      }
      v[i] = w;
    }
  }
  __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<lt_i32x4*>(lds + (tid + i * NT) * 16) = v[i];
  }
};

// workgroup id -> work: consecutive pieces go to one XCD (ids are dealt to the 8 XCDs in turn), so tiles that share
// operands share an L2; a bijection for any count
__device__ __forceinline__ unsigned lt_xcd_map(unsigned b, unsigned n) {
  const unsigned per = n >> 3, rem = n & 7, x = b & 7;
  return x * per + (x < rem ? x : rem) + (b >> 3);
}

// A wave's accumulators -> partial sums of its split, or the epilogue; (row0, col0) = the wave's corner, s = its piece of
// LDS (the tiles are no longer read).  A lane's four columns of one row would make stores of 16 bytes a row and line, so 16
// rows at a time turn through LDS and leave eight columns a lane: whole 128-byte lines of 16-bit results.
template <int FC> struct LtTurn { static constexpr int LD = 16 * FC + 4, BYTES = 16 * LD * 4; };
template <class T, int FR, int FC, int ACT, bool EVEN>
__device__ __forceinline__ void lt_tile_store_(const LtTileArgs& a, const lt_f32x4 (&acc)[FR][FC], unsigned split, int64_t row0, int col0,
                                               int lane, float* s) {
  constexpr int LD = LtTurn<FC>::LD, LPR = FC * 2, RPP = 64 / LPR < 16 ? 64 / LPR : 16, PASS = 16 / RPP;   // lanes a row, rows a pass
  const int r = lane & 15, g = lane >> 4;
  const int pr = lane / LPR, col = col0 + (lane % LPR) * 8;
  const bool use = lane < LPR * RPP;
  const int64_t nc = use ? a.cols - col : 0;
  float b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.f;
  if (a.splits == 1 && a.epi.bias && nc > 0) lt_ldv<T, 8>((const T*)a.epi.bias + col, EVEN ? 8 : nc, b);
#pragma unroll
  for (int i = 0; i < FR; ++i) {
    float res[PASS][8];
    if (a.splits == 1) {
#pragma unroll
      for (int p = 0; p < PASS; ++p) {
        const int64_t row = row0 + 16 * i + p * RPP + pr;
        lt_epi_res<T, EVEN>(a.epi, row, col, row < a.rows ? (int)nc : 0, res[p]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the rows before have been read
#pragma unroll
    for (int j = 0; j < FC; ++j) *reinterpret_cast<lt_f32x4*>(s + r * LD + 16 * j + 4 * g) = acc[i][j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int64_t row = row0 + 16 * i + p * RPP + pr;
      const int n = row < a.rows ? (int)nc : 0;
      float z[8];
      if (use) {
        const float* src = s + (p * RPP + pr) * LD + (lane % LPR) * 8;
        const lt_f32x4 u = *reinterpret_cast<const lt_f32x4*>(src), v = *reinterpret_cast<const lt_f32x4*>(src + 4);
#pragma unroll
        for (int t = 0; t < 4; ++t) z[t] = u[t], z[4 + t] = v[t];
      }
      if (a.splits > 1) {
        if (n > 0) lt_stv<float, 8>(a.part + ((int64_t)split * a.rows + row) * a.cols + col, EVEN ? 8 : n, z);
      } else {
        lt_epi8<T, ACT, EVEN>(a.epi, z, b, res[p], row, col, n);
      }
    }
  }
}

// wait for the wave's own loads and LDS reads, then for the other waves
__device__ __forceinline__ void lt_wait_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <class T, int FR, int FC, int ACT>
__device__ __forceinline__ void lt_tile_store(const LtTileArgs& a, const lt_f32x4 (&acc)[FR][FC], unsigned split, int64_t row0, int col0,
                                              int lane, float* s) {
  if (a.cols % 8 == 0) lt_tile_store_<T, FR, FC, ACT, true>(a, acc, split, row0, col0, lane, s);
  else lt_tile_store_<T, FR, FC, ACT, false>(a, acc, split, row0, col0, lane, s);
}

template <class T, bool PKM, bool QKM, int BR, int BC, int WR, int WC, bool DIRECT, bool P8, int ACT>
__global__ __launch_bounds__(64 * WR * WC) void k_dense(LtTileArgs a) {
  constexpr int BKB = 128, NBUF = 2;
  typedef LtTile<T, PKM, BC, BKB> TP;
  typedef LtTile<T, QKM, BR, BKB> TQ;
  constexpr int NW = WR * WC, NT = 64 * NW, FR = BR / WR / 16, FC = BC / WC / 16;
  constexpr int BUF = TP::BYTES + TQ::BYTES;
  extern __shared__ __attribute__((aligned(1024))) char s_tile[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // eight row tiles x all column tiles form a group: its operands stay in the L2 of the XCD that works on it
  const unsigned tiles = (unsigned)a.tr * a.tc;
  const unsigned L = lt_xcd_map(blockIdx.x, tiles * a.splits);
  const unsigned split = L / tiles, t_ = L % tiles;
  const unsigned grp = t_ / (8u * a.tc), in = t_ - grp * 8u * a.tc;
  const unsigned gr = (unsigned)a.tr - grp * 8u < 8u ? (unsigned)a.tr - grp * 8u : 8u;
  const int64_t row0 = (int64_t)(grp * 8u + in % gr) * BR;
  const int col0 = (int)(in / gr) * BC;
  const int64_t k0 = split * a.slice;
  const int64_t kend = k0 + a.slice < a.depth ? k0 + a.slice : a.depth;
  const int nk1 = (int)((kend - k0 + TP::BK - 1) / TP::BK), nk = a.Q2 ? 2 * nk1 : nk1;
  constexpr int PS = P8 ? 1 : (int)sizeof(T);
  const char* pb = a.P + (PKM ? k0 * a.ldp + (int64_t)col0 * PS : col0 * a.ldp + k0 * PS);
  const int64_t qoff = QKM ? k0 * a.ldq + row0 * (int64_t)sizeof(T) : row0 * a.ldq + k0 * (int64_t)sizeof(T);
  const int64_t pstep = PKM ? TP::BK * a.ldp : TP::BK * PS, qstep = QKM ? TQ::BK * a.ldq : BKB;
  const int64_t pn = a.cols - col0, qn = a.rows - row0;
  const uint8_t* psc = P8 ? a.ps + k0 * a.ldps : nullptr;
  auto qbase = [&](int t) { return (t < nk1 ? a.Q : a.Q2) + qoff; };   // step t of nk is step t % nk1 along k
  auto kstep = [&](int t) { return t < nk1 ? t : t - nk1; };

  lt_f32x4 acc[FR][FC];
#pragma unroll
  for (int i = 0; i < FR; ++i)
#pragma unroll
    for (int j = 0; j < FC; ++j) acc[i][j] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};
  const int wr = (wave / WC) * (BR / WR), wc = (wave % WC) * (BC / WC);

  // all of the step's fragments are asked for first, the matrix instructions start with the first that arrive; ahead() =
  // what else to set going in between
  auto compute = [&](const char* buf, auto ahead) {
    constexpr int KK = BKB / 64;
    typename LtMma<T>::frag p[KK][FC], q[KK][FR];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
      for (int j = 0; j < FC; ++j) p[kk][j] = TP::frag(buf, wc + 16 * j, kk, lane);
#pragma unroll
      for (int i = 0; i < FR; ++i) q[kk][i] = TQ::frag(buf + TP::BYTES, wr + 16 * i, kk, lane);
    }
    ahead();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) lt_mma_block<T, FR, FC>(p[kk], q[kk], acc);
  };

  if constexpr (DIRECT) {
    LtDirect<TP, PKM, NW> sp;
    LtDirect<TQ, QKM, NW> sq;
    sp.init(a.ldp, pn, wave, lane);
    sq.init(a.ldq, qn, wave, lane);
    auto issue = [&](int t) {
      const int kt = kstep(t);
      const int64_t left = kend - k0 - (int64_t)kt * TP::BK;
      char* buf = s_tile + (t % NBUF) * BUF;
      sp.load(pb + kt * pstep, buf, left, wave, lane);
      sq.load(qbase(t) + kt * qstep, buf + TP::BYTES, left, wave, lane);
    };
    issue(0);
    for (int t = 0; t < nk; ++t) {
      // this step's tiles have landed, and nobody reads the buffer of step t - 1 any more
      lt_wait_barrier();
      compute(s_tile + (t % NBUF) * BUF, [&]() {
        if (t + 1 < nk) issue(t + 1);
      });
    }
  } else {
    LtStaged<T, TP, PKM, P8, NT> sp;
    LtStaged<T, TQ, QKM, false, NT> sq;
    auto get = [&](int t) {
      const int kt = kstep(t);
      const int64_t left = kend - k0 - (int64_t)kt * TP::BK;
      sp.load(pb + kt * pstep, a.ldp, pn, left, P8 ? psc + kt * (TP::BK * a.ldps) : nullptr, a.ldps, col0, tid);
      sq.load(qbase(t) + kt * qstep, a.ldq, qn, left, nullptr, 0, 0, tid);
    };
    get(0);
    for (int t = 0; t < nk; ++t) {
      char* cur = s_tile + (t & 1) * BUF;
      sp.store(cur, tid);      // its last readers passed the barrier of step t - 1
      sq.store(cur + TP::BYTES, tid);
      __syncthreads();
      if (t + 1 < nk) get(t + 1);
      compute(cur, [] {});
    }
  }

  static_assert(NW * LtTurn<FC>::BYTES <= NBUF * BUF, "the turned rows do not fit the tiles' LDS");
  __syncthreads();
  lt_tile_store<T, FR, FC, ACT>(a, acc, split, row0 + wr, col0 + wc, lane,
                                reinterpret_cast<float*>(s_tile + wave * LtTurn<FC>::BYTES));
}

// out = epilogue(sum over the splits, in a fixed order: the same bits every time).  G threads share eight neighbours and take
// the splits in turn; one thread adding up 256 splits alone would wait for memory 256 times.
template <class T, int ACT, int G>
__global__ __launch_bounds__(256) void k_dense_join(const float* __restrict__ part, int splits, LtEpi e) {
  constexpr int EL = 256 / G;
  __shared__ float s_sum[G > 1 ? G : 1][8][EL];
  const int el = threadIdx.x % EL, sl = threadIdx.x / EL;
  const int c8 = (e.cols + 7) >> 3;
  const int64_t n = e.rows * c8, stride = (int64_t)gridDim.x * EL;
  const int64_t plane = e.rows * e.cols;
  for (int64_t b = blockIdx.x * (int64_t)EL; b < n; b += stride) {
    const int64_t i = b + el;
    int64_t row = 0;
    int col = e.cols;
    if (i < n) {
      lt_divmod(i, c8, row, col);
      col *= 8;
    }
    const int m = e.cols - col;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (m > 0) {
      const float* p = part + row * e.cols + col;
#pragma unroll 4
      for (int s = sl; s < splits; s += G) {
        float v[8];
        lt_ldv<float, 8>(p + s * plane, m, v);
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] += v[t];
      }
    }
    if constexpr (G > 1) {
      __syncthreads();   // the previous turn's sums have been read
#pragma unroll
      for (int t = 0; t < 8; ++t) s_sum[sl][t][el] = acc[t];
      __syncthreads();
      if (sl != 0) continue;
#pragma unroll
      for (int s = 1; s < G; ++s)
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] += s_sum[s][t][el];
    }
    float bias[8], res[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) bias[t] = 0.f;
    if (e.bias) lt_ldv<T, 8>((const T*)e.bias + col, m, bias);
    lt_epi_res<T, false>(e, row, col, m, res);
    lt_epi8<T, ACT, false>(e, acc, bias, res, row, col, m);
  }
}

// the eight waves' sums of 16 columns, added in wave order, and their epilogue
template <class T, int FR, int ACT>
__device__ __forceinline__ void lt_few_store(const LtTileArgs& a, const lt_f32x4 (&acc)[FR], lt_f32x4 (*s_acc)[FR][64], int col0, int wave,
                                             int lane) {
#pragma unroll
  for (int f = 0; f < FR; ++f) s_acc[wave][f][lane] = acc[f];
  __syncthreads();
  lt_f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (wave < FR) {
    s = s_acc[0][wave][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) s += s_acc[w][wave][lane];
  }
  // lane 16 g + r holds columns 4 g .. 4 g + 3 of row r; two lanes' columns make one lane's eight
  lt_f32x4 t;
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = __shfl_xor(s[i], 16, 64);
  const int g = lane >> 4;
  if (wave >= FR || (g & 1)) return;
  const int64_t row = wave * 16 + (lane & 15);
  const int col = col0 + 4 * g, n = row < a.rows ? a.cols - col : 0;
  if (n <= 0) return;
  const float z[8] = {s[0], s[1], s[2], s[3], t[0], t[1], t[2], t[3]};
  float b[8], res[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.f;
  if (a.epi.bias) lt_ldv<T, 8>((const T*)a.epi.bias + col, n, b);
  lt_epi_res<T, false>(a.epi, row, col, n, res);
  lt_epi8<T, ACT, false>(a.epi, z, b, res, row, col, n);
}

// ---- few rows: y[rows <= 32][cols].  Bound by reading P once: a workgroup takes 16 columns, its 8 waves share k in
// turns of four fragments (256 bytes of each of the 16 lines of P), operands go from memory straight into the matrix
// instructions' registers (nothing is used twice but the few rows of Q, which the caches hold), and the waves' sums are
// added through LDS in wave order.
template <class T, int FR, int ACT>
__global__ __launch_bounds__(512) void k_dense_few(LtTileArgs a) {
  typedef typename LtMma<T>::frag Frag;
  constexpr int CH = 16 / sizeof(T), KF = 4 * CH, U = 4;
  __shared__ lt_f32x4 s_acc[8][FR][64];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col0 = blockIdx.x * 16;
  const bool pok = col0 + r < a.cols;
  const T* p = (const T*)(a.P + (int64_t)(pok ? col0 + r : 0) * a.ldp);
  lt_f32x4 acc[FR];
#pragma unroll
  for (int f = 0; f < FR; ++f) acc[f] = (lt_f32x4){0.f, 0.f, 0.f, 0.f};
  auto get = [&](const T* line, bool ok, int64_t k) -> Frag {
    Frag v;
    const int64_t n = ok ? a.depth - k : 0;
    if (n >= CH) __builtin_memcpy(&v, line + k, 16);
    else {
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = j < n ? line[k + j] : (T)0.f;
    }
    return v;
  };
  for (int64_t k = (int64_t)wave * U * KF; k < a.depth; k += 8 * U * KF) {
    Frag pf[U], qf[FR][U];
#pragma unroll
    for (int u = 0; u < U; ++u) pf[u] = get(p, pok, k + u * KF + g * CH);
#pragma unroll
    for (int f = 0; f < FR; ++f) {
      const bool ok = f * 16 + r < a.rows;
      const T* q = (const T*)(a.Q + (int64_t)(ok ? f * 16 + r : 0) * a.ldq);
#pragma unroll
      for (int u = 0; u < U; ++u) qf[f][u] = get(q, ok, k + u * KF + g * CH);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < FR; ++f) acc[f] = LtMma<T>::mma(pf[u], qf[f][u], acc[f]);
  }
  lt_few_store<T, FR, ACT>(a, acc, s_acc, col0, wave, lane);
}
