// Dense operators (linear, rms_norm, 8-bit checkpoints): types, 8-bit formats, epilogue.  gfx950.
#pragma once
#include "common.h"
#include "../../include/latte_hip.h"

typedef __bf16 lt_bf16;
typedef _Float16 lt_f16;
typedef float lt_f32x4 __attribute__((ext_vector_type(4)));
typedef int lt_i32x4 __attribute__((ext_vector_type(4)));
typedef int lt_i32x8 __attribute__((ext_vector_type(8)));
typedef short lt_s16x4 __attribute__((ext_vector_type(4)));
typedef short lt_s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 lt_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lt_f16x8 __attribute__((ext_vector_type(8)));
#define LT_LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))

template <class T> struct LtType;   // kMaxExp: the exponent of the type's last binade
template <> struct LtType<float> { static constexpr int id = LT_DT_F32, kMaxExp = 127; };
template <> struct LtType<lt_bf16> { static constexpr int id = LT_DT_BF16, kMaxExp = 127; };
template <> struct LtType<lt_f16> { static constexpr int id = LT_DT_F16, kMaxExp = 15; };
static inline int lt_dt_size(int dt) { return dt == LT_DT_F32 ? 4 : 2; }

// ---- guarded vector access: n = elements that exist (<= 0: none); rows may start at any element, the hardware takes
// unaligned 16-, 8- and 4-byte accesses, so only the end of a row goes element by element
template <class T, int V>
__device__ __forceinline__ void lt_ldv(const T* p, int64_t n, float (&o)[V]) {
  if (n >= V) {
    T t[V];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < n ? (float)p[i] : 0.f;
  }
}
template <class T, int V>
__device__ __forceinline__ void lt_stv(T* p, int64_t n, const float (&o)[V]) {
  if (n >= V) {
    T t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)o[i];
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = (T)o[i];
  }
}

// i = q * d + r; 64-bit division costs some hundred instructions, so it is left to indexes that need it
__device__ __forceinline__ void lt_divmod(int64_t i, int d, int64_t& q, int& r) {
  if ((uint64_t)i >> 32 == 0) {
    const unsigned u = (unsigned)i / (unsigned)d;
    q = u;
    r = (int)((unsigned)i - u * (unsigned)d);
  } else {
    q = i / d;
    r = (int)(i - q * d);
  }
}

// ---- mx8: 32 neighbours of a row share the scale 2^E, E the smallest integer with amax <= 448 * 2^E (amax over the
// finite values; 448 is e4m3's largest), never below -126; the scale byte is E + 127.  Nothing saturates, so a value that
// is held reads back within 2^-4 of itself (2^-10 * 2^E at the bottom).  Where the block's largest value lies in the last
// binade of its type and above 1.75 times its power of two, 256 * 2^E is infinite in that type and larger than all of them:
// values are then cut at 240 * 2^E, which is within 2^-4 of everything above it.  (A y that is computed in fp32 and lies
// beyond float16 is held as it is.)  Infinities and NaN are held as NaN, each in its own place.
__device__ __forceinline__ int lt_mx8_exp(float amax) {
  const unsigned u = __float_as_uint(amax);            // finite and >= 0
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // mantissa over 1.75: one more
  return e < -126 ? -126 : e;
}
__device__ __forceinline__ float lt_two_to(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float lt_finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.4028234663852886e38f ? a : 0.f;
}
// two values at scale inv = 2^-E, |v * inv| <= 448, cut at lim -> two e4m3 bytes in the low half
__device__ __forceinline__ int lt_mx8_pack2(float a, float b, float inv, float lim) {
  const float u = __builtin_amdgcn_fmed3f(a * inv, -lim, lim) + (a - a);   // a - a: 0, or NaN where a is not finite
  const float v = __builtin_amdgcn_fmed3f(b * inv, -lim, lim) + (b - b);
  return __builtin_amdgcn_cvt_pk_fp8_f32(u, v, 0, false);
}
__device__ __forceinline__ float lt_mx8_lim(float amax, int e, int max_exp) {
  return (int)(__float_as_uint(amax) >> 23) - 127 == max_exp && e + 8 > max_exp ? 240.f : 448.f;
}
template <int WHICH>   // bytes 2 * WHICH, 2 * WHICH + 1 of a word of four e4m3 values, times s = 2^E
__device__ __forceinline__ void lt_mx8_get2(int word, float s, float& a, float& b) {
  auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, s, WHICH != 0);
  a = v[0];
  b = v[1];
}

// 8 neighbours of a row whose block of 32 the four lanes of an aligned group hold together (all four must call): n = how
// many of the 8 exist (<= 0: none, nothing is stored), q / sc = where they and the block's scale go
__device__ __forceinline__ void lt_mx8_put8(const float (&v)[8], int n, int max_exp, uint8_t* q, uint8_t* sc) {
  float a = 0.f;
#pragma unroll
  for (int t = 0; t < 8; ++t) a = fmaxf(a, t < n ? lt_finite_abs(v[t]) : 0.f);
  a = fmaxf(a, __shfl_xor(a, 1, 64));
  a = fmaxf(a, __shfl_xor(a, 2, 64));
  if (n <= 0) return;
  const int e = lt_mx8_exp(a);
  const float inv = lt_two_to(-e), lim = lt_mx8_lim(a, e, max_exp);
  int w[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
    w[t] = (lt_mx8_pack2(v[4 * t], v[4 * t + 1], inv, lim) & 0xFFFF) | (lt_mx8_pack2(v[4 * t + 2], v[4 * t + 3], inv, lim) << 16);
  if (n >= 8) __builtin_memcpy(q, w, 8);
  else
    for (int t = 0; t < n; ++t) q[t] = (uint8_t)(w[t >> 2] >> (8 * (t & 3)));
  if ((threadIdx.x & 3) == 0) *sc = (uint8_t)(e + 127);
}
__device__ __forceinline__ void lt_mx8_get8(const uint8_t* q, int n, uint8_t sc, float (&v)[8]) {
  int w[2] = {0, 0};
  if (n >= 8) __builtin_memcpy(w, q, 8);
  else
    for (int t = 0; t < n; ++t) w[t >> 2] |= (int)q[t] << (8 * (t & 3));
  const float s = __uint_as_float((unsigned)sc << 23);
  lt_mx8_get2<0>(w[0], s, v[0], v[1]);
  lt_mx8_get2<1>(w[0], s, v[2], v[3]);
  lt_mx8_get2<0>(w[1], s, v[4], v[5]);
  lt_mx8_get2<1>(w[1], s, v[6], v[7]);
}

// ---- activations and their derivatives
// act'(z) in a byte: (c - 32) / 192, c = 0..254 (0 and 1 exactly; gelu' and silu' stay inside [-0.13, 1.13]); 255 is NaN.
__device__ __forceinline__ unsigned lt_deriv_byte(float d) {
  const float c = rintf(__builtin_amdgcn_fmed3f(__fmaf_rn(d, 192.f, 32.f), 0.f, 254.f));
  return d == d ? (unsigned)c : 255u;
}
__device__ __forceinline__ float lt_deriv_value(unsigned c) {
  return c == 255u ? __builtin_nanf("") : ((float)(int)c - 32.f) * (1.f / 192.f);
}
// act'(z) beside 16-bit results, no checkpoint: the same grid in 16 bits, (c - 8192) / 49152, |error| <= 1e-5.  A 16-bit
// float would be off by up to 2^-9 of act' and, with dz rounded to the type as well, double the variance of every gradient.
__device__ __forceinline__ unsigned lt_deriv_word(float d) {
  const float c = rintf(__builtin_amdgcn_fmed3f(__fmaf_rn(d, 49152.f, 8192.f), 0.f, 65534.f));
  return d == d ? (unsigned)c : 65535u;
}
__device__ __forceinline__ float lt_deriv_word_value(unsigned c) {
  return c == 65535u ? __builtin_nanf("") : ((float)(int)c - 8192.f) * (1.f / 49152.f);
}
// y = act(z), d = act'(z).  FAST (16-bit results): the hardware's exp2 and reciprocal, and the normal distribution's tail as
// Phi(-a) = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a), P of degree 5.  Its coefficients are a linear program's least largest error
// over a = 0 .. 19, weighted so that Phi is within 4e-7 and, however small, within 3.2e-5 of itself (in fp32): for z < 0 the
// result is z Phi(z), and an error that is only small beside 1 would be several bf16 steps of it.  fp32: the library's functions.
template <int ACT, bool FAST>
__device__ __forceinline__ void lt_act(float z, float& y, float& d) {
  if constexpr (ACT == LT_ACT_RELU) {
    const bool off = z <= 0.f;   // NaN: neither value nor gradient is cut
    y = off ? 0.f : z;
    d = off ? 0.f : 1.f;
  } else if constexpr (ACT == LT_ACT_GELU) {
    float cdf, e;
    if constexpr (FAST) {
      e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);   // exp(-z^2 / 2)
      const float t = __builtin_amdgcn_rcpf(__fmaf_rn(0.3f, fabsf(z), 1.f));
      float p = __fmaf_rn(-0.0782357082f, t, 0.218392029f);
      p = __fmaf_rn(p, t, -0.0182251427f);
      p = __fmaf_rn(p, t, 0.144031808f);
      p = __fmaf_rn(p, t, 0.114006624f);
      p = __fmaf_rn(p, t, 0.12003047f);
      const float tail = p * t * e;   // Phi(-|z|)
      cdf = z < 0.f ? tail : 1.f - tail;
    } else {
      cdf = 0.5f * erfcf(z * -0.70710678118654752f);
      e = expf(-0.5f * z * z);
    }
    y = z * cdf;
    d = __fmaf_rn(z * 0.39894228040143268f, e, cdf);
  } else if constexpr (ACT == LT_ACT_SILU) {
    float s;
    if constexpr (FAST) s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
    else s = 1.f / (1.f + expf(-z));
    y = z * s;
    d = s * __fmaf_rn(z, 1.f - s, 1.f);
  } else {
    y = z;
    d = 1.f;
  }
}

// ---- epilogue of a product: y = act(z + bias) + residual, and what the backward pass keeps of act'
struct LtEpi {
  const void* bias;     // [cols], the type of y, or NULL
  const void* res;      // [rows][ldres], or NULL
  int64_t ldres;
  void* out;            // [rows][ldo]
  int64_t ldo;
  void* deriv;          // LT_DERIV_BITS: uint16 [rows][ceil(cols/16)]; _BYTE: uint8 [rows][cols]; _FULL: fp32, or
                        // uint16 beside 16-bit results, [rows][cols]
  int dkind;
  int64_t rows;
  int cols;
};

// eight neighbours (row, col..col+7) of the product, n of which exist (<= 0: nothing to do), with their residual (loaded
// ahead: the stores in between would hold the loads back)
// EVEN: n is 8 or more, or 0 and less -- straight-line code, no element by element ends
template <class T, bool EVEN>
__device__ __forceinline__ void lt_epi_res(const LtEpi& e, int64_t row, int col, int n, float (&r)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = 0.f;
  if (e.res && n > 0) lt_ldv<T, 8>((const T*)e.res + row * e.ldres + col, EVEN ? 8 : n, r);
}
template <class T, int ACT, bool EVEN>
__device__ __forceinline__ void lt_epi8(const LtEpi& e, const float (&z)[8], const float (&b)[8], const float (&r)[8], int64_t row,
                                        int col, int n_) {
  if (n_ <= 0) return;
  const int n = EVEN ? 8 : n_;
  float y[8], d[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) lt_act<ACT, sizeof(T) == 2>(z[i] + b[i], y[i], d[i]);
  if constexpr (ACT == LT_ACT_RELU) {
    if (e.dkind == LT_DERIV_BITS) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m |= d[i] != 0.f ? 1u << i : 0u;
      ((uint8_t*)e.deriv)[row * (((e.cols + 15) >> 4) * 2) + (col >> 3)] = (uint8_t)m;
    }
  } else if constexpr (ACT != LT_ACT_NONE) {
    if (e.dkind == LT_DERIV_BYTE) {
      uint8_t* p = (uint8_t*)e.deriv + row * e.cols + col;
      uint8_t c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = (uint8_t)lt_deriv_byte(d[i]);
      if (n >= 8) __builtin_memcpy(p, c, 8);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) p[i] = c[i];
    } else if (e.dkind == LT_DERIV_FULL) {
      if constexpr (sizeof(T) == 4) lt_stv<float, 8>((float*)e.deriv + row * e.cols + col, n, d);
      else {
        uint16_t* p = (uint16_t*)e.deriv + row * e.cols + col;
        uint16_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = (uint16_t)lt_deriv_word(d[i]);
        if (n >= 8) __builtin_memcpy(p, c, 16);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = c[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] += r[i];
  lt_stv<T, 8>((T*)e.out + row * e.ldo + col, n, y);
}

// out[c] = sum over slabs of part[slab][c]: 16 columns a workgroup, 16 threads a column, fixed order
template <class T>
__global__ __launch_bounds__(256) void k_col_join(const float* __restrict__ part, int slabs, int N, T* __restrict__ out) {
  __shared__ float s_sum[16][17];
  const int c = threadIdx.x & 15, l = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < N) {
#pragma unroll 8
    for (int i = l; i < slabs; i += 16) s += part[(int64_t)i * N + col];
  }
  s_sum[l][c] = s;
  __syncthreads();
  if (l == 0 && col < N) {
    for (int i = 1; i < 16; ++i) s += s_sum[i][c];
    out[col] = (T)s;
  }
}

// ---- host side
// dispatch over the value types: expression F<T>(...) with T bound
#define LT_DENSE_TYPES(dt, ...)                                    \
  do {                                                             \
    if ((dt) == LT_DT_F32) { using T = float; __VA_ARGS__; }       \
    else if ((dt) == LT_DT_BF16) { using T = lt_bf16; __VA_ARGS__; } \
    else { using T = lt_f16; __VA_ARGS__; }                        \
  } while (0)

// Launches go to `stream`'s device, whatever device the calling thread has current (the null stream: the current device).
struct LtOnStream {
  int prev = -1;
  bool switched = false;
  int enter(hipStream_t stream) {
    if (!stream) return LT_OK;
    int dev = -1;
    LT_CHECK_HIP(hipGetDevice(&prev));
    LT_CHECK_HIP(hipStreamGetDevice(stream, &dev));
    if (dev != prev) {
      LT_CHECK_HIP(hipSetDevice(dev));
      switched = true;
    }
    return LT_OK;
  }
  ~LtOnStream() {
    if (switched) (void)hipSetDevice(prev);
  }
};

// a product out[i][j] = sum_k Q(i,k) P(j,k), i < rows, j < cols, k < depth, for the dispatchers in dense_*.hip.
// *_kmajor: the operand lies [k][i or j] instead of [i or j][k].
struct LtGemm {
  const void* P;
  const void* Q;
  const void* Q2;            // or NULL: a second term of Q, laid out like it
  int64_t ldp, ldq;
  int64_t rows, depth;
  int cols;
  int dt;
  bool p_kmajor, q_kmajor;
  bool padded;               // 16-byte pieces that reach past a line's end read zeros (or nothing that an output takes)
  const uint8_t* p_scales;   // P is mx8 (k-major only): e4m3 values [k][ldp], scales [k][ceil(cols/32)]
  int act;
  LtEpi epi;
};
