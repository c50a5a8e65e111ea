// What the 16-bit products do to an element between the accumulator and memory: types,
// activations and their derivatives, loads and stores of eight neighbouring elements.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mfma.h"
#include "rtat_native.h"

namespace rtat_native {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));

// The 16-bit operand types: eight of them as one MFMA operand, and the 16x16x32 MFMA.  Operand
// lane l holds row (column) l % 16 and k = 8 * (l / 16) .. + 7; accumulator register r of lane l
// holds D[4 * (l / 16) + r][l % 16].
template <class T> struct Half;
template <> struct Half<__bf16> {
  typedef bf16x8_t vec_t;
  static constexpr int id = RTAT_TYPE_BF16;
  __device__ static inline f4_t mfma(s8_t a, s8_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec_t, a),
                                                   __builtin_bit_cast(vec_t, b), c, 0, 0, 0);
  }
  __device__ static inline void mfma_into(f4_t& c, s8_t a, s8_t b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
template <> struct Half<_Float16> {
  typedef f16x8_t vec_t;
  static constexpr int id = RTAT_TYPE_F16;
  __device__ static inline f4_t mfma(s8_t a, s8_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec_t, a),
                                                  __builtin_bit_cast(vec_t, b), c, 0, 0, 0);
  }
  __device__ static inline void mfma_into(f4_t& c, s8_t a, s8_t b) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
};
// mfma_into keeps the accumulator in the accumulation registers and its place in the program: a
// wave that holds 256 of them leaves the compiler no room to move them about, which it otherwise
// does every iteration.  The compiler does not see a matrix instruction there, so nothing but
// mfma_into may touch the accumulators until mfma_settle has passed: it waits longer than any
// matrix instruction takes, and hands every accumulator on as a new value, so that no read can
// move in front of it.
template <int M, int N>
__device__ __forceinline__ void mfma_settle(f4_t (&acc)[M][N]) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) asm volatile("" : "+a"(acc[i][j]));
  __builtin_amdgcn_sched_barrier(0);
}
// An accumulator of mfma_into, after mfma_settle.
__device__ __forceinline__ float mfma_get(float a) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
  return v;
}

// Sixteen bytes at an address that is only element-aligned (one global load: the hardware
// accepts any alignment).
struct __attribute__((packed, aligned(2))) Loose16 {
  u4_t v;
};

__device__ inline float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896f); }
__device__ inline float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// Phi(z) and the density phi(z) of the normal distribution.  The tail beyond a = |z| is exp(-a^2 / 2)
// times t q(t), t = 1 / (1 + 0.305 a): a septic fitted for the least largest relative error (9.4e-8
// over 0 <= a <= 14), so that one exponential serves both and small values of z Phi(z) keep their
// leading bits: relative to the tail at most 6.2 half steps of f32 times 1 + a^2, emulated, from
// rounding a^2.  Exactly a half at 0.
__device__ inline void normal_cdf(float z, float& Phi, float& phi) {
  const float e = __builtin_amdgcn_exp2f(z * z * -0.721347520444482f);
  const float t = rcp_fast(__builtin_fmaf(0.305f, __builtin_fabsf(z), 1.0f));
  float q = __builtin_fmaf(0.0366991985f, t, -0.152988333f);
  q = __builtin_fmaf(q, t, 0.185716919f);
  q = __builtin_fmaf(q, t, -0.0379768468f);
  q = __builtin_fmaf(q, t, 0.121021689f);
  q = __builtin_fmaf(q, t, 0.103420865f);
  q = __builtin_fmaf(q, t, 0.12246682f);
  q = __builtin_fmaf(q, t, 0.121639735f);
  const float tail = q * t * e;
  Phi = z < 0.0f ? tail : 1.0f - tail;
  phi = 0.398942280401433f * e;
}

// u of GELU_TANH with the factor two that turns (1 + tanh u) / 2 into a logistic of 2u.
constexpr float GELU_C2 = 1.59576912160573f;  // 2 sqrt(2 / pi)
constexpr float GELU_K = 0.044715f;

__device__ inline float act_value(int act, float z) {
  switch (act) {
    case RTAT_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case RTAT_ACT_GELU: {
      float Phi, phi;
      normal_cdf(z, Phi, phi);
      return z * Phi;
    }
    case RTAT_ACT_GELU_TANH: return z * rcp_fast(1.0f + exp_fast(-GELU_C2 * z * __builtin_fmaf(GELU_K * z, z, 1.0f)));
    case RTAT_ACT_SILU: return z * rcp_fast(1.0f + exp_fast(-z));
    default: return z;
  }
}

// Past +-100 every slope is 0 or 1 to the last bit; the bound keeps infinities and squares that
// overflow out of products with 0.  A NaN stays one.
__device__ inline float act_slope(int act, float z) {
  if (act != RTAT_ACT_RELU) z = z > 100.0f ? 100.0f : (z < -100.0f ? -100.0f : z);
  switch (act) {
    case RTAT_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case RTAT_ACT_GELU: {
      float Phi, phi;
      normal_cdf(z, Phi, phi);
      return __builtin_fmaf(z, phi, Phi);
    }
    case RTAT_ACT_GELU_TANH: {
      const float z2 = z * z;
      const float p = rcp_fast(1.0f + exp_fast(-GELU_C2 * z * __builtin_fmaf(GELU_K, z2, 1.0f)));
      // d(2u)/dz = 2 sqrt(2/pi) (1 + 3 * 0.044715 z^2)
      return p + z * GELU_C2 * __builtin_fmaf(3.0f * GELU_K, z2, 1.0f) * (p * (1.0f - p));
    }
    case RTAT_ACT_SILU: {
      const float p = rcp_fast(1.0f + exp_fast(-z));
      return p * __builtin_fmaf(z, 1.0f - p, 1.0f);
    }
    default: return 1.0f;
  }
}

__host__ __device__ inline int type_bytes(int type) { return type == RTAT_TYPE_F32 ? 4 : 2; }

__device__ inline float half_to_float(int type, uint16_t bits) {
  return type == RTAT_TYPE_BF16 ? (float)__builtin_bit_cast(__bf16, bits)
                                : (float)__builtin_bit_cast(_Float16, bits);
}
// Rounds to nearest even.
__device__ inline uint16_t float_to_half(int type, float x) {
  return type == RTAT_TYPE_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)x)
                                : __builtin_bit_cast(uint16_t, (_Float16)x);
}

__device__ inline float load_one(int type, const void* p, long i) {
  return type == RTAT_TYPE_F32 ? static_cast<const float*>(p)[i]
                               : half_to_float(type, static_cast<const uint16_t*>(p)[i]);
}
__device__ inline void store_one(int type, void* p, long i, float x) {
  if (type == RTAT_TYPE_F32) static_cast<float*>(p)[i] = x;
  else static_cast<uint16_t*>(p)[i] = float_to_half(type, x);
}

// Eight neighbours, at any element-aligned address.
__device__ inline u4_t load16(const void* p, long byte) {
  return reinterpret_cast<const Loose16*>(static_cast<const char*>(p) + byte)->v;
}
__device__ inline void store16(void* p, long byte, u4_t v) {
  reinterpret_cast<Loose16*>(static_cast<char*>(p) + byte)->v = v;
}
__device__ inline void unpack8(int type, u4_t raw, float (&v)[8]) {
  if (type == RTAT_TYPE_BF16) {
    const bf16x8_t h = __builtin_bit_cast(bf16x8_t, raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
  } else {
    const f16x8_t h = __builtin_bit_cast(f16x8_t, raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
  }
}
__device__ inline u4_t pack8(int type, const float (&v)[8]) {
  if (type == RTAT_TYPE_BF16) {
    bf16x8_t h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (__bf16)v[e];
    return __builtin_bit_cast(u4_t, h);
  }
  f16x8_t h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
  return __builtin_bit_cast(u4_t, h);
}
__device__ inline void load8(int type, const void* p, long i, float (&v)[8]) {
  if (type == RTAT_TYPE_F32) {
    const f4_t a = __builtin_bit_cast(f4_t, load16(p, 4 * i));
    const f4_t b = __builtin_bit_cast(f4_t, load16(p, 4 * i + 16));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
    unpack8(type, load16(p, 2 * i), v);
  }
}
__device__ inline void store8(int type, void* p, long i, const float (&v)[8]) {
  if (type == RTAT_TYPE_F32) {
    store16(p, 4 * i, __builtin_bit_cast(u4_t, f4_t{v[0], v[1], v[2], v[3]}));
    store16(p, 4 * i + 16, __builtin_bit_cast(u4_t, f4_t{v[4], v[5], v[6], v[7]}));
  } else {
    store16(p, 2 * i, pack8(type, v));
  }
}

// The first `left` of eight neighbours (all of them from 8 on, none up to 0); the others read as 0
// and are left alone in memory.
__device__ inline u4_t load16_part(const void* p, long i, int left) {
  if (left >= 8) return load16(p, 2 * i);
  const short* at = static_cast<const short*>(p) + i;
  s8_t v = {};
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < left) v[e] = at[e];
  return __builtin_bit_cast(u4_t, v);
}
__device__ inline void load8_part(int type, const void* p, long i, int left, float (&v)[8]) {
  if (left >= 8) {
    load8(type, p, i, v);
  } else if (type == RTAT_TYPE_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? static_cast<const float*>(p)[i + e] : 0.0f;
  } else {
    unpack8(type, load16_part(p, i, left), v);
  }
}
__device__ inline void store8_part(int type, void* p, long i, int left, const float (&v)[8]) {
  if (left >= 8) {
    store8(type, p, i, v);
  } else if (type == RTAT_TYPE_F32) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < left) static_cast<float*>(p)[i + e] = v[e];
  } else {
    const s8_t h = __builtin_bit_cast(s8_t, pack8(type, v));
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < left) static_cast<short*>(p)[i + e] = h[e];
  }
}

// N times eight elements, 32 apart, from element i on; PART: only the first `left` of all.
template <int N, bool PART>
__device__ inline void store_all(int type, void* p, long i, int left, const float (&v)[N][8]) {
#define RTAT_EACH(A)                                                        \
  _Pragma("unroll") for (int q = 0; q < N; ++q) {                           \
    if (PART) store8_part(A, p, i + 32 * q, left - 32 * q, v[q]);           \
    else store8(A, p, i + 32 * q, v[q]);                                    \
  }
  if (type == RTAT_TYPE_BF16) {
    RTAT_EACH(RTAT_TYPE_BF16)
  } else if (type == RTAT_TYPE_F16) {
    RTAT_EACH(RTAT_TYPE_F16)
  } else {
    RTAT_EACH(RTAT_TYPE_F32)
  }
#undef RTAT_EACH
}

// N times eight elements through an activation; the choice is made once for all of them.
// Eight at a time are enough to fill the pipe; all at once would not fit the registers.
template <int N>
__device__ inline void act_values(int act, float (&v)[N][8]) {
#define RTAT_EACH(A)                                     \
  case A:                                                \
    _Pragma("unroll") for (int q = 0; q < N; ++q) {      \
      _Pragma("unroll") for (int i = 0; i < 8; ++i)      \
        v[q][i] = act_value(A, v[q][i]);                 \
      if (N > 1) __builtin_amdgcn_sched_barrier(0);      \
    }                                                    \
    break;
  switch (act) {
    RTAT_EACH(RTAT_ACT_RELU)
    RTAT_EACH(RTAT_ACT_GELU)
    RTAT_EACH(RTAT_ACT_GELU_TANH)
    RTAT_EACH(RTAT_ACT_SILU)
    default: break;
  }
#undef RTAT_EACH
}
// v *= act'(z), z as the 16-bit values in `raw`.
template <int N>
__device__ inline void act_slopes(int act, int type, const u4_t (&raw)[N], float (&v)[N][8]) {
#define RTAT_EACH(A)                                     \
  case A:                                                \
    _Pragma("unroll") for (int q = 0; q < N; ++q) {      \
      float z[8];                                        \
      unpack8(type, raw[q], z);                          \
      _Pragma("unroll") for (int i = 0; i < 8; ++i)      \
        v[q][i] *= act_slope(A, z[i]);                   \
      if (N > 1) __builtin_amdgcn_sched_barrier(0);      \
    }                                                    \
    break;
  switch (act) {
    RTAT_EACH(RTAT_ACT_RELU)
    RTAT_EACH(RTAT_ACT_GELU)
    RTAT_EACH(RTAT_ACT_GELU_TANH)
    RTAT_EACH(RTAT_ACT_SILU)
    default: break;
  }
#undef RTAT_EACH
}
// v += factor * c, c as the 16-bit values in `raw`.
template <int N>
__device__ inline void add_scaled(int type, const u4_t (&raw)[N], float factor, float (&v)[N][8]) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    float c[8];
    unpack8(type, raw[q], c);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[q][i] = __builtin_fmaf(factor, c[i], v[q][i]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// What becomes of the product.  Elements (row, col) with row < rows and col < cols are stored.
//   forward (slope == 0): z = alpha * acc + bias[row]; aux = z; D = act(z) + beta * C
//   gradient (slope == 1): D = alpha * acc * act'(aux); sums += D along the columns
// `copy` receives what D does, in f16; `diag` is added to D(i, i).  `scale`, if given, points to a
// number r per matrix of a batch on the device: alpha is multiplied by r^r_power and, when
// scale_c, beta by r.
struct Epilogue {
  int rows, cols;
  int act, slope;
  float alpha, beta, diag;
  const void* bias;
  int bias_type;
  void* aux;
  long ldaux, aux_stride;
  int aux_type;
  const void* C;
  long ldc, c_stride;
  int c_type;
  void* D;
  long ldd, d_stride;
  int d_type;
  void* copy;
  long ldcopy, copy_stride;
  float* sums;  // gradient: one row of `rows` partial sums per wave column of the launch
  const float* scale;
  int r_power, scale_c;
  int plain;  // nothing but alpha, and D has the operands' type (set by launch_gemm16)
};

__device__ inline void add_diagonal(float diag, int row, int col, float (&v)[8]) {
  if (diag != 0.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += row + i == col ? diag : 0.0f;
  }
}

// Rows row .. row + 7 of column col, batch matrix z: v holds the accumulators and, for a
// gradient, leaves with the values that belong to the row sums (0 outside).
__device__ inline void epilogue8(const Epilogue& e, float alpha, float beta, int row, int col,
                                 long z, float (&v)[8]) {
  if (col >= e.cols || row >= e.rows) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    return;
  }
  const long d_at = z * e.d_stride + row + (long)col * e.ldd;
  const long aux_at = z * e.aux_stride + row + (long)col * e.ldaux;
  const long c_at = z * e.c_stride + row + (long)col * e.ldc;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= alpha;
  const int left = e.rows - row;
  if (e.slope) {
    if (e.act != RTAT_ACT_NONE) {
      const u4_t z8[1] = {load16_part(e.aux, aux_at, left)};
      act_slopes<1>(e.act, e.aux_type, z8, reinterpret_cast<float(&)[1][8]>(v));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? v[i] : 0.0f;
  } else {
    float w[8];
    if (e.bias != nullptr) {
      load8_part(e.bias_type, e.bias, row, left, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += w[i];
    }
    if (e.aux != nullptr) store8_part(e.aux_type, e.aux, aux_at, left, v);
    act_values<1>(e.act, reinterpret_cast<float(&)[1][8]>(v));
    if (e.C != nullptr) {
      load8_part(e.c_type, e.C, c_at, left, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(beta, w[i], v[i]);
    }
    add_diagonal(e.diag, row, col, v);
  }
  store8_part(e.d_type, e.D, d_at, left, v);
  if (e.copy != nullptr)
    store8_part(RTAT_TYPE_F16, e.copy, z * e.copy_stride + row + (long)col * e.ldcopy, left, v);
}

// One element; returns what belongs to its row's sum.
__device__ inline float epilogue1(const Epilogue& e, float alpha, float beta, int row, int col,
                                  long z, float x) {
  x *= alpha;
  if (e.slope) {
    if (e.act != RTAT_ACT_NONE)
      x *= act_slope(e.act, load_one(e.aux_type, e.aux, z * e.aux_stride + row + (long)col * e.ldaux));
  } else {
    if (e.bias != nullptr) x += load_one(e.bias_type, e.bias, row);
    if (e.aux != nullptr) store_one(e.aux_type, e.aux, z * e.aux_stride + row + (long)col * e.ldaux, x);
    x = act_value(e.act, x);
    if (e.C != nullptr)
      x = __builtin_fmaf(beta, load_one(e.c_type, e.C, z * e.c_stride + row + (long)col * e.ldc), x);
    if (row == col) x += e.diag;
  }
  store_one(e.d_type, e.D, z * e.d_stride + row + (long)col * e.ldd, x);
  if (e.copy != nullptr)
    store_one(RTAT_TYPE_F16, e.copy, z * e.copy_stride + row + (long)col * e.ldcopy, x);
  return x;
}

}  // namespace rtat_native
