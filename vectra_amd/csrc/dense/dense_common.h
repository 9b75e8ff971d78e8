// Device-side helpers of the dense operators (gfx950, wave64).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vectra_dense.h"

namespace vectra_dense {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// (HIP's min and max of 64-bit integers go through double.)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t most(int64_t a, int64_t b) { return a > b ? a : b; }

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// ------------------------------------------------------------- activations
//
// The normal distribution's tail, for a = |z|:
//   Phi(-a) = exp(-a^2 / 2) t P(t),  t = 1 / (1 + c a),
// the form of Abramowitz and Stegun 26.2.17 with polynomials of this file's own
// (least squares at Chebyshev nodes, weighted towards the least largest relative
// error over a in [0, 14]): degree 8 for fp32 (3.0e-8, half of fp32's half step;
// its coefficients were rounded one after the other, the rest fitted again each
// time), degree 6 for values that are rounded to 16 bits (8.2e-7, a 600th of
// fp16's half step).  These are the errors of the constants as they stand,
// evaluated exactly; the fp32 evaluation adds its own roundings.  It has no
// cancellation on either side: for z < 0 the tail is the value, for z > 0 it is
// subtracted from 1.  About 20 instructions (18), where erff's branches take
// about 60: at 17 million elements on 256 CUs that is 9 us of vector issue
// instead of 26.  (Degree 6 instead of 8: 66560 x 128 -> 256 bf16 21.4 -> 20.8 us,
// 7202 x 144 -> 7744 fp16 72.2 -> 69.5.)
template <typename T>
__device__ __forceinline__ void normal_tail(float a, float& tail, float& gauss) {
  float t, p;
  if constexpr (sizeof(T) == 4) {
    t = rcp_fast(__builtin_fmaf(0.21f, a, 1.f));
    p = -0.07165627926588058f;
    p = __builtin_fmaf(p, t, 0.2835884094238281f);
    p = __builtin_fmaf(p, t, -0.3302529752254486f);
    p = __builtin_fmaf(p, t, 0.34940046072006226f);
    p = __builtin_fmaf(p, t, -0.09392476826906204f);
    p = __builtin_fmaf(p, t, 0.12487250566482544f);
    p = __builtin_fmaf(p, t, 0.06919223815202713f);
    p = __builtin_fmaf(p, t, 0.08506884425878525f);
    p = __builtin_fmaf(p, t, 0.08371157199144363f);
  } else {
    t = rcp_fast(__builtin_fmaf(0.3625f, a, 1.f));
    p = 0.04806305468082428f;
    p = __builtin_fmaf(p, t, -0.17974300682544708f);
    p = __builtin_fmaf(p, t, 0.17510487139225006f);
    p = __builtin_fmaf(p, t, 0.029681770130991936f);
    p = __builtin_fmaf(p, t, 0.13925696909427643f);
    p = __builtin_fmaf(p, t, 0.1429363340139389f);
    p = __builtin_fmaf(p, t, 0.14470037817955017f);
  }
  gauss = exp2_fast(a * a * (-0.5f * kLog2e));
  tail = p * t * gauss;
}

// 1 / (1 + exp(-z)).  exp2 of a large argument is inf and its reciprocal 0.
__device__ __forceinline__ float sigmoid(float z) { return rcp_fast(1.f + exp2_fast(-kLog2e * z)); }

// The same with its complement, neither by a subtraction from 1: the slopes
// multiply the complement by up to z^3, which would magnify its rounding.
__device__ __forceinline__ void sigmoid_pair(float z, float& s, float& rest) {
  const float e = exp2_fast(-kLog2e * __builtin_fabsf(z));  // at most 1
  const float big = rcp_fast(1.f + e), small = e * big;
  s = z < 0.f ? small : big;
  rest = z < 0.f ? big : small;
}

constexpr float kTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kTanhK = 0.044715f;

// T: the type that the result is rounded to.
template <typename T>
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case VECTRA_DENSE_RELU:
      return z < 0.f ? 0.f : z;  // keeps NaN
    case VECTRA_DENSE_GELU: {
      float tail, gauss;
      normal_tail<T>(__builtin_fabsf(z), tail, gauss);
      return z * (z < 0.f ? tail : 1.f - tail);
    }
    case VECTRA_DENSE_GELU_TANH:  // (1 + tanh(y)) / 2 = sigmoid(2 y)
      return z * sigmoid(2.f * kTanhC * __builtin_fmaf(kTanhK * z * z, z, z));
    case VECTRA_DENSE_SILU:
      return z * sigmoid(z);
    default:
      return z;
  }
}

// act(z) and act'(z), for dz.  With fp32's polynomial whatever the operands' type:
// a bias's gradient may be fp32 beside 16-bit operands, and is summed from dz
// before its rounding.
__device__ __forceinline__ void act_slope(float z, int act, float& value, float& slope) {
  switch (act) {
    case VECTRA_DENSE_RELU:
      value = z < 0.f ? 0.f : z;
      slope = z > 0.f ? 1.f : 0.f;
      return;
    case VECTRA_DENSE_GELU: {
      float tail, gauss;
      normal_tail<float>(__builtin_fabsf(z), tail, gauss);
      const float cdf = z < 0.f ? tail : 1.f - tail;
      value = z * cdf;
      slope = __builtin_fmaf(z, gauss * 0.3989422804014327f, cdf);
      return;
    }
    case VECTRA_DENSE_GELU_TANH: {
      float s, rest;
      sigmoid_pair(2.f * kTanhC * __builtin_fmaf(kTanhK * z * z, z, z), s, rest);
      value = z * s;
      // (z^2 held finite: past |z| = 1.8e19 it would be inf beside a rest or value of 0.)
      slope = __builtin_fmaf(value * rest, 2.f * kTanhC * __builtin_fmaf(3.f * kTanhK, __builtin_fminf(z * z, 1e30f), 1.f), s);
      return;
    }
    case VECTRA_DENSE_SILU: {
      float s, rest;
      sigmoid_pair(z, s, rest);
      value = z * s;
      slope = __builtin_fmaf(value, rest, s);
      return;
    }
    default:
      value = z;
      slope = 1.f;
  }
}

// f with the activation as a constant: its element loops hold no branch.
template <int kAct>
struct Activation {
  static constexpr int value = kAct;
};
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case VECTRA_DENSE_RELU: return f(Activation<VECTRA_DENSE_RELU>{});
    case VECTRA_DENSE_GELU: return f(Activation<VECTRA_DENSE_GELU>{});
    case VECTRA_DENSE_GELU_TANH: return f(Activation<VECTRA_DENSE_GELU_TANH>{});
    case VECTRA_DENSE_SILU: return f(Activation<VECTRA_DENSE_SILU>{});
    default: return f(Activation<VECTRA_DENSE_NONE>{});
  }
}

// ------------------------------------------------------------ element types

template <typename T>
__device__ __forceinline__ float widen(T x) { return static_cast<float>(x); }

// fp32 -> T, round to nearest even.  The value is made opaque first, so that
// the product before it is not fused with the conversion (one rounding from
// the fp32 result).
template <typename T>
__device__ __forceinline__ T narrow(float x) {
  if constexpr (sizeof(T) < 4) asm volatile("" : "+v"(x));
  return static_cast<T>(x);
}

// Runs of four and eight consecutive elements of a row, of which `left` exist.
// Whole runs move as one 8- or 16-byte access (fp32: 16 bytes, twice for
// eight) at whatever alignment the row has: gfx950's vector memory accesses
// need none.
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int left) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (left >= 4) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
    __builtin_memcpy(&v, p, sizeof(v));
    r = __builtin_convertvector(v, f32x4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) r[i] = widen(p[i]);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v, int left) {
  if (left >= 4) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(T) < 4) asm volatile("" : "+v"(v));
    const T4 t = __builtin_convertvector(v, T4);
    __builtin_memcpy(p, &t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = narrow<T>(v[i]);
  }
}

// Zeros behind a row's `columns` elements up to its stride, at most seven: dz,
// whose rows are padded to whole 16-byte chunks for the products that read it.
template <typename T>
__device__ __forceinline__ void zero_padding(T* row, int64_t columns, int64_t stride) {
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (columns + e < stride) row[columns + e] = static_cast<T>(0.f);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, f32x4& a, f32x4& b) {
  if constexpr (sizeof(T) == 2) {
    if (left >= 8) {
      typedef T T4 __attribute__((ext_vector_type(4)));
      u32x4 w;
      __builtin_memcpy(&w, p, 16);
      a = __builtin_convertvector(__builtin_bit_cast(T4, uint2{w[0], w[1]}), f32x4);
      b = __builtin_convertvector(__builtin_bit_cast(T4, uint2{w[2], w[3]}), f32x4);
      return;
    }
  }
  a = load4(p, left);
  b = load4(p + 4, left - 4);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, f32x4 a, f32x4 b, int left) {
  if constexpr (sizeof(T) == 2) {
    if (left >= 8) {
      typedef T T4 __attribute__((ext_vector_type(4)));
      asm volatile("" : "+v"(a), "+v"(b));
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_convertvector(a, T4));
      const uint2 hi = __builtin_bit_cast(uint2, __builtin_convertvector(b, T4));
      const u32x4 w = {lo.x, lo.y, hi.x, hi.y};
      __builtin_memcpy(p, &w, 16);
      return;
    }
  }
  store4(p, a, left);
  store4(p + 4, b, left - 4);
}

// Element i of a bias, in its own type.
__device__ __forceinline__ float load_bias(const void* bias, int64_t i, int32_t dtype) {
  switch (dtype) {
    case VECTRA_DENSE_F32:
      return static_cast<const float*>(bias)[i];
    case VECTRA_DENSE_F16:
      return static_cast<float>(static_cast<const _Float16*>(bias)[i]);
    default:
      return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(bias)[i]) << 16);
  }
}

// Writes element i of a vector in the given type.
__device__ __forceinline__ void store_as(void* out, int64_t i, int32_t dtype, float v) {
  if (dtype == VECTRA_DENSE_F32)
    static_cast<float*>(out)[i] = v;
  else if (dtype == VECTRA_DENSE_F16)
    static_cast<_Float16*>(out)[i] = narrow<_Float16>(v);
  else
    static_cast<__bf16*>(out)[i] = narrow<__bf16>(v);
}

}  // namespace vectra_dense
