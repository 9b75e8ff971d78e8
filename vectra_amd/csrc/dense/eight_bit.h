// Elements in 8 bits: e4m3 codes of x / 2^e, 2^e shared by a block.
#pragma once

#include "dense_common.h"

namespace vectra_dense {

// The exponent byte of a block whose largest finite magnitude is `largest`:
// the smallest e with largest <= 448 * 2^e, at least `lowest`, plus 127.
// largest = f * 2^x with f in [1, 2): 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(float largest, int lowest) {
  const uint32_t bits = __float_as_uint(largest);
  int e;
  if (bits < 0x00800000u) {
    e = lowest;  // zero or an fp32 subnormal: far below the lowest exponent
  } else {
    e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x007fffffu) > 0x00600000u ? 1 : 0);
  }
  return max(e, lowest) + 127;
}

// 2^e as fp32 for e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// fp32 in [-448, 448] to e4m3, ties to even (v_cvt_pk_fp8_f32); NaN to NaN.
__device__ __forceinline__ uint32_t to_e4m3x4(f32x4 v) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true));
}

__device__ __forceinline__ f32x4 from_e4m3x4(uint32_t w) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}

// The largest finite magnitude of eight elements, at least `largest`; the others
// become NaN.
__device__ __forceinline__ float largest_finite(f32x4 (&v)[2], float largest) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = __builtin_fabsf(v[k / 4][k % 4]);
    if (a <= 3.4028234663852886e38f) {
      largest = a > largest ? a : largest;
    } else {
      v[k / 4][k % 4] = __builtin_nanf("");
    }
  }
  return largest;
}

// Eight elements of a block of exponent e (in [-117, 120]) as codes.  `highest`: the
// exponent at which an element of the type's largest magnitudes (fp16: 255.9 * 2^8,
// else 2^120) would round to 256 times it, which the type lacks: there, magnitudes
// of 248 and more take the code below, 240.
__device__ __forceinline__ uint2 to_codes(f32x4 (&v)[2], int e, int highest) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v[h] *= power_of_two(-e);
    if (e == highest)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (__builtin_fabsf(v[h][k]) >= 248.f) v[h][k] = __builtin_copysignf(240.f, v[h][k]);
    w[h] = to_e4m3x4(v[h]);
  }
  return uint2{w[0], w[1]};
}

}  // namespace vectra_dense
