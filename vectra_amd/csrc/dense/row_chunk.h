// 16-byte chunks of rows that need no alignment.
#pragma once

#include "dense_common.h"

namespace vectra_dense {

// What one lane feeds a matrix instruction: 16 bytes.
struct Frag {
  u32x4 w;
};

// Elements first .. of a row of `width`, zeros past its end.
template <typename T>
__device__ __forceinline__ Frag load_row_chunk(const T* row, int64_t width, int64_t first) {
  constexpr int kPer = 16 / sizeof(T);
  Frag f;
  if (first + kPer <= width) {
    __builtin_memcpy(&f.w, row + first, 16);  // unaligned
  } else {
    T v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = first + e < width ? row[first + e] : static_cast<T>(0.f);
    __builtin_memcpy(&f.w, v, 16);
  }
  return f;
}

// Eight elements of a row from `first` on, zeros past its end, as they are in
// memory and as fp32.
template <typename T>
struct Eight {
  Frag part[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* row, int64_t width, int64_t first) {
  Eight<T> r;
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) r.part[h] = load_row_chunk<T>(row, width, first + 4 * h);
  return r;
}

template <typename T>
__device__ __forceinline__ void widen_eight(const Eight<T>& r, f32x4& a, f32x4& b) {
  if constexpr (sizeof(T) == 4) {
    a = __builtin_bit_cast(f32x4, r.part[0].w);
    b = __builtin_bit_cast(f32x4, r.part[1].w);
  } else {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const u32x4 w = r.part[0].w;
    a = __builtin_convertvector(__builtin_bit_cast(T4, uint2{w[0], w[1]}), f32x4);
    b = __builtin_convertvector(__builtin_bit_cast(T4, uint2{w[2], w[3]}), f32x4);
  }
}

}  // namespace vectra_dense
