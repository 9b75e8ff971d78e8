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

}  // namespace vectra_dense
