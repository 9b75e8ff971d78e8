// Device-side helpers of the operators between a block's dense products (gfx950, wave64).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../dense/dense_common.h"
#include "../dense/eight_bit.h"
#include "../dense/row_chunk.h"
#include "../rbf_common.h"
#include "vectra_block.h"

namespace vectra_block {

using vectra_dense::Eight;
using vectra_dense::f32x4;
using vectra_dense::least;
using vectra_dense::load_eight;
using vectra_dense::most;
using vectra_dense::store8;
using vectra_dense::widen_eight;

static_assert(int{VECTRA_BLOCK_F32} == int{VECTRA_DENSE_F32} && int{VECTRA_BLOCK_F16} == int{VECTRA_DENSE_F16} &&
              int{VECTRA_BLOCK_BF16} == int{VECTRA_DENSE_BF16});

// Exponents of 8-bit blocks: the least, and the one at which codes are held below the
// next power of two (vectra_block.h).
constexpr int kLowestExponent = -117, kHighestExponent = 120;

// ----------------------------------------------------------------- dropout

struct Dropout {
  const int64_t* rng;  // seed, offset
  int32_t threshold;   // of 65536; 0: every element is kept
  uint32_t stream;
  float scale;         // 65536 / (65536 - threshold)
};

// The seed and the offset, read once per thread (uniform).
struct DropoutKey {
  uint32_t k0, k1, offset;
};

__device__ __forceinline__ DropoutKey dropout_key(const Dropout& d) {
  if (d.threshold == 0) return DropoutKey{0, 0, 0};
  const uint64_t seed = static_cast<uint64_t>(d.rng[0]);
  return DropoutKey{static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), static_cast<uint32_t>(d.rng[1])};
}

// Which of the eight elements of a group are kept, a bit each: Philox 4x32, ten
// rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3;
// SC 2011).  16 bits per element: with 32 the twenty wide multiplications, at a
// quarter of the vector rate, would be shared by four elements instead of eight,
// and dropout of 16-bit elements would be bound by them rather than by memory.
__device__ __forceinline__ uint32_t dropout_kept(const Dropout& d, const DropoutKey& key, uint64_t group) {
  uint32_t a = static_cast<uint32_t>(group), b = static_cast<uint32_t>(group >> 32), c = d.stream, e = key.offset;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p = static_cast<uint64_t>(0xD2511F53u) * a, q = static_cast<uint64_t>(0xCD9E8D57u) * c;
    a = static_cast<uint32_t>(q >> 32) ^ b ^ k0;
    b = static_cast<uint32_t>(q);
    c = static_cast<uint32_t>(p >> 32) ^ e ^ k1;
    e = static_cast<uint32_t>(p);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t words[4] = {a, b, c, e}, t = static_cast<uint32_t>(d.threshold);
  uint32_t kept = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kept |= (words[j] & 0xffffu) >= t ? 1u << 2 * j : 0u;
    kept |= (words[j] >> 16) >= t ? 2u << 2 * j : 0u;
  }
  return kept;
}

// The elements scaled, with 0 for a dropped one whatever it holds.
__device__ __forceinline__ void drop(f32x4 (&x)[2], uint32_t kept, float scale) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i / 4][i % 4] = kept >> i & 1 ? x[i / 4][i % 4] * scale : 0.f;
}

// ------------------------------------------------------------------ vectors

// Eight elements of a per-column vector from `first` on (`left` of them exist, the
// others are 0), in its own type; NULL: `missing` for those that exist.
__device__ __forceinline__ void load_vector(const void* v, int32_t dtype, int64_t first, int left, float missing,
                                            f32x4 (&out)[2]) {
  if (!v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i / 4][i % 4] = i < left ? missing : 0.f;
  } else if (left <= 0) {
    out[0] = out[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  } else if (dtype == VECTRA_BLOCK_F32) {
    vectra_dense::load8(static_cast<const float*>(v) + first, left, out[0], out[1]);
  } else if (dtype == VECTRA_BLOCK_F16) {
    vectra_dense::load8(static_cast<const _Float16*>(v) + first, left, out[0], out[1]);
  } else {
    vectra_dense::load8(static_cast<const __bf16*>(v) + first, left, out[0], out[1]);
  }
}

__device__ __forceinline__ void store_vector(void* v, int32_t dtype, int64_t first, int left, const f32x4 (&x)[2]) {
  if (left <= 0) return;
  if (dtype == VECTRA_BLOCK_F32)
    store8(static_cast<float*>(v) + first, x[0], x[1], left);
  else if (dtype == VECTRA_BLOCK_F16)
    store8(static_cast<_Float16*>(v) + first, x[0], x[1], left);
  else
    store8(static_cast<__bf16*>(v) + first, x[0], x[1], left);
}

}  // namespace vectra_block
