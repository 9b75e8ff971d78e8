// Products in 8 bits of a few rows (one token to 32) with a weight that is read once:
// the kernel template, instantiated per type in product8_<type>.hip.
//
//   y = act(x^ W^T + b) + r,  or the gated product
//
// Such a call is the weight's bytes, one for each element.  A workgroup of 8 or 16
// waves takes 16 rows of W (gated: 16 of the gate and the same 16 of the up
// projection), and its waves share out the blocks of 128 of the contraction; lane
// (g, i) of a wave loads 32 bytes of row i, so a wave reads whole 128-byte lines.  (Of
// a wide W two such tiles: launch_few8.)
// The codes are turned into bf16 together with their power of two, which is exact,
// and multiplied on the bf16 matrix cores: exact products, fp32 sums.  (The 8-bit
// cores drop bits of a product beside a large one, and would save nothing here.)
// The order of the contraction within a block is the matrix instruction's own
// affair: both operands use the same.
//
// A few rows that are short enough are brought into 8 bits by each workgroup for
// itself, in LDS, while its first rows of W are on their way: no second launch and
// nothing in the workspace.  More come as codes.
#pragma once

#include "block_common.h"
#include "product8_kernels.h"

namespace vectra_block {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 2^(byte - 127) as the conversions below take it: in the exponent's bits.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes times a power of two as bf16, by gfx950's scaled conversion of pairs:
// four bits of significand, exact (past bf16's range: infinity, or a subnormal).
__device__ __forceinline__ bf16x8 decode(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// One lane's 32 codes of a block, decoded: the operands of four matrix instructions.
struct Block8 {
  u32x4 w[2];
  float scale;
  __device__ __forceinline__ bf16x8 part(int j) const { return decode(w[j / 2][j % 2 * 2], w[j / 2][j % 2 * 2 + 1], scale); }
};

// kPair: 32 rows of W per workgroup, not gated.
template <typename T, int kRowTiles, bool kGated, bool kRaw, int kWaves, bool kPair>
__global__ __launch_bounds__(64 * kWaves) void few8_kernel(const Product8Params p) {
  static_assert(!(kGated && kPair));
  constexpr int kHalves = kGated || kPair ? 2 : 1;
  constexpr int kBatch = 2;  // blocks of W on their way
  __shared__ f32x4 part[kWaves][kHalves][kRowTiles][64];
  // x in 8 bits: rows 32 bytes apart in the banks.
  __shared__ __attribute__((aligned(16))) uint8_t x_codes[kRaw ? kRawBytes + kFewRaw8 * 32 : 16];
  __shared__ uint8_t x_bytes[kRaw ? kRawBytes / 128 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (kPair ? 32 : 16);
  const int blocks = static_cast<int>(p.depth / 128);
  // Rows past the end: W's repeat the last one (their results are not stored), x's
  // are zeros.
  const uint8_t* w_row[kHalves];
  const uint8_t* w_scale[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    const int64_t row = kPair ? least(n0 + h * 16 + i, p.n - 1) : least(n0 + i, p.n - 1) + h * p.n;
    w_row[h] = p.weight + row * p.depth + g * 32;
    w_scale[h] = p.weight_scales + row / 128 * p.scale_stride;
  }

  f32x4 acc[kHalves][kRowTiles];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  Block8 w[kBatch][kHalves];
  uint32_t w_byte[kBatch][kHalves];
  const auto load_w = [&](int first) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int at = first + b * kWaves;
      if (at >= blocks) continue;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        w[b][h].w[0] = *reinterpret_cast<const u32x4*>(w_row[h] + at * 128);
        w[b][h].w[1] = *reinterpret_cast<const u32x4*>(w_row[h] + at * 128 + 16);
        w_byte[b][h] = w_scale[h][at];
      }
    }
  };
  if constexpr (kRaw) load_w(wave);
  const int x_stride = static_cast<int>(p.depth) + 32;
  if constexpr (kRaw) {
    // A block of a row by 16 lanes, eight elements each.
    const int eights = static_cast<int>(p.depth / 8), total = static_cast<int>(p.rows) * eights;
    for (int base = wave * 64; base < total; base += 64 * kWaves) {
      const int at = base + lane;
      const bool live = at < total;  // (a block's 16 lanes alike)
      const int row = live ? at / eights : 0, column = live ? (at - row * eights) * 8 : 0;
      f32x4 v[2] = {};
      const int left = live ? static_cast<int>(most(least(p.width - column, 8), 0)) : 0;
      if (left > 0) vectra_dense::load8(static_cast<const T*>(p.x) + row * p.x_stride + column, left, v[0], v[1]);
      const float largest = vectra::reduce_low<16>(vectra_dense::largest_finite(v, 0.f), vectra::OpMax{});
      const int byte = vectra_dense::block_exponent(largest, kLowestExponent);
      const uint2 c = vectra_dense::to_codes(v, byte - 127, kHighestExponent);
      if (!live) continue;
      *reinterpret_cast<uint2*>(x_codes + row * x_stride + column) = c;
      if (lane % 16 == 0) x_bytes[row * blocks + column / 128] = static_cast<uint8_t>(byte);
    }
    __syncthreads();
  }
  for (int first = wave; first < blocks; first += kWaves * kBatch) {
    // A batch's loads, all of them before the first is used: W's blocks and, from L2
    // after the first workgroups, x's.
    if (!kRaw || first != wave) load_w(first);
    Block8 x[kBatch][kRowTiles];
    uint32_t x_byte[kBatch][kRowTiles];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int at = first + b * kWaves;
      if (at >= blocks) continue;
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) {
        const int row = t * 16 + i;
        x[b][t].w[0] = x[b][t].w[1] = u32x4{0, 0, 0, 0};
        x_byte[b][t] = 127;
        if (row < p.rows) {
          const uint8_t* const from = kRaw ? x_codes + row * x_stride + at * 128 + g * 32
                                           : p.codes + row * p.depth + static_cast<int64_t>(at) * 128 + g * 32;
          x[b][t].w[0] = *reinterpret_cast<const u32x4*>(from);
          x[b][t].w[1] = *reinterpret_cast<const u32x4*>(from + 16);
          x_byte[b][t] = kRaw ? x_bytes[row * blocks + at] : p.scales[row * p.scale_stride + at];
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (first + b * kWaves >= blocks) continue;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) w[b][h].scale = scale_of(w_byte[b][h]);
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) x[b][t].scale = scale_of(x_byte[b][t]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 wj[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) wj[h] = w[b][h].part(j);
#pragma unroll
        for (int t = 0; t < kRowTiles; ++t) {
          const bf16x8 xj = x[b][t].part(j);
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            acc[h][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wj[h], xj, acc[h][t], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) part[wave][h][t][lane] = acc[h][t];
  __syncthreads();
  // A wave finishes one row tile (of a pair's half): lane holds outputs n .. n + 3 of row m.
  if (wave >= kRowTiles * (kPair ? 2 : 1)) return;
  const int tile = wave % kRowTiles, of = wave / kRowTiles;
  const int m = tile * 16 + i;
  const int64_t n = n0 + of * 16 + 4 * g;
  const int left = static_cast<int>(least(p.n - n, 4));
  if (m >= p.rows || left <= 0) return;
  f32x4 z = {0.f, 0.f, 0.f, 0.f}, u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    z += part[k][of][tile][lane];
    if constexpr (kGated) u += part[k][1][tile][lane];
  }
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) {
        z[e] += vectra_dense::load_bias(p.bias, n + e, p.bias_dtype);
        if constexpr (kGated) u[e] += vectra_dense::load_bias(p.bias, p.n + n + e, p.bias_dtype);
      }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    z[e] = vectra_dense::act_value<T>(z[e], p.activation);
    if constexpr (kGated) z[e] *= u[e];
  }
  if (!kGated && p.residual) z += vectra_dense::load4(static_cast<const T*>(p.residual) + m * p.residual_stride + n, left);
  vectra_dense::store4(static_cast<T*>(p.out) + m * p.out_stride + n, z, left);
}

template <typename T, bool kGated, int kWaves, bool kPair>
auto few8_for(int64_t rows, bool raw) {
  if constexpr (!kPair) {
    if (raw) return few8_kernel<T, 1, kGated, true, kWaves, false>;
  }
  return rows <= 16 ? few8_kernel<T, 1, kGated, false, kWaves, kPair> : few8_kernel<T, 2, kGated, false, kWaves, kPair>;
}

template <typename T>
int launch_few8(const Product8Params& p, bool gated, hipStream_t stream) {
  // 16 waves where at most one workgroup of 8 would be on a CU.  Every workgroup reads all
  // codes of x, from L2: of 32 rows twice the weight's bytes.  Pairs halve that, where they
  // leave a workgroup for every CU (us with pairs / without: 32 x 4096 -> 16384 26.0 / 35.8,
  // 8 rows 20.6 / 21.6; 32 x 8192 -> 28672 80 / 105; 32 x 1024 -> 8192 7.7 / 8.3).
  const bool pair = !gated && !p.x && p.n >= 32 * 256;
  const int waves = p.n <= 16 * 256 ? 16 : 8;
  const dim3 grid(static_cast<uint32_t>((p.n + (pair ? 31 : 15)) / (pair ? 32 : 16)));
  const auto kernel = gated    ? (waves == 16 ? few8_for<T, true, 16, false>(p.rows, p.x) : few8_for<T, true, 8, false>(p.rows, p.x))
                      : pair   ? few8_for<T, false, 8, true>(p.rows, false)
                      : waves == 16 ? few8_for<T, false, 16, false>(p.rows, p.x)
                                    : few8_for<T, false, 8, false>(p.rows, p.x);
  kernel<<<grid, 64 * waves, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

}  // namespace vectra_block
