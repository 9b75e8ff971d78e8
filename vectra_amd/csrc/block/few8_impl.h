// Products in 8 bits of a few rows (one token to 64) with a weight that is read once:
// the kernel template, instantiated per type in product8_<type>.hip.
//
//   y = act(x^ W^T + b) + r,  or the gated product
//
// Such a call is the weight's bytes, one for each element.  A workgroup of 8 or 16
// waves takes 16 rows of W (gated: 16 of the gate and the same 16 of the up
// projection), and its waves share out the blocks of 128 of the contraction; lane
// (g, i) of a wave loads 32 bytes of row i, so a wave reads whole 128-byte lines.
// The codes are turned into bf16 together with their power of two, which is exact,
// and multiplied on the bf16 matrix cores: exact products, fp32 sums.  (The 8-bit
// cores drop bits of a product beside a large one, and would save nothing here.)
// The order of the contraction within a block is the matrix instruction's own
// affair: both operands use the same.
//
// Up to 16 rows a wave brings its own blocks of x into 8 bits, from registers to
// registers: four lanes share a row's block.  There is no second launch and nothing
// in the workspace.  More rows come as codes.
#pragma once

#include "block_common.h"
#include "product8_kernels.h"

namespace vectra_block {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 2^(byte - 127) as fp32: the exponent's own bits, but for byte 0 (2^-127, an fp32
// subnormal) and 255 (NaN).
__device__ __forceinline__ float scale_of(uint32_t byte) {
  const uint32_t bits = byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23;
  return __uint_as_float(bits);
}

// Eight codes times a power of two as bf16: four bits of significand, exact (past
// bf16's range: infinity, or a subnormal).
__device__ __forceinline__ bf16x8 decode(uint32_t lo, uint32_t hi, float scale) {
  bf16x8 r;
  const uint32_t words[2] = {lo, hi};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 v = vectra_dense::from_e4m3x4(words[h]) * scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[4 * h + e] = static_cast<__bf16>(v[e]);
  }
  return r;
}

// One lane's 32 codes of a block, decoded: the operands of four matrix instructions.
struct Block8 {
  u32x4 w[2];
  float scale;
  __device__ __forceinline__ bf16x8 part(int j) const { return decode(w[j / 2][j % 2 * 2], w[j / 2][j % 2 * 2 + 1], scale); }
};

// A lane's 32 elements of a row's block, zeros past the row's end, in 8 bits.  The
// four lanes (g = 0 .. 3) of row i find the block's largest together.
template <typename T>
__device__ __forceinline__ Block8 quantise_block(const T* row, int64_t width, int64_t first) {
  f32x4 v[4][2];
  float largest = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int left = static_cast<int>(most(least(row ? width - first - 8 * j : 0, 8), 0));
    v[j][0] = v[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (left > 0) vectra_dense::load8(row + first + 8 * j, left, v[j][0], v[j][1]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) largest = vectra_dense::largest_finite(v[j], largest);
  largest = vectra::allreduce_bit16(largest, vectra::OpMax{});
  largest = vectra::allreduce_bit32(largest, vectra::OpMax{});
  const int e = vectra_dense::block_exponent(largest, kLowestExponent) - 127;
  Block8 b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint2 c = vectra_dense::to_codes(v[j], e, kHighestExponent);
    b.w[j / 2][j % 2 * 2] = c.x;
    b.w[j / 2][j % 2 * 2 + 1] = c.y;
  }
  b.scale = vectra_dense::power_of_two(e);
  return b;
}

template <typename T, int kRowTiles, bool kGated, bool kRaw, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void few8_kernel(const Product8Params p) {
  constexpr int kHalves = kGated ? 2 : 1;
  constexpr int kBatch = 2;  // blocks of W on their way
  __shared__ f32x4 part[kWaves][kHalves][kRowTiles][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int blocks = static_cast<int>(p.depth / 128);
  // Rows past the end: W's repeat the last one (their results are not stored), x's
  // are zeros.
  const uint8_t* w_row[kHalves];
  const uint8_t* w_scale[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    const int64_t row = least(n0 + i, p.n - 1) + h * p.n;
    w_row[h] = p.weight + row * p.depth + g * 32;
    w_scale[h] = p.weight_scales + row / 128 * p.scale_stride;
  }

  f32x4 acc[kHalves][kRowTiles];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int first = wave; first < blocks; first += kWaves * kBatch) {
    Block8 w[kBatch][kHalves];
    uint32_t byte[kBatch][kHalves];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int at = first + b * kWaves;
      if (at >= blocks) continue;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const u32x4* const from = reinterpret_cast<const u32x4*>(w_row[h] + at * 128);
        w[b][h].w[0] = from[0];
        w[b][h].w[1] = from[1];
        byte[b][h] = w_scale[h][at];
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int at = first + b * kWaves;
      if (at >= blocks) continue;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) w[b][h].scale = scale_of(byte[b][h]);
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) {
        const int row = t * 16 + i;
        Block8 x;
        if constexpr (kRaw) {
          x = quantise_block<T>(row < p.rows ? static_cast<const T*>(p.x) + row * p.x_stride : nullptr, p.width,
                                static_cast<int64_t>(at) * 128 + g * 32);
        } else {
          x.w[0] = x.w[1] = u32x4{0, 0, 0, 0};
          x.scale = 0.f;
          if (row < p.rows) {
            const u32x4* const from = reinterpret_cast<const u32x4*>(p.codes + row * p.depth + static_cast<int64_t>(at) * 128 + g * 32);
            x.w[0] = from[0];
            x.w[1] = from[1];
            x.scale = scale_of(p.scales[row * p.scale_stride + at]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8 xj = x.part(j);
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            acc[h][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[b][h].part(j), xj, acc[h][t], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) part[wave][h][t][lane] = acc[h][t];
  __syncthreads();
  // A wave finishes one row tile: lane holds outputs n .. n + 3 of row m.
  if (wave >= kRowTiles) return;
  const int m = wave * 16 + i;
  const int64_t n = n0 + 4 * g;
  const int left = static_cast<int>(least(p.n - n, 4));
  if (m >= p.rows || left <= 0) return;
  f32x4 z = {0.f, 0.f, 0.f, 0.f}, u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    z += part[k][0][wave][lane];
    if constexpr (kGated) u += part[k][1][wave][lane];
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

template <typename T, bool kGated, int kWaves>
auto few8_for(int64_t rows, bool raw) {
  if (raw) return few8_kernel<T, 1, kGated, true, kWaves>;
  return rows <= 16   ? few8_kernel<T, 1, kGated, false, kWaves>
         : rows <= 32 ? few8_kernel<T, 2, kGated, false, kWaves>
                      : few8_kernel<T, 4, kGated, false, kWaves>;
}

template <typename T>
int launch_few8(const Product8Params& p, bool gated, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((p.n + 15) / 16));
  // 16 waves where at most one workgroup of 8 would be on a CU.
  const int waves = p.n <= 16 * 256 ? 16 : 8;
  const auto kernel = gated ? (waves == 16 ? few8_for<T, true, 16>(p.rows, p.x) : few8_for<T, true, 8>(p.rows, p.x))
                            : (waves == 16 ? few8_for<T, false, 16>(p.rows, p.x) : few8_for<T, false, 8>(p.rows, p.x));
  kernel<<<grid, 64 * waves, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

}  // namespace vectra_block
