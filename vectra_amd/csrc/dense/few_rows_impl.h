// Products of a few rows (one token to 32) with a weight that is read once:
// the kernel template, instantiated per element type in few_rows_<type>.hip.
//
//   y = act(x W^T + b) + r,  or the gated product
//
// Such a call is the weight's bytes.  A workgroup of 8 or 16 waves takes 16
// rows of W (16 of the gate and the same 16 of the up projection), and its
// waves share out the contraction: of 8, wave w takes the 64-byte steps w,
// w + 8, ... of those rows, so the workgroup reads 512 consecutive bytes of
// each row at a time.  A
// wave loads a batch of steps straight into the registers of the matrix
// instruction's first operand (lane l: row l % 16, 16-byte chunk l / 16), x
// likewise into the second's (from L2 after the first workgroups), and has up
// to 8 KB in flight.  The waves' sums meet in LDS and are added in a fixed
// order; there is no second launch and nothing in the workspace.
//
// Measured: one row, 4096 -> 4096 fp16 with a residual 8.8 us, 3.8 TB/s of a large
// copy's 5.1; 4 rows, 4096 -> 2 x 11008 bf16 gated 39.8 us, 4.5 TB/s.
//
// Rows need no alignment: full chunks are loaded as 16 unaligned bytes, a
// row's last partial chunk element by element.
#pragma once

#include "resident_impl.h"

namespace vectra_dense {

template <typename T, int kRowTiles, bool kGated, int kFewWaves>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(const FewRowsParams p) {
  constexpr int kHalves = kGated ? 2 : 1;
  constexpr int kBatch = kGated || kRowTiles > 1 ? 4 : 8;
  constexpr int kPer = 16 / sizeof(T);
  __shared__ f32x4 part[kFewWaves][kHalves][kRowTiles][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int steps = static_cast<int>((p.width + 4 * kPer - 1) / (4 * kPer));
  const T* const x = static_cast<const T*>(p.x);
  // Rows past the end: W's repeat the last one (their results are not
  // stored), x's are zeros.
  const T* w_row[kHalves];
  w_row[0] = static_cast<const T*>(p.w) + least(n0 + i, p.n - 1) * p.ldw;
  if constexpr (kGated) w_row[1] = w_row[0] + p.n * p.ldw;

  f32x4 acc[kHalves][kRowTiles];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int t = 0; t < kRowTiles; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int first = wave; first < steps; first += kFewWaves * kBatch) {
    Frag fw[kBatch][kHalves], fx[kBatch][kRowTiles];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int at = ((first + b * kFewWaves) * 4 + g) * kPer;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        fw[b][h].w = u32x4{0, 0, 0, 0};
        if (at < p.width) fw[b][h] = load_row_chunk<T>(w_row[h], p.width, at);
      }
#pragma unroll
      for (int t = 0; t < kRowTiles; ++t) {
        fx[b][t].w = u32x4{0, 0, 0, 0};
        if (t * 16 + i < p.rows && at < p.width) fx[b][t] = load_row_chunk<T>(x + (t * 16 + i) * p.ldx, p.width, at);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int t = 0; t < kRowTiles; ++t) acc[h][t] = Mma<T>::run(fw[b][h], fx[b][t], acc[h][t]);
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
  const int left = static_cast<int>(p.n - n);
  if (m >= p.rows || left <= 0) return;
  f32x4 z = {0.f, 0.f, 0.f, 0.f}, u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kFewWaves; ++k) {
    z += part[k][0][wave][lane];
    if constexpr (kGated) u += part[k][1][wave][lane];
  }
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) {
        z[e] += load_bias(p.bias, n + e, p.bias_dtype);
        if constexpr (kGated) u[e] += load_bias(p.bias, p.n + n + e, p.bias_dtype);
      }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    z[e] = act_value<T>(z[e], p.activation);
    if constexpr (kGated) z[e] *= u[e];
  }
  if (!kGated && p.residual) z += load4(static_cast<const T*>(p.residual) + m * p.ldr + n, left);
  store4(static_cast<T*>(p.out) + m * p.ldo + n, z, left);
}

template <typename T>
int launch_few_rows(const FewRowsParams& p, bool gated, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((p.n + 15) / 16));
  // 16 waves where at most one workgroup of 8 would be on a CU.
  const int waves = p.n <= 16 * 256 ? 16 : 8;
  const auto kernel = p.rows <= 16 ? (gated ? (waves == 16 ? few_rows_kernel<T, 1, true, 16> : few_rows_kernel<T, 1, true, 8>)
                                            : (waves == 16 ? few_rows_kernel<T, 1, false, 16> : few_rows_kernel<T, 1, false, 8>))
                                   : (gated ? (waves == 16 ? few_rows_kernel<T, 2, true, 16> : few_rows_kernel<T, 2, true, 8>)
                                            : (waves == 16 ? few_rows_kernel<T, 2, false, 16> : few_rows_kernel<T, 2, false, 8>));
  kernel<<<grid, 64 * waves, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? VECTRA_DENSE_OK : VECTRA_DENSE_ERR_LAUNCH;
}

}  // namespace vectra_dense
