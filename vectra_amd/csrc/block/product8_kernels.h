// What the host code launches for products in 8 bits.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vectra_block.h"

namespace vectra_block {

struct Product8Params {
  const void* x;           // few rows only: the input itself, or NULL with codes and scales
  int64_t x_stride;
  const uint8_t* codes;    // [rows, depth]
  const uint8_t* scales;   // [rows, scale_stride]
  const uint8_t* weight;   // [n_w, depth]
  const uint8_t* weight_scales;  // [ceil(n_w / 128), scale_stride]
  int64_t rows, n, width, depth, scale_stride;  // n: outputs (gated: of a half)
  const void* bias;
  int32_t bias_dtype, activation;
  const void* residual;
  int64_t residual_stride;
  void* out;  // kPartial: fp32 planes [parts, rows, out_stride]
  int64_t out_stride;
  int32_t tiles_m, tiles_n, k_tiles, k_tiles_per_part;  // (of several parts: a multiple of 4)
};

enum { kStore8 = 0, kGated8 = 1, kPartial8 = 2 };
enum { kLarge8 = 0, kMedium8 = 1, kSmall8 = 2, kTiles8 = 3 };
constexpr int kTile8[kTiles8] = {256, 128, 64};  // rows and columns

// Rows up to which a product reads the weight straight into registers, and rows and
// bytes of them up to which its workgroups bring the input into 8 bits themselves.  The
// bound is part of the contract (exact sums), and no rule on time: 32 rows so and 33 on
// tiles, bf16 from codes, us: 4096 -> 4096 11.0 and 12.1, 4096 -> 16384 24.3 and 26.1, but
// 8192 -> 8192 24.4 and 22.5, 16384 -> 4096 33.9 and 23.4, 8192 -> 28672 81.5 and 68.5,
// gated 2048 -> 2 x 5632 12.4 and 13.8, 4096 -> 2 x 11008 33.8 and 31.2; 17 rows so 9.0,
// 21.3, 22.9, 25.8, 68.8, 10.9 and 29.1.  (64 rows so: 4096 -> 4096 18.9, 8192 -> 8192 56.)
constexpr int kFewRows8 = 32, kFewRaw8 = 16, kRawBytes = 16384;

// One definition per type of result.
int launch_product8_f32(const Product8Params& p, int tile, int epilogue, int parts, hipStream_t stream);
int launch_product8_f16(const Product8Params& p, int tile, int epilogue, int parts, hipStream_t stream);
int launch_product8_bf16(const Product8Params& p, int tile, int epilogue, int parts, hipStream_t stream);

int launch_few8_f32(const Product8Params& p, bool gated, hipStream_t stream);
int launch_few8_f16(const Product8Params& p, bool gated, hipStream_t stream);
int launch_few8_bf16(const Product8Params& p, bool gated, hipStream_t stream);

}  // namespace vectra_block
