// What the dense library's host code launches.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vectra_dense.h"

namespace vectra_dense {

// Epilogues of the tiled product.
enum {
  kEpiStore = 0,       // act(D + bias) + residual, in the element type
  kEpiPartial = 1,     // D in fp32, one plane per split of the contraction
  kEpiGated = 2,       // act(D_gate + bias) * (D_up + bias)
  kEpiSlope = 3,       // grad * act'(D + bias)
  kEpiGatedSlope = 4,  // both factors' gradients
};

struct GemmParams {
  const void* a;  // row operand
  const void* b;  // column operand
  int64_t lda, ldb;
  int64_t a_width, b_width;  // wide operands: elements per stored row (whole chunks)
  int64_t m, n;              // output rows and columns (gated: outputs)
  int64_t depth;             // contraction, as A's rows hold it (zero padded to whole chunks)
  int64_t depth_b;           // contraction rows of a wide B (at most depth: rows past it are zeros)
  int32_t tiles_m, tiles_n;
  int32_t k_tiles, k_tiles_per_split;
  void* out;
  int64_t ldo;
  const void* bias;
  const void* residual;
  int64_t ldr;
  const void* grad;
  int64_t ldg;
  // Slope epilogues: column sums of dz, [tiles_m, columns].  Weight layout: sums
  // of A over the contraction (the bias's gradient), [parts, m].  Several rows
  // are fp32, to be added up; a single one is the result itself.  NULL: not
  // wanted (always on the big tiles' weight products).
  void* sums;
  int32_t sums_dtype;
  int32_t bias_dtype;
  int32_t activation;
};

// The shapes of one tiled product's kernels.
enum { kLayoutForward = 0, kLayoutInput = 1, kLayoutWeight = 2 };
enum { kTileLarge = 0, kTileTall = 1, kTileMedium = 2, kTileSmall = 3, kTileCount = 4 };
constexpr int kTileRows[kTileCount] = {256, 192, 128, 64}, kTileColumns[kTileCount] = {256, 256, 128, 64};
// The small ones take operands of any alignment and sum the bias's gradient
// beside the weight's; the tall one is for 16-bit types.
constexpr bool kTileBig[kTileCount] = {true, true, false, false};

// Launches the product with the given layout, tile and epilogue on `splits`
// contraction parts; `any`: operands of any alignment (not on the big tiles),
// for which depth, depth_b and the widths are the true sizes.  One definition per element type.
int launch_gemm_bf16(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream);
int launch_gemm_f16(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream);
int launch_gemm_f32(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream);

// A product with a weight that stays in LDS (resident_impl.h).
struct ResidentParams {
  const void* x;
  int64_t ldx, rows, width;  // width: contraction
  const void* w;
  int64_t ldw;
  int32_t n, n_pad;  // outputs (gated: of a half), and rounded up to 32
  const void* bias;
  int32_t bias_dtype, activation;
  const void* residual;
  int64_t ldr;
  const void* grad;  // slope epilogues
  int64_t ldg;
  void* out;  // y, or dz (NULL: not wanted)
  int64_t ldo;
  void* dx;
  int64_t lddx;
};

// Contraction steps (of 64 bytes) that a resident kernel exists for, the LDS a
// workgroup may use, and the steps up to which it can form dx as well.
constexpr int kResidentSteps16[] = {2, 4, 8};
constexpr int kResidentSteps32[] = {2, 4, 6, 9, 12, 16};
constexpr int kResidentLds = 160 * 1024;
constexpr int kResidentDxSteps = 4;

int launch_resident_bf16(const ResidentParams& p, int steps, int epi, bool with_dx, int workgroups, hipStream_t stream);
int launch_resident_f16(const ResidentParams& p, int steps, int epi, bool with_dx, int workgroups, hipStream_t stream);
int launch_resident_f32(const ResidentParams& p, int steps, int epi, bool with_dx, int workgroups, hipStream_t stream);

// A product of a few rows (few_rows_impl.h).
struct FewRowsParams {
  const void* x;
  int64_t ldx;
  int32_t rows;
  const void* w;
  int64_t ldw, n, width;  // outputs (gated: of a half), contraction
  const void* bias;
  int32_t bias_dtype, activation;
  const void* residual;
  int64_t ldr;
  void* out;
  int64_t ldo;
};
constexpr int kFewRows = 32;

int launch_few_rows_bf16(const FewRowsParams& p, bool gated, hipStream_t stream);
int launch_few_rows_f16(const FewRowsParams& p, bool gated, hipStream_t stream);
int launch_few_rows_f32(const FewRowsParams& p, bool gated, hipStream_t stream);

}  // namespace vectra_dense
