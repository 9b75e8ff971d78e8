// What the block library's host code launches.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vectra_block.h"

namespace vectra_block {

struct Vector {
  const void* p;
  int32_t dtype;
};

struct NormParams {
  const void* x;
  const void* residual;
  Vector weight, bias, gate, post_weight, post_bias;
  const int64_t* rng;
  void* h;
  void* n;
  uint8_t* codes;
  uint8_t* scales;
  int32_t norm, post, threshold;
  uint32_t stream_id;
  float eps, residual_scale, drop_scale, inverse_width;
  int64_t rows, width, gate_rows, depth, scale_stride;
  int64_t x_stride, residual_stride, gate_stride, h_stride, n_stride;
};

struct NormGradParams {
  const void* grad_h;
  const void* grad_n;
  const void* x;
  const void* residual;
  const void* h;
  Vector weight, gate, post_weight, post_bias;
  const int64_t* rng;
  void* dx;
  void* dresidual;
  // The vectors' sums over each workgroup's rows, fp32 [workgroups, width] each;
  // NULL: not wanted.
  float* weight_sums;
  float* bias_sums;
  float* post_weight_sums;
  float* post_bias_sums;
  // The gate's gradient: its own rows where one workgroup sums all of a gate row's
  // (dgate), else sums over each part of them, fp32 [units, width] (gate_sums).
  void* dgate;
  float* gate_sums;
  int32_t dgate_dtype;
  int32_t norm, post, threshold;
  uint32_t stream_id;
  float eps, residual_scale, drop_scale, inverse_width;
  int64_t rows, width, gate_rows;
  int64_t grad_h_stride, grad_n_stride, x_stride, residual_stride, h_stride, gate_stride;
  int64_t dx_stride, dresidual_stride, dgate_stride;
  // Units of work: of the unit_rows rows from (u / parts) * unit_rows on, those from
  // (u % parts) * rows_per_part on.  unit_rows: gate_rows where a gate row's gradient
  // is a sum over several rows, else all rows.
  int64_t units, unit_rows, rows_per_part;
  int32_t parts;
};

// Rows of a workgroup, by the lanes a row takes: 8 columns each.  Up to 64 lanes a
// workgroup of 256 holds several rows; more lanes are a workgroup of their own.
// The widest rows take two chunks per lane.
constexpr int kNormLanes[] = {16, 32, 64, 128, 256, 512, 1024};
constexpr int kNormWidths[] = {128, 256, 512, 1024, 2048, 4096, 8192};

inline int norm_lanes(int64_t width) {
  for (int i = 0; i < 7; ++i)
    if (width <= kNormWidths[i]) return kNormLanes[i];
  return 1024;
}

// One definition per pair of types (of the branch, of the stream).
int launch_norm_f32_f32(const NormParams& p, int cus, hipStream_t stream);
int launch_norm_f16_f16(const NormParams& p, int cus, hipStream_t stream);
int launch_norm_f16_f32(const NormParams& p, int cus, hipStream_t stream);
int launch_norm_bf16_bf16(const NormParams& p, int cus, hipStream_t stream);
int launch_norm_bf16_f32(const NormParams& p, int cus, hipStream_t stream);

int launch_norm_grad_f32_f32(const NormGradParams& p, int workgroups, hipStream_t stream);
int launch_norm_grad_f16_f16(const NormGradParams& p, int workgroups, hipStream_t stream);
int launch_norm_grad_f16_f32(const NormGradParams& p, int workgroups, hipStream_t stream);
int launch_norm_grad_bf16_bf16(const NormGradParams& p, int workgroups, hipStream_t stream);
int launch_norm_grad_bf16_f32(const NormGradParams& p, int workgroups, hipStream_t stream);

}  // namespace vectra_block
