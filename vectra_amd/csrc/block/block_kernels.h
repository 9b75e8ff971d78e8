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

// How a row of a norm lies in a workgroup: on 16, 32 or 64 lanes, several rows in one
// of 256 threads, or on all lanes of a workgroup of as many waves as its width takes
// (1152 fp16 on 3 waves instead of 4: 52 -> 50 us forward); eight columns per lane and
// chunk, past 8 waves more chunks.
struct NormShape {
  int lanes, chunks, threads, rows;
};

inline NormShape norm_shape(int64_t width) {
  for (int lanes = 16; lanes <= 64; lanes *= 2)
    if (width <= lanes * 8) return NormShape{lanes, 1, 256, 256 / lanes};
  const int chunks = width <= 4096 ? 1 : width <= 8192 ? 2 : 4;
  const int lanes = static_cast<int>((width + 512 * chunks - 1) / (512 * chunks)) * 64;
  return NormShape{lanes > 64 ? lanes : 128, chunks, lanes > 64 ? lanes : 128, 1};
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
