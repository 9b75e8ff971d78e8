// The residual stream with a branch's output, and its norm: forward and backward
// kernel templates, instantiated per pair of types in norm_<branch>_<stream>.hip.
//
//   h = s r + gate * k * post(x),  n = norm(h)
//
// A row of `width` elements is held in registers by 16 to 1024 lanes, eight
// consecutive columns each (two such chunks past 8192 columns): 16 bytes of a
// 16-bit row per lane and access.  Everything between the loads and the stores of
// a row happens there, so each tensor is moved once; the per-column vectors are
// loaded once per workgroup, and the next row's loads are issued before a row is
// worked on.  What bounds it is HBM; the sums of a row cross lanes by DPP moves and
// lane swaps, and waves through LDS with one barrier each.
//
// Layer norm's variance is the mean of (x - mean)^2, not a difference of squares:
// within a wave from the wave's own mean, the waves' joined by
//   sum (x - mean)^2 = sum over waves of [sum (x - mean_w)^2 + count_w (mean_w - mean)^2].
//
// The backward pass computes the normalised rows again, from x and r where a gate
// or a post norm needs them anyway (h is then not read: the same bytes, and in
// fp32 as the forward pass had it), else from h as it was rounded; statistics are
// not kept.  The vectors' gradients are summed over the rows of a workgroup in
// registers, then over the workgroups by a second launch in a fixed order.
#pragma once

#include "block_common.h"
#include "block_kernels.h"

namespace vectra_block {

using vectra::OpMax;
using vectra::OpSum;
using vectra::reduce_low;

// Threads of the workgroup that holds rows of so many lanes.
constexpr int row_threads(int lanes) { return lanes > 64 ? lanes : 256; }

template <int kLanes_, int kChunks_>
struct Row {
  static constexpr int kLanes = kLanes_, kChunks = kChunks_;
  static constexpr bool kMany = kLanes > 64;  // several waves per row, one row per workgroup
  static constexpr int kThreads = row_threads(kLanes);
  static constexpr int kRows = kThreads / kLanes;
  static constexpr int kWaves = kMany ? kLanes / 64 : 1;

  typedef f32x4 Values[kChunks][2];  // a lane's part of a row; 0 past the row's end

  int lane, slot;
  int64_t width;
  int64_t column[kChunks];
  int left[kChunks];  // elements of the chunk that exist
  f32x4* lds;         // 2 kWaves of them
  int turn = 0;

  __device__ __forceinline__ Row(int64_t width_, f32x4* lds_) : width(width_), lds(lds_) {
    lane = threadIdx.x % kLanes;
    slot = threadIdx.x / kLanes;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      column[j] = (static_cast<int64_t>(j) * kLanes + lane) * 8;
      left[j] = static_cast<int>(most(least(width - column[j], 8), 0));
    }
  }

  // What each wave of the row holds, for all of them to read.  Two buffers: a wave
  // may write the next while another still reads this one, and no further.
  __device__ __forceinline__ const f32x4* share(f32x4 mine) {
    f32x4* const at = lds + turn * kWaves;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = mine;
    __syncthreads();
    return at;
  }

  static __device__ __forceinline__ float wave_sum(float v) { return reduce_low<kLanes < 64 ? kLanes : 64>(v, OpSum{}); }

  // Sums of two quantities over the row's lanes.
  __device__ __forceinline__ void sum(float& a, float& b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (kMany) {
      const f32x4* const at = share(f32x4{a, b, 0.f, 0.f});
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f32x4 v = at[w];
        a += v[0];
        b += v[1];
      }
    }
  }

  // v / sqrt(mean(v^2) + eps) in place, and that factor.
  __device__ __forceinline__ float normalise_rms(Values& v, float inverse_width, float eps) {
    float s = 0.f, none = 0.f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s = __builtin_fmaf(v[j][i / 4][i % 4], v[j][i / 4][i % 4], s);
    sum(s, none);
    const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(s, inverse_width, eps));
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      v[j][0] *= r;
      v[j][1] *= r;
    }
    return r;
  }

  // (v - mean) / sqrt(var + eps) in place (0 past the row's end), and the factor.
  __device__ __forceinline__ float normalise_layer(Values& v, float inverse_width, float eps) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[j][i / 4][i % 4];
    s = wave_sum(s);
    float mean = s * inverse_width, count = 0.f;
    if constexpr (kMany) {  // of this wave's elements first
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
        count += static_cast<float>(most(least(width - (column[j] - (lane & 63) * 8), 512), 0));
      mean = count > 0.f ? s / count : 0.f;
    }
    float m2 = 0.f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = i < left[j] ? v[j][i / 4][i % 4] - mean : 0.f;
        m2 = __builtin_fmaf(d, d, m2);
      }
    m2 = wave_sum(m2);
    if constexpr (kMany) {
      const f32x4* const at = share(f32x4{s, m2, count, mean});
      s = m2 = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += at[w][0];
      mean = s * inverse_width;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f32x4 u = at[w];
        const float d = u[3] - mean;
        m2 += __builtin_fmaf(u[2] * d, d, u[1]);
      }
    }
    const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(m2, inverse_width, eps));
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i / 4][i % 4] = i < left[j] ? (v[j][i / 4][i % 4] - mean) * r : 0.f;
    return r;
  }

  __device__ __forceinline__ float normalise(Values& v, int kind, float inverse_width, float eps) {
    return kind == VECTRA_BLOCK_RMS ? normalise_rms(v, inverse_width, eps) : normalise_layer(v, inverse_width, eps);
  }

  // The norm's transpose: of g, the gradient before the affine part, to the
  // gradient of the norm's input.  g <- r (g - hat mean(g hat) [- mean(g)]).
  __device__ __forceinline__ void transpose(Values& g, const Values& hat, float r, int kind, float inverse_width) {
    float along = 0.f, total = 0.f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        along = __builtin_fmaf(g[j][i / 4][i % 4], hat[j][i / 4][i % 4], along);
        total += g[j][i / 4][i % 4];
      }
    sum(along, total);
    along *= inverse_width;
    total = kind == VECTRA_BLOCK_LAYER ? total * inverse_width : 0.f;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) g[j][h] = (g[j][h] - hat[j][h] * along - total) * r;
  }

  __device__ __forceinline__ void load_vector_of(const Vector& v, int64_t at, float missing, Values& out) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const void* const row =
          v.p ? static_cast<const char*>(v.p) + at * (v.dtype == VECTRA_BLOCK_F32 ? 4 : 2) : nullptr;
      load_vector(row, v.dtype, column[j], left[j], missing, out[j]);
    }
  }

  template <typename T>
  __device__ __forceinline__ void load(const void* p, int64_t row, int64_t stride, Eight<T> (&out)[kChunks]) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if (left[j] > 0)
        out[j] = load_eight<T>(static_cast<const T*>(p) + row * stride, width, column[j]);
      else
        out[j] = Eight<T>{};
    }
  }

  template <typename T>
  __device__ __forceinline__ void store(void* p, int64_t row, int64_t stride, const Values& v) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      if (left[j] > 0) store8(static_cast<T*>(p) + row * stride + column[j], v[j][0], v[j][1], left[j]);
  }
};

template <typename T, int kChunks>
__device__ __forceinline__ void widen_row(const Eight<T> (&in)[kChunks], f32x4 (&out)[kChunks][2]) {
#pragma unroll
  for (int j = 0; j < kChunks; ++j) widen_eight(in[j], out[j][0], out[j][1]);
}

// -------------------------------------------------------------------- forward

template <typename T, typename R, int kLanes, int kChunks>
__global__ __launch_bounds__(row_threads(kLanes)) void norm_kernel(const NormParams p) {
  using Row = Row<kLanes, kChunks>;
  typedef typename Row::Values Values;
  __shared__ f32x4 lds[2 * Row::kWaves];
  Row row(p.width, lds);
  Values weight, bias, gate, post_weight, post_bias;
  row.load_vector_of(p.weight, 0, 1.f, weight);
  row.load_vector_of(p.bias, 0, 0.f, bias);
  row.load_vector_of(p.post_weight, 0, 1.f, post_weight);
  row.load_vector_of(p.post_bias, 0, 0.f, post_bias);
  const bool gate_each = p.gate.p && p.gate_rows < p.rows;
  row.load_vector_of(p.gate, 0, 1.f, gate);
  const Dropout dropout{p.rng, p.threshold, p.stream_id, p.drop_scale};
  const DropoutKey key = dropout_key(dropout);
  const uint32_t groups = static_cast<uint32_t>((p.width + 7) / 8);

  const int64_t step = static_cast<int64_t>(gridDim.x) * Row::kRows;
  Eight<T> x_next[kChunks];
  Eight<R> r_next[kChunks];
  const auto fetch = [&](int64_t base) {
    const int64_t at = least(base + row.slot, p.rows - 1);  // (rows past the end repeat the last; they are not stored)
    row.load(p.x, at, p.x_stride, x_next);
    row.load(p.residual, at, p.residual_stride, r_next);
  };
  int64_t base = static_cast<int64_t>(blockIdx.x) * Row::kRows;
  if (base < p.rows) fetch(base);
  for (; base < p.rows; base += step) {
    const bool live = base + row.slot < p.rows;
    const int64_t at = live ? base + row.slot : p.rows - 1;
    Values v, h;
    widen_row(x_next, v);
    widen_row(r_next, h);
    if (base + step < p.rows) fetch(base + step);
    if (gate_each)
      row.load_vector_of(p.gate, static_cast<uint32_t>(at) / static_cast<uint32_t>(p.gate_rows) * p.gate_stride, 1.f, gate);
    if (p.post != VECTRA_BLOCK_NO_NORM) {
      row.normalise(v, p.post, p.inverse_width, p.eps);
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) v[j][e] = v[j][e] * post_weight[j][e] + post_bias[j][e];
    }
    if (p.threshold) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        f32x4 k[2];
        dropout_factors(dropout, key, static_cast<uint64_t>(at) * groups + (row.column[j] >> 3), k);
        drop(v[j], k);
      }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) h[j][e] = h[j][e] * p.residual_scale + v[j][e] * gate[j][e];
    if (live) row.template store<R>(p.h, at, p.h_stride, h);
    row.normalise(h, p.norm, p.inverse_width, p.eps);
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) h[j][e] = h[j][e] * weight[j][e] + bias[j][e];
    if (p.n) {
      if (live) row.template store<T>(p.n, at, p.n_stride, h);
    } else {
      // 8-bit rows: a block of 128 is held by 16 adjacent lanes.
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const float largest = reduce_low<16>(vectra_dense::largest_finite(h[j], 0.f), OpMax{});
        const int byte = vectra_dense::block_exponent(largest, kLowestExponent);
        const uint2 w = vectra_dense::to_codes(h[j], byte - 127, kHighestExponent);
        if (!live || row.column[j] >= p.depth) continue;
        *reinterpret_cast<uint2*>(p.codes + at * p.depth + row.column[j]) = w;
        if (row.lane % 16 == 0) p.scales[at * p.scale_stride + row.column[j] / 128] = static_cast<uint8_t>(byte);
      }
      if (live)
        for (int64_t k = p.depth / 128 + row.lane; k < p.scale_stride; k += kLanes) p.scales[at * p.scale_stride + k] = 0;
    }
  }
}

// ------------------------------------------------------------------- backward

// kBranch: the branch's output matters, by a gate or a post norm; x and r are read,
// else h.
template <typename T, typename R, int kLanes, int kChunks, bool kBranch>
__global__ __launch_bounds__(row_threads(kLanes)) void norm_grad_kernel(const NormGradParams p) {
  using Row = Row<kLanes, kChunks>;
  typedef typename Row::Values Values;
  __shared__ f32x4 lds[2 * Row::kWaves];
  __shared__ float slots[Row::kMany ? 1 : Row::kRows][Row::kMany ? 1 : kLanes * 8 + 4];
  Row row(p.width, lds);
  Values weight, gate, post_weight, post_bias;
  row.load_vector_of(p.weight, 0, 1.f, weight);
  if constexpr (kBranch) {
    row.load_vector_of(p.post_weight, 0, 1.f, post_weight);
    row.load_vector_of(p.post_bias, 0, 0.f, post_bias);
    row.load_vector_of(p.gate, 0, 1.f, gate);
  }
  const bool gate_full = p.gate.p && p.gate_rows == 1;  // a gate row, and its gradient, for each row
  const bool gate_each = p.gate.p && p.unit_rows == p.gate_rows;
  const Dropout dropout{p.rng, p.threshold, p.stream_id, p.drop_scale};
  const DropoutKey key = dropout_key(dropout);
  const uint32_t groups = static_cast<uint32_t>((p.width + 7) / 8);

  Values d_weight = {}, d_bias = {}, d_gate = {}, d_post_weight = {}, d_post_bias = {};

  // The sum over the workgroup's slots of what each holds of a vector's gradient.
  // To all threads' d of slot 0; a workgroup with one slot has it already.
  const auto over_slots = [&](Values& d) {
    if constexpr (!Row::kMany) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) slots[row.slot][row.lane * 8 + e] = d[0][e / 4][e % 4];
      __syncthreads();
      if (row.slot == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < Row::kRows; ++k) s += slots[k][row.lane * 8 + e];
          d[0][e / 4][e % 4] = s;
        }
      }
    }
  };
  const auto write_sums = [&](Values& d, float* to) {
    over_slots(d);
    if (row.slot == 0)
#pragma unroll
      for (int j = 0; j < kChunks; ++j) store_vector(to, VECTRA_BLOCK_F32, row.column[j], row.left[j], d[j]);
  };

  Eight<T> g_next[kChunks], x_next[kBranch ? kChunks : 1];
  Eight<R> gh_next[kChunks], r_next[kChunks];
  const auto fetch = [&](int64_t at) {
    if (p.grad_n) row.load(p.grad_n, at, p.grad_n_stride, g_next);
    if (p.grad_h) row.load(p.grad_h, at, p.grad_h_stride, gh_next);
    if constexpr (kBranch) {
      row.load(p.x, at, p.x_stride, x_next);
      row.load(p.residual, at, p.residual_stride, r_next);
    } else {
      row.load(p.h, at, p.h_stride, r_next);
    }
  };
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    g_next[j] = Eight<T>{};
    gh_next[j] = Eight<R>{};
  }

  const int64_t unit_first = p.units * blockIdx.x / gridDim.x, unit_last = p.units * (blockIdx.x + 1) / gridDim.x;
  for (int64_t unit = unit_first; unit < unit_last; ++unit) {
    const int64_t group = unit / p.parts, part = unit - group * p.parts;
    const int64_t first = group * p.unit_rows + part * p.rows_per_part;
    const int64_t last = least(least(first + p.rows_per_part, (group + 1) * p.unit_rows), p.rows);
    if constexpr (kBranch) {
      if (gate_each && !gate_full) row.load_vector_of(p.gate, group * p.gate_stride, 1.f, gate);
    }
    if (first < last) fetch(least(first + row.slot, last - 1));
    for (int64_t base = first; base < last; base += Row::kRows) {
      const bool live = base + row.slot < last;
      const int64_t at = live ? base + row.slot : last - 1;
      Values g, gt, x, h;
      widen_row(g_next, g);
      widen_row(gh_next, gt);
      widen_row(r_next, h);
      if constexpr (kBranch) {
        widen_row(x_next, x);
        if (gate_full) row.load_vector_of(p.gate, at * p.gate_stride, 1.f, gate);
      }
      if (base + Row::kRows < last) fetch(least(base + Row::kRows + row.slot, last - 1));
      if (!live) {  // (a row of another slot: it must not be summed twice)
#pragma unroll
        for (int j = 0; j < kChunks; ++j) g[j][0] = g[j][1] = gt[j][0] = gt[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      f32x4 k[kChunks][2];
      if (p.threshold) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
          dropout_factors(dropout, key, static_cast<uint64_t>(at) * groups + (row.column[j] >> 3), k[j]);
      }
      float post_r = 1.f;
      Values v;  // the branch before its gate
      if constexpr (kBranch) {
        if (p.post != VECTRA_BLOCK_NO_NORM) post_r = row.normalise(x, p.post, p.inverse_width, p.eps);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            v[j][e] = p.post != VECTRA_BLOCK_NO_NORM ? x[j][e] * post_weight[j][e] + post_bias[j][e] : x[j][e];
          if (p.threshold) drop(v[j], k[j]);
#pragma unroll
          for (int e = 0; e < 2; ++e) h[j][e] = h[j][e] * p.residual_scale + v[j][e] * gate[j][e];
        }
      }
      if (p.grad_n) {
        const float r = row.normalise(h, p.norm, p.inverse_width, p.eps);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            d_weight[j][e] += g[j][e] * h[j][e];
            d_bias[j][e] += g[j][e];
            g[j][e] *= weight[j][e];
          }
        row.transpose(g, h, r, p.norm, p.inverse_width);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) gt[j][e] += g[j][e];
      }
      if (p.dresidual && live) {
        Values d;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) d[j][e] = gt[j][e] * p.residual_scale;
        row.template store<R>(p.dresidual, at, p.dresidual_stride, d);
      }
      if constexpr (kBranch) {
        Values own;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            own[j][e] = gt[j][e] * v[j][e];
            d_gate[j][e] += own[j][e];
            gt[j][e] *= gate[j][e];
          }
        if (p.dgate && gate_full && live) {
#pragma unroll
          for (int j = 0; j < kChunks; ++j)
            store_vector(static_cast<char*>(p.dgate) + at * p.dgate_stride * (p.dgate_dtype == VECTRA_BLOCK_F32 ? 4 : 2),
                         p.dgate_dtype, row.column[j], row.left[j], own[j]);
        }
      }
      if (p.threshold) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) drop(gt[j], k[j]);
      }
      if constexpr (kBranch) {
        if (p.post != VECTRA_BLOCK_NO_NORM) {
#pragma unroll
          for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              d_post_weight[j][e] += gt[j][e] * x[j][e];
              d_post_bias[j][e] += gt[j][e];
              gt[j][e] *= post_weight[j][e];
            }
          row.transpose(gt, x, post_r, p.post, p.inverse_width);
        }
      }
      if (p.dx && live) row.template store<T>(p.dx, at, p.dx_stride, gt);
    }
    if constexpr (kBranch) {
      if (p.gate_sums || (p.dgate && !gate_full)) {
        over_slots(d_gate);
        if (row.slot == 0) {
#pragma unroll
          for (int j = 0; j < kChunks; ++j) {
            if (p.gate_sums)
              store_vector(p.gate_sums + unit * p.width, VECTRA_BLOCK_F32, row.column[j], row.left[j], d_gate[j]);
            else
              store_vector(static_cast<char*>(p.dgate) + group * p.dgate_stride * (p.dgate_dtype == VECTRA_BLOCK_F32 ? 4 : 2),
                           p.dgate_dtype, row.column[j], row.left[j], d_gate[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j) d_gate[j][0] = d_gate[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  const int64_t plane = static_cast<int64_t>(blockIdx.x) * p.width;
  if (p.weight_sums) write_sums(d_weight, p.weight_sums + plane);
  if (p.bias_sums) write_sums(d_bias, p.bias_sums + plane);
  if constexpr (kBranch) {
    if (p.post_weight_sums) write_sums(d_post_weight, p.post_weight_sums + plane);
    if (p.post_bias_sums) write_sums(d_post_bias, p.post_bias_sums + plane);
  }
}

// ----------------------------------------------------------------------- host

template <int kLanes_, int kChunks_>
struct Shape {
  static constexpr int kLanes = kLanes_, kChunks = kChunks_;
};

template <typename F>
void with_shape(int64_t width, F&& f) {
  switch (norm_lanes(width)) {
    case 16: return f(Shape<16, 1>{});
    case 32: return f(Shape<32, 1>{});
    case 64: return f(Shape<64, 1>{});
    case 128: return f(Shape<128, 1>{});
    case 256: return f(Shape<256, 1>{});
    case 512: return f(Shape<512, 1>{});
    default: return width <= 8192 ? f(Shape<1024, 1>{}) : f(Shape<1024, 2>{});
  }
}

template <typename T, typename R>
int launch_norm(const NormParams& p, int cus, hipStream_t stream) {
  with_shape(p.width, [&](auto shape) {
    using S = decltype(shape);
    using Geometry = Row<S::kLanes, S::kChunks>;
    const int64_t blocks = (p.rows + Geometry::kRows - 1) / Geometry::kRows;
    const int64_t most_blocks = static_cast<int64_t>(cus) * (2048 / Geometry::kThreads);
    norm_kernel<T, R, S::kLanes, S::kChunks>
        <<<static_cast<uint32_t>(blocks < most_blocks ? blocks : most_blocks), Geometry::kThreads, 0, stream>>>(p);
  });
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

template <typename T, typename R>
int launch_norm_grad(const NormGradParams& p, int workgroups, hipStream_t stream) {
  with_shape(p.width, [&](auto shape) {
    using S = decltype(shape);
    constexpr int kThreads = Row<S::kLanes, S::kChunks>::kThreads;
    const auto kernel = p.x ? norm_grad_kernel<T, R, S::kLanes, S::kChunks, true>
                            : norm_grad_kernel<T, R, S::kLanes, S::kChunks, false>;
    kernel<<<static_cast<uint32_t>(workgroups), kThreads, 0, stream>>>(p);
  });
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

}  // namespace vectra_block
