// The residual stream with a branch's output, and its norm: forward and backward
// kernel templates, instantiated per pair of types in norm_<branch>_<stream>.hip.
//
//   h = s r + gate * k * post(x),  n = norm(h)
//
// A row of `width` elements is held in registers by 16, 32 or 64 lanes or by up to 8
// waves, eight consecutive columns per lane (past 4096 columns two or four such
// chunks): 16 bytes of a 16-bit row per lane and access.  Everything between the loads
// and the stores of a row happens there, so each tensor is moved once; the per-column
// vectors are loaded once per workgroup, and the next row's loads are issued before a
// row is worked on.  The sums of a row cross lanes by DPP moves and lane swaps, and
// waves through LDS with one barrier each.  What bounds it is HBM: 8192 x 4096 bf16 on
// an fp32 stream, rms norms on both sides and a gate over all rows, 82 us forward
// (4.9 TB/s) and 140 backward with the joining of its sums (4.3).  Short rows are bound by
// vector issue beside it: 66560 x 128 bf16, layer norm and dropout, 18.8 us and 34.7
// (3.6, 2.9 TB/s).  Past 4096 columns the registers do not hold a row, its
// gradients and their sums over the rows: most of the sums are in LDS there, and no row
// is loaded ahead; past 8192 columns, and in the backward pass with a gate and a post norm,
// the vectors over the columns are read again for every row.  4096 x 8192, both norms and
// a gate, 82 us and 214 (all in registers, spilled: 139 and 405; the vectors read again
// 100 forward); 2048 x 16384 108 us and 337 (184, 1740).
//
// Layer norm's variance is the mean of (x - mean)^2, not a difference of squares:
// within a wave from the wave's own mean, the waves' joined by
//   sum (x - mean)^2 = sum over waves of [sum (x - mean_w)^2 + count_w (mean_w - mean)^2].
//
// The backward pass computes the normalised rows again, from x and r (h is then not
// read) or from an fp32 h, in fp32 as the forward pass had them; statistics are
// not kept.  The vectors' gradients are summed over the rows of a workgroup, then over the
// workgroups by a second launch in a fixed order.
#pragma once

#include "block_common.h"
#include "block_kernels.h"

namespace vectra_block {

using vectra::OpMax;
using vectra::OpSum;
using vectra::reduce_low;
using vectra_dense::u32x4;

// How a row's last chunk is read.  Whole: rows are whole chunks.  Ragged: as the row's
// last eight elements, moved into place afterwards; read element by element, it would
// be waited for before the next load (6000 x 1001 bf16 backward 46 -> 36 us, of 5 rows read or written).  Narrow:
// rows of fewer than eight elements, by those.  (Kinds of their own, because a branch
// among the loads of the row ahead waits for them where its sides meet: 8192 x 4096
// forward 77 us, with such a branch 112.)
enum { kWhole = 0, kRagged = 1, kNarrow = 2 };

// 1 / sqrt(v); the instruction takes subnormals for zero.
__device__ __forceinline__ float inverse_root(float v) {
  const bool small = v < 0x1p-126f;
  return __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v) * (small ? 0x1p32f : 1.f);
}

// kLanes: of a row, or 0: all of the workgroup's (kMany).
constexpr int kMany = 0;
constexpr int kMostLanes = 512;
constexpr int row_threads(int lanes) { return lanes == kMany ? kMostLanes : 256; }  // at most

// kKeep: the vectors over the columns stay in registers (Held).
template <int kLanes, int kChunks_, int kKind, bool kKeep>
struct Row {
  static constexpr int kChunks = kChunks_;
  static constexpr bool kWaves = kLanes == kMany;  // several waves per row, one row per workgroup
  static constexpr int kRows = kWaves ? 1 : 256 / kLanes;
  static constexpr int kLds = kWaves ? 2 * kMostLanes / 64 : 1;

  typedef f32x4 Values[kChunks][2];  // a lane's part of a row; 0 past the row's end

  int lane, slot, lanes, waves;
  int64_t width;
  int32_t column[kChunks];
  int left[kChunks];  // elements of the chunk that exist
  f32x4* lds;         // kLds of them
  int turn = 0;

  __device__ __forceinline__ Row(int64_t width_, f32x4* lds_) : width(width_), lds(lds_) {
    lanes = kWaves ? static_cast<int>(blockDim.x) : kLanes;
    waves = lanes / 64;
    lane = kWaves ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % kLanes;
    slot = kWaves ? 0 : static_cast<int>(threadIdx.x) / kLanes;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      column[j] = (j * lanes + lane) * 8;
      left[j] = max(min(static_cast<int>(width) - column[j], 8), 0);
    }
  }

  // What each wave of the row holds, for all of them to read.  Two buffers: a wave
  // may write the next while another still reads this one, and no further.
  __device__ __forceinline__ const f32x4* share(f32x4 mine) {
    f32x4* const at = lds + turn;
    turn ^= kMostLanes / 64;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = mine;
    __syncthreads();
    return at;
  }

  static __device__ __forceinline__ float wave_sum(float v) { return reduce_low<kWaves ? 64 : kLanes>(v, OpSum{}); }

  // Sums of two quantities over the row's lanes.
  __device__ __forceinline__ void sum(float& a, float& b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (kWaves) {
      const f32x4* const at = share(f32x4{a, b, 0.f, 0.f});
      a = b = 0.f;
#pragma unroll 2
      for (int w = 0; w < waves; ++w) {
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
    const float r = inverse_root(__builtin_fmaf(s, inverse_width, eps));
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
    if constexpr (kWaves) {  // of this wave's elements first
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
        count += static_cast<float>(max(min(static_cast<int>(width) - (column[j] - (lane & 63) * 8), 512), 0));
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
    if constexpr (kWaves) {
      const f32x4* const at = share(f32x4{s, m2, count, mean});
      s = m2 = 0.f;
#pragma unroll 2
      for (int w = 0; w < waves; ++w) s += at[w][0];
      mean = s * inverse_width;
#pragma unroll 2
      for (int w = 0; w < waves; ++w) {
        const f32x4 u = at[w];
        const float d = u[3] - mean;
        m2 += __builtin_fmaf(u[2] * d, d, u[1]);
      }
    }
    const float r = inverse_root(__builtin_fmaf(m2, inverse_width, eps));
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

  // A vector over the columns, from element `at` of it on: held in registers (kKeep), or,
  // where they are full, read where it is used (from L1 and L2: every row reads the
  // same).
  struct Held {
    Vector from;
    int64_t at;
    float missing;
    f32x4 value[kKeep ? kChunks * 2 : 1];
  };
  // Chunk j's first column; with several chunks, whose registers are full, known anew at
  // each use: an address for every vector, chunk and type would be held over the loop.
  __device__ __forceinline__ int column_of(int j) const {
    int at = column[j];
    if constexpr (kChunks > 1) asm volatile("" : "+v"(at));
    return at;
  }
  __device__ __forceinline__ void load_chunk(const Held& v, int j, f32x4(&out)[2]) const {
    const void* const row =
        v.from.p ? static_cast<const char*>(v.from.p) + v.at * (v.from.dtype == VECTRA_BLOCK_F32 ? 4 : 2) : nullptr;
    load_vector(row, v.from.dtype, column_of(j), left[j], v.missing, out);
  }
  __device__ __forceinline__ void hold(const Vector& from, int64_t at, float missing, Held& v) const {
    v.from = from;
    v.at = at;
    v.missing = missing;
    if constexpr (kKeep)
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        f32x4 chunk[2];
        load_chunk(v, j, chunk);
        v.value[j * 2] = chunk[0];
        v.value[j * 2 + 1] = chunk[1];
      }
  }
  __device__ __forceinline__ void use(const Held& v, int j, f32x4(&out)[2]) const {
    if constexpr (kKeep) {
      out[0] = v.value[j * 2];
      out[1] = v.value[j * 2 + 1];
    } else {
      load_chunk(v, j, out);
    }
  }
  // The same in two steps, the loads and the conversion: a gate's row on its way while
  // the row before is worked on.
  struct Coming {
    u32x4 w[2];
  };
  __device__ __forceinline__ void fetch(const Held& v, Coming& c) const {
    if (v.from.dtype == VECTRA_BLOCK_F32) {
      const Eight<float> e = load_chunk_of(static_cast<const float*>(v.from.p) + v.at, 0);
      c.w[0] = e.part[0].w;
      c.w[1] = e.part[1].w;
    } else {
      c.w[0] = load_chunk_of(static_cast<const _Float16*>(v.from.p) + v.at, 0).part[0].w;
    }
  }
  __device__ __forceinline__ void take(const Coming& c, Held& v) const {
    if (v.from.dtype == VECTRA_BLOCK_F32) {
      Eight<float> e;
      e.part[0].w = c.w[0];
      e.part[1].w = c.w[1];
      widen_chunk(e, 0, reinterpret_cast<f32x4(&)[2]>(v.value));
    } else if (v.from.dtype == VECTRA_BLOCK_F16) {
      Eight<_Float16> e;
      e.part[0].w = c.w[0];
      widen_chunk(e, 0, reinterpret_cast<f32x4(&)[2]>(v.value));
    } else {
      Eight<__bf16> e;
      e.part[0].w = c.w[0];
      widen_chunk(e, 0, reinterpret_cast<f32x4(&)[2]>(v.value));
    }
  }
  // x * weight + bias in place.
  __device__ __forceinline__ void affine(f32x4(&x)[2], const Held& weight, const Held& bias, int j) const {
    f32x4 w[2], b[2];
    use(weight, j, w);
    use(bias, j, b);
#pragma unroll
    for (int e = 0; e < 2; ++e) x[e] = x[e] * w[e] + b[e];
  }

  // Chunk j of a row as it is in memory.
  template <typename T>
  __device__ __forceinline__ Eight<T> load_chunk_of(const T* row, int j) const {
    Eight<T> e{};
    if (left[j] > 0) {
      if constexpr (kKind == kNarrow) {
        e = load_eight<T>(row, width, column[j]);
      } else {
        const int at = column_of(j);
        const T* const from = row + (kKind == kRagged ? min(at, static_cast<int>(width) - 8) : at);
        __builtin_memcpy(&e, from, sizeof(e));  // unaligned
      }
    }
    return e;
  }
  template <typename T>
  __device__ __forceinline__ void load(const void* p, int64_t row, int64_t stride, Eight<T> (&out)[kChunks]) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) out[j] = load_chunk_of(static_cast<const T*>(p) + row * stride, j);
  }
  __device__ __forceinline__ void settle_chunk(f32x4(&v)[2], int j) const {
    const int shift = left[j] > 0 ? 8 - left[j] : 0;
#pragma unroll
    for (int by = 1; by < 8; by *= 2)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float from = i + by < 8 ? v[(i + by) / 4 % 2][(i + by) % 4] : 0.f;
        v[i / 4][i % 4] = shift & by ? from : v[i / 4][i % 4];
      }
  }
  template <typename T>
  __device__ __forceinline__ void widen_chunk(const Eight<T>& in, int j, f32x4(&out)[2]) const {
    widen_eight(in, out[0], out[1]);
    if constexpr (kKind == kRagged) settle_chunk(out, j);
  }
  template <typename T>
  __device__ __forceinline__ void widen(const Eight<T> (&in)[kChunks], Values& out) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) widen_chunk(in[j], j, out[j]);
  }

  template <typename T>
  __device__ __forceinline__ void store(void* p, int64_t row, int64_t stride, const Values& v) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      if (left[j] > 0) store8(static_cast<T*>(p) + row * stride + column_of(j), v[j][0], v[j][1], left[j]);
  }
};

// -------------------------------------------------------------------- forward

template <typename T, typename R, int kLanes, int kChunks, int kKind>
__global__ __launch_bounds__(row_threads(kLanes)) void norm_kernel(const NormParams p) {
  using Row = Row<kLanes, kChunks, kKind, kChunks <= 2>;
  typedef typename Row::Values Values;
  __shared__ f32x4 lds[Row::kLds];
  Row row(p.width, lds);
  typename Row::Held weight, bias, gate, post_weight, post_bias;
  row.hold(p.weight, 0, 1.f, weight);
  row.hold(p.bias, 0, 0.f, bias);
  row.hold(p.post_weight, 0, 1.f, post_weight);
  row.hold(p.post_bias, 0, 0.f, post_bias);
  const bool gate_each = p.gate.p && p.gate_rows < p.rows;
  row.hold(p.gate, 0, 1.f, gate);
  const Dropout dropout{p.rng, p.threshold, p.stream_id, p.drop_scale};
  const DropoutKey key = dropout_key(dropout);
  const uint32_t groups = static_cast<uint32_t>((p.width + 7) / 8);

  const int64_t step = static_cast<int64_t>(gridDim.x) * Row::kRows;
  Eight<T> x_next[kChunks];
  Eight<R> r_next[kChunks];
  typename Row::Coming gate_next;
  const auto fetch = [&](int64_t base) {
    const int64_t at = least(base + row.slot, p.rows - 1);  // (rows past the end repeat the last; they are not stored)
    row.load(p.x, at, p.x_stride, x_next);
    row.load(p.residual, at, p.residual_stride, r_next);
    if (gate_each) {
      gate.at = static_cast<uint32_t>(at) / static_cast<uint32_t>(p.gate_rows) * p.gate_stride;
      if constexpr (kChunks == 1) row.fetch(gate, gate_next);
      if constexpr (kChunks == 2) row.hold(p.gate, gate.at, 1.f, gate);
    }
  };
  int64_t base = static_cast<int64_t>(blockIdx.x) * Row::kRows;
  if constexpr (kChunks == 1) {  // (the registers of more have no room for a row ahead)
    if (base < p.rows) fetch(base);
  }
  for (; base < p.rows; base += step) {
    const bool live = base + row.slot < p.rows;
    const int64_t at = live ? base + row.slot : p.rows - 1;
    Values v, h;
    if constexpr (kChunks > 1) fetch(base);
    row.widen(x_next, v);
    row.widen(r_next, h);
    if constexpr (kChunks == 1) {
      if (gate_each) row.take(gate_next, gate);
      if (base + step < p.rows) fetch(base + step);
    }
    if (p.post != VECTRA_BLOCK_NO_NORM) {
      row.normalise(v, p.post, p.inverse_width, p.eps);
#pragma unroll
      for (int j = 0; j < kChunks; ++j) row.affine(v[j], post_weight, post_bias, j);
    }
    if (p.threshold) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        drop(v[j], dropout_kept(dropout, key, static_cast<uint64_t>(at) * groups + (row.column[j] >> 3)), p.drop_scale);
      }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      f32x4 k[2];
      row.use(gate, j, k);
#pragma unroll
      for (int e = 0; e < 2; ++e) h[j][e] = h[j][e] * p.residual_scale + v[j][e] * k[e];
    }
    if (live) row.template store<R>(p.h, at, p.h_stride, h);
    row.normalise(h, p.norm, p.inverse_width, p.eps);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) row.affine(h[j], weight, bias, j);
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
        for (int64_t k = p.depth / 128 + row.lane; k < p.scale_stride; k += row.lanes) p.scales[at * p.scale_stride + k] = 0;
    }
  }
}

// ------------------------------------------------------------------- backward

// A lane's sums over the rows of a workgroup: in registers, or, past 4096 columns, whose
// registers are full, in LDS, at kMostLanes vectors apart from `at` on.  A lane's own, which
// no other reads, so nothing waits for them.
template <int kChunks, bool kInLds>
struct Total {
  f32x4 held[kInLds ? 1 : kChunks * 2];
  f32x4* at;
  __device__ __forceinline__ Total(f32x4* mine, int plane) : at(mine + plane * (kChunks * 2 * kMostLanes)) {}
  __device__ __forceinline__ f32x4& of(int j, int e) { return kInLds ? at[(j * 2 + e) * kMostLanes] : held[kInLds ? 0 : j * 2 + e]; }
  __device__ __forceinline__ void add(int j, int e, f32x4 v) { of(j, e) += v; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) of(j, 0) = of(j, 1) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void get(f32x4 (&out)[kChunks][2]) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) out[j][e] = of(j, e);
  }
};

// With a gate or a post norm the branch's output matters: x and r are read.  With a
// stream of 16 bits too, because h as it was rounded is not what the forward pass
// normalised: the weight's gradient, a sum over the rows, would be off by 1.3e-3 of its
// norm (a fifth more bytes: 16384 x 2048 bf16 90 us from x and r, 74 from h).
template <typename T, typename R, int kLanes, int kChunks, int kKind, bool kGate, bool kPost>
__global__ __launch_bounds__(row_threads(kLanes)) void norm_grad_kernel(const NormGradParams p) {
  constexpr bool kBranch = kGate || kPost || sizeof(R) == 2;
  using Row = Row<kLanes, kChunks, kKind, kChunks == 1 || (kChunks == 2 && !(kGate && kPost))>;
  typedef typename Row::Values Values;
  __shared__ f32x4 lds[Row::kLds];
  // The vectors' sums that are in LDS, in order: the weight's, the gate's, the post
  // norm's, the bias's.
  constexpr int kSums = 2 + kGate + 2 * kPost, kFits = kChunks == 1 ? 0 : 8 / kChunks, kInLds = kFits < kSums ? kFits : kSums;
  __shared__ f32x4 planes[kInLds ? kInLds * kChunks * 2 * kMostLanes : 1];
  __shared__ float slots[Row::kRows][Row::kWaves ? 1 : kLanes * 8 + 4];
  Row row(p.width, lds);
  typename Row::Held weight, gate, post_weight, post_bias;
  row.hold(p.weight, 0, 1.f, weight);
  if constexpr (kPost) {
    row.hold(p.post_weight, 0, 1.f, post_weight);
    row.hold(p.post_bias, 0, 0.f, post_bias);
  }
  if constexpr (kGate) row.hold(p.gate, 0, 1.f, gate);
  const bool gate_full = p.gate.p && p.gate_rows == 1;  // a gate row, and its gradient, for each row
  const bool gate_each = p.gate.p && p.unit_rows == p.gate_rows;
  const Dropout dropout{p.rng, p.threshold, p.stream_id, p.drop_scale};
  const DropoutKey key = dropout_key(dropout);
  const uint32_t groups = static_cast<uint32_t>((p.width + 7) / 8);

  f32x4* const mine = planes + (kInLds ? threadIdx.x : 0);
  Total<kChunks, (0 < kInLds)> d_weight(mine, 0);
  Total<kChunks, (1 < kInLds)> d_gate(mine, 1);
  Total<kChunks, (1 + kGate < kInLds)> d_post_weight(mine, 1 + kGate);
  Total<kChunks, (2 + kGate < kInLds)> d_post_bias(mine, 2 + kGate);
  Total<kChunks, (kSums - 1 < kInLds)> d_bias(mine, kSums - 1);
  d_weight.clear();
  d_bias.clear();
  if constexpr (kGate) d_gate.clear();
  if constexpr (kPost) {
    d_post_weight.clear();
    d_post_bias.clear();
  }

  // The sum over the workgroup's slots of what each holds of a vector's gradient.
  // To all threads' d of slot 0; a workgroup with one slot has it already.
  const auto over_slots = [&](Values& d) {
    if constexpr (!Row::kWaves) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) slots[row.slot][row.lane * 8 + e] = d[0][e / 4][e % 4];
      __syncthreads();
      if (row.slot == 0) {
        d[0][0] = d[0][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
        for (int k = 0; k < Row::kRows; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) d[0][e / 4][e % 4] += slots[k][row.lane * 8 + e];
      }
    }
  };
  const auto write_sums = [&](auto& total, float* to) {
    Values d;
    total.get(d);
    over_slots(d);
    if (row.slot == 0)
#pragma unroll
      for (int j = 0; j < kChunks; ++j) store_vector(to, VECTRA_BLOCK_F32, row.column[j], row.left[j], d[j]);
  };

  Eight<T> g_next[kChunks], x_next[kBranch ? kChunks : 1];
  Eight<R> gh_next[kChunks], r_next[kChunks];
  // With four chunks per lane the gradients are loaded where they are used, that of h
  // onto what comes from n's: three rows of values in registers instead of four.
  constexpr bool kLate = kChunks > 2;
  const auto fetch = [&](int64_t at) {
    if constexpr (!kLate) {
      if (p.grad_n) row.load(p.grad_n, at, p.grad_n_stride, g_next);
      if (p.grad_h) row.load(p.grad_h, at, p.grad_h_stride, gh_next);
    }
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
    if constexpr (kGate) {
      if (gate_each && !gate_full) row.hold(p.gate, group * p.gate_stride, 1.f, gate);
    }
    if constexpr (kChunks == 1) {
      if (first < last) fetch(least(first + row.slot, last - 1));
    }
    for (int64_t base = first; base < last; base += Row::kRows) {
      const bool live = base + row.slot < last;
      const int64_t at = live ? base + row.slot : last - 1;
      if constexpr (kChunks > 1) fetch(at);
      Values g, gt, x, h;
      if constexpr (!kLate) {
        row.widen(g_next, g);
        row.widen(gh_next, gt);
      }
      row.widen(r_next, h);
      if constexpr (kBranch) row.widen(x_next, x);
      if constexpr (kGate) {
        if (gate_full) row.hold(p.gate, at * p.gate_stride, 1.f, gate);
      }
      if constexpr (kChunks == 1) {
        if (base + Row::kRows < last) fetch(least(base + Row::kRows + row.slot, last - 1));
      }
      if constexpr (!Row::kWaves) {
        if (!live) {  // (a row of another slot: it must not be summed twice)
#pragma unroll
          for (int j = 0; j < kChunks; ++j) g[j][0] = g[j][1] = gt[j][0] = gt[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
      uint32_t kept[kChunks];
      if (p.threshold) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
          kept[j] = dropout_kept(dropout, key, static_cast<uint64_t>(at) * groups + (row.column[j] >> 3));
      }
      // The branch before its gate, of chunk j: from the normalised x where it has a norm.
      const auto branch = [&](int j, f32x4(&v)[2]) {
        v[0] = x[j][0];
        v[1] = x[j][1];
        if constexpr (kPost) row.affine(v, post_weight, post_bias, j);
        if (p.threshold) drop(v, kept[j], p.drop_scale);
      };
      float post_r = 1.f;
      if constexpr (kPost) post_r = row.normalise(x, p.post, p.inverse_width, p.eps);
      if constexpr (kBranch) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          f32x4 v[2], k[2];
          branch(j, v);
          if constexpr (kGate) row.use(gate, j, k);
#pragma unroll
          for (int e = 0; e < 2; ++e) h[j][e] = h[j][e] * p.residual_scale + (kGate ? v[e] * k[e] : v[e]);
        }
      }
      if (p.grad_n) {
        const float r = row.normalise(h, p.norm, p.inverse_width, p.eps);
        if constexpr (kLate) {
          row.load(p.grad_n, at, p.grad_n_stride, g_next);
          row.widen(g_next, g);
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          f32x4 w[2];
          row.use(weight, j, w);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            d_weight.add(j, e, g[j][e] * h[j][e]);
            d_bias.add(j, e, g[j][e]);
            g[j][e] *= w[e];
          }
        }
        row.transpose(g, h, r, p.norm, p.inverse_width);
        if constexpr (!kLate) {
#pragma unroll
          for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) gt[j][e] += g[j][e];
        }
      }
      if constexpr (kLate) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          gt[j][0] = gt[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (p.grad_h) row.widen_chunk(row.load_chunk_of(static_cast<const R*>(p.grad_h) + at * p.grad_h_stride, j), j, gt[j]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (p.grad_n) gt[j][e] += g[j][e];
        }
      }
      if (p.dresidual && live) {
        Values d;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) d[j][e] = gt[j][e] * p.residual_scale;
        row.template store<R>(p.dresidual, at, p.dresidual_stride, d);
      }
      if constexpr (kGate) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          f32x4 v[2], k[2];
          branch(j, v);
          row.use(gate, j, k);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            v[e] *= gt[j][e];
            d_gate.add(j, e, v[e]);
            gt[j][e] *= k[e];
          }
          if (p.dgate && gate_full && live)
            store_vector(static_cast<char*>(p.dgate) + at * p.dgate_stride * (p.dgate_dtype == VECTRA_BLOCK_F32 ? 4 : 2),
                         p.dgate_dtype, row.column_of(j), row.left[j], v);
        }
      }
      if (p.threshold) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) drop(gt[j], kept[j], p.drop_scale);
      }
      if constexpr (kPost) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          f32x4 w[2];
          row.use(post_weight, j, w);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            d_post_weight.add(j, e, gt[j][e] * x[j][e]);
            d_post_bias.add(j, e, gt[j][e]);
            gt[j][e] *= w[e];
          }
        }
        row.transpose(gt, x, post_r, p.post, p.inverse_width);
      }
      if (p.dx && live) row.template store<T>(p.dx, at, p.dx_stride, gt);
    }
    if constexpr (kGate) {
      if (p.gate_sums || (p.dgate && !gate_full)) {
        Values d;
        d_gate.get(d);
        over_slots(d);
        if (row.slot == 0) {
#pragma unroll
          for (int j = 0; j < kChunks; ++j) {
            if (p.gate_sums)
              store_vector(p.gate_sums + unit * p.width, VECTRA_BLOCK_F32, row.column[j], row.left[j], d[j]);
            else
              store_vector(static_cast<char*>(p.dgate) + group * p.dgate_stride * (p.dgate_dtype == VECTRA_BLOCK_F32 ? 4 : 2),
                           p.dgate_dtype, row.column[j], row.left[j], d[j]);
          }
        }
        d_gate.clear();
      }
    }
  }
  const int64_t plane = static_cast<int64_t>(blockIdx.x) * p.width;
  if (p.weight_sums) write_sums(d_weight, p.weight_sums + plane);
  if (p.bias_sums) write_sums(d_bias, p.bias_sums + plane);
  if constexpr (kPost) {
    if (p.post_weight_sums) write_sums(d_post_weight, p.post_weight_sums + plane);
    if (p.post_bias_sums) write_sums(d_post_bias, p.post_bias_sums + plane);
  }
}

// ----------------------------------------------------------------------- host

template <int kLanes_, int kChunks_, int kKind_>
struct Shape {
  static constexpr int kLanes = kLanes_, kChunks = kChunks_, kKind = kKind_;
};

template <int kKind, typename F>
void with_kind(const NormShape& shape, F&& f) {
  switch (shape.lanes) {
    case 16: return f(Shape<16, 1, kKind>{});
    case 32: return f(Shape<32, 1, kKind>{});
    case 64: return f(Shape<64, 1, kKind>{});
    default:
      return shape.chunks == 1   ? f(Shape<kMany, 1, kKind>{})
             : shape.chunks == 2 ? f(Shape<kMany, 2, kKind>{})
                                 : f(Shape<kMany, 4, kKind>{});
  }
}

template <typename F>
void with_shape(const NormShape& shape, int64_t width, F&& f) {
  if (width < 8) return f(Shape<16, 1, kNarrow>{});
  return width % 8 ? with_kind<kRagged>(shape, f) : with_kind<kWhole>(shape, f);
}

template <typename T, typename R>
int launch_norm(const NormParams& p, int cus, hipStream_t stream) {
  const NormShape shape = norm_shape(p.width);
  const int64_t blocks = (p.rows + shape.rows - 1) / shape.rows;
  // (A CU's 2048 threads; at 111 to 121 registers of one chunk per lane half of these
  // workgroups are there at once, and the others follow.)
  const int64_t most_blocks = static_cast<int64_t>(cus) * (2048 / shape.threads);
  with_shape(shape, p.width, [&](auto s) {
    using S = decltype(s);
    norm_kernel<T, R, S::kLanes, S::kChunks, S::kKind>
        <<<static_cast<uint32_t>(blocks < most_blocks ? blocks : most_blocks), shape.threads, 0, stream>>>(p);
  });
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

template <typename T, typename R>
int launch_norm_grad(const NormGradParams& p, int workgroups, hipStream_t stream) {
  const NormShape shape = norm_shape(p.width);
  with_shape(shape, p.width, [&](auto s) {
    using S = decltype(s);
    const bool post = p.post != VECTRA_BLOCK_NO_NORM;
    const auto kernel = p.gate.p ? (post ? norm_grad_kernel<T, R, S::kLanes, S::kChunks, S::kKind, true, true>
                                         : norm_grad_kernel<T, R, S::kLanes, S::kChunks, S::kKind, true, false>)
                                 : (post ? norm_grad_kernel<T, R, S::kLanes, S::kChunks, S::kKind, false, true>
                                         : norm_grad_kernel<T, R, S::kLanes, S::kChunks, S::kKind, false, false>);
    kernel<<<static_cast<uint32_t>(workgroups), shape.threads, 0, stream>>>(p);
  });
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

}  // namespace vectra_block
