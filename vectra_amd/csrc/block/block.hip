// C ABI of the operators between a block's dense products (include/vectra_block.h):
// argument checks, the plan of a call, and the small kernels.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "block_common.h"
#include "block_kernels.h"
#include "product8_kernels.h"

namespace vectra_block {
namespace {

// ----------------------------------------------------------------- kernels

// y = k * x: a thread takes kGroups groups of eight elements, 256 groups apart,
// their loads issued together.
template <typename T, typename Index, int kGroups>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, int64_t rows, int64_t width, int64_t x_stride, T* y,
                                                      int64_t y_stride, Dropout d) {
  const DropoutKey key = dropout_key(d);
  const Index groups = static_cast<Index>((width + 7) / 8), total = static_cast<Index>(rows) * groups;
  const Index first = static_cast<Index>(blockIdx.x) * (256 * kGroups) + threadIdx.x;
  Eight<T> in[kGroups];
  Index at[kGroups], row[kGroups];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    at[j] = first + j * 256;
    row[j] = at[j] / groups;
    if (at[j] < total)
      in[j] = load_eight<T>(x + static_cast<int64_t>(row[j]) * x_stride, width, static_cast<int64_t>(at[j] - row[j] * groups) * 8);
  }
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    if (at[j] >= total) continue;
    const int64_t column = static_cast<int64_t>(at[j] - row[j] * groups) * 8;
    f32x4 v[2];
    widen_eight(in[j], v[0], v[1]);
    if (d.threshold) {
      drop(v, dropout_kept(d, key, at[j]), d.scale);
    }
    store8(y + static_cast<int64_t>(row[j]) * y_stride + column, v[0], v[1], static_cast<int>(least(width - column, 8)));
  }
}

// Adds up the workgroups' (a gate's: the parts') sums of the vectors' gradients in a
// fixed order.  blockIdx.y: the vector, then the gate's rows; a workgroup takes 32
// columns, 8 quads by 32 lanes that each add every 32nd plane, eight in flight.
struct SumOf {
  const float* planes;
  int64_t count;  // of planes, `width` apart
  void* out;
  int32_t dtype;
};
struct SumParams {
  SumOf vectors[4];
  int32_t vector_count;
  const float* gate;  // [gate rows, parts, width]
  int64_t parts, dgate_stride;
  void* dgate;
  int32_t dgate_dtype;
  int64_t width;
};

__global__ __launch_bounds__(256) void sum_kernel(const SumParams p) {
  __shared__ f32x4 part[32][8];
  const int q = threadIdx.x % 8, lane = threadIdx.x / 8;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + q * 4;
  const int left = static_cast<int>(most(least(p.width - column, 4), 0));
  const bool vector = static_cast<int>(blockIdx.y) < p.vector_count;
  const int64_t gate_row = static_cast<int64_t>(blockIdx.y) - p.vector_count;
  SumOf s;
  if (vector) {
    s = p.vectors[blockIdx.y];
  } else {
    s.planes = p.gate + gate_row * p.parts * p.width;
    s.count = p.parts;
    s.dtype = p.dgate_dtype;
    s.out = static_cast<char*>(p.dgate) + gate_row * p.dgate_stride * (s.dtype == VECTRA_BLOCK_F32 ? 4 : 2);
  }
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
  if (left > 0) {
    const float* const from = s.planes + column;
    int64_t k = lane;
    for (; k + 7 * 32 < s.count; k += 8 * 32) {
      f32x4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = vectra_dense::load4(from + (k + j * 32) * p.width, left);
#pragma unroll
      for (int j = 0; j < 8; ++j) total += v[j];
    }
    for (; k < s.count; k += 32) total += vectra_dense::load4(from + k * p.width, left);
  }
  part[lane][q] = total;
  __syncthreads();
  if (lane != 0 || left <= 0) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) total += part[k][q];
  if (s.dtype == VECTRA_BLOCK_F32)
    vectra_dense::store4(static_cast<float*>(s.out) + column, total, left);
  else if (s.dtype == VECTRA_BLOCK_F16)
    vectra_dense::store4(static_cast<_Float16*>(s.out) + column, total, left);
  else
    vectra_dense::store4(static_cast<__bf16*>(s.out) + column, total, left);
}

// 8-bit rows: 16 lanes per block of 128.  blockIdx covers the padded scales too.
template <typename T, typename Index>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* x, int64_t rows, int64_t width, int64_t x_stride,
                                                            uint8_t* codes, uint8_t* scales, int64_t depth,
                                                            int64_t scale_stride) {
  const Index at = static_cast<Index>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const bool live = at < static_cast<Index>(rows) * static_cast<Index>(scale_stride);
  const Index row = live ? at / static_cast<Index>(scale_stride) : 0;
  const int64_t block = live ? at - row * static_cast<Index>(scale_stride) : 0;
  const int64_t column = block * 128 + (threadIdx.x & 15) * 8;
  const int left = live ? static_cast<int>(most(least(width - column, 8), 0)) : 0;
  f32x4 v[2] = {};
  if (left > 0) vectra_dense::load8(x + static_cast<int64_t>(row) * x_stride + column, left, v[0], v[1]);
  const float largest = vectra::reduce_low<16>(vectra_dense::largest_finite(v, 0.f), vectra::OpMax{});
  const int byte = vectra_dense::block_exponent(largest, kLowestExponent);
  const uint2 w = vectra_dense::to_codes(v, byte - 127, kHighestExponent);
  if (!live) return;
  if (column < depth) *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(row) * depth + column) = w;
  if ((threadIdx.x & 15) == 0) scales[at] = static_cast<uint8_t>(column < depth ? byte : 0);
}

// 8-bit tiles: a workgroup per tile of 128 x 128, a thread's elements in registers
// between the largest and the codes.
template <typename T>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(const T* x, int64_t rows, int64_t width, int64_t x_stride,
                                                             uint8_t* codes, uint8_t* scales, int64_t depth,
                                                             int64_t scale_stride) {
  __shared__ float of_wave[4];
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * 128 + (threadIdx.x >> 4);
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 128 + (threadIdx.x & 15) * 8;
  const int left = static_cast<int>(most(least(width - column, 8), 0));
  f32x4 v[8][2] = {};
  float largest = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (row0 + j * 16 < rows && left > 0) vectra_dense::load8(x + (row0 + j * 16) * x_stride + column, left, v[j][0], v[j][1]);
#pragma unroll
  for (int j = 0; j < 8; ++j) largest = vectra_dense::largest_finite(v[j], largest);
  largest = vectra::reduce_low<64>(largest, vectra::OpMax{});
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = largest;
  __syncthreads();
  largest = fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
  const int byte = vectra_dense::block_exponent(largest, kLowestExponent);
  const bool inside = column < depth;
  if (threadIdx.x == 0) scales[blockIdx.y * scale_stride + blockIdx.x] = static_cast<uint8_t>(inside ? byte : 0);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (row0 + j * 16 < rows && inside)
      *reinterpret_cast<uint2*>(codes + (row0 + j * 16) * depth + column) = vectra_dense::to_codes(v[j], byte - 127, kHighestExponent);
}

// Adds up a split product's planes in a fixed order and finishes it with the layer's
// epilogue: a thread per four columns (a gated layer: of both halves).
template <typename T, bool kGated>
__global__ __launch_bounds__(256) void join8_kernel(const float* planes, int parts, int64_t plane_stride, Product8Params p) {
  constexpr int kHalves = kGated ? 2 : 1;
  const int64_t quads = (p.n + 3) / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= p.rows * quads) return;
  const int64_t row = at / quads, column = (at - row * quads) * 4;
  const int left = static_cast<int>(least(p.n - column, 4));
  f32x4 z[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    const float* const from = planes + row * plane_stride + h * p.n + column;
    z[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      f32x4 v;  // (the up half starts at any column; its rows are long enough)
      __builtin_memcpy(&v, from + k * p.rows * plane_stride, 16);
      z[h] += v;
    }
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) z[h][e] += vectra_dense::load_bias(p.bias, h * p.n + column + e, p.bias_dtype);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    z[0][e] = vectra_dense::act_value<T>(z[0][e], p.activation);
    if constexpr (kGated) z[0][e] *= z[1][e];
  }
  if (!kGated && p.residual) z[0] += vectra_dense::load4(static_cast<const T*>(p.residual) + row * p.residual_stride + column, left);
  vectra_dense::store4(static_cast<T*>(p.out) + row * p.out_stride + column, z[0], left);
}

// -------------------------------------------------------------------- host

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// CUs of the current device (an atomic per device id, filled once).
int compute_units() {
  static std::atomic<int> known[64];
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return 256;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) n = 256;
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

bool known_dtype(int32_t t) { return t == VECTRA_BLOCK_F32 || t == VECTRA_BLOCK_F16 || t == VECTRA_BLOCK_BF16; }

template <typename F>
void typed(int32_t dtype, F&& f) {
  switch (dtype) {
    case VECTRA_BLOCK_F32: return f(static_cast<float*>(nullptr));
    case VECTRA_BLOCK_F16: return f(static_cast<_Float16*>(nullptr));
    default: return f(static_cast<__bf16*>(nullptr));
  }
}

int launched() { return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH; }

constexpr int64_t kMostRows = int64_t{1} << 30;
constexpr int64_t kMostWidth = int64_t{1} << 21;

int check_sizes(int64_t rows, int64_t width) {
  if (rows < 0 || width < 0) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  // Elementwise kernels: a thread per eight elements, fewer than 2^32 threads.
  if (rows > kMostRows || width > kMostWidth || rows * (width + 512) >= int64_t{1} << 35) return VECTRA_BLOCK_ERR_TOO_LARGE;
  return VECTRA_BLOCK_OK;
}

// A row stride covers the row (that of a single row is not read).
int check_stride(int64_t stride, int64_t width, int64_t rows) {
  if (rows > 1 && stride < width) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  if (stride < 0) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  if (rows > 1 && stride > (int64_t{1} << 40)) return VECTRA_BLOCK_ERR_TOO_LARGE;
  return VECTRA_BLOCK_OK;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool known_threshold(int32_t t) { return t >= 0 && t <= 65535; }

float drop_scale(int32_t threshold) { return static_cast<float>(65536.0 / (65536 - threshold)); }

int quantize(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, bool tiles, void* codes,
             void* scales, hipStream_t stream) {
  const int64_t depth = ceil_div(width, 128) * 128, scale_stride = ceil_div(width, 512) * 4;
  uint8_t* const c = static_cast<uint8_t*>(codes);
  uint8_t* const s = static_cast<uint8_t*>(scales);
  typed(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const T* const from = static_cast<const T*>(x);
    if (tiles) {
      // (Tile rows in launches of at most 65,535, a grid's limit.)
      for (int64_t first = 0; first < rows; first += 128 * int64_t{65535}) {
        const int64_t some = std::min(rows - first, 128 * int64_t{65535});
        quantize_tiles_kernel<T><<<dim3(static_cast<uint32_t>(scale_stride), static_cast<uint32_t>(ceil_div(some, 128))), 256, 0, stream>>>(
            from + first * x_stride, some, width, x_stride, c + first * depth, s + first / 128 * scale_stride, depth, scale_stride);
      }
      return;
    }
    const int64_t total = rows * scale_stride;
    const auto kernel = total < (int64_t{1} << 31) - 16 ? quantize_rows_kernel<T, uint32_t> : quantize_rows_kernel<T, int64_t>;
    kernel<<<static_cast<uint32_t>(ceil_div(total, 16)), 256, 0, stream>>>(from, rows, width, x_stride, c, s, depth, scale_stride);
  });
  return launched();
}

// What the two norm calls share.
template <typename Args>
int check_norm(const Args& a) {
  if (!known_dtype(a.dtype)) return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (a.stream_dtype != a.dtype && a.stream_dtype != VECTRA_BLOCK_F32) return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (a.norm != VECTRA_BLOCK_RMS && a.norm != VECTRA_BLOCK_LAYER) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (a.post < VECTRA_BLOCK_NO_NORM || a.post > VECTRA_BLOCK_LAYER) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (!known_threshold(a.threshold)) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (!(a.eps >= 0.f) || std::isinf(a.eps)) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (int st = check_sizes(a.rows, a.width)) return st;
  if (a.width > VECTRA_BLOCK_NORM_WIDTH) return VECTRA_BLOCK_ERR_TOO_LARGE;
  return VECTRA_BLOCK_OK;
}

// Gate rows of a call; one serves at most all rows.  (gate_rows is at least 1.)
int64_t count_gate_rows(int64_t rows, int64_t gate_rows) { return ceil_div(rows, std::min(gate_rows, std::max<int64_t>(rows, 1))); }

// Whether the gradients read the branch and the residual, or h: h where it tells all that
// matters, without a gate and a post norm and as the forward pass had it, in fp32.
bool reads_branch(const vectra_norm_grad_args& a) {
  return a.gate || a.post != VECTRA_BLOCK_NO_NORM || a.stream_dtype != VECTRA_BLOCK_F32;
}

// A vector that is given has the branch's type or fp32.
bool vector_dtype(const void* p, int32_t dtype, int32_t of) { return !p || dtype == of || dtype == VECTRA_BLOCK_F32; }

int check_forward(const vectra_norm_args* a) {
  if (!a) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->struct_size != static_cast<int64_t>(sizeof(vectra_norm_args))) return VECTRA_BLOCK_ERR_BAD_STRUCT;
  if (int st = check_norm(*a)) return st;
  if (!vector_dtype(a->weight, a->weight_dtype, a->dtype) || !vector_dtype(a->bias, a->bias_dtype, a->dtype) ||
      !vector_dtype(a->gate, a->gate_dtype, a->dtype) || !vector_dtype(a->post_weight, a->post_weight_dtype, a->dtype) ||
      !vector_dtype(a->post_bias, a->post_bias_dtype, a->dtype))
    return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (a->rows == 0 || a->width == 0) return VECTRA_BLOCK_OK;
  if (!a->x || !a->residual || !a->h || (!a->n && (!a->codes || !a->scales))) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->threshold && !a->rng) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (!a->n && !aligned(a->codes, 16)) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  if (int st = check_stride(a->x_stride, a->width, a->rows)) return st;
  if (int st = check_stride(a->residual_stride, a->width, a->rows)) return st;
  if (int st = check_stride(a->h_stride, a->width, a->rows)) return st;
  if (a->n)
    if (int st = check_stride(a->n_stride, a->width, a->rows)) return st;
  if (a->gate) {
    if (a->gate_rows < 1) return VECTRA_BLOCK_ERR_BAD_SHAPE;
    if (int st = check_stride(a->gate_stride, a->width, count_gate_rows(a->rows, a->gate_rows))) return st;
  }
  return VECTRA_BLOCK_OK;
}

int forward(const vectra_norm_args& a, hipStream_t stream) {
  if (a.rows == 0 || a.width == 0) return VECTRA_BLOCK_OK;
  NormParams p{};
  p.x = a.x;
  p.residual = a.residual;
  p.weight = {a.weight, a.weight_dtype};
  p.bias = {a.bias, a.bias_dtype};
  p.gate = {a.gate, a.gate_dtype};
  p.post_weight = {a.post_weight, a.post_weight_dtype};
  p.post_bias = {a.post_bias, a.post_bias_dtype};
  p.rng = a.rng;
  p.h = a.h;
  p.n = a.n;
  p.codes = static_cast<uint8_t*>(a.codes);
  p.scales = static_cast<uint8_t*>(a.scales);
  p.norm = a.norm;
  p.post = a.post;
  p.threshold = a.threshold;
  p.stream_id = a.stream_id;
  p.eps = a.eps;
  p.residual_scale = a.residual_scale;
  p.drop_scale = drop_scale(a.threshold);
  p.inverse_width = 1.f / static_cast<float>(a.width);
  p.rows = a.rows;
  p.width = a.width;
  p.gate_rows = a.gate ? std::min(a.gate_rows, a.rows) : a.rows;
  p.depth = ceil_div(a.width, 128) * 128;
  p.scale_stride = ceil_div(a.width, 512) * 4;
  p.x_stride = a.x_stride;
  p.residual_stride = a.residual_stride;
  p.gate_stride = a.gate_stride;
  p.h_stride = a.h_stride;
  p.n_stride = a.n_stride;
  const bool wide = a.stream_dtype == VECTRA_BLOCK_F32;
  const auto f = a.dtype == VECTRA_BLOCK_F32   ? launch_norm_f32_f32
                 : a.dtype == VECTRA_BLOCK_F16 ? (wide ? launch_norm_f16_f32 : launch_norm_f16_f16)
                                               : (wide ? launch_norm_bf16_f32 : launch_norm_bf16_bf16);
  return f(p, compute_units(), stream);
}

int check_backward(const vectra_norm_grad_args* a) {
  if (!a) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->struct_size != static_cast<int64_t>(sizeof(vectra_norm_grad_args))) return VECTRA_BLOCK_ERR_BAD_STRUCT;
  if (int st = check_norm(*a)) return st;
  const auto fits = [&](const void* p, const void* d, int32_t dtype) {
    return vector_dtype(p, dtype, a->dtype) && vector_dtype(d, dtype, a->dtype);
  };
  if (!fits(a->weight, a->dweight, a->weight_dtype) || !fits(nullptr, a->dbias, a->bias_dtype) ||
      !fits(a->gate, a->dgate, a->gate_dtype) || !fits(a->post_weight, a->dpost_weight, a->post_weight_dtype) ||
      !fits(a->post_bias, a->dpost_bias, a->post_bias_dtype))
    return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (a->width == 0) return VECTRA_BLOCK_OK;
  const bool branch = reads_branch(*a);
  if (a->dgate && !a->gate) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if ((a->dpost_weight || a->dpost_bias) && a->post == VECTRA_BLOCK_NO_NORM) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (a->gate && a->gate_rows < 1) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  if (a->dgate)
    if (int st = check_stride(a->dgate_stride, a->width, count_gate_rows(a->rows, a->gate_rows))) return st;
  if (a->rows == 0) return VECTRA_BLOCK_OK;
  if (branch ? !a->x || !a->residual : !a->h) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->threshold && !a->rng) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->gate)
    if (int st = check_stride(a->gate_stride, a->width, count_gate_rows(a->rows, a->gate_rows))) return st;
  const struct {
    const void* p;
    int64_t stride;
  } rows[] = {{a->grad_h, a->grad_h_stride}, {a->grad_n, a->grad_n_stride}, {branch ? a->x : nullptr, a->x_stride},
              {branch ? a->residual : nullptr, a->residual_stride}, {branch ? nullptr : a->h, a->h_stride},
              {a->dx, a->dx_stride}, {a->dresidual, a->dresidual_stride}};
  for (const auto& r : rows)
    if (r.p)
      if (int st = check_stride(r.stride, a->width, a->rows)) return st;
  return VECTRA_BLOCK_OK;
}

// Scratch memory in order of use.  Without a base only the size is found.
struct Scratch {
  char* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* const p = base ? base + used : reinterpret_cast<void*>(256);
    used += (bytes + 255) & ~int64_t{255};
    return p;
  }
};

int backward(const vectra_norm_grad_args& a, Scratch& scratch, bool launch, int cus, hipStream_t stream) {
  if (a.width == 0) return VECTRA_BLOCK_OK;
  const bool sums = a.dweight || a.dbias || a.dpost_weight || a.dpost_bias;
  if (!sums && (a.rows == 0 || (!a.dx && !a.dresidual && !a.dgate))) return VECTRA_BLOCK_OK;
  NormGradParams p{};
  const bool branch = reads_branch(a);
  const int64_t gate_rows = a.gate ? std::max<int64_t>(1, std::min(a.gate_rows, a.rows)) : std::max<int64_t>(1, a.rows);
  const bool gate_full = a.gate && gate_rows == 1;
  p.grad_h = a.grad_h;
  p.grad_n = a.grad_n;
  p.x = branch ? a.x : nullptr;
  p.residual = a.residual;
  p.h = a.h;
  p.weight = {a.weight, a.weight_dtype};
  p.gate = {a.gate, a.gate_dtype};
  p.post_weight = {a.post_weight, a.post_weight_dtype};
  p.post_bias = {a.post_bias, a.post_bias_dtype};
  p.rng = a.rng;
  p.dx = a.dx;
  p.dresidual = a.dresidual;
  p.dgate_dtype = a.gate_dtype;
  p.norm = a.norm;
  p.post = a.post;
  p.threshold = a.threshold;
  p.stream_id = a.stream_id;
  p.eps = a.eps;
  p.residual_scale = a.residual_scale;
  p.drop_scale = drop_scale(a.threshold);
  p.inverse_width = 1.f / static_cast<float>(a.width);
  p.rows = a.rows;
  p.width = a.width;
  p.gate_rows = gate_rows;
  p.grad_h_stride = a.grad_h_stride;
  p.grad_n_stride = a.grad_n_stride;
  p.x_stride = a.x_stride;
  p.residual_stride = a.residual_stride;
  p.h_stride = a.h_stride;
  p.gate_stride = a.gate_stride;
  p.dx_stride = a.dx_stride;
  p.dresidual_stride = a.dresidual_stride;
  p.dgate_stride = a.dgate_stride;

  // Units: the rows, or a gate's groups of rows, in parts: as many as the registers let
  // the card hold at once (2 waves per SIMD with a gate and a post norm, 3 with one of
  // them, 4 with neither), and where there are rows enough for the card no more than
  // leave a workgroup's slots eight each, beside which its sums, 8 bytes a column written
  // and read, are little.
  const NormShape shape = norm_shape(a.width);
  const int threads = a.gate ? (a.post ? 512 : 768) : a.post ? 768 : 1024;  // of a CU
  const int64_t wanted = static_cast<int64_t>(cus) * std::max(1, threads / shape.threads);
  p.unit_rows = gate_full ? a.rows : gate_rows;
  const int64_t groups = a.rows ? ceil_div(a.rows, p.unit_rows) : 0;
  const int64_t each = std::max<int64_t>(1, std::min<int64_t>(8, a.rows / (2 * shape.rows * cus)));
  const int64_t parts = groups ? std::min(ceil_div(wanted, groups), ceil_div(p.unit_rows, each * shape.rows)) : 1;
  p.rows_per_part = std::max<int64_t>(1, ceil_div(p.unit_rows, parts));
  p.parts = static_cast<int32_t>(ceil_div(p.unit_rows, p.rows_per_part));
  if (a.rows == 0) p.parts = 0;
  p.units = groups * p.parts;
  const int64_t workgroups = std::min(p.units, wanted);

  SumParams s{};
  s.width = a.width;
  const auto vector = [&](void* out, int32_t dtype) -> float* {
    if (!out) return nullptr;
    float* const planes = static_cast<float*>(scratch.take(workgroups * a.width * 4));
    s.vectors[s.vector_count++] = SumOf{planes, workgroups, out, dtype};
    return planes;
  };
  p.weight_sums = vector(a.dweight, a.weight_dtype);
  p.bias_sums = vector(a.dbias, a.bias_dtype);
  p.post_weight_sums = vector(a.dpost_weight, a.post_weight_dtype);
  p.post_bias_sums = vector(a.dpost_bias, a.post_bias_dtype);
  int64_t gate_planes = 0;  // gate rows whose parts are to be added up
  if (a.dgate && a.rows) {
    if (gate_full || p.parts == 1) {
      p.dgate = a.dgate;
    } else {
      s.gate = p.gate_sums = static_cast<float*>(scratch.take(p.units * a.width * 4));
      s.parts = p.parts;
      s.dgate = a.dgate;
      s.dgate_stride = a.dgate_stride;
      s.dgate_dtype = a.gate_dtype;
      gate_planes = groups;
    }
  }
  if (!launch) return VECTRA_BLOCK_OK;
  (void)hipGetLastError();  // an error left by other work is not this call's
  if (a.rows) {
    const bool wide = a.stream_dtype == VECTRA_BLOCK_F32;
    const auto f = a.dtype == VECTRA_BLOCK_F32   ? launch_norm_grad_f32_f32
                   : a.dtype == VECTRA_BLOCK_F16 ? (wide ? launch_norm_grad_f16_f32 : launch_norm_grad_f16_f16)
                                                 : (wide ? launch_norm_grad_bf16_f32 : launch_norm_grad_bf16_bf16);
    if (int st = f(p, static_cast<int>(workgroups), stream)) return st;
  }
  const int64_t across = s.vector_count + gate_planes;
  if (across > 0)
    sum_kernel<<<dim3(static_cast<uint32_t>(ceil_div(a.width, 32)), static_cast<uint32_t>(across)), 256, 0, stream>>>(s);
  return launched();
}

// ------------------------------------------------------------- products in 8 bits

int check_linear8(const vectra_linear8_args* a) {
  if (!a) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->struct_size != static_cast<int64_t>(sizeof(vectra_linear8_args))) return VECTRA_BLOCK_ERR_BAD_STRUCT;
  if (!known_dtype(a->dtype)) return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (!vector_dtype(a->bias, a->bias_dtype, a->dtype)) return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (a->activation < VECTRA_DENSE_NONE || a->activation > VECTRA_DENSE_SILU) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if ((a->gated != 0 && a->gated != 1) || (a->gated && a->residual)) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  if (int st = check_sizes(a->rows, a->width)) return st;
  if (int st = check_sizes(a->rows, a->width_out)) return st;
  if (int st = check_sizes(a->rows, a->width_out * (1 + a->gated))) return st;
  if (a->rows == 0 || a->width_out == 0) return VECTRA_BLOCK_OK;
  if (!a->out || (a->width && (!a->weight || !a->weight_scales || (!a->x && (!a->codes || !a->scales)))))
    return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (a->width) {
    if (!aligned(a->weight, 16) || !aligned(a->weight_scales, 4)) return VECTRA_BLOCK_ERR_BAD_SHAPE;
    if (!a->x && (!aligned(a->codes, 16) || !aligned(a->scales, 4))) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  }
  // Offsets within a tile's operands, and from a gate's row to its up row, have 31 bits.
  const int64_t depth = ceil_div(a->width, 128) * 128;
  if ((a->gated * a->width_out + 256) * depth >= int64_t{1} << 31) return VECTRA_BLOCK_ERR_TOO_LARGE;
  if (a->x)
    if (int st = check_stride(a->x_stride, a->width, a->rows)) return st;
  if (a->residual)
    if (int st = check_stride(a->residual_stride, a->width_out, a->rows)) return st;
  return check_stride(a->out_stride, a->width_out, a->rows);
}

// The tile and the number of contraction parts with the least estimated time.
//   kRate      of all CUs, full, by tile (16-bit results; fp32's), as a line in the
//              contraction: 8192 x K -> 16384 takes 1.45, 0.69 and 0.28 us per block and
//              tile on 256, 128 and 64
//   kResident  workgroups that a CU holds; one that holds fewer runs at kPart of the rate
//   kBatch     a CU's first loads and epilogues: the line's intercept, 10.4, 2.1 and 0.5
//              us per tile
// A split costs its fp32 planes, written and read at 5 TB/s, and the joining launch.
//   chosen / others, bf16, us: 4096 x 4096 -> 4096 65 on 256 (91 on 128); 1024 x 4096 ->
//   4096 25 on 128 (49 on 256, 43 on 64); 128 x 4096 -> 4096 9.5 and a join on 64 in 4
//   parts (15 in one, 10.3 on 128 in 4)
void choose8(const Product8Params& p, int64_t columns, int32_t dtype, int cus, int& tile, int& parts) {
  static constexpr double kRate16[kTiles8] = {2.9e15, 1.55e15, 0.95e15}, kRate32[kTiles8] = {0, 0.72e15, 0.55e15};
  static constexpr int kResident[kTiles8] = {1, 2, 5};
  static constexpr double kPart[kTiles8][5] = {{1.0}, {0.95, 1.0}, {0.63, 0.75, 0.8, 0.86, 1.0}};
  static constexpr double kBatch[kTiles8] = {10.4e-6, 4.2e-6, 2.6e-6};
  const bool precise = dtype == VECTRA_BLOCK_F32;
  double best = 1e30;
  tile = kSmall8;
  parts = 1;
  for (int t = precise ? kMedium8 : kLarge8; t < kTiles8; ++t) {
    const int64_t tiles = ceil_div(p.rows, kTile8[t]) * ceil_div(columns, kTile8[t]);
    const double rate = (precise ? kRate32[t] : kRate16[t]) / 256;
    for (int k = 1; k <= std::max(1, std::min(16, p.k_tiles / 4)); k *= 2) {
      const int64_t depth = ceil_div(p.k_tiles, k) * 128;
      const int64_t per_cu = ceil_div(tiles * k, cus);
      const int together = static_cast<int>(std::min<int64_t>(per_cu, kResident[t]));
      const double products = per_cu * 2.0 * kTile8[t] * kTile8[t] * depth / (rate * kPart[t][together - 1]);
      const double join = k > 1 ? 8.0 * k * p.rows * columns / 5e12 + 4e-6 : 0;
      const double time = products + ceil_div(per_cu, kResident[t]) * kBatch[t] + join;
      if (time < best * 0.98) {
        best = time;
        tile = t;
        parts = k;
      }
    }
  }
}

int linear8(const vectra_linear8_args& a, Scratch& scratch, bool launch, int cus, hipStream_t stream) {
  if (a.rows == 0 || a.width_out == 0) return VECTRA_BLOCK_OK;
  Product8Params p{};
  p.rows = a.rows;
  p.n = a.width_out;
  p.width = a.width;
  p.depth = ceil_div(a.width, 128) * 128;
  p.scale_stride = ceil_div(a.width, 512) * 4;
  p.weight = static_cast<const uint8_t*>(a.weight);
  p.weight_scales = static_cast<const uint8_t*>(a.weight_scales);
  p.codes = static_cast<const uint8_t*>(a.codes);
  p.scales = static_cast<const uint8_t*>(a.scales);
  p.bias = a.bias;
  p.bias_dtype = a.bias_dtype;
  p.activation = a.activation;
  p.residual = a.residual;
  p.residual_stride = a.residual_stride;
  p.out = a.out;
  p.out_stride = a.out_stride;
  if (launch) (void)hipGetLastError();  // an error left by other work is not this call's
  if (a.x && a.rows <= kFewRaw8 && a.rows * p.depth <= kRawBytes) {
    p.x = a.x;
    p.x_stride = a.x_stride;
  } else if (a.x) {
    uint8_t* const codes = static_cast<uint8_t*>(scratch.take(a.rows * p.depth));
    uint8_t* const scales = static_cast<uint8_t*>(scratch.take(a.rows * p.scale_stride));
    p.codes = codes;
    p.scales = scales;
    if (launch && a.width)
      if (int st = quantize(a.x, a.dtype, a.rows, a.width, a.x_stride, false, codes, scales, stream)) return st;
  }
  if (a.rows <= kFewRows8) {
    if (!launch) return VECTRA_BLOCK_OK;
    const auto f = a.dtype == VECTRA_BLOCK_F32 ? launch_few8_f32 : a.dtype == VECTRA_BLOCK_F16 ? launch_few8_f16 : launch_few8_bf16;
    return f(p, a.gated, stream);
  }
  const int64_t columns = a.gated ? 2 * p.n : p.n;
  p.k_tiles = static_cast<int32_t>(p.depth / 128);
  int tile, parts;
  choose8(p, columns, a.dtype, cus, tile, parts);
  p.tiles_m = static_cast<int32_t>(ceil_div(p.rows, kTile8[tile]));
  p.tiles_n = static_cast<int32_t>(ceil_div(columns, kTile8[tile]));
  // (A part begins with a word of scales.)
  p.k_tiles_per_part = static_cast<int32_t>(std::max<int64_t>(1, parts == 1 ? p.k_tiles : ceil_div(ceil_div(p.k_tiles, parts), 4) * 4));
  parts = static_cast<int>(std::max<int64_t>(1, ceil_div(p.k_tiles, p.k_tiles_per_part)));
  const auto f = a.dtype == VECTRA_BLOCK_F32   ? launch_product8_f32
                 : a.dtype == VECTRA_BLOCK_F16 ? launch_product8_f16
                                               : launch_product8_bf16;
  if (parts == 1) return launch ? f(p, tile, a.gated ? kGated8 : kStore8, 1, stream) : VECTRA_BLOCK_OK;
  // Planes of four-column pieces; the join reads such pieces of the up half from
  // column n on.
  const int64_t ld = ceil_div(a.gated ? p.n + ceil_div(p.n, 4) * 4 : columns, 4) * 4;
  Product8Params q = p;
  q.n = columns;
  q.out = scratch.take(parts * p.rows * ld * 4);
  q.out_stride = ld;
  if (!launch) return VECTRA_BLOCK_OK;
  if (int st = f(q, tile, kPartial8, parts, stream)) return st;
  typed(a.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const auto kernel = a.gated ? join8_kernel<T, true> : join8_kernel<T, false>;
    kernel<<<static_cast<uint32_t>(ceil_div(p.rows * ceil_div(p.n, 4), 256)), 256, 0, stream>>>(
        static_cast<const float*>(q.out), parts, ld, p);
  });
  return launched();
}

}  // namespace
}  // namespace vectra_block

using namespace vectra_block;

extern "C" {

int vectra_dropout(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, void* y,
                   int64_t y_stride, int32_t threshold, const int64_t* rng, uint32_t stream_id,
                   vectra_block_stream_t stream) {
  if (!known_dtype(dtype)) return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (!known_threshold(threshold)) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (int st = check_sizes(rows, width)) return st;
  if (rows == 0 || width == 0) return VECTRA_BLOCK_OK;
  if (!x || !y || (threshold && !rng)) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (int st = check_stride(x_stride, width, rows)) return st;
  if (int st = check_stride(y_stride, width, rows)) return st;
  const Dropout d{rng, threshold, stream_id, drop_scale(threshold)};
  const int64_t total = rows * ceil_div(width, 8);
  (void)hipGetLastError();
  typed(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int kGroups = sizeof(T) == 2 ? 4 : 2;
    const auto kernel = total < (int64_t{1} << 31) - 256 * kGroups ? dropout_kernel<T, uint32_t, kGroups>
                                                                   : dropout_kernel<T, int64_t, kGroups>;
    kernel<<<static_cast<uint32_t>(ceil_div(total, 256 * kGroups)), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        static_cast<const T*>(x), rows, width, x_stride, static_cast<T*>(y), y_stride, d);
  });
  return launched();
}

int vectra_norm_forward(const vectra_norm_args* args, vectra_block_stream_t stream) {
  if (int st = check_forward(args)) return st;
  (void)hipGetLastError();
  return forward(*args, reinterpret_cast<hipStream_t>(stream));
}

int vectra_norm_backward(const vectra_norm_grad_args* args, void* workspace, int64_t workspace_bytes,
                         vectra_block_stream_t stream) {
  if (int st = check_backward(args)) return st;
  const int cus = compute_units();
  Scratch sized{nullptr, 0};
  if (int st = backward(*args, sized, false, cus, nullptr)) return st;
  if (sized.used > 0 && (!workspace || workspace_bytes < sized.used || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return VECTRA_BLOCK_ERR_WORKSPACE;
  Scratch scratch{static_cast<char*>(workspace), 0};
  return backward(*args, scratch, true, cus, reinterpret_cast<hipStream_t>(stream));
}

int64_t vectra_norm_backward_workspace_bytes(const vectra_norm_grad_args* args) {
  if (int st = check_backward(args)) return -st;
  Scratch sized{nullptr, 0};
  if (int st = backward(*args, sized, false, compute_units(), nullptr)) return -st;
  return sized.used;
}

int vectra_blocks_quantize(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, int32_t tiles,
                           void* codes, void* scales, vectra_block_stream_t stream) {
  if (!known_dtype(dtype)) return VECTRA_BLOCK_ERR_BAD_DTYPE;
  if (tiles != 0 && tiles != 1) return VECTRA_BLOCK_ERR_BAD_OPTION;
  if (int st = check_sizes(rows, width)) return st;
  if (rows == 0 || width == 0) return VECTRA_BLOCK_OK;
  if (!x || !codes || !scales) return VECTRA_BLOCK_ERR_NULL_ARGUMENT;
  if (!aligned(codes, 16)) return VECTRA_BLOCK_ERR_BAD_SHAPE;
  if (int st = check_stride(x_stride, width, rows)) return st;
  (void)hipGetLastError();
  return quantize(x, dtype, rows, width, x_stride, tiles, codes, scales, reinterpret_cast<hipStream_t>(stream));
}

int vectra_linear8_forward(const vectra_linear8_args* args, void* workspace, int64_t workspace_bytes,
                           vectra_block_stream_t stream) {
  if (int st = check_linear8(args)) return st;
  const int cus = compute_units();
  Scratch sized{nullptr, 0};
  if (int st = linear8(*args, sized, false, cus, nullptr)) return st;
  if (sized.used > 0 && (!workspace || workspace_bytes < sized.used || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return VECTRA_BLOCK_ERR_WORKSPACE;
  Scratch scratch{static_cast<char*>(workspace), 0};
  return linear8(*args, scratch, true, cus, reinterpret_cast<hipStream_t>(stream));
}

int64_t vectra_linear8_workspace_bytes(const vectra_linear8_args* args) {
  if (int st = check_linear8(args)) return -st;
  Scratch sized{nullptr, 0};
  if (int st = linear8(*args, sized, false, compute_units(), nullptr)) return -st;
  return sized.used;
}

const char* vectra_block_status_string(int status) {
  switch (status) {
    case VECTRA_BLOCK_OK: return "ok";
    case VECTRA_BLOCK_ERR_NULL_ARGUMENT: return "a required pointer is NULL";
    case VECTRA_BLOCK_ERR_BAD_DTYPE: return "unsupported dtype combination";
    case VECTRA_BLOCK_ERR_BAD_SHAPE: return "negative or inconsistent sizes or strides";
    case VECTRA_BLOCK_ERR_BAD_STRUCT: return "struct_size does not match this build of the library";
    case VECTRA_BLOCK_ERR_TOO_LARGE: return "a size exceeds the kernels' range";
    case VECTRA_BLOCK_ERR_LAUNCH: return "HIP kernel launch failed";
    case VECTRA_BLOCK_ERR_BAD_OPTION: return "unknown norm or activation, or a threshold or eps out of range";
    case VECTRA_BLOCK_ERR_WORKSPACE: return "workspace missing, too small or not 256-byte aligned";
    default: return "unknown status";
  }
}

int vectra_block_abi_version(void) { return (1 << 16) | 0; }

}  // extern "C"
