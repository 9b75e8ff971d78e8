// The dense operators' C ABI (include/vectra_dense.h): argument checks, the
// plan of a call (which products, on which tiles, through which scratch) and
// the small kernels around the products.
//
// A backward pass is
//   [x^ = the 8-bit rows' values]       where the input was kept in 8 bits
//   [dz, sums of dz] = slope epilogue of x W^T      (an activation or a gate)
//   dx = dz W;   dW = dz^T x;   db = the sums, added up.
// z is computed again rather than kept: that is one more product, but no
// [rows, width_out] tensor lives from the forward to the backward pass, and at
// the price model's widths (128 to 256) reading x again is cheaper than
// reading z back.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "dense_common.h"
#include "dense_kernels.h"
#include "row_chunk.h"

namespace vectra_dense {
namespace {

constexpr int kBlock = 32;  // elements that share a power of two

// ----------------------------------------------------------------- kernels

// Copies rows into rows of whole 16-byte chunks (zero padded): operands whose
// rows are not 16-byte aligned or hold part of a chunk at their end.  One
// thread per output chunk, read as unaligned 16 bytes; Index as in the 8-bit
// rows' kernels below (80981 x 327 bf16: 24 us, 29 with elements read one by one).
template <typename T, typename Index>
__global__ __launch_bounds__(256) void pack_kernel(const T* x, int64_t stride, int64_t rows, int64_t width, T* out,
                                                   int64_t chunks) {
  constexpr int kPer = 16 / sizeof(T);
  const Index at = static_cast<Index>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<Index>(rows * chunks)) return;
  const Index row = at / static_cast<Index>(chunks);
  const int64_t first = static_cast<int64_t>(at - row * static_cast<Index>(chunks)) * kPer;
  const Frag f = load_row_chunk<T>(x + row * stride, width, first);
  *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(at) * kPer) = f.w;
}

// Adds up the planes of a split product in a fixed order and finishes it with
// the product's epilogue.  A thread adds every kLanes-th plane of four columns
// (a gated layer: of both halves), four planes in flight; the kLanes threads of
// a quad are joined in LDS.  One lane per quad where there are few planes or
// many quads; 16 where one thread would walk hundreds of planes (a [256, 128]
// weight gradient of 208 parts: 57.8 us with one lane, each load waiting for
// the one before; 5 with 16).
template <typename T, int kLanes, int kEpi>
__global__ __launch_bounds__(256) void join_kernel(const float* parts, int splits, int64_t m, int64_t n, int64_t ld,
                                                   GemmParams p, int quad_blocks, void* sums_out,
                                                   int32_t sums_dtype) {
  constexpr int kQuads = 256 / kLanes;
  constexpr bool kGated = kEpi == kEpiGated || kEpi == kEpiGatedSlope;
  constexpr int kHalves = kGated ? 2 : 1;
  if (static_cast<int>(blockIdx.x) >= quad_blocks) {  // the sums' planes: 16 lanes per sum, 16 sums
    __shared__ float sum_part[16][16];
    const int c = threadIdx.x % 16, lane = threadIdx.x / 16;
    const int64_t at = static_cast<int64_t>(blockIdx.x - quad_blocks) * 16 + c;
    float s = 0.f;
    if (at < m) {
#pragma unroll 4
      for (int k = lane; k < splits; k += 16) s += static_cast<const float*>(p.sums)[k * m + at];
    }
    sum_part[lane][c] = s;
    __syncthreads();
    if (lane != 0 || at >= m) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) s += sum_part[k][c];
    store_as(sums_out, at, sums_dtype, s);
    return;
  }
  __shared__ f32x4 part[kLanes > 1 ? kLanes : 1][kHalves][kQuads];
  const int q = threadIdx.x % kQuads, lane = threadIdx.x / kQuads;
  const int64_t quads = (n + 3) / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kQuads + q;
  const bool live = at < m * quads;
  const int64_t row = live ? at / quads : 0, col = live ? (at - row * quads) * 4 : 0;
  const int64_t plane = m * ld;
  f32x4 s[kHalves] = {};
  if (live) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const float* const from = parts + row * ld + h * n + col;
      const auto load = [&](int k) {  // (the up half starts at any column)
        f32x4 v;
        __builtin_memcpy(&v, from + k * plane, 16);
        return v;
      };
      int k = lane;
      for (; k + 3 * kLanes < splits; k += 4 * kLanes) {
        f32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load(k + j * kLanes);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[h] += v[j];
      }
      for (; k < splits; k += kLanes) s[h] += load(k);
    }
  }
  if constexpr (kLanes > 1) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) part[lane][h][q] = s[h];
    __syncthreads();
    if (lane != 0) return;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int k = 1; k < kLanes; ++k) s[h] += part[k][h][q];
  }
  if (!live) return;
  const int left = static_cast<int>(least(n - col, 4));
  if (p.bias) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) s[h][e] += load_bias(p.bias, h * n + col + e, p.bias_dtype);
  }
  T* const out = static_cast<T*>(p.out) + row * p.ldo + col;
  if constexpr (kEpi == kEpiStore || kEpi == kEpiGated) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[0][e] = act_value<T>(s[0][e], p.activation);
      if constexpr (kGated) s[0][e] *= s[1][e];
    }
    if (p.residual) s[0] += load4(static_cast<const T*>(p.residual) + row * p.ldr + col, left);
    store4(out, s[0], left);
  } else {
    const f32x4 dy = load4(static_cast<const T*>(p.grad) + row * p.ldg + col, left);
    f32x4 up;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float value, slope;
      act_slope(s[0][e], p.activation, value, slope);
      s[0][e] = dy[e] * slope;
      if constexpr (kGated) {
        s[0][e] *= s[1][e];
        up[e] = dy[e] * value;
      }
    }
    store4(out, s[0], left);
    if constexpr (kGated) store4(out + n, up, left);
    if (col + 4 >= n) zero_padding(static_cast<T*>(p.out) + row * p.ldo, n * kHalves, p.ldo);
  }
}

template <typename T, int kLanes>
auto join_for(int epi) {
  return epi == kEpiStore   ? join_kernel<T, kLanes, kEpiStore>
         : epi == kEpiGated ? join_kernel<T, kLanes, kEpiGated>
         : epi == kEpiSlope ? join_kernel<T, kLanes, kEpiSlope>
                            : join_kernel<T, kLanes, kEpiGatedSlope>;
}

// Column sums of rows [blockIdx.y * per, ...): a thread adds up a 16-byte
// chunk of every kRows-th row, four rows in flight; 2^lanes_log2 threads side by
// side cover a row's chunks (64 at most, as many as a narrow row has), and the
// block's row lanes are joined in LDS in a fixed order.  Out: one row of
// partial sums per blockIdx.y, or with one of them the result itself.
template <typename In>
__global__ __launch_bounds__(256) void column_sums_kernel(const In* x, int64_t stride, int64_t rows, int64_t n,
                                                          int64_t per, int lanes_log2, void* out, int64_t out_stride,
                                                          int32_t out_dtype) {
  constexpr int kPer = 16 / sizeof(In);
  __shared__ float part[256][kPer + 1];
  const int lanes = 1 << lanes_log2, row_lanes = 256 >> lanes_log2;
  const int c = threadIdx.x & (lanes - 1), r = threadIdx.x >> lanes_log2;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * lanes + c) * kPer;
  const int64_t first = blockIdx.y * per, last = least(first + per, rows);
  float s[kPer] = {};
  const auto add = [&](const Frag& f) {
    In v[kPer];
    __builtin_memcpy(v, &f.w, 16);
#pragma unroll
    for (int e = 0; e < kPer; ++e) s[e] += widen(v[e]);
  };
  if (col < n) {
    int64_t row = first + r;
    for (; row + 3 * row_lanes < last; row += 4 * row_lanes) {
      Frag f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = load_row_chunk(x + (row + j * row_lanes) * stride, n, col);
#pragma unroll
      for (int j = 0; j < 4; ++j) add(f[j]);
    }
    for (; row < last; row += row_lanes) add(load_row_chunk(x + row * stride, n, col));
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) part[threadIdx.x][e] = s[e];
  __syncthreads();
  for (int at = threadIdx.x; at < lanes * kPer; at += 256) {
    const int64_t to = static_cast<int64_t>(blockIdx.x) * lanes * kPer + at;
    if (to >= n) continue;
    float total = 0.f;
    for (int k = 0; k < row_lanes; ++k) total += part[k * lanes + at / kPer][at % kPer];
    store_as(out, blockIdx.y * out_stride + to, out_dtype, total);
  }
}

// ------------------------------------------------------------- 8-bit rows

// The exponent byte of a block whose largest finite magnitude is `largest`:
// the smallest e with largest <= 448 * 2^e, at least `lowest`, plus 127.
// largest = f * 2^x with f in [1, 2): 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(float largest, int lowest) {
  const uint32_t bits = __float_as_uint(largest);
  int e;
  if (bits < 0x00800000u) {
    e = lowest;  // zero or an fp32 subnormal: far below the lowest exponent
  } else {
    e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x007fffffu) > 0x00600000u ? 1 : 0);
  }
  return max(e, lowest) + 127;
}

// 2^e as fp32 for e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// fp32 in [-448, 448] to e4m3, ties to even (v_cvt_pk_fp8_f32); NaN to NaN.
__device__ __forceinline__ uint32_t to_e4m3x4(f32x4 v) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true));
}

__device__ __forceinline__ f32x4 from_e4m3x4(uint32_t w) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Both kernels move eight elements per thread and turn, 16 bytes of a 16-bit
// row, and turn their work's index into a row and a column by 32-bit division
// (Index) where the counts allow: a 64-bit one costs more than the rest of a
// turn (66560 x 256 bf16: 16.6 us with it and four elements per thread; now 22
// us for both kernels, 103 MB).

// Four lanes per block of 32.
template <typename T, typename Index>
__global__ __launch_bounds__(256) void quantize_kernel(const T* x, int64_t rows, int64_t width, int64_t stride,
                                                       uint8_t* codes, int64_t codes_stride, uint8_t* scales,
                                                       int64_t scales_stride, int64_t blocks) {
  constexpr int kLowest = __is_same(T, _Float16) ? -15 : -117, kHighest = __is_same(T, _Float16) ? 8 : 120;
  const Index at = static_cast<Index>(blockIdx.x) * 64 + (threadIdx.x >> 2);
  const bool live = at < static_cast<Index>(rows * blocks);
  const Index row = live ? at / static_cast<Index>(blocks) : 0;
  const int64_t block = live ? at - row * static_cast<Index>(blocks) : 0;
  const int64_t col = block * kBlock + (threadIdx.x & 3) * 8;
  const int left = live ? static_cast<int>(most(least(width - col, 8), 0)) : 0;
  f32x4 v[2] = {};
  if (left > 0) load8(x + row * stride + col, left, v[0], v[1]);
  float largest = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = __builtin_fabsf(v[k / 4][k % 4]);
    if (a <= 3.4028234663852886e38f) {
      largest = a > largest ? a : largest;
    } else {
      v[k / 4][k % 4] = __builtin_nanf("");
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
  const int byte = block_exponent(largest, kLowest);
  const int e = byte - 127;
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v[h] *= power_of_two(-e);  // e in [-117, 120]
    // The type's largest value, 255.9 * 2^8 (fp16) or 2^120, would round to
    // 256 times that, which the type lacks: at its exponent, magnitudes of
    // 248 and more take the code below, 240.
    if (e == kHighest)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (__builtin_fabsf(v[h][k]) >= 248.f) v[h][k] = __builtin_copysignf(240.f, v[h][k]);
    w[h] = to_e4m3x4(v[h]);
  }
  uint8_t* const out = codes + row * codes_stride + col;
  if (left == 8) {
    __builtin_memcpy(out, w, 8);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) out[k] = static_cast<uint8_t>(w[k / 4] >> (8 * (k % 4)));
  }
  if (live && (threadIdx.x & 3) == 0) scales[row * scales_stride + block] = static_cast<uint8_t>(byte);
}

// The output has `columns` columns; those from `width` on are zeros (the
// workspace's padded rows).
template <typename T, typename Index>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* codes, int64_t codes_stride,
                                                         const uint8_t* scales, int64_t scales_stride, int64_t rows,
                                                         int64_t width, T* out, int64_t out_stride, int64_t columns) {
  const Index eights = static_cast<Index>((columns + 7) / 8);
  const Index at = static_cast<Index>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<Index>(rows) * eights) return;
  const Index row = at / eights;
  const int64_t col = static_cast<int64_t>(at - row * eights) * 8;
  const int left = static_cast<int>(most(least(width - col, 8), 0));
  const uint8_t* const p = codes + row * codes_stride + col;
  uint2 w = {0, 0};
  if (left == 8) {
    __builtin_memcpy(&w, p, 8);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) (k < 4 ? w.x : w.y) |= static_cast<uint32_t>(p[k]) << (8 * (k % 4));
  }
  f32x4 a = from_e4m3x4(w.x), b = from_e4m3x4(w.y);
  if (left > 0) {
    const int e = static_cast<int>(scales[row * scales_stride + col / kBlock]) - 127;
    const float s = e == 128 ? __builtin_nanf("") : e == -127 ? 5.877471754111438e-39f : power_of_two(e);
    a *= s;
    b *= s;
  }
  store8(out + row * out_stride + col, a, b, static_cast<int>(least(columns - col, 8)));
}

// -------------------------------------------------------------------- host

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t element_size(int32_t dtype) { return dtype == VECTRA_DENSE_F32 ? 4 : 2; }

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

// Scratch memory in order of use.  Without a base only the size is found.
struct Scratch {
  char* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* const p = base ? base + used : nullptr;
    used += (bytes + 255) & ~int64_t{255};
    return p;
  }
};

// An operand of products as the caller (or this call) has it, and, once a
// product needs it, its zero-padded copy with whole 16-byte chunks per row.
struct Operand {
  const void* p = nullptr;
  int64_t ld = 0, rows = 0, width = 0;
  bool padded = false;  // a matrix of this call's own: rows of whole chunks, the padding zeros
  const void* packed = nullptr;
  int64_t packed_ld = 0;
};

// A caller's matrix.  One row may come with any stride, which the products'
// bounds, (rows - 1) strides and a row, must not take for another's.
Operand operand(const void* p, int64_t stride, int64_t rows, int64_t width) {
  return Operand{p, rows > 1 ? stride : width, rows, width};
}

// One call: the element type, the scratch and whether kernels are launched.
struct Call {
  int32_t dtype;
  Scratch scratch;
  bool launch;
  hipStream_t stream;
  int cus;
  int status = VECTRA_DENSE_OK;

  int64_t esize() const { return element_size(dtype); }
  int64_t per() const { return 16 / esize(); }
  void check() {
    if (hipGetLastError() != hipSuccess && status == VECTRA_DENSE_OK) status = VECTRA_DENSE_ERR_LAUNCH;
  }
  bool go() const { return launch && status == VECTRA_DENSE_OK; }

  template <typename F>
  void typed(F&& f) {
    switch (dtype) {
      case VECTRA_DENSE_F32: f(static_cast<float*>(nullptr)); break;
      case VECTRA_DENSE_F16: f(static_cast<_Float16*>(nullptr)); break;
      default: f(static_cast<__bf16*>(nullptr)); break;
    }
    check();
  }

  bool whole_chunks(const void* p, int64_t ld, int64_t width) const {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % per() == 0 && width % per() == 0;
  }

  int64_t padded(int64_t width) const { return ceil_div(width, per()) * per(); }

  bool whole(const Operand& o) const { return o.rows == 0 || o.width == 0 || o.padded || whole_chunks(o.p, o.ld, o.width); }

  // Estimated time of the copy that pack() would make.
  double copy_time(const Operand& o) const {
    return o.packed || whole(o) ? 0.0 : 4e-6 + 2.0 * o.rows * o.width * esize() / 4.5e12;
  }

  // Makes `o` readable in whole chunks: as it is, or by a copy that later
  // products of this call use too.
  void pack(Operand& o) {
    if (o.packed) return;
    o.packed = o.p;
    o.packed_ld = o.ld;
    if (whole(o)) return;
    o.packed_ld = padded(o.width);
    const int64_t chunks = o.packed_ld / per();
    o.packed = scratch.take(o.rows * o.packed_ld * esize());
    if (go())
      typed([&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto kernel = o.rows * chunks < (int64_t{1} << 31) - 256 ? pack_kernel<T, uint32_t> : pack_kernel<T, int64_t>;
        kernel<<<static_cast<uint32_t>(ceil_div(o.rows * chunks, 256)), 256, 0, stream>>>(
            static_cast<const T*>(o.p), o.ld, o.rows, o.width, const_cast<T*>(static_cast<const T*>(o.packed)), chunks);
      });
    if (!launch) o.packed = &o;  // sizing: only that there is one counts
  }

  // The tile and the number of contraction parts with the least estimated
  // time, and that time.  Measured, 16 bits, 8192 x K -> 4096, as a line in K:
  //   slope      tile 256 x 256: 1.5 PFLOP/s; 192 x 256: 1.42; 128: 1.14 (1.0 with
  //              a wide operand); 64: 0.79; fp32: 0.12 on any of them
  //   intercept  what the epilogue moves at 4.5 TB/s, and 0.42 ps per result
  //              where it evaluates activations; a part of it (kShown) is not
  //              hidden behind other workgroups' products: all of it with one
  //              workgroup per CU (the big tiles, by LDS), 0.8 of it with 2 or 5
  // A CU holding fewer workgroups than it could runs at a part of its rate
  // (kPart).  The tiles' operands pass from L2 to LDS at 16 TB/s.  A split
  // costs its fp32 planes, written and read at 5 TB/s, and the joining launch.
  //   chosen / other tiles, us: 8192 x 4096 -> 4096 bf16 200 on 256 (225 on 192,
  //   237 on 128); 9216 x 4096 -> 4096 241 on 192 (275 on 256, whose 576 tiles
  //   are 2.25 per CU; 272 on 128); 2051 x 2048 -> 2 x 5632 fp16 gated 84 on 192
  //   (98 on 256, 95 on 128); dx of 10007 x 1000 -> 2 x 2730 bf16 109 on 192
  //   (130 on 256, 154 on 128); 300 x 1024 -> 1024 10 on 64 (14 on 128);
  //   66560 x 128 -> 256 weight gradient 18 on 64 in 64 parts (20 on 128 in 128).
  //
  // a_row_bytes: of a deep row operand, whose tile the kernels address with 31
  // bits (dz of a gated layer in fp32 has rows of up to 16 MB, twice those of
  // the gradient that the caller's stride was checked for); 0 for a wide one.
  double choose(const GemmParams& p, int64_t columns, int layout, int epi, int64_t a_row_bytes, int& tile, int& splits) const {
    static constexpr double kRate16[kTileCount] = {1.5e15, 1.42e15, 1.14e15, 0.79e15}, kRate32 = 0.12e15;
    static constexpr int kResident[kTileCount] = {1, 1, 2, 5};
    static constexpr double kPart[kTileCount][5] = {{1.0}, {1.0}, {0.65, 1.0}, {0.35, 0.6, 0.8, 0.9, 1.0}};
    static constexpr double kShown[kTileCount] = {1.0, 1.0, 0.8, 0.85}, kBatch[kTileCount] = {2e-6, 2e-6, 0.5e-6, 0.5e-6};
    const bool busy = epi > kEpiPartial || p.activation != VECTRA_DENSE_NONE;
    const int moved = 1 + (p.residual || p.grad ? 1 : 0) + (epi == kEpiGatedSlope ? 1 : 0);  // values per result
    const double finish = static_cast<double>(p.m) * p.n * (moved * esize() / 4.5e12 + (busy ? 0.42e-12 : 0));
    const int most_splits = std::min(256, p.k_tiles / 2);
    double best = 1e30;
    splits = 1;
    tile = kTileCount - 1;
    for (int t = 0; t < kTileCount; ++t) {
      if (t == kTileTall && dtype == VECTRA_DENSE_F32) continue;
      if (kTileRows[t] * a_row_bytes >= int64_t{1} << 31) continue;  // (the small tile's 64 rows always fit)
      const int64_t tiles = ceil_div(p.m, kTileRows[t]) * ceil_div(columns, kTileColumns[t]);
      const double rate16 = t == kTileMedium && layout != kLayoutForward ? 1.0e15 : kRate16[t];
      const double rate = (dtype == VECTRA_DENSE_F32 ? kRate32 : rate16) / 256;  // of a full CU
      for (int k = 1; k <= std::max(1, most_splits); k *= 2) {
        const int64_t depth = ceil_div(p.k_tiles, k) * (128 / esize());
        const int64_t per_cu = ceil_div(tiles * k, cus);
        const int together = static_cast<int>(std::min<int64_t>(per_cu, kResident[t]));
        const double products = per_cu * 2.0 * kTileRows[t] * kTileColumns[t] * depth / (rate * kPart[t][together - 1]);
        const double traffic = tiles * k * static_cast<double>(kTileRows[t] + kTileColumns[t]) * depth * esize() / 16e12;
        const double join = k > 1 ? 8.0 * k * p.m * columns / 5e12 + 6e-6 : 0;
        const double time = std::max(products, traffic) + kShown[t] * finish + ceil_div(per_cu, kResident[t]) * kBatch[t] + join;
        if (time < best * 0.98) {
          best = time;
          tile = t;
          splits = k;
        }
      }
    }
    return best;
  }

  // One product: A [p.m or contraction rows], B, the contraction p.depth, all in
  // true sizes.  sums_out: where the sums of A over the contraction go (weight
  // layout), or the column sums of dz (slope epilogues); NULL: not wanted.
  // False where they were wanted and are left to the caller.
  bool product(GemmParams p, Operand& a, Operand& b, int layout, int epi, void* sums_out = nullptr,
               int32_t sums_dtype = 0) {
    const bool gated = epi == kEpiGated || epi == kEpiGatedSlope;
    const bool slope = epi == kEpiSlope || epi == kEpiGatedSlope;
    const int64_t columns = gated ? 2 * p.n : p.n;
    const int deep = static_cast<int>(128 / esize());
    p.k_tiles = static_cast<int32_t>(ceil_div(p.depth, deep));
    int tile, splits;
    const int64_t a_row_bytes = layout == kLayoutWeight ? 0 : std::max(a.ld, padded(a.width)) * esize();
    const double time = choose(p, columns, layout, epi, a_row_bytes, tile, splits);
    p.tiles_m = static_cast<int32_t>(ceil_div(p.m, kTileRows[tile]));
    p.tiles_n = static_cast<int32_t>(ceil_div(columns, kTileColumns[tile]));
    p.k_tiles_per_split = static_cast<int32_t>(std::max<int64_t>(1, ceil_div(p.k_tiles, splits)));
    splits = static_cast<int>(std::max<int64_t>(1, ceil_div(p.k_tiles, p.k_tiles_per_split)));
    // Unaligned operands through registers run at about 0.6 of the rate
    // (80981 x 728 -> 327 bf16 with an odd W: 136 us, 81 with W copied): that
    // is taken where copying them would cost more.
    const bool any = !kTileBig[tile] && copy_time(a) + copy_time(b) > 0.6 * time;
    p.depth_b = p.depth;
    if (any) {
      p.a = a.p;
      p.lda = a.ld;
      p.b = b.p;
      p.ldb = b.ld;
    } else {
      pack(a);
      pack(b);
      p.a = a.packed;
      p.lda = a.packed_ld;
      p.b = b.packed;
      p.ldb = b.packed_ld;
      p.a_width = padded(a.width);
      p.b_width = padded(b.width);
      if (layout != kLayoutWeight) p.depth = padded(p.depth);  // deep rows are read to the end of their last chunk
      if (layout == kLayoutForward) p.depth_b = p.depth;
    }
    const int64_t kept = scratch.used;
    // The big tiles leave the sums to a pass of their own: their few adds per
    // product cost its loop 85 us of 325 (8192 x 4096 -> 4096 bf16), the pass 20.
    if (sums_out && layout == kLayoutWeight && kTileBig[tile]) {
      column_sums_of(a, p.m, sums_out, sums_dtype);
      sums_out = nullptr;
    }
    const bool sums_left = sums_out && slope && splits > 1;  // the joining launch does not sum dz
    if (sums_left) sums_out = nullptr;
    // The sums' planes: of the contraction's parts, or of the tile rows.
    const int64_t planes = layout == kLayoutWeight ? splits : p.tiles_m, sum_width = layout == kLayoutWeight ? p.m : columns;
    if (sums_out) {
      p.sums = planes == 1 ? sums_out : scratch.take(planes * sum_width * 4);
      p.sums_dtype = planes == 1 ? sums_dtype : VECTRA_DENSE_F32;
    }
    if (splits == 1) {
      run(p, layout, tile, any, epi, 1);
      if (sums_out && planes > 1)
        column_sums<float>(static_cast<const float*>(p.sums), sum_width, planes, sum_width, sums_out, sums_dtype);
    } else {
      // Rows of four-column pieces; the join reads such pieces of the up half
      // from column n on.
      const int64_t ld = ceil_div(gated ? p.n + ceil_div(p.n, 4) * 4 : columns, 4) * 4;
      GemmParams q = p;
      q.n = columns;  // (a gated weight's halves side by side)
      q.out = scratch.take(splits * p.m * ld * 4);
      q.ldo = ld;
      run(q, layout, tile, any, kEpiPartial, splits);
      if (go())
        typed([&](auto* t) {
          using T = std::remove_pointer_t<decltype(t)>;
          const int64_t quads = p.m * ceil_div(p.n, 4);
          const bool lanes = splits > 8 && quads < 64 * 256 * 4;
          const int64_t blocks = ceil_div(quads, lanes ? 16 : 256), sum_blocks = sums_out ? ceil_div(p.m, 16) : 0;
          const auto kernel = lanes ? join_for<T, 16>(epi) : join_for<T, 1>(epi);
          kernel<<<static_cast<uint32_t>(blocks + sum_blocks), 256, 0, stream>>>(
              static_cast<const float*>(q.out), splits, p.m, p.n, ld, p, static_cast<int>(blocks), sums_out, sums_dtype);
        });
    }
    most = std::max(most, scratch.used);
    scratch.used = kept;  // the next product may use it again: launches of one stream run in order
    return !sums_left;
  }

  // Column sums of an operand's n columns.
  void column_sums_of(const Operand& o, int64_t n, void* out, int32_t out_dtype) {
    typed([&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      column_sums<T>(static_cast<const T*>(o.p), o.ld, o.rows, n, out, out_dtype);
    });
  }
  int64_t most = 0;          // of scratch, over all products

  void run(const GemmParams& p, int layout, int tile, bool any, int epi, int splits) {
    if (!go()) return;
    const auto f = dtype == VECTRA_DENSE_F32 ? launch_gemm_f32 : dtype == VECTRA_DENSE_F16 ? launch_gemm_f16 : launch_gemm_bf16;
    const int st = f(p, layout, tile, any, epi, splits, stream);
    if (st != VECTRA_DENSE_OK) status = st;
  }

  // Contraction steps of the resident kernel that serves these sizes, or 0.
  // Its workgroups copy the whole weight first, so it needs rows enough for
  // the 16 waves of a quarter of the CUs, a unit of 16 rows each.
  int resident_steps(int64_t rows, int64_t width, int64_t n, bool gated) const {
    if (rows < 16 * 16 * cus / 4) return 0;
    const int64_t bytes = width * esize(), n_pad = ceil_div(n, 32) * 32 * (1 + gated);
    const auto fits = [&](int steps) {
      const int64_t row = steps * 64 + ((steps & (steps - 1)) ? 16 : 0) + 4;  // and the bias
      return bytes <= steps * 64 && n_pad * row <= kResidentLds;
    };
    if (esize() == 2) {
      for (int s : kResidentSteps16)
        if (fits(s)) return s;
    } else {
      for (int s : kResidentSteps32)
        if (fits(s)) return s;
    }
    return 0;
  }

  void resident(ResidentParams p, int steps, int epi, bool with_dx) {
    if (!go()) return;
    p.n_pad = static_cast<int32_t>(ceil_div(p.n, 32) * 32);
    const auto f = dtype == VECTRA_DENSE_F32 ? launch_resident_f32 : dtype == VECTRA_DENSE_F16 ? launch_resident_f16 : launch_resident_bf16;
    const int workgroups = static_cast<int>(std::min<int64_t>(cus, ceil_div(ceil_div(p.rows, 16), 16)));
    const int st = f(p, steps, epi, with_dx, workgroups, stream);
    if (st != VECTRA_DENSE_OK) status = st;
  }

  // Column sums of [rows, n] into the bias's gradient.
  template <typename In>
  void column_sums(const In* x, int64_t stride, int64_t rows, int64_t n, void* out, int32_t out_dtype) {
    const int64_t chunks = ceil_div(n, 16 / static_cast<int64_t>(sizeof(In)));
    int lanes_log2 = 0;
    while (lanes_log2 < 6 && (1 << lanes_log2) < chunks) ++lanes_log2;
    const uint32_t across = static_cast<uint32_t>(ceil_div(chunks, 1 << lanes_log2));
    // Enough parts for four blocks per CU, of at least eight turns of four rows.
    int64_t parts = std::min<int64_t>(ceil_div(rows, 32 * (256 >> lanes_log2)), ceil_div(4 * cus, across));
    parts = std::max<int64_t>(1, parts);
    if (parts == 1) {
      if (go())
        column_sums_kernel<In><<<dim3(across, 1), 256, 0, stream>>>(x, stride, rows, n, rows, lanes_log2, out, 0, out_dtype);
      check();
      return;
    }
    const int64_t per = ceil_div(rows, parts), kept = scratch.used;
    float* const sums = static_cast<float*>(scratch.take(parts * n * 4));
    if (go())
      column_sums_kernel<In><<<dim3(across, static_cast<uint32_t>(parts)), 256, 0, stream>>>(
          x, stride, rows, n, per, lanes_log2, sums, n, VECTRA_DENSE_F32);
    check();
    column_sums<float>(sums, n, parts, n, out, out_dtype);
    most = std::max(most, scratch.used);
    scratch.used = kept;
  }
};

// The 8-bit form's kernels, for the operators and for a backward pass.
template <typename T>
void quantize(const void* x, int64_t rows, int64_t width, int64_t stride, void* codes, int64_t codes_stride, void* scales,
              int64_t scales_stride, Call& c) {
  const int64_t blocks = ceil_div(width, kBlock), grid = ceil_div(rows * blocks, 64);
  const auto kernel = rows * blocks < (int64_t{1} << 31) - 64 ? quantize_kernel<T, uint32_t> : quantize_kernel<T, int64_t>;
  kernel<<<static_cast<uint32_t>(grid), 256, 0, c.stream>>>(
      static_cast<const T*>(x), rows, width, stride, static_cast<uint8_t*>(codes), codes_stride,
      static_cast<uint8_t*>(scales), scales_stride, blocks);
}

template <typename T>
void dequantize(const void* codes, int64_t codes_stride, const void* scales, int64_t scales_stride, int64_t rows,
                int64_t width, const void* out, int64_t out_stride, int64_t columns, Call& c) {
  const int64_t work = rows * ceil_div(columns, 8);
  const auto kernel = work < (int64_t{1} << 31) - 256 ? dequantize_kernel<T, uint32_t> : dequantize_kernel<T, int64_t>;
  kernel<<<static_cast<uint32_t>(ceil_div(work, 256)), 256, 0, c.stream>>>(
      static_cast<const uint8_t*>(codes), codes_stride, static_cast<const uint8_t*>(scales), scales_stride, rows, width,
      const_cast<T*>(static_cast<const T*>(out)), out_stride, columns);
}

constexpr int64_t kMostRows = int64_t{1} << 30;
constexpr int64_t kMostWidth = int64_t{1} << 21;

bool known_dtype(int32_t t) { return t == VECTRA_DENSE_F32 || t == VECTRA_DENSE_F16 || t == VECTRA_DENSE_BF16; }

// Sizes that the kernels' grids cover (offsets within a tile: check_stride, and
// for dz of a gated layer Call::choose).
int check_sizes(int64_t rows, int64_t width_in, int64_t width_out, int gated) {
  if (rows < 0 || width_in < 0 || width_out < 0) return VECTRA_DENSE_ERR_BAD_SHAPE;
  if (rows > kMostRows || width_in > kMostWidth || width_out > kMostWidth) return VECTRA_DENSE_ERR_TOO_LARGE;
  // Elementwise kernels: a thread per four elements, fewer than 2^32 threads.
  const int64_t widest = std::max(width_in, width_out * (1 + gated)) + 64;
  if (rows * widest >= int64_t{1} << 34) return VECTRA_DENSE_ERR_TOO_LARGE;
  return VECTRA_DENSE_OK;
}

// A row stride covers the row, and 256 rows of it, or of a copy in whole chunks
// (a gated weight's tile: a whole half and 256 rows), span less than 2^31 bytes.
int check_stride(int64_t stride, int64_t width, int64_t rows, int64_t span_rows, int64_t esize) {
  if (rows > 1 && stride < width) return VECTRA_DENSE_ERR_BAD_SHAPE;
  if (stride < 0) return VECTRA_DENSE_ERR_BAD_SHAPE;
  if (stride > (int64_t{1} << 40) || span_rows * std::max<int64_t>({stride, width + 8, 64}) * esize >= (int64_t{1} << 31))
    return VECTRA_DENSE_ERR_TOO_LARGE;
  return VECTRA_DENSE_OK;
}

bool known_activation(int32_t a) { return a >= VECTRA_DENSE_NONE && a <= VECTRA_DENSE_SILU; }

int check_forward(const vectra_dense_args* a) {
  if (!a) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  if (a->struct_size != static_cast<int64_t>(sizeof(vectra_dense_args))) return VECTRA_DENSE_ERR_BAD_STRUCT;
  if (!known_dtype(a->dtype)) return VECTRA_DENSE_ERR_BAD_DTYPE;
  if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != VECTRA_DENSE_F32) return VECTRA_DENSE_ERR_BAD_DTYPE;
  if (!known_activation(a->activation)) return VECTRA_DENSE_ERR_BAD_ACTIVATION;
  if (a->gated != 0 && a->gated != 1) return VECTRA_DENSE_ERR_BAD_SHAPE;
  if (a->gated && a->residual) return VECTRA_DENSE_ERR_BAD_SHAPE;
  const int64_t es = element_size(a->dtype);
  if (int st = check_sizes(a->rows, a->width_in, a->width_out, a->gated)) return st;
  if (a->rows == 0 || a->width_out == 0) return VECTRA_DENSE_OK;
  if (!a->out || (a->width_in && (!a->x || !a->weight))) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  const int64_t n_w = a->width_out * (1 + a->gated);
  if (int st = check_stride(a->x_stride, a->width_in, a->rows, 256, es)) return st;
  if (int st = check_stride(a->weight_stride, a->width_in, n_w, a->gated ? a->width_out + 256 : 256, es)) return st;
  if (int st = check_stride(a->out_stride, a->width_out, a->rows, 1, es)) return st;
  if (a->residual)
    if (int st = check_stride(a->residual_stride, a->width_out, a->rows, 1, es)) return st;
  return VECTRA_DENSE_OK;
}

void forward(const vectra_dense_args& a, Call& c) {
  if (a.rows == 0 || a.width_out == 0) return;
  const int64_t n_w = a.width_out * (1 + a.gated);
  if (const int steps = a.width_in ? c.resident_steps(a.rows, a.width_in, a.width_out, a.gated) : 0) {
    ResidentParams p{};
    p.x = a.x;
    p.ldx = a.x_stride;
    p.rows = a.rows;
    p.width = a.width_in;
    p.w = a.weight;
    p.ldw = a.weight_stride;
    p.n = static_cast<int32_t>(a.width_out);
    p.bias = a.bias;
    p.bias_dtype = a.bias_dtype;
    p.activation = a.activation;
    p.residual = a.residual;
    p.ldr = a.residual_stride;
    p.out = a.out;
    p.ldo = a.out_stride;
    c.resident(p, steps, a.gated ? kEpiGated : kEpiStore, false);
    return;
  }
  if (a.rows <= kFewRows && a.width_in) {
    if (!c.go()) return;
    FewRowsParams p{};
    p.x = a.x;
    p.ldx = a.x_stride;
    p.rows = static_cast<int32_t>(a.rows);
    p.w = a.weight;
    p.ldw = a.weight_stride;
    p.n = a.width_out;
    p.width = a.width_in;
    p.bias = a.bias;
    p.bias_dtype = a.bias_dtype;
    p.activation = a.activation;
    p.residual = a.residual;
    p.ldr = a.residual_stride;
    p.out = a.out;
    p.ldo = a.out_stride;
    const auto f = a.dtype == VECTRA_DENSE_F32 ? launch_few_rows_f32 : a.dtype == VECTRA_DENSE_F16 ? launch_few_rows_f16 : launch_few_rows_bf16;
    c.status = f(p, a.gated, c.stream);
    return;
  }
  Operand x = operand(a.x, a.x_stride, a.rows, a.width_in), w = operand(a.weight, a.weight_stride, n_w, a.width_in);
  GemmParams p{};
  p.m = a.rows;
  p.n = a.width_out;
  p.depth = a.width_in;
  p.out = a.out;
  p.ldo = a.out_stride;
  p.bias = a.bias;
  p.bias_dtype = a.bias_dtype;
  p.activation = a.activation;
  p.residual = a.residual;
  p.ldr = a.residual_stride;
  c.product(p, x, w, kLayoutForward, a.gated ? kEpiGated : kEpiStore);
}

int check_backward(const vectra_dense_grad_args* a) {
  if (!a) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  if (a->struct_size != static_cast<int64_t>(sizeof(vectra_dense_grad_args))) return VECTRA_DENSE_ERR_BAD_STRUCT;
  if (!known_dtype(a->dtype)) return VECTRA_DENSE_ERR_BAD_DTYPE;
  if ((a->bias || a->dbias) && a->bias_dtype != a->dtype && a->bias_dtype != VECTRA_DENSE_F32)
    return VECTRA_DENSE_ERR_BAD_DTYPE;
  if (!known_activation(a->activation)) return VECTRA_DENSE_ERR_BAD_ACTIVATION;
  if (a->gated != 0 && a->gated != 1) return VECTRA_DENSE_ERR_BAD_SHAPE;
  const int64_t es = element_size(a->dtype);
  if (int st = check_sizes(a->rows, a->width_in, a->width_out, a->gated)) return st;
  const int64_t n_w = a->width_out * (1 + a->gated);
  const bool any = a->rows && a->width_out;
  const bool use_x = a->gated || a->activation != VECTRA_DENSE_NONE || a->dweight;
  if (any && !a->grad) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  if (any && a->width_in) {
    if (!a->weight) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
    if (use_x && !a->x && !(a->codes && a->scales)) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  }
  if (any) {
    if (!use_x) {
    } else if (a->x) {
      if (int st = check_stride(a->x_stride, a->width_in, a->rows, 256, es)) return st;
    } else {
      if (int st = check_stride(a->codes_stride, a->width_in, a->rows, 1, 1)) return st;
      if (int st = check_stride(a->scales_stride, ceil_div(a->width_in, kBlock), a->rows, 1, 1)) return st;
    }
    if (int st = check_stride(a->weight_stride, a->width_in, n_w, a->gated ? a->width_out + 256 : 256, es)) return st;
    if (int st = check_stride(a->grad_stride, a->width_out, a->rows, 256, es)) return st;
  }
  if (a->dx && a->rows && a->width_in)
    if (int st = check_stride(a->dx_stride, a->width_in, a->rows, 1, es)) return st;
  if (a->dweight && n_w && a->width_in)
    if (int st = check_stride(a->dweight_stride, a->width_in, n_w, 1, es)) return st;
  return VECTRA_DENSE_OK;
}

void backward(const vectra_dense_grad_args& a, Call& c) {
  const int64_t n_w = a.width_out * (1 + a.gated);
  const bool slope = a.gated || a.activation != VECTRA_DENSE_NONE;
  const bool want_dx = a.dx && a.rows && a.width_in, want_dw = a.dweight && n_w && a.width_in;
  const bool want_db = a.dbias && n_w;
  if (!want_dx && !want_dw && !want_db) return;
  const bool use_x = slope || want_dw;
  const bool use_dz = want_dw || want_db;
  const bool any = a.rows && a.width_in && n_w;
  Operand x = operand(a.x, a.x_stride, a.rows, a.width_in), w = operand(a.weight, a.weight_stride, n_w, a.width_in);
  Operand dz = operand(a.grad, a.grad_stride, a.rows, n_w);
  // A layer with a slope whose weight fits LDS: dz and dx in one pass over x and grad.
  const int steps = slope && any ? c.resident_steps(a.rows, a.width_in, a.width_out, a.gated) : 0;
  const bool dx_with_dz = steps > 0 && want_dx && c.esize() == 2 && steps <= kResidentDxSteps;
  if (use_x && any && !a.x) {
    const int64_t ld = c.padded(a.width_in);
    x.p = c.scratch.take(a.rows * ld * c.esize());
    x.ld = ld;
    x.padded = true;
    if (c.go())
      c.typed([&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        dequantize<T>(a.codes, a.codes_stride, a.scales, a.scales_stride, a.rows, a.width_in, x.p, ld, ld, c);
      });
  }
  bool db_done = false;
  if (slope && a.rows && n_w && (use_dz || want_dx)) {
    const bool keep_dz = use_dz || !dx_with_dz;
    const int64_t n_pad = c.padded(n_w);
    if (keep_dz) dz = Operand{c.scratch.take(a.rows * n_pad * c.esize()), n_pad, a.rows, n_w, true};
    if (steps > 0) {
      ResidentParams p{};
      p.x = x.p;
      p.ldx = x.ld;
      p.rows = a.rows;
      p.width = a.width_in;
      p.w = a.weight;
      p.ldw = a.weight_stride;
      p.n = static_cast<int32_t>(a.width_out);
      p.bias = a.bias;
      p.bias_dtype = a.bias_dtype;
      p.activation = a.activation;
      p.grad = a.grad;
      p.ldg = a.grad_stride;
      p.out = keep_dz ? const_cast<void*>(dz.p) : nullptr;
      p.ldo = n_pad;
      p.dx = dx_with_dz ? a.dx : nullptr;
      p.lddx = a.dx_stride;
      c.resident(p, steps, a.gated ? kEpiGatedSlope : kEpiSlope, dx_with_dz);
    } else {
      GemmParams p{};
      p.m = a.rows;
      p.n = a.width_out;
      p.depth = a.width_in;
      p.out = const_cast<void*>(dz.p);
      p.ldo = n_pad;
      p.bias = a.bias;
      p.bias_dtype = a.bias_dtype;
      p.activation = a.activation;
      p.grad = a.grad;
      p.ldg = a.grad_stride;
      const bool summed = c.product(p, x, w, kLayoutForward, a.gated ? kEpiGatedSlope : kEpiSlope,
                                    want_db ? a.dbias : nullptr, a.bias_dtype);
      db_done = want_db && summed;
    }
  }
  // db, where the product that made dz has not summed it: with dW where that is
  // formed too (the sums of its first operand).
  if (want_db && !db_done && !want_dw) c.column_sums_of(dz, n_w, a.dbias, a.bias_dtype);
  if (want_dx && !dx_with_dz) {
    GemmParams p{};
    p.m = a.rows;
    p.n = a.width_in;
    p.depth = n_w;
    p.out = a.dx;
    p.ldo = a.dx_stride;
    c.product(p, dz, w, kLayoutInput, kEpiStore);
  }
  if (want_dw) {
    GemmParams p{};
    p.m = n_w;
    p.n = a.width_in;
    p.depth = a.rows;
    p.out = a.dweight;
    p.ldo = a.dweight_stride;
    c.product(p, dz, x, kLayoutWeight, kEpiStore, want_db && !db_done ? a.dbias : nullptr, a.bias_dtype);
  }
}

// Runs a plan twice where a workspace is needed: once to find its size, once
// to launch.  Launches nothing before the size is known to fit.
template <typename Args, typename F>
int run_call(const Args& a, F&& plan, void* workspace, int64_t workspace_bytes, vectra_dense_stream_t stream) {
  Call sized{a.dtype, {nullptr, 0}, false, nullptr, compute_units()};
  plan(a, sized);
  const int64_t need = std::max(sized.most, sized.scratch.used);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return VECTRA_DENSE_ERR_WORKSPACE;
  Call c{a.dtype, {static_cast<char*>(workspace), 0}, true, reinterpret_cast<hipStream_t>(stream), sized.cus};
  (void)hipGetLastError();  // an error left by other work is not this call's
  plan(a, c);
  return c.status;
}

template <typename Args, typename F>
int64_t need_of(const Args& a, F&& plan) {
  Call sized{a.dtype, {nullptr, 0}, false, nullptr, compute_units()};
  plan(a, sized);
  return std::max(sized.most, sized.scratch.used);
}

}  // namespace
}  // namespace vectra_dense

using namespace vectra_dense;

extern "C" {

int vectra_dense_forward(const vectra_dense_args* args, void* workspace, int64_t workspace_bytes,
                         vectra_dense_stream_t stream) {
  if (int st = check_forward(args)) return st;
  return run_call(*args, forward, workspace, workspace_bytes, stream);
}

int64_t vectra_dense_forward_workspace_bytes(const vectra_dense_args* args) {
  if (int st = check_forward(args)) return -st;
  return need_of(*args, forward);
}

int vectra_dense_backward(const vectra_dense_grad_args* args, void* workspace, int64_t workspace_bytes,
                          vectra_dense_stream_t stream) {
  if (int st = check_backward(args)) return st;
  return run_call(*args, backward, workspace, workspace_bytes, stream);
}

int64_t vectra_dense_backward_workspace_bytes(const vectra_dense_grad_args* args) {
  if (int st = check_backward(args)) return -st;
  return need_of(*args, backward);
}

int vectra_rows_quantize(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, void* codes,
                         int64_t codes_stride, void* scales, int64_t scales_stride, vectra_dense_stream_t stream) {
  if (!known_dtype(dtype)) return VECTRA_DENSE_ERR_BAD_DTYPE;
  if (int st = check_sizes(rows, width, 0, 0)) return st;
  if (rows == 0 || width == 0) return VECTRA_DENSE_OK;
  if (!x || !codes || !scales) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  const int64_t blocks = ceil_div(width, kBlock);
  if (int st = check_stride(x_stride, width, rows, 1, element_size(dtype))) return st;
  if (int st = check_stride(codes_stride, width, rows, 1, 1)) return st;
  if (int st = check_stride(scales_stride, blocks, rows, 1, 1)) return st;
  Call c{dtype, {nullptr, 0}, true, reinterpret_cast<hipStream_t>(stream), 0};
  (void)hipGetLastError();
  c.typed([&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    quantize<T>(x, rows, width, x_stride, codes, codes_stride, scales, scales_stride, c);
  });
  return c.status;
}

int vectra_rows_dequantize(const void* codes, int64_t codes_stride, const void* scales, int64_t scales_stride,
                           int32_t dtype, int64_t rows, int64_t width, void* out, int64_t out_stride,
                           vectra_dense_stream_t stream) {
  if (!known_dtype(dtype)) return VECTRA_DENSE_ERR_BAD_DTYPE;
  if (int st = check_sizes(rows, width, 0, 0)) return st;
  if (rows == 0 || width == 0) return VECTRA_DENSE_OK;
  if (!out || !codes || !scales) return VECTRA_DENSE_ERR_NULL_ARGUMENT;
  if (int st = check_stride(out_stride, width, rows, 1, element_size(dtype))) return st;
  if (int st = check_stride(codes_stride, width, rows, 1, 1)) return st;
  if (int st = check_stride(scales_stride, ceil_div(width, kBlock), rows, 1, 1)) return st;
  Call c{dtype, {nullptr, 0}, true, reinterpret_cast<hipStream_t>(stream), 0};
  (void)hipGetLastError();
  c.typed([&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    dequantize<T>(codes, codes_stride, scales, scales_stride, rows, width, out, out_stride, width, c);
  });
  return c.status;
}

const char* vectra_dense_status_string(int status) {
  switch (status) {
    case VECTRA_DENSE_OK: return "ok";
    case VECTRA_DENSE_ERR_NULL_ARGUMENT: return "a required pointer is NULL";
    case VECTRA_DENSE_ERR_BAD_DTYPE: return "unsupported dtype combination";
    case VECTRA_DENSE_ERR_BAD_SHAPE: return "negative or inconsistent sizes or strides";
    case VECTRA_DENSE_ERR_BAD_STRUCT: return "struct_size does not match this build of the library";
    case VECTRA_DENSE_ERR_TOO_LARGE: return "a size exceeds the kernels' index range";
    case VECTRA_DENSE_ERR_LAUNCH: return "HIP kernel launch failed";
    case VECTRA_DENSE_ERR_BAD_ACTIVATION: return "unknown activation";
    case VECTRA_DENSE_ERR_WORKSPACE: return "workspace missing, too small or not 256-byte aligned";
    default: return "unknown status";
  }
}

int vectra_dense_abi_version(void) { return (1 << 16) | 0; }

}  // extern "C"
