// Tiled products in 8 bits on gfx950 matrix cores, with the layers' epilogues: the
// kernel template, instantiated per type of result in product8_<type>.hip.
//
//   D[m, n] = sum_k x^(m, k) W(n, k)
//
// Both operands are e4m3 codes with the contraction contiguous, in whole blocks of
// 128.  A workgroup of kWM x kWN waves computes a kBM x kBN tile of D, a wave kTM x
// kTN tiles of 32 x 32.  W is the matrix instruction's first operand and x its second,
// so a lane holds runs of four consecutive n of one m.
//
// 16-bit results run on the 8-bit matrix cores (v_mfma_scale_f32_32x32x64_f8f6f4,
// twice the bf16 rate), which take each lane's power of two with its 32 codes: the
// blocks' scales cost no vector work but a shift.  A row's scales of four blocks are
// loaded as one word, four tiles ahead.  These cores add the 16 products of a group
// after dropping the bits below 2^-13 of the largest one's power of two: beside it,
// not relative to the sum.  Measured over 4096 elements of normal operands that is
// 1.6e-5 of the result, a hundredth of bf16's half step and a fifteenth of fp16's.
//
// fp32 results (kPrecise) take no part in that: the codes are turned into bf16
// with their powers of two, which is exact, on their way from LDS, and run on the
// bf16 cores: exact products, fp32 sums.
//
// Staging as in the dense products (dense/gemm_impl.h): tiles go from global memory
// straight into LDS one ahead of the one being multiplied, two of them there, the
// fragments of one step of 64 ahead in registers, one barrier per tile of 128.
// Buffer bounds turn rows past the operand into zeros.
#pragma once

#include "../dense/gemm_impl.h"
#include "few8_impl.h"

namespace vectra_block {

using vectra_dense::lds_char;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// A lane's 32 codes of a row: chunks (16 bytes) 2 j + half, j = 0, 1, of a step's four.
struct Frag8 {
  u32x4 w[2];
};

template <int kBM_, int kBN_, int kWM_, int kWN_, int kEpi_, bool kPrecise_>
struct Config8 {
  static constexpr int kBM = kBM_, kBN = kBN_, kWM = kWM_, kWN = kWN_, kEpi = kEpi_;
  static constexpr bool kPrecise = kPrecise_, kGated = kEpi == kGated8;
  static constexpr int kThreads = 64 * kWM * kWN;
  static constexpr int kTM = kBM / kWM / 32, kTN = kBN / kWN / 32;
  using A = vectra_dense::Tile<uint8_t, false, kBM, 128, kThreads>;
  using B = vectra_dense::Tile<uint8_t, false, kBN, 128, kThreads>;
  static constexpr int kStageBytes = A::kBytes + B::kBytes;
  static constexpr int kBandStride = kTN * 32 + 4;  // rows 16 bytes apart in the banks
  static constexpr int kBandBytes = kEpi == kPartial8 ? 0 : kWM * kWN * 32 * kBandStride * 4;
  static constexpr int kLdsBytes = 2 * kStageBytes > kBandBytes ? 2 * kStageBytes : kBandBytes;
  static_assert(kLdsBytes <= 160 * 1024, "LDS");
};

template <typename T, typename C>
__global__ __launch_bounds__(C::kThreads, 2) void product8_kernel(const Product8Params p) {
  __shared__ __attribute__((aligned(256))) char smem_generic[C::kLdsBytes];
  lds_char* const smem = (lds_char*)smem_generic;
  using A = typename C::A;
  using B = typename C::B;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, i = lane & 31;
  const int wm = wave / C::kWN, wn = wave % C::kWN;

  int part, tm, tn;
  vectra_dense::tile_of(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, part, tm, tn);
  const int64_t m0 = static_cast<int64_t>(tm) * C::kBM;
  constexpr int kOutN = C::kGated ? C::kBN / 2 : C::kBN;  // outputs per tile
  const int64_t n0 = static_cast<int64_t>(tn) * kOutN;
  const int k_first = part * p.k_tiles_per_part;
  const int k_last = min(k_first + p.k_tiles_per_part, p.k_tiles);

  // The weight's row behind row `at` of the tile.  Gated: a wave's columns are kTN / 2
  // tiles of gate rows, then the up rows of the same outputs.
  const auto weight_row = [&](int at, bool& there) -> int64_t {
    if constexpr (C::kGated) {
      constexpr int kSeg = C::kTN * 32, kHalf = kSeg / 2;
      const int in = at % kSeg;
      const int64_t out = n0 + at / kSeg * kHalf + in % kHalf;
      there = out < p.n;
      return out + (in >= kHalf ? p.n : 0);
    } else {
      there = n0 + at < p.n;
      return n0 + at;
    }
  };

  // ---- per-lane load offsets (bytes from the tile's base)
  const uint8_t* a = p.codes + m0 * p.depth + static_cast<int64_t>(k_first) * 128;
  const uint8_t* b = p.weight + n0 * p.depth + static_cast<int64_t>(k_first) * 128;
  int64_t a_bytes = least(p.rows - m0, C::kBM) * p.depth - static_cast<int64_t>(k_first) * 128;
  int64_t b_bytes = ((C::kGated ? p.n : 0) + least(p.n - n0, kOutN)) * p.depth - static_cast<int64_t>(k_first) * 128;
  uint32_t a_off[A::kSlots], b_off[B::kSlots], a_chunk[A::kSlots], b_chunk[B::kSlots];
#pragma unroll
  for (int s = 0; s < A::kSlots; ++s) {
    int row, chunk;
    A::slot(s, tid, row, chunk);
    a_off[s] = m0 + row < p.rows ? static_cast<uint32_t>(row * p.depth) + chunk * 16 : vectra_dense::kOutside;
    a_chunk[s] = 0;  // (whole blocks: every chunk of a tile exists)
  }
#pragma unroll
  for (int s = 0; s < B::kSlots; ++s) {
    int row, chunk;
    B::slot(s, tid, row, chunk);
    bool there;
    const int64_t w_row = weight_row(row, there);
    b_off[s] = there ? static_cast<uint32_t>((w_row - n0) * p.depth) + chunk * 16 : vectra_dense::kOutside;
    b_chunk[s] = 0;
  }
  const auto load = [&](int kt, int buf) {
    lds_char* const at = smem + buf * C::kStageBytes;
    const bool there = kt < k_last;
    vectra_dense::stage<A, uint8_t, false, C::kThreads, false>(at, a, a_off, there ? least(a_bytes, 0x7fffffff) : 0, 1, a_chunk, wave);
    vectra_dense::stage<B, uint8_t, false, C::kThreads, false>(at + A::kBytes, b, b_off, there ? least(b_bytes, 0x7fffffff) : 0, 1,
                                                               b_chunk, wave);
    a += 128;
    b += 128;
    a_bytes -= 128;
    b_bytes -= 128;
  };

  // ---- the scales of this lane's rows (clamped: those past the end are not stored),
  // as offsets in words from the tile's first
  const uint32_t* const a_scales = reinterpret_cast<const uint32_t*>(p.scales + m0 * p.scale_stride);
  const uint32_t* const b_scales = reinterpret_cast<const uint32_t*>(p.weight_scales);
  const int words = static_cast<int>(p.scale_stride / 4);
  uint32_t a_scale[C::kTM], b_scale[C::kTN];
#pragma unroll
  for (int t = 0; t < C::kTM; ++t)
    a_scale[t] = static_cast<uint32_t>(least((wm * C::kTM + t) * 32 + i, p.rows - 1 - m0)) * words;
#pragma unroll
  for (int t = 0; t < C::kTN; ++t) {
    bool there;
    const int64_t row = weight_row((wn * C::kTN + t) * 32 + i, there);
    b_scale[t] = static_cast<uint32_t>(there ? row / 128 : 0) * words;
  }
  struct Scales {
    uint32_t a[C::kTM], b[C::kTN];
  } now;
  const auto load_scales = [&](Scales& s, int word) {
    const int at = min(word, words - 1);
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) s.a[t] = a_scales[a_scale[t] + at];
#pragma unroll
    for (int t = 0; t < C::kTN; ++t) s.b[t] = b_scales[b_scale[t] + at];
  };

  f32x16 acc[C::kTN][C::kTM];
#pragma unroll
  for (int u = 0; u < C::kTN; ++u)
#pragma unroll
    for (int t = 0; t < C::kTM; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][t][e] = 0.f;

  const auto read_one = [&](const lds_char* tile, int row0, int step) {
    Frag8 f;
    const int row = row0 + i;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      f.w[j] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
          tile + row * 128 + (((step * 4 + 2 * j + half) ^ A::swizzle(i)) * 16));
    return f;
  };
  // The products of a step, and the fragments of the step after it: W's first, x's
  // each into the registers of the one just used, so that little more than one step's
  // are held at a time.
  Frag8 fa[C::kTM], fb[C::kTN];
  const auto read_b = [&](Frag8(&f)[C::kTN], int buf, int step) {
    const lds_char* const tb = smem + buf * C::kStageBytes + A::kBytes;
#pragma unroll
    for (int u = 0; u < C::kTN; ++u) f[u] = read_one(tb, (wn * C::kTN + u) * 32, step);
  };
  const auto read_a = [&](int t, int buf, int step) {
    return read_one(smem + buf * C::kStageBytes, (wm * C::kTM + t) * 32, step);
  };
  const auto step = [&](int shift, int buf, int next_step) {
    Frag8 fb_next[C::kTN];
    read_b(fb_next, buf, next_step);
    if constexpr (C::kPrecise) {
      float sb[C::kTN];
#pragma unroll
      for (int u = 0; u < C::kTN; ++u) sb[u] = scale_of(now.b[u] >> shift & 255);
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        const float sa = scale_of(now.a[t] >> shift & 255);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8 xa = decode(fa[t].w[j / 2][j % 2 * 2], fa[t].w[j / 2][j % 2 * 2 + 1], sa);
#pragma unroll
          for (int u = 0; u < C::kTN; ++u)
            acc[u][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                decode(fb[u].w[j / 2][j % 2 * 2], fb[u].w[j / 2][j % 2 * 2 + 1], sb[u]), xa, acc[u][t], 0, 0, 0);
        }
        fa[t] = read_a(t, buf, next_step);
      }
    } else {
      const auto codes = [](const Frag8& f) {
        return i32x8{static_cast<int>(f.w[0][0]), static_cast<int>(f.w[0][1]), static_cast<int>(f.w[0][2]),
                     static_cast<int>(f.w[0][3]), static_cast<int>(f.w[1][0]), static_cast<int>(f.w[1][1]),
                     static_cast<int>(f.w[1][2]), static_cast<int>(f.w[1][3])};
      };
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
#pragma unroll
        for (int u = 0; u < C::kTN; ++u)
          acc[u][t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes(fb[u]), codes(fa[t]), acc[u][t], 0, 0, 0,
                                                                      static_cast<int>(now.b[u] >> shift), 0,
                                                                      static_cast<int>(now.a[t] >> shift));
        fa[t] = read_a(t, buf, next_step);
      }
      // (The order above, which the scheduler would otherwise undo: LDS reads first.)
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * C::kTN, 0);
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x008, C::kTN, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, (A::kSlots + B::kSlots + C::kTM - 1) / C::kTM, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < C::kTN; ++u) fb[u] = fb_next[u];
  };

  // Two tiles in LDS, two steps per tile, the fragments of one step ahead.  While the
  // products of step 0 run, step 1 is read; then one barrier, after which nobody reads
  // this tile any more and the next one is there; while the products of step 1 run, the
  // tile after next is loaded over this one and step 0 of the next is read.  Loads past
  // the last tile go out of bounds (zeros, never multiplied).
  if (k_first < k_last) {
    load_scales(now, k_first / 4);
    load(k_first, 0);
    vectra_dense::wait_loads();
    __builtin_amdgcn_s_barrier();
    load(k_first + 1, 1);
    read_b(fb, 0, 0);
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) fa[t] = read_a(t, 0, 0);
    for (int kt = k_first; kt < k_last; ++kt) {
      const int buf = (kt - k_first) & 1, shift = (kt & 3) * 8;
      Scales next;  // (each tile's own load of the word: a branch every fourth would part the products from their reads)
      load_scales(next, (kt + 1) / 4);
      step(shift, buf, 1);
      vectra_dense::wait_all();
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      load(kt + 2, buf);
      step(shift, buf ^ 1, 0);
      now = next;
      __builtin_amdgcn_sched_barrier(0);
    }
    vectra_dense::wait_all();  // nothing is on its way into LDS when it is used again
  }

  // ---- epilogue.  A lane holds, of each tile, m = i and n = 8 q + 4 half + 0 .. 3 for
  // q = 0 .. 3.
  const auto quad = [&](const f32x16& v, int q) { return f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]}; };
  if constexpr (C::kEpi == kPartial8) {
    // (out_stride is a multiple of 4 and at least n rounded up to it.)
    float* const out = static_cast<float*>(p.out) + static_cast<int64_t>(part) * p.rows * p.out_stride;
#pragma unroll
    for (int u = 0; u < C::kTN; ++u)
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        const int64_t m = m0 + (wm * C::kTM + t) * 32 + i;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t n = n0 + (wn * C::kTN + u) * 32 + 8 * q + 4 * half;
          if (m < p.rows && n < p.n) *reinterpret_cast<f32x4*>(out + m * p.out_stride + n) = quad(acc[u][t], q);
        }
      }
  } else {
    // Through LDS, 32 rows of the wave's tile at a time (each wave in its own part: no
    // barrier but the first): afterwards a lane holds eight consecutive columns, so
    // rows of the result and the residual move in whole cache lines.
    constexpr int kCols = C::kTN * 32, kStride = C::kBandStride;
    constexpr int kOut = C::kGated ? kCols / 2 : kCols, kLanes = kOut / 8, kRows = 64 / kLanes;
    __attribute__((address_space(3))) float* const band =
        (__attribute__((address_space(3))) float*)smem + wave * 32 * kStride;
    const int col = (lane % kLanes) * 8;
    const int64_t n = n0 + wn * kOut + col;
    const int left = static_cast<int>(most(least(p.n - n, 8), 0));
    f32x4 bias[2] = {}, bias_up[2] = {};
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) {
          bias[e / 4][e % 4] = vectra_dense::load_bias(p.bias, n + e, p.bias_dtype);
          if constexpr (C::kGated) bias_up[e / 4][e % 4] = vectra_dense::load_bias(p.bias, p.n + n + e, p.bias_dtype);
        }
    }
    __syncthreads();  // all waves are done with the tiles
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) {
      const int64_t m_band = m0 + (wm * C::kTM + t) * 32 + lane / kLanes;
#pragma unroll
      for (int u = 0; u < C::kTN; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(band + i * kStride + u * 32 + 8 * q + 4 * half) =
              quad(acc[u][t], q);
      vectra_dense::with_activation(p.activation, [&](auto act) {
        constexpr int kAct = decltype(act)::value;
#pragma unroll 2
        for (int r = 0; r < 32; r += kRows) {
          const int64_t m = m_band + r;
          const __attribute__((address_space(3))) f32x4* const from =
              (const __attribute__((address_space(3))) f32x4*)(band + (r + lane / kLanes) * kStride + col);
          f32x4 z[2] = {from[0] + bias[0], from[1] + bias[1]}, up[2];
          if constexpr (C::kGated) {
            up[0] = from[kOut / 4] + bias_up[0];
            up[1] = from[kOut / 4 + 1] + bias_up[1];
          }
          if (m >= p.rows || left <= 0) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            z[e / 4][e % 4] = vectra_dense::act_value<T>(z[e / 4][e % 4], kAct);
            if constexpr (C::kGated) z[e / 4][e % 4] *= up[e / 4][e % 4];
          }
          if constexpr (!C::kGated) {
            if (p.residual) {
              f32x4 near[2];
              vectra_dense::load8(static_cast<const T*>(p.residual) + m * p.residual_stride + n, left, near[0], near[1]);
              z[0] += near[0];
              z[1] += near[1];
            }
          }
          store8(static_cast<T*>(p.out) + m * p.out_stride + n, z[0], z[1], left);
        }
      });
    }
  }
}

template <typename T, typename C>
int launch_one8(const Product8Params& p, int parts, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(p.tiles_m) * static_cast<uint32_t>(p.tiles_n) * static_cast<uint32_t>(parts);
  product8_kernel<T, C><<<grid, C::kThreads, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? VECTRA_BLOCK_OK : VECTRA_BLOCK_ERR_LAUNCH;
}

template <typename T, int kEpi>
int launch_tile8(const Product8Params& p, int tile, int parts, hipStream_t stream) {
  constexpr bool kPrecise = sizeof(T) == 4;
  switch (tile) {
    case kLarge8:
      // (fp32 does not choose it: the decoded operands would not fit its registers.)
      if constexpr (!kPrecise) return launch_one8<T, Config8<256, 256, 2, 4, kEpi, false>>(p, parts, stream);
      return VECTRA_BLOCK_ERR_LAUNCH;
    case kMedium8:
      return launch_one8<T, Config8<128, 128, 2, 2, kEpi, kPrecise>>(p, parts, stream);
    default:
      // (A wave of 32 columns holds no gate and up half: two waves side by side in m.)
      if constexpr (kEpi == kGated8) return launch_one8<T, Config8<64, 64, 2, 1, kEpi, kPrecise>>(p, parts, stream);
      return launch_one8<T, Config8<64, 64, 2, 2, kEpi, kPrecise>>(p, parts, stream);
  }
}

template <typename T>
int launch_product8(const Product8Params& p, int tile, int epilogue, int parts, hipStream_t stream) {
  switch (epilogue) {
    case kStore8: return launch_tile8<T, kStore8>(p, tile, parts, stream);
    case kGated8: return launch_tile8<T, kGated8>(p, tile, parts, stream);
    default: return launch_tile8<T, kPartial8>(p, tile, parts, stream);
  }
}

}  // namespace vectra_block
