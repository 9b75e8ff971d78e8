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
// Staging: tiles go from global memory straight into LDS, and the fragments of one step
// of 64 ahead of the products into registers.  The 256-tile takes 128 of the contraction
// per stage, three stages of x and two of W in LDS, one barrier each; the smaller ones 64,
// four stages of both, three of them on their way or ahead, one barrier each.  Buffer
// bounds turn rows past the operand into zeros.
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

template <int kByte>
struct Byte {
  static constexpr int value = kByte;
};

// kDeep: of the contraction per stage, 64 or 128.  In LDS: four stages of 64, or three
// of x and two of W of 128.
template <int kBM_, int kBN_, int kWM_, int kWN_, int kDeep_, int kEpi_, bool kPrecise_>
struct Config8 {
  static constexpr int kBM = kBM_, kBN = kBN_, kWM = kWM_, kWN = kWN_, kEpi = kEpi_;
  static constexpr bool kPrecise = kPrecise_, kGated = kEpi == kGated8;
  static constexpr int kThreads = 64 * kWM * kWN;
  static constexpr int kTM = kBM / kWM / 32, kTN = kBN / kWN / 32;
  static constexpr int kDeep = kDeep_, kStagesA = kDeep == 64 ? 4 : 3, kStagesB = kDeep == 64 ? 4 : 2;
  using A = vectra_dense::Tile<uint8_t, false, kBM, kDeep, kThreads>;
  using B = vectra_dense::Tile<uint8_t, false, kBN, kDeep, kThreads>;
  static constexpr int kLoads = A::kSlots + B::kSlots;  // of a thread, for a stage
  static constexpr int kBandStride = kTN * 32 + 4;  // rows 16 bytes apart in the banks
  static constexpr int kBandBytes = kEpi == kPartial8 ? 0 : kWM * kWN * 32 * kBandStride * 4;
  static constexpr int kStageBytes = kStagesA * A::kBytes + kStagesB * B::kBytes;
  static constexpr int kLdsBytes = kStageBytes > kBandBytes ? kStageBytes : kBandBytes;
  static_assert(kLdsBytes <= 160 * 1024, "LDS");
};

// Waits until at most `kLeft` of this wave's vector memory operations are on their way
// (kReads: and no LDS reads).
template <int kLeft, bool kReads = false>
__device__ __forceinline__ void wait_but() {
  static_assert(kLeft < 64);
  __builtin_amdgcn_s_waitcnt((kReads ? 0x0070 : 0x0f70) | (kLeft & 15) | (kLeft >> 4) << 14);
}

// Loads a stage of one operand into LDS, 16 bytes per lane and slot: `offset` from
// `base` (out of bounds: zeros), `at` further along the contraction.
__device__ __forceinline__ void load8_to_lds(__amdgpu_buffer_rsrc_t rsrc, lds_char* to, uint32_t offset, int at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)to, 16, offset, at, 0, 0);
}

template <typename TileT, int kThreads>
__device__ __forceinline__ void stage8(lds_char* stage, const uint8_t* base, int64_t bytes,
                                       const uint32_t (&offset)[TileT::kSlots], int at, int wave) {
#pragma unroll
  for (int s = 0; s < TileT::kSlots; ++s)
    load8_to_lds(vectra::plane_rsrc(base, static_cast<uint32_t>(least(bytes, 0x7fffffff))),
                 stage + (s * kThreads + wave * 64) * 16, offset[s], at);
}

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

  // ---- per-lane load offsets (bytes from the tile's first row; rows past the operand's
  // end out of bounds).  The contraction's offset is the loads' scalar one.
  uint32_t a_off[A::kSlots], b_off[B::kSlots];
#pragma unroll
  for (int s = 0; s < A::kSlots; ++s) {
    int row, chunk;
    A::slot(s, tid, row, chunk);
    a_off[s] = m0 + row < p.rows ? static_cast<uint32_t>(row * p.depth) + chunk * 16 : vectra_dense::kOutside;
  }
#pragma unroll
  for (int s = 0; s < B::kSlots; ++s) {
    int row, chunk;
    B::slot(s, tid, row, chunk);
    bool there;
    const int64_t w_row = weight_row(row, there);
    b_off[s] = there ? static_cast<uint32_t>((w_row - n0) * p.depth) + chunk * 16 : vectra_dense::kOutside;
  }
  const uint8_t* const a_base = p.codes + m0 * p.depth;
  const uint8_t* const b_base = p.weight + n0 * p.depth;
  const int64_t a_bytes = least(p.rows - m0, C::kBM) * p.depth;
  const int64_t b_bytes = ((C::kGated ? p.n : 0) + least(p.n - n0, kOutN)) * p.depth;
  const int last_stage = k_last * (128 / C::kDeep) - 1;
  // (Past the last stage: that one again, into a buffer that nobody reads.)
  const auto load_a = [&](int stage, int buf) {
    stage8<A, C::kThreads>(smem + buf * A::kBytes, a_base, a_bytes, a_off, min(stage, last_stage) * C::kDeep, wave);
  };
  const auto load_b = [&](int stage, int buf) {
    stage8<B, C::kThreads>(smem + C::kStagesA * A::kBytes + buf * B::kBytes, b_base, b_bytes, b_off,
                           min(stage, last_stage) * C::kDeep, wave);
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
  } now, next;
  // (Loads that the waits below count: relaxed atomics of this wave's scope, which are
  // ordinary loads to the memory, but which the compiler may not move past another
  // access, join or leave out.)
  const auto load_word = [](const uint32_t* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT); };
  const auto load_scales = [&](Scales& s, int word) {
    const int at = min(word, words - 1);
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) s.a[t] = load_word(a_scales + a_scale[t] + at);
#pragma unroll
    for (int t = 0; t < C::kTN; ++t) s.b[t] = load_word(b_scales + b_scale[t] + at);
  };

  f32x16 acc[C::kTN][C::kTM];
#pragma unroll
  for (int u = 0; u < C::kTN; ++u)
#pragma unroll
    for (int t = 0; t < C::kTM; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][t][e] = 0.f;

  // LDS holds the stages of x, then those of W.  A lane's address within one, but for
  // the row block and the step: a fragment's chunks are three bits of it at most, so
  // they are this with constants XORed in.  (Opaque in each step: hoisted out of the
  // loop, every step's addresses would be registers of their own, and the large tile
  // has none left.)
  const uint32_t in_block = i * C::kDeep + ((half ^ A::swizzle(i)) * 16);
  const uint32_t a_at = wm * C::kTM * 32 * C::kDeep + in_block;
  const uint32_t b_at = C::kStagesA * A::kBytes + wn * C::kTN * 32 * C::kDeep + in_block;
  const auto read_one = [&](uint32_t at, int offset, int step) {
    Frag8 f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      f.w[j] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(smem + (at ^ ((step * 4 + 2 * j) * 16)) + offset);
    return f;
  };

  // The products of a step, and the fragments of the step after it: W's first, x's
  // each into the registers of the one just used, so that little more than one step's
  // are held at a time.
  Frag8 fa[C::kTM], fb[C::kTN];
  const auto read_b = [&](Frag8(&f)[C::kTN], uint32_t at, int buf, int step) {
#pragma unroll
    for (int u = 0; u < C::kTN; ++u) f[u] = read_one(at, buf * B::kBytes + u * 32 * C::kDeep, step);
  };
  const auto read_a = [&](int t, uint32_t at, int step) { return read_one(at, t * 32 * C::kDeep, step); };
  const auto multiply = [&](auto which, int next_a, int next_b, int next_step) {
    constexpr int kByte = decltype(which)::value;
    uint32_t from_a = a_at + next_a * A::kBytes, from_b = b_at;
    if constexpr (C::kDeep == 128) asm volatile("" : "+v"(from_a), "+v"(from_b));
    Frag8 fb_next[C::kTN];
    read_b(fb_next, from_b, next_b, next_step);
    if constexpr (C::kPrecise) {
      float sb[C::kTN];
#pragma unroll
      for (int u = 0; u < C::kTN; ++u) sb[u] = scale_of(now.b[u] >> (8 * kByte) & 255);
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        const float sa = scale_of(now.a[t] >> (8 * kByte) & 255);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8 xa = decode(fa[t].w[j / 2][j % 2 * 2], fa[t].w[j / 2][j % 2 * 2 + 1], sa);
#pragma unroll
          for (int u = 0; u < C::kTN; ++u)
            acc[u][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                decode(fb[u].w[j / 2][j % 2 * 2], fb[u].w[j / 2][j % 2 * 2 + 1], sb[u]), xa, acc[u][t], 0, 0, 0);
        }
        fa[t] = read_a(t, from_a, next_step);
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
          acc[u][t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes(fb[u]), codes(fa[t]), acc[u][t], 0, 0, kByte,
                                                                      static_cast<int>(now.b[u]), kByte,
                                                                      static_cast<int>(now.a[t]));
        fa[t] = read_a(t, from_a, next_step);
      }
      // (The order above, which the scheduler would otherwise undo: LDS reads first.)
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * C::kTN, 0);
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x008, C::kTN, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, (C::kLoads + C::kTM - 1) / C::kTM, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < C::kTN; ++u) fb[u] = fb_next[u];
  };

  // The fragments of one step of 64 ahead in registers; a word holds a row's scales of
  // four blocks, the byte is the matrix instruction's own selection, so four blocks are
  // a turn, and the next word, loaded in the first, has the others' time to arrive.
  const auto turns = [&](auto&& block) {
    for (int kt = k_first;; kt += 4) {
      block(kt, Byte<0>{});
      if (kt + 1 >= k_last) break;
      block(kt + 1, Byte<1>{});
      if (kt + 2 >= k_last) break;
      block(kt + 2, Byte<2>{});
      if (kt + 3 >= k_last) break;
      block(kt + 3, Byte<3>{});
      if (kt + 4 >= k_last) break;
    }
  };
  const auto read_first = [&] {
    read_b(fb, b_at, 0, 0);
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) fa[t] = read_a(t, a_at, 0);
  };
  if (k_first < k_last) {
    load_scales(now, k_first / 4);
    if constexpr (C::kDeep == 128) {
      // A stage is a block, two steps.  While the products of step 0 run, step 1 is
      // read; then one barrier, after which nobody reads this stage any more and the
      // next one is there; while the products of step 1 run, step 0 of the next is
      // read, and W's block after next and x's third from here are loaded over this
      // one: as much on its way as LDS holds.
      load_b(k_first, 0);
      load_a(k_first, 0);
      __builtin_amdgcn_sched_barrier(0);
      load_a(k_first + 1, 1);
      load_b(k_first + 1, 1);
      __builtin_amdgcn_sched_barrier(0);
      load_a(k_first + 2, 2);
      __builtin_amdgcn_sched_barrier(0);
      wait_but<2 * A::kSlots + B::kSlots>();
      __builtin_amdgcn_s_barrier();
      read_first();
      int buf_a = 0;
      turns([&](int kt, auto which) {
        constexpr int kByte = decltype(which)::value, kBuf = kByte & 1;
        multiply(which, buf_a, kBuf, 1);
        // (x's block after next stays on its way; a word of scales issued with it is
        // waited for.)
        wait_but<A::kSlots, true>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kByte == 0) load_scales(next, kt / 4 + 1);
        load_b(kt + 2, kBuf);
        __builtin_amdgcn_sched_barrier(0x0007);  // (arithmetic may pass: the loads' order is what the wait counts on)
        load_a(kt + 3, buf_a);
        buf_a = buf_a == 2 ? 0 : buf_a + 1;
        multiply(which, buf_a, kBuf ^ 1, 0);
        if constexpr (kByte == 3) now = next;
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      constexpr int kStages = C::kStagesA;
      // kStages steps in LDS or on their way there.  A step: wait for the next one's
      // loads, of this wave, then at the barrier of all; nobody reads the stage before
      // this one any more, and the step kStages - 1 ahead is loaded over it; the next
      // step is read while this one is multiplied.
#pragma unroll
      for (int s = 0; s < kStages - 1; ++s) {
        load_a(2 * k_first + s, s);
        load_b(2 * k_first + s, s);
      }
      wait_but<(kStages - 2) * C::kLoads>();
      __builtin_amdgcn_s_barrier();
      read_first();
      const auto step = [&](int at, auto which) {
        constexpr int kStep = decltype(which)::value, kAhead = kStages - 1;
        // Younger than the next step's loads: those of the steps behind it, and the
        // scales' while they are (not counted where both were issued in one step, in an
        // order that is the compiler's).
        constexpr int kScales = kStep >= 1 && kStep < kAhead - 1 ? C::kTM + C::kTN : 0;
        wait_but<(kStages - 3) * C::kLoads + kScales>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        load_a(at + kAhead, (kStep + kAhead) % kStages);
        load_b(at + kAhead, (kStep + kAhead) % kStages);
        if constexpr (kStep == 0) load_scales(next, at / 8 + 1);
        multiply(Byte<kStep / 2>{}, (kStep + 1) % kStages, (kStep + 1) % kStages, 0);
        if constexpr (kStep == 7) now = next;
        __builtin_amdgcn_sched_barrier(0);
      };
      turns([&](int kt, auto which) {
        constexpr int kByte = decltype(which)::value;
        step(2 * kt, Byte<2 * kByte>{});
        step(2 * kt + 1, Byte<2 * kByte + 1>{});
      });
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
      if constexpr (!kPrecise) return launch_one8<T, Config8<256, 256, 2, 4, 128, kEpi, false>>(p, parts, stream);
      return VECTRA_BLOCK_ERR_LAUNCH;
    case kMedium8:
      return launch_one8<T, Config8<128, 128, 2, 2, 64, kEpi, kPrecise>>(p, parts, stream);
    default:
      // (A wave of 32 columns holds no gate and up half: two waves side by side in m.)
      if constexpr (kEpi == kGated8) return launch_one8<T, Config8<64, 64, 2, 1, 64, kEpi, kPrecise>>(p, parts, stream);
      return launch_one8<T, Config8<64, 64, 2, 2, 64, kEpi, kPrecise>>(p, parts, stream);
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
