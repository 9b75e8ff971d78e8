// Tiled matrix products on gfx950 matrix cores, with the operators' epilogues:
// the kernel template, instantiated per element type in gemm_<type>.hip.
//
//   D[m, n] = sum_c A(m, c) B(n, c)
//
// A is the row operand and B the column operand.  Each is stored either with
// the contraction c contiguous ("deep" rows: element (m, c) at m ld + c) or
// with it strided ("wide" rows: element (m, c) at c ld + m), which covers
//   forward  x W^T     both deep
//   dx       dz W      A deep, B wide
//   dW       dz^T x    both wide
//
// A workgroup of kWM x kWN waves computes a kBM x kBN tile of D, a wave
// kTM x kTN tiles of 16 x 16.  B is the matrix instruction's first operand and
// A its second, so a lane holds four consecutive n of one m: rows of D are
// stored in 8- or 16-byte pieces.
//
// Staging: the tiles go from global memory straight into LDS in 16-byte chunks
// (buffer loads with the LDS bit: no registers, no LDS write instructions),
// one tile ahead of the one being multiplied.  Such a load writes LDS in lane
// order, so the swizzle that keeps LDS reads free of bank conflicts is applied
// to the global address each lane loads: LDS chunk p of a row holds the row's
// chunk p ^ f(row).  Buffer bounds turn rows past the operand into zeros;
// chunks past the contraction's end are sent out of bounds on the last tile.
// This wants operands with 16-byte aligned rows of whole chunks.  Others are
// copied first, zero padded, or, on the tiles of 128 and 64 rows and where the
// copy would cost more, pass through registers (kAny): full chunks as unaligned
// 16-byte loads, a row's last partial chunk element by element.
//
// Measured, 8192 x 4096 -> 4096 bf16, four sets of operands, in turn with the
// library's products: forward 215 us against 179 (1.28 and 1.53 PFLOP/s), dx 221
// against 208 (1.25 and 1.32), dW 221 against 243 (1.25 and 1.13).  The matrix
// cores are busy 61 to 62% of the launch: what a tile of 256 x 256 leaves idle is
// its first loads and its epilogue, with one workgroup per CU, and the clock
// falls under full load.
//
// LDS reads: deep 16-bit and 32-bit operands read 16 bytes per lane.  Wide
// 16-bit operands are read with the transposing LDS read (rbf_mfma_ops.h
// describes its lane mapping), wide fp32 operands element by element.  fp32
// products use a permuted contraction (lane group g takes elements 4g .. 4g+3
// of 16), the same for both operands.
#pragma once

#include "dense_common.h"
#include "dense_kernels.h"
#include "row_chunk.h"

namespace vectra_dense {

typedef short lds_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

template <bool kFlag>
struct Flag {
  static constexpr bool value = kFlag;
};

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a.w), __builtin_bit_cast(V, b.w), c, 0, 0, 0);
  }
  // s + the fragment's elements, in fp32: one v_dot2 per pair.  The ones come
  // from a scalar register: as an inline constant the compiler encodes a bf16
  // pair as the 32-bit constant of one of its halves.
  static __device__ __forceinline__ float sum(Frag a, float s) {
    typedef __bf16 V2 __attribute__((ext_vector_type(2)));
    uint32_t ones;
    asm("s_mov_b32 %0, 0x3f803f80" : "=s"(ones));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = a.w[j];  // (a bit cast of the element itself takes element 0)
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(V2, pair), __builtin_bit_cast(V2, ones), s, false);
    }
    return s;
  }
};
template <>
struct Mma<_Float16> {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a.w), __builtin_bit_cast(V, b.w), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum(Frag a, float s) {
    typedef _Float16 V2 __attribute__((ext_vector_type(2)));
    const V2 ones = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = a.w[j];
      s = __builtin_amdgcn_fdot2(__builtin_bit_cast(V2, pair), ones, s, false);
    }
    return s;
  }
};
template <>
struct Mma<float> {
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w[j]), __uint_as_float(b.w[j]), c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float sum(Frag a, float s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s += __uint_as_float(a.w[j]);
    return s;
  }
};

// One operand's tile in LDS: kRows rows of the output dimension, kDeep of the
// contraction.
template <typename T, bool kWide, int kRows, int kDeep, int kThreads>
struct Tile {
  static constexpr int kPer = 16 / sizeof(T);                       // elements per chunk
  static constexpr int kLdsRows = kWide ? kDeep : kRows;            // rows as stored
  static constexpr int kChunks = (kWide ? kRows : kDeep) / kPer;    // chunks per stored row
  static constexpr int kRowBytes = kChunks * 16;
  static constexpr int kBytes = kLdsRows * kRowBytes;
  static constexpr int kSlots = kLdsRows * kChunks / kThreads;      // loads per thread
  static constexpr int kStep = 4 * kPer;                            // contraction per fragment
  static constexpr int kReads = !kWide ? 1 : sizeof(T) == 2 ? 2 : 4;  // LDS reads per fragment
  static_assert(kSlots * kThreads == kLdsRows * kChunks, "whole loads");
  static_assert(kWide || kChunks == 8 || kChunks == 4, "64- or 128-byte deep rows");

  // The chunk XOR of a stored row.
  //  deep, 128-byte rows: 16 lanes read one chunk of 16 consecutive rows; with
  //    64 banks (256 bytes) two rows share a bank line, so rows r and r + 1
  //    differ already and (r >> 1) & 7 separates the pairs.
  //  deep, 64-byte rows: four rows share a line; (r >> 2) & 3 likewise.
  //  wide, 16-bit: a transposing read takes 32-byte pieces of rows {0..3} and
  //    {8..11} (then {4..7}, {12..15}) at once: piece index ^ f, f from row
  //    bits 0, 1 and 3 (rows of 128 or 384 bytes hold bit 0 by their address).
  //  wide, fp32: 64-byte pieces of the rows 4g + j, g = 0..3: piece ^ g.
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!kWide) {
      return kChunks == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
    } else if constexpr (sizeof(T) == 2) {
      if constexpr (kRowBytes % 256 == 0) return ((row & 3) | ((row >> 1) & 4)) << 1;
      return (((row >> 1) & 1) | ((row >> 2) & 2)) << 1;
    } else {
      return kRowBytes >= 256 ? ((row >> 2) & 3) << 2 : ((row >> 3) & 1) << 2;
    }
  }

  // Slot s of a thread: the stored row and the row's chunk that it loads.
  static __device__ __forceinline__ void slot(int s, int tid, int& row, int& chunk) {
    const int at = s * kThreads + tid;
    row = at / kChunks;
    chunk = (at % kChunks) ^ swizzle(row);
  }

  // The fragment of 16 rows from `row0` (a multiple of 16) of contraction step
  // `step`, for lane group g, lane i of it.
  static __device__ __forceinline__ Frag read(const lds_char* tile, int row0, int step, int g, int i) {
    Frag f;
    if constexpr (!kWide) {
      const int row = row0 + i;
      f.w = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
          tile + row * kRowBytes + (((step * 4 + g) ^ swizzle(i)) * 16));
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = step * 32 + 8 * g + 4 * h + i / 4;
        const int chunk = (row0 / 8 + (i % 4) / 2) ^ swizzle(8 * g + i / 4);
        const lds_v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) lds_v4s*)(const_cast<lds_char*>(tile) + row * kRowBytes + chunk * 16 +
                                                         (i & 1) * 8));
        const uint2 u = __builtin_bit_cast(uint2, v);
        f.w[2 * h] = u.x;
        f.w[2 * h + 1] = u.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = step * 16 + 4 * g + j;
        const int chunk = (row0 / 4 + i / 4) ^ swizzle(4 * g);
        f.w[j] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(tile + row * kRowBytes +
                                                                                      chunk * 16 + (i % 4) * 4);
      }
    }
    return f;
  }
};

// The part of the contraction and the tile that workgroup `id` computes.
// Workgroups are dealt round-robin to the 8 XCDs: each XCD takes one contiguous
// run of the tiles of all parts, part by part (the tiles of a part read the
// same operand rows), and within a part bands of kBand tile rows are walked
// column by column, so that the operands of the tiles in flight on an XCD stay
// in its L2.
constexpr int kBand = 4;
__device__ __forceinline__ void tile_of(int id, int total, int tiles_m, int tiles_n, int& part, int& tm, int& tn) {
  const int xcd = id & 7, each = total >> 3, more = total & 7;
  int t = xcd * each + (xcd < more ? xcd : more) + (id >> 3);
  part = t / (tiles_m * tiles_n);
  t -= part * tiles_m * tiles_n;
  const int per_band = kBand * tiles_n;
  const int band = t / per_band, in = t - band * per_band;
  const int height = min(kBand, tiles_m - band * kBand);
  tn = in / height;
  tm = band * kBand + (in - tn * height);
}

// Waits for this wave's loads into LDS (they count as vector memory
// operations; a workgroup barrier by itself orders LDS instructions only).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// The same, and for LDS reads.
__device__ __forceinline__ void wait_all() { __builtin_amdgcn_s_waitcnt(0x0070); }  // vmcnt(0) lgkmcnt(0)

// Asks the scheduler to spread a phase's LDS reads (and loads) over its
// products.
template <typename C, bool kLoads>
__device__ __forceinline__ void interleave() {
  constexpr int kReads = C::kTM * C::A::kReads + C::kTN * C::B::kReads;
  constexpr int kProducts = C::kTM * C::kTN * C::kMmas;
  constexpr int kLoadCount = kLoads ? C::A::kSlots + C::B::kSlots : 0;
  constexpr int kGroups = kReads;
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
    constexpr int kEach = kProducts / kGroups;
    __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);  // matrix
    if (kLoadCount > 0 && j * kLoadCount / kGroups != (j + 1) * kLoadCount / kGroups)
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // load
  }
}

constexpr uint32_t kOutside = 0x80000000u;  // past any buffer (host checks: tiles span less than 2^31 bytes)

// The 16-byte load into LDS that stage() issues.
//
// kOpaque: written as an instruction rather than through the builtin.  The
// compiler waits for every outstanding load of the builtin's kind before a
// transposing LDS read, whose address it cannot tell apart from theirs: the
// loads just issued for the tile after next would be waited for at once.
// Here the kernel's own waits (wait_loads, wait_all before the barrier that
// hands a tile over) order them.  The instruction writes no register; M0
// holds the wave's LDS address (one wait state before its use, five for a
// scalar register of the descriptor that a vector instruction wrote).
template <bool kOpaque>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, u32x4 words, lds_char* to, uint32_t at) {
  if constexpr (kOpaque) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to))), "v"(at), "s"(words)
        : "memory", "m0");
  } else {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)to, 16, at, 0, 0, 0);
  }
}

// Loads the tile of one operand.  `base`: the operand's element (first row of
// the tile, first contraction element of the tile), wave-uniform.
template <typename TileT, typename T, bool kWide, int kThreads, bool kOpaque>
__device__ __forceinline__ void stage(lds_char* tile, const T* base, const uint32_t (&offset)[TileT::kSlots],
                                      int64_t bytes, int valid_chunks, const uint32_t (&chunk)[TileT::kSlots],
                                      int wave) {
  const uint32_t size = static_cast<uint32_t>(bytes > 0 ? bytes : 0);
  __amdgpu_buffer_rsrc_t rsrc;
  u32x4 words;
  if constexpr (kOpaque) {
    const uint64_t address = reinterpret_cast<uintptr_t>(base);
    const auto uniform = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); };
    words = u32x4{uniform(static_cast<uint32_t>(address)), uniform(static_cast<uint32_t>(address >> 32)), uniform(size),
                  0x00020000u};
  } else {
    rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, static_cast<int>(size), 0x00020000);
  }
#pragma unroll
  for (int s = 0; s < TileT::kSlots; ++s) {
    uint32_t at = offset[s];
    if constexpr (!kWide) at = static_cast<int>(chunk[s]) < valid_chunks ? at : kOutside;
    load_to_lds<kOpaque>(rsrc, words, tile + (s * kThreads + wave * 64) * 16, at);
  }
}

template <typename T, int kBM_, int kBN_, int kWM_, int kWN_, bool kWideA_, bool kWideB_, int kEpi_,
          bool kPhased_ = false, bool kAny_ = false>
struct GemmConfig {
  static constexpr int kBM = kBM_, kBN = kBN_, kWM = kWM_, kWN = kWN_, kEpi = kEpi_;
  static constexpr bool kWideA = kWideA_, kWideB = kWideB_;
  static constexpr int kThreads = 64 * kWM * kWN;
  static constexpr int kDeep = 128 / sizeof(T);  // contraction per tile
  static constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16;
  static constexpr bool kGated = kEpi == kEpiGated || kEpi == kEpiGatedSlope;
  // The weight's gradient, and with it the bias's: where the registers have
  // room for it (the big tiles have none).
  static constexpr bool kSums = kWideA && kWideB && kTM * kTN <= 16 && (kPhased_ || kAny_);
  using A = Tile<T, kWideA, kBM, kDeep, kThreads>;
  using B = Tile<T, kWideB, kBN, kDeep, kThreads>;
  static constexpr int kStageBytes = A::kBytes + B::kBytes;
  static constexpr int kMmas = sizeof(T) == 2 ? 1 : 4;  // matrix instructions per fragment pair
  static constexpr bool kPhased = kPhased_;
  static constexpr bool kAny = kAny_;  // operands of any alignment, staged through registers
  static constexpr bool kOpaque = kPhased && sizeof(T) == 2 && (kWideA || kWideB);
  static constexpr int kBandTiles = kTM % 4 == 0 ? 4 : kTM % 3 == 0 ? 3 : kTM;  // 16-row tiles per epilogue band
  static constexpr int kBandStride = kTN * 16 + 4;      // rows 16 bytes apart in the banks
  static constexpr int kBandBytes = kEpi == kEpiPartial ? 0 : kWM * kWN * kBandTiles * 16 * kBandStride * 4;
  static constexpr int kLdsBytes = 2 * kStageBytes > kBandBytes ? 2 * kStageBytes : kBandBytes;
  static_assert(kLdsBytes <= 160 * 1024, "LDS");
};

template <typename T, typename C>
__global__ __launch_bounds__(C::kThreads, 2) void gemm_kernel(const GemmParams p) {
  __shared__ __attribute__((aligned(256))) char smem_generic[C::kLdsBytes];
  lds_char* const smem = (lds_char*)smem_generic;
  using A = typename C::A;
  using B = typename C::B;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int wm = wave / C::kWN, wn = wave % C::kWN;

  int part, tm, tn;
  tile_of(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, part, tm, tn);
  const int64_t m0 = static_cast<int64_t>(tm) * C::kBM;
  constexpr int kOutN = C::kGated ? C::kBN / 2 : C::kBN;  // output columns per tile
  const int64_t n0 = static_cast<int64_t>(tn) * kOutN;
  const int k_first = part * p.k_tiles_per_split;
  const int k_last = min(k_first + p.k_tiles_per_split, p.k_tiles);

  // ---- per-lane load offsets (bytes from the tile's base) and base pointers
  // (kAny: row pointers, below)
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  uint32_t a_off[A::kSlots], b_off[B::kSlots], a_chunk[A::kSlots], b_chunk[B::kSlots];
  int64_t a_bytes, b_bytes, a_step, b_step;  // bytes left in the operand from the base, bytes per contraction tile
  if constexpr (C::kWideA) {
    a += static_cast<int64_t>(k_first) * C::kDeep * p.lda + m0;
    a_bytes = ((p.depth - static_cast<int64_t>(k_first) * C::kDeep - 1) * p.lda + (p.a_width - m0)) * sizeof(T);
    a_step = static_cast<int64_t>(C::kDeep) * p.lda * sizeof(T);
  } else {
    a += m0 * p.lda + static_cast<int64_t>(k_first) * C::kDeep;
    const int64_t rows = least(p.m - m0, C::kBM);
    a_bytes = ((rows - 1) * p.lda + p.depth - static_cast<int64_t>(k_first) * C::kDeep) * sizeof(T);
    a_step = C::kDeep * sizeof(T);
  }
  if constexpr (C::kWideB) {
    b += static_cast<int64_t>(k_first) * C::kDeep * p.ldb + n0;
    b_bytes = ((p.depth_b - static_cast<int64_t>(k_first) * C::kDeep - 1) * p.ldb + (p.b_width - n0)) * sizeof(T);
    b_step = static_cast<int64_t>(C::kDeep) * p.ldb * sizeof(T);
  } else {
    b += n0 * p.ldb + static_cast<int64_t>(k_first) * C::kDeep;
    const int64_t rows = (C::kGated ? p.n : 0) + least(p.n - n0, kOutN);
    b_bytes = ((rows - 1) * p.ldb + p.depth - static_cast<int64_t>(k_first) * C::kDeep) * sizeof(T);
    b_step = C::kDeep * sizeof(T);
  }
#pragma unroll
  for (int s = 0; s < A::kSlots; ++s) {
    int row, chunk;
    A::slot(s, tid, row, chunk);
    a_off[s] = static_cast<uint32_t>(row * p.lda * sizeof(T)) + chunk * 16;
    a_chunk[s] = chunk;
    if constexpr (C::kWideA) {
      if (m0 + chunk * A::kPer >= p.a_width) a_off[s] = kOutside;
    }
  }
#pragma unroll
  for (int s = 0; s < B::kSlots; ++s) {
    int row, chunk;
    B::slot(s, tid, row, chunk);
    b_chunk[s] = chunk;
    if constexpr (C::kGated) {
      // A wave's columns are kTN / 2 tiles of gate rows, then the up rows of
      // the same outputs: one wave holds both factors of its outputs.
      constexpr int kSeg = C::kTN * 16, kHalf = kSeg / 2;
      const int seg = row / kSeg, in = row % kSeg;
      const int out = seg * kHalf + in % kHalf;
      const int64_t w_row = out + (in >= kHalf ? p.n : 0);
      b_off[s] = n0 + out < p.n ? static_cast<uint32_t>(w_row * p.ldb * sizeof(T)) + chunk * 16 : kOutside;
    } else {
      b_off[s] = static_cast<uint32_t>(row * p.ldb * sizeof(T)) + chunk * 16;
      if constexpr (C::kWideB) {
        if (n0 + chunk * B::kPer >= p.b_width) b_off[s] = kOutside;
      }
    }
  }
  // kAny: the row of each slot (deep operands: of the output dimension, fixed;
  // wide ones: of the contraction, a tile further each time), NULL past the
  // operand's rows, and the loads of one tile into registers.
  const T* a_row[C::kAny ? A::kSlots : 1];
  const T* b_row[C::kAny ? B::kSlots : 1];
  Frag a_next[C::kAny ? A::kSlots : 1], b_next[C::kAny ? B::kSlots : 1];
  if constexpr (C::kAny) {
#pragma unroll
    for (int s = 0; s < A::kSlots; ++s) {
      int row, chunk;
      A::slot(s, tid, row, chunk);
      if constexpr (C::kWideA)
        a_row[s] = static_cast<const T*>(p.a) + (static_cast<int64_t>(k_first) * C::kDeep + row) * p.lda;
      else
        a_row[s] = m0 + row < p.m ? static_cast<const T*>(p.a) + (m0 + row) * p.lda : nullptr;
    }
#pragma unroll
    for (int s = 0; s < B::kSlots; ++s) {
      int row, chunk;
      B::slot(s, tid, row, chunk);
      if constexpr (C::kWideB) {
        b_row[s] = static_cast<const T*>(p.b) + (static_cast<int64_t>(k_first) * C::kDeep + row) * p.ldb;
      } else if constexpr (C::kGated) {
        constexpr int kSeg = C::kTN * 16, kHalf = kSeg / 2;
        const int in = row % kSeg;
        const int64_t out = n0 + row / kSeg * kHalf + in % kHalf;
        b_row[s] = out < p.n ? static_cast<const T*>(p.b) + (out + (in >= kHalf ? p.n : 0)) * p.ldb : nullptr;
      } else {
        b_row[s] = n0 + row < p.n ? static_cast<const T*>(p.b) + (n0 + row) * p.ldb : nullptr;
      }
    }
  }
  const auto fetch = [&](int kt) {
    const int64_t k0 = static_cast<int64_t>(kt) * C::kDeep;
    const auto one = [&](auto wide, const T*& at, int row, int chunk, int64_t ld, int64_t first, int64_t width) {
      Frag f;
      f.w = u32x4{0, 0, 0, 0};
      if constexpr (decltype(wide)::value) {
        if (k0 + row < p.depth && first < width) f = load_row_chunk<T>(at, width, first);
        at += C::kDeep * ld;
      } else {
        const int64_t k = k0 + chunk * A::kPer;
        if (at && k < p.depth) f = load_row_chunk<T>(at, p.depth, k);
      }
      return f;
    };
#pragma unroll
    for (int s = 0; s < (C::kAny ? A::kSlots : 0); ++s) {
      int row, chunk;
      A::slot(s, tid, row, chunk);
      a_next[s] = one(Flag<C::kWideA>{}, a_row[s], row, chunk, p.lda, m0 + chunk * A::kPer, p.m);
    }
#pragma unroll
    for (int s = 0; s < (C::kAny ? B::kSlots : 0); ++s) {
      int row, chunk;
      B::slot(s, tid, row, chunk);
      b_next[s] = one(Flag<C::kWideB>{}, b_row[s], row, chunk, p.ldb, n0 + chunk * B::kPer, p.n);
    }
  };
  const auto put = [&](int buf) {
    lds_char* const at = smem + buf * C::kStageBytes;
#pragma unroll
    for (int s = 0; s < (C::kAny ? A::kSlots : 0); ++s)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(at + (s * C::kThreads + tid) * 16) = a_next[s].w;
#pragma unroll
    for (int s = 0; s < (C::kAny ? B::kSlots : 0); ++s)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(at + A::kBytes + (s * C::kThreads + tid) * 16) =
          b_next[s].w;
  };
  // (The chunks of a tile that hold contraction elements: all but on the last.)
  const int depth_chunks = static_cast<int>((p.depth + A::kPer - 1) / A::kPer);
  const auto load = [&](int kt, int buf) {
    lds_char* const at = smem + buf * C::kStageBytes;
    const int left = depth_chunks - kt * (C::kDeep / A::kPer);
    const bool there = kt < k_last;
    stage<A, T, C::kWideA, C::kThreads, C::kOpaque>(at, a, a_off, there ? least(a_bytes, 0x7fffffff) : 0, left, a_chunk, wave);
    stage<B, T, C::kWideB, C::kThreads, C::kOpaque>(at + A::kBytes, b, b_off, there ? least(b_bytes, 0x7fffffff) : 0, left, b_chunk, wave);
    a = reinterpret_cast<const T*>(reinterpret_cast<const char*>(a) + a_step);
    b = reinterpret_cast<const T*>(reinterpret_cast<const char*>(b) + b_step);
    a_bytes -= a_step;
    b_bytes -= b_step;
  };

  f32x4 acc[C::kTN][C::kTM];
#pragma unroll
  for (int tn_ = 0; tn_ < C::kTN; ++tn_)
#pragma unroll
    for (int tm_ = 0; tm_ < C::kTM; ++tm_) acc[tn_][tm_] = f32x4{0.f, 0.f, 0.f, 0.f};

  float sums[C::kSums ? C::kTM : 1] = {};

  const auto read = [&](Frag(&fa)[C::kTM], Frag(&fb)[C::kTN], int buf, int step) {
    const lds_char* const ta = smem + buf * C::kStageBytes;
    const lds_char* const tb = ta + A::kBytes;
#pragma unroll
    for (int t = 0; t < C::kTN; ++t) fb[t] = B::read(tb, (wn * C::kTN + t) * 16, step, g, i);
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) fa[t] = A::read(ta, (wm * C::kTM + t) * 16, step, g, i);
  };
  const auto multiply = [&](const Frag(&fa)[C::kTM], const Frag(&fb)[C::kTN]) {
#pragma unroll
    for (int t = 0; t < C::kTM; ++t)
#pragma unroll
      for (int u = 0; u < C::kTN; ++u) acc[u][t] = Mma<T>::run(fb[u], fa[t], acc[u][t]);
  };
  const auto add_sums = [&](const Frag(&fa)[C::kTM]) {
#pragma unroll
    for (int t = 0; t < C::kTM; ++t) sums[t] = Mma<T>::sum(fa[t], sums[t]);
  };

  if constexpr (C::kPhased) {
    // Two tiles in LDS, two steps per tile, the fragments of one step ahead in
    // registers.  While the products of step 0 run, step 1 is read; then one
    // barrier, after which nobody reads this tile any more and the next one is
    // there; while the products of step 1 run, the tile after next is loaded
    // over this one and step 0 of the next is read.  Loads past the last tile
    // go out of bounds (zeros, never multiplied).
    static_assert(C::kDeep / A::kStep == 2, "two steps per tile");
    if (k_first < k_last) {
      Frag fa0[C::kTM], fb0[C::kTN], fa1[C::kTM], fb1[C::kTN];
      load(k_first, 0);
      wait_loads();
      __builtin_amdgcn_s_barrier();
      load(k_first + 1, 1);
      read(fa0, fb0, 0, 0);
      const auto one = [&](int kt, auto with_sums) {
        const int buf = (kt - k_first) & 1;
        read(fa1, fb1, buf, 1);
        multiply(fa0, fb0);
        if constexpr (decltype(with_sums)::value) add_sums(fa0);
        interleave<C, false>();
        wait_all();
        __builtin_amdgcn_s_barrier();
        load(kt + 2, buf);
        read(fa0, fb0, buf ^ 1, 0);
        multiply(fa1, fb1);
        if constexpr (decltype(with_sums)::value) add_sums(fa1);
        interleave<C, true>();
      };
      bool with_sums = false;
      if constexpr (C::kSums) with_sums = p.sums && tn == 0;
      if constexpr (C::kSums) {
        if (with_sums)
          for (int kt = k_first; kt < k_last; ++kt) one(kt, Flag<true>{});
      }
      if (!with_sums)
        for (int kt = k_first; kt < k_last; ++kt) one(kt, Flag<false>{});
      wait_all();  // nothing is on its way into LDS when it is used again
    }
  } else if constexpr (C::kAny) {
    // Registers hold the next tile while this one is multiplied; one barrier
    // per tile (the buffer written is the one read two tiles ago).
    if (k_first < k_last) fetch(k_first);
    for (int kt = k_first; kt < k_last; ++kt) {
      const int buf = (kt - k_first) & 1;
      put(buf);
      __syncthreads();
      if (kt + 1 < k_last) fetch(kt + 1);
#pragma unroll
      for (int step = 0; step < C::kDeep / A::kStep; ++step) {
        Frag fa[C::kTM], fb[C::kTN];
        read(fa, fb, buf, step);
        multiply(fa, fb);
        if constexpr (C::kSums) {
          if (p.sums && tn == 0) add_sums(fa);
        }
      }
    }
  } else {
    static_assert(!C::kSums);
    if (k_first < k_last) load(k_first, 0);
    for (int kt = k_first; kt < k_last; ++kt) {
      const int buf = (kt - k_first) & 1;
      wait_loads();
      __syncthreads();  // tile kt is in LDS, and nobody reads the other buffer any more
      if (kt + 1 < k_last) load(kt + 1, buf ^ 1);
#pragma unroll
      for (int step = 0; step < C::kDeep / A::kStep; ++step) {
        Frag fa[C::kTM], fb[C::kTN];
        read(fa, fb, buf, step);
        multiply(fa, fb);
      }
    }
  }

  // ---- epilogue
  if constexpr (C::kEpi == kEpiPartial) {
    // A lane holds D[m, n .. n + 3] of every 16 x 16 tile; ldo is a multiple of 4.
    float* const out = static_cast<float*>(p.out) + static_cast<int64_t>(part) * p.m * p.ldo;
#pragma unroll
    for (int u = 0; u < C::kTN; ++u) {
      const int64_t n = n0 + (wn * C::kTN + u) * 16 + 4 * g;
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        const int64_t m = m0 + (wm * C::kTM + t) * 16 + i;
        if (m < p.m && n < p.n) *reinterpret_cast<f32x4*>(out + m * p.ldo + n) = acc[u][t];
      }
    }
  } else {
    // Through LDS, a band of up to 64 rows of the wave's tile at a time (each
    // wave in its own part: no barrier but the first): afterwards a lane holds
    // eight consecutive columns, so rows of the result, the residual and the
    // gradient move in whole cache lines.
    constexpr int kBandTiles = C::kBandTiles, kCols = C::kTN * 16;
    constexpr int kStride = C::kBandStride;  // floats per row
    constexpr int kOut = C::kGated ? kCols / 2 : kCols, kLanes = kOut / 8, kRows = 64 / kLanes;
    __attribute__((address_space(3))) float* const band =
        (__attribute__((address_space(3))) float*)smem + wave * kBandTiles * 16 * kStride;
    const int col = (lane % kLanes) * 8;
    const int64_t n = n0 + wn * kOut + col;
    const int left = static_cast<int>(least(p.n - n, 8));
    f32x4 bias[2] = {}, bias_up[2] = {};
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) {
          bias[e / 4][e % 4] = load_bias(p.bias, n + e, p.bias_dtype);
          if constexpr (C::kGated) bias_up[e / 4][e % 4] = load_bias(p.bias, p.n + n + e, p.bias_dtype);
        }
    }
    // Slope epilogues: the lane's columns of dz (and of the up half's), added up
    // over the wave's rows.
    constexpr bool kSlope = C::kEpi == kEpiSlope || C::kEpi == kEpiGatedSlope;
    f32x4 column[kSlope ? (C::kGated ? 4 : 2) : 1] = {};
    __syncthreads();  // all waves are done with the tiles
    // The residual's or the gradient's rows, kAhead of them on their way.
    constexpr int kTurns = kBandTiles * 16 / kRows;
    constexpr int kAhead = kTurns % 2 == 0 ? 2 : 1;
    Eight<T> ahead[kAhead];
    const T* const beside = static_cast<const T*>(kSlope ? p.grad : C::kEpi == kEpiStore ? p.residual : nullptr);
    const int64_t ld_beside = kSlope ? p.ldg : p.ldr;
    const auto fetch_beside = [&](int64_t m, int slot) {
      if (beside && m < p.m && left > 0) ahead[slot] = load_eight<T>(beside + m * ld_beside, p.n, n);
    };
#pragma unroll
    for (int first = 0; first < C::kTM; first += kBandTiles) {
      const int64_t m_band = m0 + (wm * C::kTM + first) * 16 + lane / kLanes;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) fetch_beside(m_band + j * kRows, j);
#pragma unroll
      for (int t = 0; t < kBandTiles; ++t)
#pragma unroll
        for (int u = 0; u < C::kTN; ++u)
          *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(band + (t * 16 + i) * kStride + u * 16 + 4 * g) =
              acc[u][first + t];
      with_activation(p.activation, [&](auto act) {
        constexpr int kAct = decltype(act)::value;
        // Rows r .. of the band; `near`: the residual's or the gradient's.
        const auto finish = [&](int r, const f32x4(&near)[2], auto with) {
          const int64_t m = m_band + r;
          const __attribute__((address_space(3))) f32x4* const from =
              (const __attribute__((address_space(3))) f32x4*)(band + (r + lane / kLanes) * kStride + col);
          f32x4 z[2] = {from[0] + bias[0], from[1] + bias[1]}, u[2];
          if constexpr (C::kGated) {
            u[0] = from[kOut / 4] + bias_up[0];
            u[1] = from[kOut / 4 + 1] + bias_up[1];
          }
          if (m >= p.m || left <= 0) return;
          if constexpr (C::kEpi == kEpiStore || C::kEpi == kEpiGated) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              z[e / 4][e % 4] = act_value<T>(z[e / 4][e % 4], kAct);
              if constexpr (C::kGated) z[e / 4][e % 4] *= u[e / 4][e % 4];
            }
            if constexpr (decltype(with)::value) {
              z[0] += near[0];
              z[1] += near[1];
            }
            store8(static_cast<T*>(p.out) + m * p.ldo + n, z[0], z[1], left);
          } else {
            f32x4 up[2];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float value, slope;
              act_slope(z[e / 4][e % 4], kAct, value, slope);
              z[e / 4][e % 4] = near[e / 4][e % 4] * slope;
              if constexpr (C::kGated) {
                z[e / 4][e % 4] *= u[e / 4][e % 4];
                up[e / 4][e % 4] = near[e / 4][e % 4] * value;
              }
            }
            T* const out = static_cast<T*>(p.out) + m * p.ldo + n;
            store8(out, z[0], z[1], left);
            if constexpr (C::kGated) store8(out + p.n, up[0], up[1], left);
            if (n + 8 >= p.n) zero_padding(static_cast<T*>(p.out) + m * p.ldo, p.n * (C::kGated ? 2 : 1), p.ldo);
            if constexpr (kSlope) {
              column[0] += z[0];
              column[1] += z[1];
              if constexpr (C::kGated) {
                column[2] += up[0];
                column[3] += up[1];
              }
            }
          }
        };
        // (Two loops: a branch around the loads would wait for them in its own
        // block, one loop without it costs the plain store 10%.)
        if (kSlope || (C::kEpi == kEpiStore && beside)) {
          if constexpr (kSlope || C::kEpi == kEpiStore) {
#pragma unroll 1
            for (int turn = 0; turn < kTurns; turn += kAhead) {
#pragma unroll
              for (int j = 0; j < kAhead; ++j) {
                const int r = (turn + j) * kRows;
                f32x4 near[2];
                widen_eight(ahead[j], near[0], near[1]);
                if (turn + kAhead < kTurns) fetch_beside(m_band + r + kAhead * kRows, j);
                finish(r, near, Flag<true>{});
              }
            }
          }
        } else {
          const f32x4 none[2] = {};
#pragma unroll 2
          for (int r = 0; r < kTurns * kRows; r += kRows) finish(r, none, Flag<false>{});
        }
      });
    }
    // Over the lanes of a column, then over the rows of waves, in a fixed
    // order: row tm of p.sums.
    if constexpr (kSlope) {
      if (p.sums) {
        constexpr int kSumCols = C::kWN * kOut;  // of one half
        __attribute__((address_space(3))) float* const sums_lds = (__attribute__((address_space(3))) float*)smem;
        __syncthreads();  // the bands are read
#pragma unroll
        for (int q = 0; q < (C::kGated ? 4 : 2); ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = column[q][e];
#pragma unroll
            for (int d = kLanes; d < 64; d <<= 1) v += __shfl_xor(v, d);
            if (lane < kLanes)
              sums_lds[(wm * (C::kGated ? 2 : 1) + q / 2) * kSumCols + wn * kOut + col + (q % 2) * 4 + e] = v;
          }
        __syncthreads();
        for (int at = tid; at < kSumCols * (C::kGated ? 2 : 1); at += C::kThreads) {
          const int half = at / kSumCols;
          const int64_t to = n0 + at % kSumCols;
          if (to >= p.n) continue;
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < C::kWM; ++w) v += sums_lds[(w * (C::kGated ? 2 : 1) + half) * kSumCols + at % kSumCols];
          store_as(p.sums, static_cast<int64_t>(tm) * (C::kGated ? 2 * p.n : p.n) + half * p.n + to, p.sums_dtype, v);
        }
      }
    }
  }

  // The sums of A, by the workgroups of the first tile column: lane group g
  // holds those of its own elements.
  if constexpr (C::kSums) {
    if (p.sums && tn == 0 && wn == 0) {
#pragma unroll
      for (int t = 0; t < C::kTM; ++t) {
        float s = sums[t];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        const int64_t m = m0 + (wm * C::kTM + t) * 16 + i;
        if (g == 0 && m < p.m) store_as(p.sums, static_cast<int64_t>(part) * p.m + m, p.sums_dtype, s);
      }
    }
  }
}

}  // namespace vectra_dense
