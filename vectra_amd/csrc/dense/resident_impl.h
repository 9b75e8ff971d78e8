// Products with a weight that fits LDS, over many rows: the kernel template,
// instantiated per element type in resident_<type>.hip.
//
//   forward      y = act(x W^T + b) + r,  or the gated product
//   slope        dz = g * act'(x W^T + b) (or both of a gated layer's), and
//                with it dx = dz W
//
// At the price model's widths (128 in, 256 out) these calls are bound by the
// bytes of x, y, g and dz, not by the products, so the kernel is built around
// streaming rows: a workgroup of 16 waves copies W into LDS once, then every
// wave walks units of 16 rows by itself, without barriers.  A unit's x goes
// from global memory straight into the registers of the matrix instruction's
// second operand (lane l: row l % 16, 16-byte chunk l / 16 of each step), W
// fragments come from LDS, and the result leaves in the layout it has.  While
// some waves of a SIMD wait for rows, others evaluate activations, which is
// what the vector units are busy with: a GELU takes about 24 issue slots of
// four cycles per 64 elements, 10 us for 17 million elements on 256 CUs.
//
// Measured, 66560 rows, 128 -> 256 bf16: forward with a GELU 21 us (51 MB; the
// vector units are busy 77% of it, the matrix cores 11%), dz and dx 35 us;
// gated with SiLU 22 and 46 us; 65536 rows, 141 -> 256 fp32 with a GELU 56 us
// (matrix cores 59% busy, 31 us of work).  One unit of 16 rows per wave and 16
// waves are the fastest of what was tried: two units per wave, or 8 and 12
// waves with more registers each, were 5-20% slower, loads one pair ahead the
// same.
//
// W's rows are stored in an order that gives a lane eight consecutive outputs
// of its row: LDS row 32 p + 16 j + i holds output 32 p + 8 (i / 4) + 4 j + i % 4,
// so the tiles j = 0, 1 of pair p leave lane group g the outputs
// 32 p + 8 g .. + 7, one 16-byte store for 16-bit types.
//
// dx needs no exchange between lanes: the values of dz that a lane holds for a
// pair (outputs 4 g .. 4 g + 3 of both tiles) are eight elements of its row,
// which is what the matrix instruction wants from lane group g for 32
// contraction elements, in an order of its own; the other operand, W with the
// contraction along its rows, is read from the same LDS copy by transposing
// reads of the same four rows per group.
//
// Units that are left when the others came out even over all waves are shared:
// their pairs of output tiles go to several waves of a workgroup (66560 rows
// are 16.25 units per CU: 256 -> 128 bf16 with a residual 18.6 -> 17.1 us).  Not
// with dx, whose sums would have to be joined: that took registers the kernel
// does not have (36 -> 42 us).
//
// Rows need no alignment: full chunks are loaded as 16 unaligned bytes, a
// row's last partial chunk element by element.
#pragma once

#include "gemm_impl.h"

namespace vectra_dense {

template <typename T, int kSteps_, int kEpi_, bool kDx_>
struct ResidentConfig {
  static constexpr int kSteps = kSteps_, kEpi = kEpi_;
  static constexpr bool kDx = kDx_;
  static constexpr int kPer = 16 / sizeof(T);
  static constexpr int kDeep = kSteps * 4 * kPer;  // contraction elements, padded
  static constexpr int kChunks = kSteps * 4;       // per LDS row
  static constexpr bool kPowerOfTwo = (kSteps & (kSteps - 1)) == 0;
  // Power-of-two rows are swizzled, others padded by a chunk.
  static constexpr int kRowBytes = kChunks * 16 + (kPowerOfTwo ? 0 : 16);
  static constexpr bool kGated = kEpi == kEpiGated || kEpi == kEpiGatedSlope;
  static constexpr bool kSlope = kEpi == kEpiSlope || kEpi == kEpiGatedSlope;
};

constexpr int kResidentWaves = 16;

// The chunk XOR of an LDS row.  Deep reads take one chunk of 16 consecutive
// rows, transposing reads two (32 bytes) of 8 consecutive rows; 256 bytes are
// one line of banks.
template <int kChunks>
__device__ __forceinline__ int resident_swizzle(int row) {
  if constexpr (kChunks >= 16) return ((row & 7) << 1) | ((row >> 3) & 1);
  if constexpr (kChunks == 8) return (((row >> 1) & 3) << 1) | ((row >> 3) & 1);
  return (row >> 2) & 3;
}

// kAct: the activation, fixed per instantiation of the body so that no branch
// sits in the element loops.
template <typename T, typename C, int kAct>
__device__ __forceinline__ void resident_body(const ResidentParams& p, const lds_char* w_lds,
                                              const __attribute__((address_space(3))) float* bias_lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int64_t units = (p.rows + 15) / 16;
  const int64_t hop = static_cast<int64_t>(gridDim.x) * kResidentWaves, rounds = units / hop;
  const int pairs = p.n_pad / 32;
  const T* const x = static_cast<const T*>(p.x);

  // After the rounds of whole units, at most `last` units are left for this
  // workgroup: `share` waves each.
  const int last = static_cast<int>((units - rounds * hop + gridDim.x - 1) / gridDim.x);
  int share = 1;
  if constexpr (!C::kDx)
    while (2 * share * last <= kResidentWaves && 2 * share <= pairs) share *= 2;

  for (int64_t round = 0; round <= rounds; ++round) {
    const int waves = round == rounds ? share : 1;
    const int first_pair = wave % waves;
    const int64_t unit = round * hop + static_cast<int64_t>(wave / waves) * gridDim.x + blockIdx.x;
    if (unit >= units) break;
    const int64_t row = unit * 16 + i;
    const bool live = row < p.rows;
    const int64_t row_read = live ? row : p.rows - 1;
    Frag fx[C::kSteps];
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s)
      fx[s] = load_row_chunk<T>(x + row_read * p.ldx, p.width, (s * 4 + g) * C::kPer);

    f32x4 dx[C::kDx ? C::kDeep / 16 : 1];
    if constexpr (C::kDx) {
#pragma unroll
      for (int t = 0; t < C::kDeep / 16; ++t) dx[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // z of the 16 outputs of LDS rows `first` ..
    const auto product = [&](int first) {
      f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < C::kSteps; ++s) {
        Frag fw;
        const int chunk = C::kPowerOfTwo ? (s * 4 + g) ^ resident_swizzle<C::kChunks>(i) : s * 4 + g;
        fw.w = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(w_lds + (first + i) * C::kRowBytes + chunk * 16);
        z = Mma<T>::run(fw, fx[s], z);
      }
      return z;
    };
    // dx += dz W for the 32 outputs of LDS rows `first` ..
    const auto gradient = [&](int first, f32x4 a, f32x4 b) {
      if constexpr (C::kDx) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const uint2 lo = __builtin_bit_cast(uint2, __builtin_convertvector(a, T4));
        const uint2 hi = __builtin_bit_cast(uint2, __builtin_convertvector(b, T4));
        Frag fz;
        fz.w = u32x4{lo.x, lo.y, hi.x, hi.y};
        // Row 4 g + i / 4, chunk (i % 4) / 2 of pair t = 0; rows are powers of
        // two apart, so pair t is an XOR away.  Opaque: as loop invariants the
        // addresses of all t are more than the registers hold.
        const int r = 4 * g + i / 4;
        int at = r * C::kRowBytes + ((((i % 4) / 2) ^ resident_swizzle<C::kChunks>(r)) * 16) + (i & 1) * 8;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int t = 0; t < C::kDeep / 16; ++t) {
          Frag fw;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const lds_v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) lds_v4s*)(const_cast<lds_char*>(w_lds) + first * C::kRowBytes + (at ^ (t * 32)) +
                                                             16 * j * C::kRowBytes));
            const uint2 u = __builtin_bit_cast(uint2, v);
            fw.w[2 * j] = u.x;
            fw.w[2 * j + 1] = u.y;
          }
          dx[t] = Mma<T>::run(fw, fz, dx[t]);
        }
      }
    };

    for (int pair = first_pair; pair < pairs; pair += waves) {
      const int n = pair * 32 + 8 * g;
      const int left = static_cast<int>(p.n - n);
      f32x4 za = product(pair * 32), zb = product(pair * 32 + 16);
      f32x4 ua, ub;
      if constexpr (C::kGated) {
        ua = product(p.n_pad + pair * 32);
        ub = product(p.n_pad + pair * 32 + 16);
      }
      if (p.bias) {
        za += *reinterpret_cast<const __attribute__((address_space(3))) f32x4*>(bias_lds + n);
        zb += *reinterpret_cast<const __attribute__((address_space(3))) f32x4*>(bias_lds + n + 4);
        if constexpr (C::kGated) {
          ua += *reinterpret_cast<const __attribute__((address_space(3))) f32x4*>(bias_lds + p.n_pad + n);
          ub += *reinterpret_cast<const __attribute__((address_space(3))) f32x4*>(bias_lds + p.n_pad + n + 4);
        }
      }
      if constexpr (!C::kSlope) {
        f32x4 ya, yb;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ya[e] = act_value<T>(za[e], kAct);
          yb[e] = act_value<T>(zb[e], kAct);
          if constexpr (C::kGated) {
            ya[e] *= ua[e];
            yb[e] *= ub[e];
          }
        }
        if (live && left > 0) {
          if (!C::kGated && p.residual) {
            f32x4 ra, rb;
            load8(static_cast<const T*>(p.residual) + row * p.ldr + n, left, ra, rb);
            ya += ra;
            yb += rb;
          }
          store8(static_cast<T*>(p.out) + row * p.ldo + n, ya, yb, left);
        }
      } else {
        f32x4 ga = {0.f, 0.f, 0.f, 0.f}, gb = {0.f, 0.f, 0.f, 0.f};
        if (live && left > 0)
          load8(static_cast<const T*>(p.grad) + row * p.ldg + n, left, ga, gb);
        f32x4 da, db, ea = {}, eb = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float value, slope;
          act_slope(za[e], kAct, value, slope);
          da[e] = ga[e] * slope;
          if constexpr (C::kGated) {
            da[e] *= ua[e];
            ea[e] = ga[e] * value;
          }
          act_slope(zb[e], kAct, value, slope);
          db[e] = gb[e] * slope;
          if constexpr (C::kGated) {
            db[e] *= ub[e];
            eb[e] = gb[e] * value;
          }
        }
        if constexpr (sizeof(T) == 2) {  // one rounding from the fp32 value
          asm volatile("" : "+v"(da), "+v"(db));
          if constexpr (C::kGated) asm volatile("" : "+v"(ea), "+v"(eb));
        }
        // Outputs past n have weights and biases of zero in LDS, so z and dz are
        // zero there, but for an x that is not finite (inf * 0): dx adds them up.
        if (left < 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e >= left) da[e] = ea[e] = 0.f;
            if (e + 4 >= left) db[e] = eb[e] = 0.f;
          }
        gradient(pair * 32, da, db);
        if constexpr (C::kGated) gradient(p.n_pad + pair * 32, ea, eb);
        if (p.out && live && left > 0) {
          T* const out = static_cast<T*>(p.out) + row * p.ldo + n;
          store8(out, da, db, left);
          if constexpr (C::kGated) store8(out + p.n, ea, eb, left);
        }
      }
    }
    if constexpr (C::kSlope) {
      if (p.out && live && g == 0 && first_pair == 0)
        zero_padding(static_cast<T*>(p.out) + row * p.ldo, p.n * (C::kGated ? 2 : 1), p.ldo);
    }
    if constexpr (C::kDx) {
      if (live && p.dx) {
        T* const out = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
        for (int t = 0; t < C::kDeep / 16; ++t)
          store4(out + t * 16 + 4 * g, dx[t], static_cast<int>(p.width) - (t * 16 + 4 * g));
      }
    }
  }
}

template <typename T, typename C>
__global__ __launch_bounds__(64 * kResidentWaves) void resident_kernel(const ResidentParams p) {
  extern __shared__ __attribute__((aligned(256))) char resident_smem[];
  lds_char* const w_lds = (lds_char*)resident_smem;
  const int rows_lds = p.n_pad * (C::kGated ? 2 : 1);
  __attribute__((address_space(3))) float* const bias_lds =
      (__attribute__((address_space(3))) float*)(w_lds + rows_lds * C::kRowBytes);

  // W into LDS: a chunk per thread and turn.  LDS row r of a half holds the
  // output given above; outputs past n are zeros.
  const T* const w = static_cast<const T*>(p.w);
  for (int at = threadIdx.x; at < rows_lds * C::kChunks; at += 64 * kResidentWaves) {
    const int r = at / C::kChunks, chunk = at % C::kChunks;
    const bool up = C::kGated && r >= p.n_pad;
    const int in = up ? r - p.n_pad : r;
    const int n = (in & ~31) + 8 * ((in >> 2) & 3) + 4 * ((in >> 4) & 1) + (in & 3);
    Frag f;
    f.w = u32x4{0, 0, 0, 0};
    if (n < p.n) {
      const int64_t w_row = n + (up ? p.n : 0);
      f = load_row_chunk<T>(w + w_row * p.ldw, p.width, chunk * C::kPer);
    }
    const int to = C::kPowerOfTwo ? chunk ^ resident_swizzle<C::kChunks>(r & 15) : chunk;
    *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(w_lds + r * C::kRowBytes + to * 16) = f.w;
  }
  if (p.bias)
    for (int r = threadIdx.x; r < rows_lds; r += 64 * kResidentWaves) {
      const bool up = C::kGated && r >= p.n_pad;
      const int n = up ? r - p.n_pad : r;
      bias_lds[r] = n < p.n ? load_bias(p.bias, n + (up ? p.n : 0), p.bias_dtype) : 0.f;
    }
  __syncthreads();
  switch (p.activation) {
    case VECTRA_DENSE_RELU: return resident_body<T, C, VECTRA_DENSE_RELU>(p, w_lds, bias_lds);
    case VECTRA_DENSE_GELU: return resident_body<T, C, VECTRA_DENSE_GELU>(p, w_lds, bias_lds);
    case VECTRA_DENSE_GELU_TANH: return resident_body<T, C, VECTRA_DENSE_GELU_TANH>(p, w_lds, bias_lds);
    case VECTRA_DENSE_SILU: return resident_body<T, C, VECTRA_DENSE_SILU>(p, w_lds, bias_lds);
    default: return resident_body<T, C, VECTRA_DENSE_NONE>(p, w_lds, bias_lds);
  }
}

template <typename T, typename C>
int launch_resident_one(const ResidentParams& p, int workgroups, hipStream_t stream) {
  const int rows_lds = p.n_pad * (C::kGated ? 2 : 1);
  const int lds = rows_lds * C::kRowBytes + rows_lds * 4;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(&resident_kernel<T, C>), hipFuncAttributeMaxDynamicSharedMemorySize,
                          kResidentLds) != hipSuccess)
    return VECTRA_DENSE_ERR_LAUNCH;
  resident_kernel<T, C><<<workgroups, 64 * kResidentWaves, lds, stream>>>(p);
  return hipGetLastError() == hipSuccess ? VECTRA_DENSE_OK : VECTRA_DENSE_ERR_LAUNCH;
}

template <typename T, int kSteps>
int launch_resident_steps(const ResidentParams& p, int epi, bool with_dx, int workgroups, hipStream_t stream) {
  if constexpr (sizeof(T) == 2 && kSteps <= 4) {
    if (with_dx)
      return epi == kEpiSlope ? launch_resident_one<T, ResidentConfig<T, kSteps, kEpiSlope, true>>(p, workgroups, stream)
                              : launch_resident_one<T, ResidentConfig<T, kSteps, kEpiGatedSlope, true>>(p, workgroups, stream);
  }
  if (with_dx) return VECTRA_DENSE_ERR_LAUNCH;
  switch (epi) {
    case kEpiStore: return launch_resident_one<T, ResidentConfig<T, kSteps, kEpiStore, false>>(p, workgroups, stream);
    case kEpiGated: return launch_resident_one<T, ResidentConfig<T, kSteps, kEpiGated, false>>(p, workgroups, stream);
    case kEpiSlope: return launch_resident_one<T, ResidentConfig<T, kSteps, kEpiSlope, false>>(p, workgroups, stream);
    default: return launch_resident_one<T, ResidentConfig<T, kSteps, kEpiGatedSlope, false>>(p, workgroups, stream);
  }
}

}  // namespace vectra_dense
