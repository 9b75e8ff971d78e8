// Host side of the tiled product: from layout, tile and epilogue to a kernel.
#pragma once

#include "gemm_impl.h"

namespace vectra_dense {

template <typename T, typename C>
int launch_one(const GemmParams& p, int splits, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(p.tiles_m) * static_cast<uint32_t>(p.tiles_n) * static_cast<uint32_t>(splits);
  gemm_kernel<T, C><<<grid, C::kThreads, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? VECTRA_DENSE_OK : VECTRA_DENSE_ERR_LAUNCH;
}

template <typename T, bool kWideA, bool kWideB, int kEpi>
int launch_tile(const GemmParams& p, int tile, bool any, int splits, hipStream_t stream) {
  // One or two workgroups per CU need the phased loop; so do the transposing
  // reads of wide operands at any tile (10007 x 1000 -> 5464 bf16 weight
  // gradient on medium tiles: 174 us with the plain loop, 123 phased).
  // Forward products on medium and small tiles keep the plain loop: their
  // workgroups overlap each other (8192 x 4096 -> 4096: 245 us either way,
  // 10007 x 1000 -> 2 x 2730 gated: 143 plain, 151 phased).
  constexpr bool kWide = kWideA || kWideB;
  switch (tile) {
    case kTileLarge:
      return launch_one<T, GemmConfig<T, 256, 256, 2, 4, kWideA, kWideB, kEpi, true>>(p, splits, stream);
    case kTileTall:
      // (fp32 does not choose it: its rate is the same on any tile.)
      if constexpr (sizeof(T) == 2)
        return launch_one<T, GemmConfig<T, 192, 256, 2, 4, kWideA, kWideB, kEpi, true>>(p, splits, stream);
      return VECTRA_DENSE_ERR_LAUNCH;
    case kTileMedium:
      if (any) return launch_one<T, GemmConfig<T, 128, 128, 2, 2, kWideA, kWideB, kEpi, false, true>>(p, splits, stream);
      return launch_one<T, GemmConfig<T, 128, 128, 2, 2, kWideA, kWideB, kEpi, kWide>>(p, splits, stream);
    default:
      if (any) return launch_one<T, GemmConfig<T, 64, 64, 2, 2, kWideA, kWideB, kEpi, false, true>>(p, splits, stream);
      return launch_one<T, GemmConfig<T, 64, 64, 2, 2, kWideA, kWideB, kEpi, kWide>>(p, splits, stream);
  }
}

template <typename T>
int launch_gemm(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream) {
  if (layout == kLayoutForward) {
    switch (epi) {
      case kEpiStore: return launch_tile<T, false, false, kEpiStore>(p, tile, any, splits, stream);
      case kEpiPartial: return launch_tile<T, false, false, kEpiPartial>(p, tile, any, splits, stream);
      case kEpiGated: return launch_tile<T, false, false, kEpiGated>(p, tile, any, splits, stream);
      case kEpiSlope: return launch_tile<T, false, false, kEpiSlope>(p, tile, any, splits, stream);
      default: return launch_tile<T, false, false, kEpiGatedSlope>(p, tile, any, splits, stream);
    }
  }
  if (layout == kLayoutInput)
    return epi == kEpiStore ? launch_tile<T, false, true, kEpiStore>(p, tile, any, splits, stream)
                            : launch_tile<T, false, true, kEpiPartial>(p, tile, any, splits, stream);
  return epi == kEpiStore ? launch_tile<T, true, true, kEpiStore>(p, tile, any, splits, stream)
                          : launch_tile<T, true, true, kEpiPartial>(p, tile, any, splits, stream);
}

}  // namespace vectra_dense
