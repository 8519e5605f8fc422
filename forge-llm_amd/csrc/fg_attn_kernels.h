// The attention kernels of one 16-bit type: items of few rows, of many, and both in one launch.
#pragma once

#include "fg_attn_rows.h"
#include "fg_attn_tile.h"

namespace fg {

template <bool BF16, bool FP8, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attn_rows_kernel(const AttnArgs a) {
  __shared__ __align__(16) uint8_t lds[RowsLds<FP8, DP>::kBytes];
  attn_rows<BF16, FP8, DP>(a, blockIdx.x, lds);
}

template <bool BF16, bool FP8, bool DIRECT, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attn_tile_kernel(const AttnArgs a) {
  __shared__ __align__(16) uint8_t lds[TileLds<DP>::kBytes];
  attn_tile<BF16, FP8, DIRECT, DP>(a, blockIdx.x, lds);
}

// The prefix's items of many rows, bound by the matrix products, and the sequences' items of few rows, bound by their reads.
// Spread evenly among each other, in groups of eight workgroups (one for each XCD), both kinds share the CUs; or the
// prefix's go first, where they would outlast the others.
template <bool BF16, bool FP8, bool DIRECT, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attn_mixed_kernel(const AttnArgs a) {
  constexpr int kBytes = TileLds<DP>::kBytes > RowsLds<FP8, DP>::kBytes ? TileLds<DP>::kBytes : RowsLds<FP8, DP>::kBytes;
  __shared__ __align__(16) uint8_t lds[kBytes];
  const int many = (a.items_p + 7) / 8, all = gridDim.x / 8, at = blockIdx.x / 8, xcd = blockIdx.x % 8;
  int before = (int)((int64_t)at * many / all), after = (int)((int64_t)(at + 1) * many / all);
  if (a.lead) {
    before = min(at, many);
    after = min(at + 1, many);
  }
  if (after > before) {
    const int id = before * 8 + xcd;
    if (id < a.items_p) attn_tile<BF16, FP8, DIRECT, DP>(a, id, lds);
  } else {
    const int id = a.items_p + (at - before) * 8 + xcd;
    if (id < a.items) attn_rows<BF16, FP8, DP>(a, id, lds);
  }
}

template <bool BF16>
static hipError_t launch_attn_items(const AttnArgs& a, bool fp8, int kind, hipStream_t st) {
  auto run = [&](auto f_tag, auto direct_tag, auto d_tag) {
    constexpr bool F = decltype(f_tag)::value, DI = decltype(direct_tag)::value;
    constexpr int DP = decltype(d_tag)::value;
    if (kind == kAttnTile) {
      hipLaunchKernelGGL((attn_tile_kernel<BF16, F, DI, DP>), dim3((unsigned)a.items), dim3(256), 0, st, a);
    } else {
      const int groups = (a.items_p + 7) / 8 + (a.items - a.items_p + 7) / 8;
      hipLaunchKernelGGL((attn_mixed_kernel<BF16, F, DI, DP>), dim3((unsigned)groups * 8), dim3(256), 0, st, a);
    }
    return hipGetLastError();
  };
  auto by_kind = [&](auto f_tag, auto d_tag) {
    constexpr bool F = decltype(f_tag)::value;
    constexpr int DP = decltype(d_tag)::value;
    if (kind == kAttnRows) {
      hipLaunchKernelGGL((attn_rows_kernel<BF16, F, DP>), dim3((unsigned)a.items), dim3(256), 0, st, a);
      return hipGetLastError();
    }
    if constexpr (!F) {
      if (a.D == DP) return run(f_tag, std::true_type{}, d_tag);
    }
    return run(f_tag, std::false_type{}, d_tag);
  };
  auto by_d = [&](auto f_tag) {
    if (a.D <= 64) return by_kind(f_tag, std::integral_constant<int, 64>{});
    if (a.D <= 128) return by_kind(f_tag, std::integral_constant<int, 128>{});
    return by_kind(f_tag, std::integral_constant<int, 256>{});
  };
  return fp8 ? by_d(std::true_type{}) : by_d(std::false_type{});
}

}  // namespace fg
