// The attention kernels over a block-scaled cache of one 16-bit type.
#pragma once

#include "fg_mx_rows.h"
#include "fg_mx_tile.h"

namespace fg {

template <bool BF16>
static hipError_t launch_mx_items(const MxAttnArgs& m, hipStream_t st) {
  const dim3 grid((unsigned)m.a.items), block(256);
  auto go = [&](auto bits_tag, auto c_tag, auto d_tag) {
    constexpr int BITS = decltype(bits_tag)::value, DP = decltype(d_tag)::value;
    constexpr bool CAP = decltype(c_tag)::value;
    if (m.tile) hipLaunchKernelGGL((mx_tile_kernel<BF16, BITS, CAP, DP>), grid, block, 0, st, m);
    else if (m.a.page % 16 == 0 && m.a.c_token < 1u << 24) hipLaunchKernelGGL((mx_rows_kernel<BF16, BITS, CAP, DP, true>), grid, block, 0, st, m);
    else hipLaunchKernelGGL((mx_rows_kernel<BF16, BITS, CAP, DP, false>), grid, block, 0, st, m);
    return hipGetLastError();
  };
  auto by_d = [&](auto bits_tag, auto c_tag) {
    if (m.a.D <= 64) return go(bits_tag, c_tag, std::integral_constant<int, 64>{});
    if (m.a.D <= 128) return go(bits_tag, c_tag, std::integral_constant<int, 128>{});
    return go(bits_tag, c_tag, std::integral_constant<int, 256>{});
  };
  auto by_cap = [&](auto bits_tag) { return m.cap_in != 0.f ? by_d(bits_tag, std::true_type{}) : by_d(bits_tag, std::false_type{}); };
  return m.bits == 4 ? by_cap(std::integral_constant<int, 4>{}) : by_cap(std::integral_constant<int, 8>{});
}

}  // namespace fg
