// A paged cache in 4 or 8 bits with a power-of-two scale for each 32 columns (the OCP microscaling formats: e2m1 or e4m3 elements,
// e8m0 scales): arguments and the scale's arithmetic.
//
// A row of D columns (a whole number of blocks) is D BITS / 8 bytes of codes, 4-bit ones in pairs with the even column low, and
// D / 32 bytes of scales: byte b stands for 2^(b - 127), 255 for NaN.  The scales lie in the codes' order, so that a row's place among
// them is its place among the codes divided by 4 BITS, the bytes of one block.
#pragma once

#include "fg_device.h"

namespace fg {

constexpr int kMxBlock = 32;  // columns per scale
constexpr int kMxAxes = 4;    // axes of positions

struct MxCache {
  uint8_t *k, *v, *ks, *vs;
  int64_t page, head, token;  // byte strides of the codes
  int64_t n_slots;
  int page_size, Hk, D;
};

struct MxAppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;  // element strides of tokens and heads
  uint16_t* qo;
  int64_t qo_t, qo_h;
  const void* pos;  // [axes][T], ld_pos elements from axis to axis
  int pos64;
  int64_t ld_pos;
  int axes, ends[kMxAxes];  // axis a turns the pairs in front of ends[a]
  const float* table;       // [max_pos][rot]: cosines of the pairs, then sines
  int64_t ld_table, max_pos;
  const void* slots;
  int slots64;
  MxCache cache;
  int Hq, rot;
};

struct MxReadArgs {
  MxCache cache;
  const void* slots;
  int slots64;
  uint16_t *ko, *vo;  // [n][Hk][D], adjacent
  int64_t n;
};

hipError_t launch_mx_append(const MxAppendArgs& a, int64_t T, bool bf16, int bits, bool inter, hipStream_t st);
hipError_t launch_mx_read(const MxReadArgs& a, bool bf16, int bits, hipStream_t st);

// The scale byte of a block whose largest magnitude has these fp32 bits: the smallest power of two, from 2^-126 on, that brings
// it to half a step past the largest code at most (6 + 1 in e2m1, 448 + 16 in e4m3), so that no value is off by more than half
// a step of its own; 255 where it is not finite.
template <int BITS>
__device__ __forceinline__ uint32_t mx_byte(uint32_t amax) {
  constexpr int kTop = BITS == 4 ? 2 : 8;                           // the largest code's exponent
  constexpr uint32_t kRoom = BITS == 4 ? 0x600000u : 0x680000u;     // 1.75, 1.8125: seven, and 464, by their powers of two
  if (amax >= 0x7f800000u) return 255;
  const int e = (int)(amax >> 23) - kTop + ((amax & 0x7fffffu) > kRoom);
  return (uint32_t)(e < 1 ? 1 : e);
}

__device__ __forceinline__ float mx_scale(uint32_t byte) { return byte == 255 ? __builtin_nanf("") : __uint_as_float(byte << 23); }

// Two 16-bit floats from codes: byte `i` of a word of e2m1, half `i` of a word of e4m3.  Exact where the type can hold the value.
template <bool BF16, int BITS, int I>
__device__ __forceinline__ uint32_t mx_pair(uint32_t word, float scale) {
  if constexpr (BITS == 4) {
    if constexpr (BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, I));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, I));
  } else {
    if constexpr (BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)word, scale, I != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)word, scale, I != 0));
  }
}

// Eight columns as 16-bit floats from their codes (one word of e2m1, two of e4m3).
template <bool BF16, int BITS>
__device__ __forceinline__ uint4 mx_eight(uint32_t lo, uint32_t hi, float scale) {
  if constexpr (BITS == 4)
    return make_uint4(mx_pair<BF16, 4, 0>(lo, scale), mx_pair<BF16, 4, 1>(lo, scale), mx_pair<BF16, 4, 2>(lo, scale),
                      mx_pair<BF16, 4, 3>(lo, scale));
  else
    return make_uint4(mx_pair<BF16, 8, 0>(lo, scale), mx_pair<BF16, 8, 1>(lo, scale), mx_pair<BF16, 8, 0>(hi, scale),
                      mx_pair<BF16, 8, 1>(hi, scale));
}

}  // namespace fg
