// 8-bit codes of activations, shared by the quantisers and the kernels that quantise what they compute: the e4m3 cast, the
// exact quotient by a row's scale, 8 values at a time in 16-byte units.
#pragma once

#include "fg_device.h"

namespace fg {

__device__ __forceinline__ uint8_t f32_to_e4m3(float v) {
  // v_cvt_pk_fp8_f32: OCP e4m3 (gfx950), round to nearest even; inputs are pre-clamped to +-448.  A NaN becomes the
  // e4m3fn NaN code with its sign (0x7F / 0xFF), as torch's cast writes it.
  const int packed = __builtin_amdgcn_cvt_pk_fp8_f32(v, 0.f, 0, false);
  const uint8_t nan_code = (__float_as_uint(v) >> 24 & 0x80) | 0x7F;
  return __builtin_isnan(v) ? nan_code : (uint8_t)(packed & 0xff);
}

// RN(a / b) from y = RN(1 / b): q0 = a y is within two units in the last place, one correction brings it within one,
// and the second correction of a quotient that close is the correctly rounded one (Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990, theorem on division with a fused multiply-add).
// It holds while no intermediate leaves the normal range: the callers use it for 2^-60 <= b <= 2^60.  There a residual
// can only lose bits for |a| < 2^-102, where the quotient is below 2^-42 and its code is zero either way.
__device__ __forceinline__ float div_by(float a, float b, float y) {
  const float q0 = a * y;
  const float q1 = __builtin_fmaf(__builtin_fmaf(-b, q0, a), y, q0);
  return __builtin_fmaf(__builtin_fmaf(-b, q1, a), y, q1);
}
__device__ __forceinline__ bool div_by_ok(float b) { return b >= 0x1p-60f && b <= 0x1p60f; }

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      f[2 * i] = f16_bits_to_f32((uint16_t)w[i]);
      f[2 * i + 1] = f16_bits_to_f32((uint16_t)(w[i] >> 16));
    }
  }
}

// Codes of 4 values as they lie in memory.  `fast`: div_by applies (finite values, a scale in its range).
template <bool FP8>
__device__ __forceinline__ uint32_t encode4(const float* v, float scale, float y, bool fast) {
  float d[4];
  if (fast) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float q = div_by(v[i], scale, y);
      // the corrections turn -0 into +0; an e4m3 code keeps the sign of a zero
      d[i] = FP8 ? __builtin_copysignf(fminf(fmaxf(q, -448.f), 448.f), v[i]) : fminf(fmaxf(q, -127.f), 127.f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float q = __fdiv_rn(v[i], scale);
      if (FP8)
        d[i] = __builtin_isnan(q) ? q : fminf(fmaxf(q, -448.f), 448.f);
      else
        d[i] = __builtin_isnan(q) ? 0.f : fminf(fmaxf(q, -127.f), 127.f);
    }
  }
  if (FP8) {
    if (fast) {
      const int p = __builtin_amdgcn_cvt_pk_fp8_f32(d[0], d[1], 0, false);
      return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(d[2], d[3], p, true);
    }
    return (uint32_t)f32_to_e4m3(d[0]) | (uint32_t)f32_to_e4m3(d[1]) << 8 | (uint32_t)f32_to_e4m3(d[2]) << 16 |
           (uint32_t)f32_to_e4m3(d[3]) << 24;
  }
  // |d| <= 127: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low byte
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(d[i] + 12582912.f);
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u),
                               __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
}

template <bool FP8>
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float scale, float y, bool fast) {
  return make_uint2(encode4<FP8>(v, scale, y, fast), encode4<FP8>(v + 4, scale, y, fast));
}

__device__ __forceinline__ void load8_f(const void* p, int dt, int64_t i, float (&f)[8]) {
  if (dt == FG_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    if (dt == FG_BF16) unpack8<true>(u, f);
    else unpack8<false>(u, f);
  }
}

}  // namespace fg
