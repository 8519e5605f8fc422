// One row of a norm in registers, shared by the kernels that norm rows: 8 columns per thread and unit in any float type, and what
// follows the products h w: the norm, and the row in 16 or 32 bits or as 8-bit codes.
#pragma once

#include "fg_codes.h"
#include "fg_decoder.h"

namespace fg {

// 16- and 8-byte accesses at any element's address
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// DT: FG_F32 / FG_F16 / FG_BF16.  Eight values as they lie in memory.
template <int DT>
struct Raw8 {
  u32x4_any w[DT == FG_F32 ? 2 : 1];
};

// Columns [i, i + n) of a row, n = 8 or, in its last unit, fewer (the rest are zeros).
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* p, int64_t i, int n) {
  Raw8<DT> r;
  constexpr int item = DT == FG_F32 ? 4 : 2;
  if (n >= 8) {
    const char* a = static_cast<const char*>(p) + i * item;
    r.w[0] = *reinterpret_cast<const u32x4_any*>(a);
    if constexpr (DT == FG_F32) r.w[1] = *reinterpret_cast<const u32x4_any*>(a + 16);
  } else {
    uint32_t e[8] = {};
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) e[j] = load_raw(p, DT, i + j);
    if constexpr (DT == FG_F32) {
      r.w[0] = (u32x4_any){e[0], e[1], e[2], e[3]};
      r.w[1] = (u32x4_any){e[4], e[5], e[6], e[7]};
    } else {
      r.w[0] = (u32x4_any){e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&f)[8]) {
  if constexpr (DT == FG_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(r.w[j / 4][j % 4]);
  } else {
    unpack8<DT == FG_BF16>(make_uint4(r.w[0][0], r.w[0][1], r.w[0][2], r.w[0][3]), f);
  }
}

// Eight values rounded to DT, to nearest even.
template <int DT>
__device__ __forceinline__ Raw8<DT> narrow8(const float (&f)[8]) {
  Raw8<DT> r;
  if constexpr (DT == FG_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.w[j / 4][j % 4] = __float_as_uint(f[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == FG_BF16) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        r.w[0][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){f[2 * j], f[2 * j + 1]}, bf16x2));
      } else {
        r.w[0][j] = (uint32_t)f32_to_f16_bits(f[2 * j]) | (uint32_t)f32_to_f16_bits(f[2 * j + 1]) << 16;
      }
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void store_raw8(void* p, int64_t i, int n, const Raw8<DT>& r) {
  constexpr int item = DT == FG_F32 ? 4 : 2;
  char* a = static_cast<char*>(p) + i * item;
  if (n >= 8) {
    *reinterpret_cast<u32x4_any*>(a) = r.w[0];
    if constexpr (DT == FG_F32) *reinterpret_cast<u32x4_any*>(a + 16) = r.w[1];
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      if (j >= n) continue;
      if constexpr (DT == FG_F32)
        static_cast<uint32_t*>(p)[i + j] = r.w[j / 4][j % 4];
      else
        static_cast<uint16_t*>(p)[i + j] = (uint16_t)(r.w[0][j / 2] >> (16 * (j % 2)));
    }
  }
}

__device__ __forceinline__ void store_codes8(uint8_t* p, int64_t i, int n, const uint2& c) {
  if (n >= 8) {
    *reinterpret_cast<u32x2_any*>(p + i) = (u32x2_any){c.x, c.y};
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) p[i + j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j % 4)));
  }
}

// Weights of the columns [i, i + n) from a row of type dt: ones without a row.
__device__ __forceinline__ void weights8(const void* p, int dt, int i, int n, float (&w)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = 1.f;
  if (!p) return;
  if (dt == FG_F32) widen8<FG_F32>(load_raw8<FG_F32>(p, i, n), w);
  else if (dt == FG_BF16) widen8<FG_BF16>(load_raw8<FG_BF16>(p, i, n), w);
  else widen8<FG_F16>(load_raw8<FG_F16>(p, i, n), w);
}

// What the wavefronts of a row exchange.
struct NormRed {
  float ss[16];
  uint32_t max[16];
};

// y of a row whose products t = h w, whose sum of squares of h so far (ss) and whose units' largest |t| (m, as bits: a NaN's are
// above every number's) the threads hold.  XT: y's type where it is no codes.  KT: the type of the row of h in memory at `kept`
// (each thread's own columns), which a row with a product past fp32's range reads again.
template <int XT, int KT, int C>
__device__ __forceinline__ void norm_row(const NormArgs& a, int64_t row, const char* kept, float (&t)[C][8], float ss, uint32_t (&m)[C],
                                         NormRed& red) {
  const int T = blockDim.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = T >> 6, K = a.K;
  auto at = [&](int c) { return 8 * (int)(threadIdx.x + c * T); };
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) top = max(top, m[c]);
  ss = wave_sum(ss);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, kWave));
  if (waves > 1) {
    if (lane == 0) {
      red.ss[wave] = ss;
      red.max[wave] = top;
    }
    __syncthreads();
    ss = red.ss[0];
    top = red.max[0];
    for (int w = 1; w < waves; ++w) {
      ss += red.ss[w];
      top = max(top, red.max[w]);
    }
  }
  float rs = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)K) + a.eps));
  if (top >= 0x7f800000u) {
    // a product h w passed fp32's range (or is no number): y as it is defined, h rs first, from what this thread kept or read
    top = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int n = K - at(c);
      if (n <= 0) continue;
      float h[8], w[8];
      widen8<KT>(load_raw8<KT>(kept, at(c), n), h);
      weights8(a.w, a.wdt, at(c), n, w);
      m[c] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t[c][j] = h[j] * rs * w[j];
        m[c] = max(m[c], __float_as_uint(t[c][j]) & 0x7fffffffu);
      }
      top = max(top, m[c]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, kWave));
    if (waves > 1) {
      __syncthreads();  // everyone has read the first maxima
      if (lane == 0) red.max[wave] = top;
      __syncthreads();
      for (int w = 0; w < waves; ++w) top = max(top, red.max[w]);
    }
    rs = 1.f;
  }
  const bool int8 = a.ydt == FG_I8;
  auto scale_of = [&](uint32_t bits) {  // a NaN is not above 0: such rows take scale 1
    const float amax = __uint_as_float(bits) * rs;
    return amax > 0.f ? __fdiv_rn(amax, int8 ? 127.f : 448.f) : 1.f;
  };
  if (a.ydt != FG_I8 && a.ydt != FG_E4M3) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int n = K - at(c);
      if (n <= 0) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[c][j] *= rs;
      store_raw8<XT>(static_cast<char*>(a.y) + row * a.ldy * (XT == FG_F32 ? 4 : 2), at(c), n, narrow8<XT>(t[c]));
    }
    return;
  }
  float scale = 1.f, inv = 1.f;
  bool fast = true;
  if (a.log_l < 0) {
    scale = scale_of(top);
    inv = __fdiv_rn(1.f, scale);
    if (threadIdx.x == 0) a.s[row * a.s_row] = scale;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int n = K - at(c);
    uint32_t bits = m[c];
    if (a.log_l >= 0) {  // the block's lanes are neighbours: T is a multiple of 64
      for (int off = (1 << a.log_l) >> 1; off > 0; off >>= 1)
        bits = max(bits, (uint32_t)__shfl_xor((int)bits, off, kWave));
      scale = scale_of(bits);
      inv = __fdiv_rn(1.f, scale);
      if (n > 0 && (threadIdx.x & ((1 << a.log_l) - 1)) == 0)
        a.s[row * a.s_row + ((threadIdx.x + c * T) >> a.log_l) * a.s_block] = scale;
    } else {
      bits = top;
    }
    // the exact quotient by multiply-adds: finite values, a scale in its range
    fast = __uint_as_float(bits) * rs < __builtin_inff() && div_by_ok(scale);
    if (n <= 0) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) t[c][j] *= rs;
    const uint2 codes = int8 ? encode8<false>(t[c], scale, inv, fast) : encode8<true>(t[c], scale, inv, fast);
    store_codes8(static_cast<uint8_t*>(a.y) + row * a.ldy, at(c), n, codes);
  }
}

}  // namespace fg
