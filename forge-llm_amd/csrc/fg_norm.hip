// Residual addition, RMSNorm and quantisation of one row in one pass:
//   h = rnd(x + r)            fp32 sum, rounded to the residual's type (h = x without a residual); h is the new residual
//   y = (h w) / sqrt(mean(h^2) + eps)          fp32
//   y in x's type, or codes by y's largest magnitude a per row or per 1 x block columns: scale s = a / 127 or a / 448 (IEEE
//   quotient; 1 where a > 0 is false), code = round(y / s), ties to even, to int8 or e4m3.
// The norm is that of h as it is kept, so the fused call gives what an addition, a norm and a quantiser give one by one.
//
// One workgroup per row, 8 columns per thread and unit, the row in registers from its one read to its one write.  With the
// weight multiplied in first, y = t rs for t = h w and the row's rs: rounding is monotonic, so max |y| = |max |t| rs| exactly,
// and one exchange between the wavefronts carries both the sum of squares and the maximum.  A row with a product past fp32's
// range takes a second turn, h rs w.  What bounds it is the latency of
// that chain for few rows and HBM for many.
//
// Rows need no alignment: 16-byte accesses at any address of their element type (the hardware takes them), and the last
// unit of a row that is no multiple of 8 columns goes element by element.
#include <algorithm>

#include "fg_codes.h"
#include "fg_decoder.h"

namespace fg {

namespace {

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

// Weights of the columns [i, i + n): ones without a weight.
__device__ __forceinline__ void weights8(const NormArgs& a, int i, int n, float (&w)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = 1.f;
  if (!a.w) return;
  if (a.wdt == FG_F32) widen8<FG_F32>(load_raw8<FG_F32>(a.w, i, n), w);
  else if (a.wdt == FG_BF16) widen8<FG_BF16>(load_raw8<FG_BF16>(a.w, i, n), w);
  else widen8<FG_F16>(load_raw8<FG_F16>(a.w, i, n), w);
}

}  // namespace

// RT: the residual's type, -1 for none.  A thread holds the row's units t, t + T, .. (C of them at most, T threads).
template <int XT, int RT, int C>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const NormArgs a) {
  constexpr int HT = RT < 0 ? XT : RT;
  __shared__ float red_ss[16];
  __shared__ uint32_t red_max[16];
  const int64_t row = blockIdx.x;
  const int T = blockDim.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = T >> 6, K = a.K;
  auto at = [&](int c) { return 8 * (int)(threadIdx.x + c * T); };
  const char* xrow = static_cast<const char*>(a.x) + row * a.ldx * (XT == FG_F32 ? 4 : 2);
  const char* rrow = static_cast<const char*>(a.r) + row * a.ldr * (HT == FG_F32 ? 4 : 2);
  Raw8<XT> xv[C];
  Raw8<HT> rv[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int n = K - at(c);
    if (n > 0) {
      xv[c] = load_raw8<XT>(xrow, at(c), n);
      if constexpr (RT >= 0) rv[c] = load_raw8<HT>(rrow, at(c), n);
    }
  }
  float t[C][8], ss = 0.f;
  uint32_t m[C];  // bit pattern of each unit's largest |h w|: a NaN's is above every number's
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int n = K - at(c);
    m[c] = 0;
    if (n <= 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[c][j] = 0.f;
      continue;
    }
    float h[8];
    widen8<XT>(xv[c], h);
    if constexpr (RT >= 0) {
      float r[8];
      widen8<HT>(rv[c], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += r[j];
      const Raw8<HT> kept = narrow8<HT>(h);
      widen8<HT>(kept, h);
      store_raw8<HT>(static_cast<char*>(a.ro) + row * a.ldro * (HT == FG_F32 ? 4 : 2), at(c), n, kept);
    }
    float w[8];
    weights8(a, at(c), n, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = __builtin_fmaf(h[j], h[j], ss);
      t[c][j] = h[j] * w[j];  // columns past the row's end are zeros
      m[c] = max(m[c], __float_as_uint(t[c][j]) & 0x7fffffffu);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) top = max(top, m[c]);
  ss = wave_sum(ss);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, kWave));
  if (waves > 1) {
    if (lane == 0) {
      red_ss[wave] = ss;
      red_max[wave] = top;
    }
    __syncthreads();
    ss = red_ss[0];
    top = red_max[0];
    for (int w = 1; w < waves; ++w) {
      ss += red_ss[w];
      top = max(top, red_max[w]);
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
      if constexpr (RT >= 0)
        widen8<HT>(load_raw8<HT>(static_cast<char*>(a.ro) + row * a.ldro * (HT == FG_F32 ? 4 : 2), at(c), n), h);
      else
        widen8<XT>(load_raw8<XT>(xrow, at(c), n), h);
      weights8(a, at(c), n, w);
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
      if (lane == 0) red_max[wave] = top;
      __syncthreads();
      for (int w = 0; w < waves; ++w) top = max(top, red_max[w]);
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

// Threads per row and units per thread: one unit per thread while the rows are too few to fill the CUs (a row's latency
// counts), else about two (rows in flight count; us, units per thread 1 / 2 / 4: 8192 x 4096 bf16 to e4m3 in blocks 48.1 /
// 45.2 / 51.3, to bf16 44.9 / 44.5 / 47.2, 2048 x 8192 to e4m3 24.5 / 23.1 / 22.9, 1111 x 5001 fp16 on an fp32 residual 16.4 /
// 13.6 / 13.8; non-temporal loads 52.7 for the first, with four).
static int norm_plan(int64_t M, int64_t K, int* C) {
  const int64_t units = (K + 7) / 8, per = M <= 2 * device_cus() ? 1 : 2;
  const int64_t t = std::min<int64_t>(1024, ((units + per - 1) / per + kWave - 1) / kWave * kWave);
  const int64_t c = (units + t - 1) / t;
  *C = c <= 1 ? 1 : (c <= 2 ? 2 : 4);
  return (int)t;
}

bool norm_fits(int64_t M, int64_t K) {
  int C = 0;
  return launchable(M, norm_plan(M, K, &C));
}

hipError_t launch_add_rmsnorm(const NormArgs& a, int xdt, int rdt, int64_t M, hipStream_t st) {
  int C = 0;
  const int T = norm_plan(M, a.K, &C);
  auto go = [&](auto x_tag, auto r_tag, auto c_tag) {
    constexpr int XT = decltype(x_tag)::value, RT = decltype(r_tag)::value, CC = decltype(c_tag)::value;
    note_kernel("add_rmsnorm_kernel<%d,%d,%d> T=%d", XT, RT, CC, T);
    hipLaunchKernelGGL((add_rmsnorm_kernel<XT, RT, CC>), dim3((unsigned)M), dim3(T), 0, st, a);
    return hipGetLastError();
  };
  auto pick = [&](auto x_tag, auto r_tag) {
    if (C == 1) return go(x_tag, r_tag, std::integral_constant<int, 1>{});
    if (C == 2) return go(x_tag, r_tag, std::integral_constant<int, 2>{});
    return go(x_tag, r_tag, std::integral_constant<int, 4>{});
  };
  auto by_residual = [&](auto x_tag) {
    if (!a.r) return pick(x_tag, std::integral_constant<int, -1>{});
    if (rdt == FG_F32) return pick(x_tag, std::integral_constant<int, FG_F32>{});
    if constexpr (decltype(x_tag)::value == FG_F32)
      return hipErrorInvalidValue;  // refused by the entry point
    else
      return pick(x_tag, x_tag);
  };
  if (xdt == FG_F32) return by_residual(std::integral_constant<int, FG_F32>{});
  if (xdt == FG_BF16) return by_residual(std::integral_constant<int, FG_BF16>{});
  return by_residual(std::integral_constant<int, FG_F16>{});
}

}  // namespace fg
