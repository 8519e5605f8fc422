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

#include "fg_norm_row.h"

namespace fg {

// RT: the residual's type, -1 for none.  A thread holds the row's units t, t + T, .. (C of them at most, T threads).
template <int XT, int RT, int C>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const NormArgs a) {
  constexpr int HT = RT < 0 ? XT : RT;
  __shared__ NormRed red;
  const int64_t row = blockIdx.x;
  const int T = blockDim.x, K = a.K;
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
  uint32_t m[C];
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
    weights8(a.w, a.wdt, at(c), n, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = __builtin_fmaf(h[j], h[j], ss);
      t[c][j] = h[j] * w[j];  // columns past the row's end are zeros
      m[c] = max(m[c], __float_as_uint(t[c][j]) & 0x7fffffffu);
    }
  }
  norm_row<XT, HT, C>(a, row, RT >= 0 ? static_cast<const char*>(a.ro) + row * a.ldro * (HT == FG_F32 ? 4 : 2) : xrow, t, ss, m, red);
}

// Threads per row and units per thread: one unit per thread while the rows are too few to fill the CUs (a row's latency
// counts), else about two (rows in flight count; us, units per thread 1 / 2 / 4: 8192 x 4096 bf16 to e4m3 in blocks 48.1 /
// 45.2 / 51.3, to bf16 44.9 / 44.5 / 47.2, 2048 x 8192 to e4m3 24.5 / 23.1 / 22.9, 1111 x 5001 fp16 on an fp32 residual 16.4 /
// 13.6 / 13.8; non-temporal loads 52.7 for the first, with four).
int norm_plan(int64_t M, int64_t K, int* C) {
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
