// The step between two blocks of a decoder layer that norms a block's output as well as the next one's input, one row in one pass:
//   b = x / sqrt(mean(x^2) + eps_post) * post_weight * residual_scale * gate      fp32, in this order, an IEEE quotient: a sum next
//                                          to a border of the residual's type goes to the side that the same steps one by one give
//   h = rnd(r + b)                         rounded to the residual's type; the new residual
//   y = (h w) / sqrt(mean(h^2) + eps)      fp32, stored in x's type or as codes, as add_rmsnorm does
//
// One workgroup per row, as in add_rmsnorm, whose second half this shares: x and r stay in registers from their one read, so a row
// costs two exchanges between the wavefronts and no memory traffic beyond its inputs and outputs.  What bounds it is HBM for many
// rows and, for few, the chain load -> sum -> sum -> store: there the weights and the gate are loaded in front of the first exchange.
#include "fg_norm_row.h"

namespace fg {

constexpr int kStrides = 4096;  // columns of a row whose squares are added up by strides

// STRIDES: the squares of x are added up in the order of a wavefront that reads four columns a lane, columns 256 apart one after the
// other, then each four neighbours, then lanes, neighbours first.  It is the order in which the sum of such rows is taken where the
// steps run one by one, so that rms, and with it every h next to a border of its type, comes out the same to the bit; x goes through
// LDS for it (8192 x 4096 in bf16 to e4m3 blocks: 60 us either way).
template <int XT, int RT, int C, bool STRIDES>
__global__ void __launch_bounds__(1024) postnorm_add_rmsnorm_kernel(const PostNormArgs p) {
  __shared__ __align__(16) float red_post[STRIDES ? 256 : 16];
  __shared__ __align__(16) uint8_t kept_x[STRIDES ? kStrides * (XT == FG_F32 ? 4 : 2) : 16];
  __shared__ NormRed red;
  const NormArgs& a = p.norm;
  const int64_t row = blockIdx.x;
  const int T = blockDim.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = T >> 6, K = a.K;
  auto at = [&](int c) { return 8 * (int)(threadIdx.x + c * T); };
  const char* xrow = static_cast<const char*>(a.x) + row * a.ldx * (XT == FG_F32 ? 4 : 2);
  const char* rrow = static_cast<const char*>(a.r) + row * a.ldr * (RT == FG_F32 ? 4 : 2);
  char* hrow = static_cast<char*>(a.ro) + row * a.ldro * (RT == FG_F32 ? 4 : 2);
  const char* grow = p.gate ? static_cast<const char*>(p.gate) + row * p.ldg * (p.gdt == FG_F32 ? 4 : 2) : nullptr;
  Raw8<XT> xv[C];
  Raw8<RT> rv[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int n = K - at(c);
    if (n > 0) {
      xv[c] = load_raw8<XT>(xrow, at(c), n);
      rv[c] = load_raw8<RT>(rrow, at(c), n);
    }
  }
  constexpr bool kEarly = C == 1;  // few rows: nobody else's work hides these loads
  float pw[8], g[8], w[8];
  auto factors = [&](int c) __attribute__((always_inline)) {
    const int n = K - at(c);
    weights8(p.pw, p.pwdt, at(c), n, pw);
    weights8(grow, p.gdt, at(c), n, g);
    weights8(a.w, a.wdt, at(c), n, w);
  };
  if (kEarly && K > at(0)) factors(0);
  float ss = 0.f;
  if constexpr (STRIDES) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (K > at(c)) {
        uint4* to = reinterpret_cast<uint4*>(kept_x + at(c) * (XT == FG_F32 ? 4 : 2));  // a row's last unit ends in zeros
        to[0] = make_uint4(xv[c].w[0][0], xv[c].w[0][1], xv[c].w[0][2], xv[c].w[0][3]);
        if constexpr (XT == FG_F32) to[1] = make_uint4(xv[c].w[1][0], xv[c].w[1][1], xv[c].w[1][2], xv[c].w[1][3]);
      }
    __syncthreads();
    for (int r = threadIdx.x; r < 256; r += T) {
      float sum = 0.f;
      for (int i = r; i < K; i += 1024) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = load_f(kept_x, XT, i + 256 * j);
          sum += i + 256 * j < K ? x * x : 0.f;
        }
      }
      red_post[r] = sum;
    }
    __syncthreads();
    const float4 four = reinterpret_cast<const float4*>(red_post)[lane];
    ss = ((four.x + four.y) + four.z) + four.w;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) ss += __shfl_xor(ss, off, kWave);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (K <= at(c)) continue;
      float x[8];
      widen8<XT>(xv[c], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
    }
    ss = wave_sum(ss);
    if (waves > 1) {
      if (lane == 0) red_post[wave] = ss;
      __syncthreads();
      ss = red_post[0];
      for (int i = 1; i < waves; ++i) ss += red_post[i];
    }
  }
  // x / rms by multiply-adds: both by the power of two that brings rms into their range; one that is infinite gives zeros
  float rms = __builtin_sqrtf(__fdiv_rn(ss, (float)K) + p.eps_post);
  const float by = div_by_ok(rms) ? 1.f : (rms > 1.f ? 0x1p-64f : 0x1p64f);
  rms *= by;
  const float rs = __fdiv_rn(1.f, rms);
  rms = rms == __builtin_inff() ? 0.f : rms;
  float t[C][8];
  uint32_t m[C];
  ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int n = K - at(c);
    m[c] = 0;
    if (n <= 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[c][j] = 0.f;
      continue;
    }
    if (!kEarly) factors(c);
    float x[8], h[8];
    widen8<XT>(xv[c], x);
    widen8<RT>(rv[c], h);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] += div_by(x[j] * by, rms, rs) * pw[j] * p.scale * g[j];
    const Raw8<RT> kept = narrow8<RT>(h);
    widen8<RT>(kept, h);
    store_raw8<RT>(hrow, at(c), n, kept);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= n) h[j] = 0.f;  // columns past the row's end: a factor that is no number does not show in the sum
      ss = __builtin_fmaf(h[j], h[j], ss);
      t[c][j] = h[j] * w[j];
      m[c] = max(m[c], __float_as_uint(t[c][j]) & 0x7fffffffu);
    }
  }
  norm_row<XT, RT, C>(a, row, hrow, t, ss, m, red);
}

hipError_t launch_postnorm_add_rmsnorm(const PostNormArgs& p, int xdt, int rdt, int64_t M, hipStream_t st) {
  int C = 0;
  const int T = norm_plan(M, p.norm.K, &C);
  auto go = [&](auto x_tag, auto r_tag, auto c_tag) {
    constexpr int XT = decltype(x_tag)::value, RT = decltype(r_tag)::value, CC = decltype(c_tag)::value;
    note_kernel("postnorm_add_rmsnorm_kernel<%d,%d,%d> T=%d", XT, RT, CC, T);
    // two units a thread: the rows are many
    if (CC == 2 && p.norm.K % 4 == 0 && p.norm.K <= kStrides)
      hipLaunchKernelGGL((postnorm_add_rmsnorm_kernel<XT, RT, CC, CC == 2>), dim3((unsigned)M), dim3(T), 0, st, p);
    else
      hipLaunchKernelGGL((postnorm_add_rmsnorm_kernel<XT, RT, CC, false>), dim3((unsigned)M), dim3(T), 0, st, p);
    return hipGetLastError();
  };
  auto pick = [&](auto x_tag, auto r_tag) {
    if (C == 1) return go(x_tag, r_tag, std::integral_constant<int, 1>{});
    if (C == 2) return go(x_tag, r_tag, std::integral_constant<int, 2>{});
    return go(x_tag, r_tag, std::integral_constant<int, 4>{});
  };
  auto by_residual = [&](auto x_tag) {
    if (rdt == FG_F32) return pick(x_tag, std::integral_constant<int, FG_F32>{});
    return pick(x_tag, x_tag);  // the entry point takes x's type or fp32 only
  };
  if (xdt == FG_F32) return by_residual(std::integral_constant<int, FG_F32>{});
  if (xdt == FG_BF16) return by_residual(std::integral_constant<int, FG_BF16>{});
  return by_residual(std::integral_constant<int, FG_F16>{});
}

}  // namespace fg
