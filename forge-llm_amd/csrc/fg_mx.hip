// The way into a block-scaled cache and back out of it.
//
// mx_append: rotary embedding of a projection's queries and keys, and the keys' and values' codes and scales, in one launch.  A
// thread holds 8 columns of a head, so the 32 columns of a scale are four neighbours, and a head lies in one wavefront: all its
// loads come in front of its stores, which lets the rotated queries stand in the queries' place although a rotation takes the
// other half's columns too.  The thread keeps its columns' cosines and sines and walks the token's heads with them.
// Keys are rotated in fp64, where the products of a 16-bit value and an fp32 cosine are exact, and rounded to fp32 once: which code or
// scale a value next to a border gets does not hang on how the sum is formed.  Values go to their codes as they are.
// mx_read: rows of 16-bit values from the slots' codes.
// Both are bound by one read and one write of the tokens for prompts (8192 tokens of 32 + 2 x 8 heads of 128 into 4 bits 46 us, 3.9
// TB/s; read back 12.9 us) and by latency for few tokens (64 of 64 + 2 x 8 heads: 5 us; 3.3).
#include <algorithm>

#include "fg_codes.h"
#include "fg_decoder.h"
#include "fg_mx.h"

namespace fg {

namespace {

typedef uint32_t u32x4_by2 __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any 16-bit element
typedef float f32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMxThreads = 128;

__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  const u32x4_by2 w = *reinterpret_cast<const u32x4_by2*>(p);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool BF16>
__device__ __forceinline__ float one_f(uint16_t b) {
  return BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// Codes and scale of this lane's 8 columns, of which four neighbouring lanes make a block.
template <int BITS>
__device__ __forceinline__ void put_codes(const float (&f)[8], int u, uint8_t* codes, uint8_t* scales) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  top = max(top, __float_as_uint(dpp_partner<1>(__uint_as_float(top))));
  top = max(top, __float_as_uint(dpp_partner<2>(__uint_as_float(top))));
  const uint32_t byte = mx_byte<BITS>(top);
  uint32_t w[2] = {0, 0};
  if (byte != 255) {
    if constexpr (BITS == 4) {
      const float s = mx_scale(byte);
      w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], f[0], f[1], s, 0);
      w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], f[2], f[3], s, 1);
      w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], f[4], f[5], s, 2);
      w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], f[6], f[7], s, 3);
    } else {
      const float inv = __uint_as_float((254 - byte) << 23);  // the products are exact
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = fminf(fmaxf(f[4 * i + j] * inv, -448.f), 448.f);
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], p, true);
      }
    }
  }
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(codes + 4 * u) = w[0];
  else *reinterpret_cast<uint2*>(codes + 8 * u) = make_uint2(w[0], w[1]);
  if (u % 4 == 0) scales[u / 4] = (uint8_t)byte;
}

}  // namespace

// WIDE: a unit's partner columns are a unit too (rotary halves, or interleaved pairs, of whole units).
// Eight wavefronts to a SIMD hide a turn's loads best (8192 tokens: 46 us; 5 wavefronts 53, and 61 with the next turn's loads ahead of
// this one's work).
template <bool BF16, int BITS, bool INTER, bool WIDE>
__global__ void __launch_bounds__(kMxThreads, 8) mx_append_kernel(const MxAppendArgs a) {
  const int64_t t = blockIdx.x;
  const MxCache& c = a.cache;
  const int items = c.D / 8, per_wave = 64 / items, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int u = lane % items, r = lane / items, rows = per_wave * (blockDim.x >> 6);
  if (r >= per_wave) return;
  const int64_t slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[t] : static_cast<const int32_t*>(a.slots)[t];
  const bool keep = slot >= 0 && slot < c.n_slots;  // any other slot is padding
  const int64_t page = keep ? slot / c.page_size : 0, off = keep ? slot - page * c.page_size : 0;
  const int64_t place = page * c.page + off * c.token;
  const int c0 = 8 * u, half = a.rot / 2;
  float cs[8], sn[8];  // column j turns to x cs + partner sn
  if (c0 < a.rot) {
    int64_t row[kMxAxes];
#pragma unroll
    for (int x = 0; x < kMxAxes; ++x) {
      row[x] = -1;
      if (x >= a.axes) continue;
      const int64_t at = x * a.ld_pos + t;
      const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.pos)[at] : static_cast<const int32_t*>(a.pos)[at];
      if (p >= 0 && p < a.max_pos) row[x] = p * a.ld_table;  // a position that the table lacks shows as NaN
    }
    const float nan = __builtin_nanf("");
    if (WIDE && a.axes == 1) {
      const int pair = INTER ? c0 / 2 : (c0 < half ? c0 : c0 - half);
      f32x4_by4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // cosines of the unit's pairs, then sines (4 pairs of an interleaved unit, else 8)
        if (INTER && i % 2) continue;
        const float* p = a.table + row[0] + (i < 2 ? 0 : half) + pair + 4 * (i % 2);
        w[i] = row[0] < 0 ? (f32x4_by4)(nan) : *reinterpret_cast<const f32x4_by4*>(p);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = INTER ? w[0][j / 2] : w[j / 4][j % 4];
        sn[j] = INTER ? w[2][j / 2] : w[2 + j / 4][j % 4];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = c0 + j, pair = INTER ? col / 2 : (col < half ? col : col - half);
        int64_t at = row[0];
#pragma unroll
        for (int x = 1; x < kMxAxes; ++x)
          if (x < a.axes && pair >= a.ends[x - 1]) at = row[x];
        const bool in = col < a.rot && at >= 0;
        cs[j] = in ? a.table[at + pair] : nan;
        sn[j] = in ? a.table[at + half + pair] : nan;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (INTER ? j % 2 == 0 : c0 + j < half) sn[j] = -sn[j];
  }
  const int H = a.Hq + 2 * c.Hk;
  for (int h = blockIdx.y * rows + wave * per_wave + r; h < H; h += gridDim.y * rows) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + c.Hk;
    const int hk = is_v ? h - a.Hq - c.Hk : h - a.Hq;
    if (!is_q && !keep) continue;
    const uint16_t* src = is_q ? a.q + t * a.q_t + h * a.q_h : (is_v ? a.v + t * a.v_t + hk * a.v_h : a.k + t * a.k_t + hk * a.k_h);
    float x[8];
    unpack8<BF16>(load16(src + c0), x);
    if (!is_v && c0 < a.rot) {
      float p[8];
      if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = x[j ^ 1];
      } else if constexpr (WIDE) {
        unpack8<BF16>(load16(src + (c0 < half ? c0 + half : c0 - half)), p);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = c0 + j;
          p[j] = one_f<BF16>(src[col < half ? col + half : (col < a.rot ? col - half : col)]);
        }
      }
      float y[8];
      if (is_q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[j] * cs[j] + p[j] * sn[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (float)((double)x[j] * cs[j] + (double)p[j] * sn[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = WIDE || c0 + j < a.rot ? y[j] : x[j];
    }
    __builtin_amdgcn_wave_barrier();  // the head's loads are behind us: its place may be written
    if (is_q) {
      u32x4_by2 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (BF16) w[j] = (uint32_t)f32_to_bf16_bits_hw(x[2 * j]) | (uint32_t)f32_to_bf16_bits_hw(x[2 * j + 1]) << 16;
        else w[j] = (uint32_t)f32_to_f16_bits(x[2 * j]) | (uint32_t)f32_to_f16_bits(x[2 * j + 1]) << 16;
      }
      *reinterpret_cast<u32x4_by2*>(a.qo + t * a.qo_t + h * a.qo_h + c0) = w;
    } else {
      const int64_t at = place + hk * c.head;
      put_codes<BITS>(x, u, (is_v ? c.v : c.k) + at, (is_v ? c.vs : c.ks) + at / (4 * BITS));
    }
  }
}

hipError_t launch_mx_append(const MxAppendArgs& a, int64_t T, bool bf16, int bits, bool inter, hipStream_t st) {
  const int items = a.cache.D / 8, per_wave = 64 / items, H = a.Hq + 2 * a.cache.Hk;
  const int waves = std::min(kMxThreads / 64, (H + per_wave - 1) / per_wave), rows = waves * per_wave;
  // few tokens: the turns over a token's heads are workgroups
  const unsigned gy = T <= 2 * device_cus() ? (unsigned)((H + rows - 1) / rows) : 1u;
  if (gy > 65535 || !launchable(T * gy, waves * 64)) return hipErrorInvalidConfiguration;
  const bool wide = inter ? a.rot % 8 == 0 : a.rot % 16 == 0;
  auto go = [&](auto b_tag, auto bits_tag, auto i_tag, auto w_tag) {
    note_kernel("mx_append_kernel<%d> heads/%u", bits, gy);
    hipLaunchKernelGGL((mx_append_kernel<decltype(b_tag)::value, decltype(bits_tag)::value, decltype(i_tag)::value,
                                         decltype(w_tag)::value>),
                       dim3((unsigned)T, gy), dim3(waves * 64), 0, st, a);
    return hipGetLastError();
  };
  auto by_w = [&](auto b_tag, auto bits_tag, auto i_tag) {
    return wide ? go(b_tag, bits_tag, i_tag, std::true_type{}) : go(b_tag, bits_tag, i_tag, std::false_type{});
  };
  auto by_i = [&](auto b_tag, auto bits_tag) {
    return inter ? by_w(b_tag, bits_tag, std::true_type{}) : by_w(b_tag, bits_tag, std::false_type{});
  };
  auto by_bits = [&](auto b_tag) {
    return bits == 4 ? by_i(b_tag, std::integral_constant<int, 4>{}) : by_i(b_tag, std::integral_constant<int, 8>{});
  };
  return bf16 ? by_bits(std::true_type{}) : by_bits(std::false_type{});
}

template <bool BF16, int BITS>
__global__ void __launch_bounds__(256) mx_read_kernel(const MxReadArgs a) {
  const MxCache& c = a.cache;
  const int items = c.D / 8, all = 2 * c.Hk * items;
  const int64_t t = blockIdx.x;
  const int64_t slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[t] : static_cast<const int32_t*>(a.slots)[t];
  const bool in = slot >= 0 && slot < c.n_slots;
  const int64_t page = in ? slot / c.page_size : 0, place = page * c.page + (slot - page * c.page_size) * c.token;
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const int u = i % items, h = i / items, hk = h < c.Hk ? h : h - c.Hk;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (in) {
      const int64_t at = place + hk * c.head;
      const uint8_t* codes = (h < c.Hk ? c.k : c.v) + at + u * BITS;
      const uint32_t byte = ((h < c.Hk ? c.ks : c.vs) + at / (4 * BITS))[u / 4];
      uint2 raw = make_uint2(0, 0);
      if constexpr (BITS == 4) raw.x = *reinterpret_cast<const uint32_t*>(codes);
      else raw = *reinterpret_cast<const uint2*>(codes);
      w = mx_eight<BF16, BITS>(raw.x, raw.y, mx_scale(byte));
      if (byte == 255) w.x = w.y = w.z = w.w = 0x7fff7fffu;  // NaN in either type
    }
    *reinterpret_cast<uint4*>((h < c.Hk ? a.ko : a.vo) + (t * c.Hk + hk) * c.D + 8 * u) = w;
  }
}

hipError_t launch_mx_read(const MxReadArgs& a, bool bf16, int bits, hipStream_t st) {
  const int all = 2 * a.cache.Hk * (a.cache.D / 8), threads = std::min(256, (all + 63) / 64 * 64);
  if (!launchable(a.n, threads)) return hipErrorInvalidConfiguration;
  auto go = [&](auto b_tag, auto bits_tag) {
    note_kernel("mx_read_kernel<%d>", bits);
    hipLaunchKernelGGL((mx_read_kernel<decltype(b_tag)::value, decltype(bits_tag)::value>), dim3((unsigned)a.n), dim3(threads), 0, st, a);
    return hipGetLastError();
  };
  auto by_bits = [&](auto b_tag) {
    return bits == 4 ? go(b_tag, std::integral_constant<int, 4>{}) : go(b_tag, std::integral_constant<int, 8>{});
  };
  return bf16 ? by_bits(std::true_type{}) : by_bits(std::false_type{});
}

}  // namespace fg
