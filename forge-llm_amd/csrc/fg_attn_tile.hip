// Attention over a paged cache for work items of many rows: the shared prefix of a batch, or prompts of several tokens.
//
// Four wavefronts of 32 rows share tiles of 64 keys (32 for heads of more than 128 columns) in LDS.  The products are those of
// attn_rows_kernel in 32 x 32 x 16 form: S^T = K Q^T leaves a row's scores in the two lanes l, l + 32, keys 8 a + 4 (l / 32) + b
// in register 4 a + b, and O^T += V^T P^T takes them as they are, V^T by transposing reads in the same key order.  The next
// tile's keys and values are on their way to registers while this one is computed, and go to the other LDS buffer after it: one
// barrier per tile.  e4m3 keys and values become 16-bit on that way, once per workgroup.
//
// Bound by the matrix products and, beside them, by the exponentials and the LDS reads: per 64 keys and wavefront 32 products
// (1024 cycles), 32 exponentials and 32 KiB from LDS.  Two workgroups per CU fill each other's waits.
#include <algorithm>

#include "fg_attn.h"

namespace fg {

namespace {

constexpr int kTileRows = 128;
constexpr int kTabHalf = 1024;  // keys per half of the row table: one half is read while the other is filled

// Unit u of key t in a tile whose rows hold U 16-byte units: the reads of 16 keys of one unit (keys) and of 4 keys x 4 units
// (values, transposed) both spread over all banks.
template <int U>
__device__ __forceinline__ int tile_unit(int t, int u) {
  if constexpr (U >= 16) return u ^ ((t & 3) << 2 | (t >> 2 & 3));
  return u ^ ((t >> 1 & 1) << 2 | (t >> 2 & 3));
}

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(const s16x8& x, const s16x8& y, const f32x16& c) {
  if constexpr (BF16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, x), __builtin_bit_cast(v8, y), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, x), __builtin_bit_cast(v8, y), c, 0, 0, 0);
  }
}

}  // namespace

template <bool BF16, bool FP8, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attn_tile_kernel(const AttnArgs a, int first, int count) {
  constexpr int KT = DP > 128 ? 32 : 64, U = DP / 8, C = DP / 16, DB = DP / 32, TB = KT / 32;
  constexpr int SU = FP8 ? DP / 16 : U;                // 16-byte units per key in memory
  constexpr int TP = 256 / SU, PASS = KT / TP;         // keys per pass of the workgroup, passes
  constexpr int kBuf = KT * DP * 2;
  __shared__ __align__(16) uint8_t lds[2][2][kBuf];    // [buffer][keys, values]
  __shared__ uint32_t tab[2 * kTabHalf];

  // items that share keys (row tiles of one part) go to one XCD, one after the other
  int id = blockIdx.x;
  const int per = count / 8;
  if (id < per * 8) id = (id % 8) * per + id / 8;
  AttnItem it;
  if (!attn_item<kTileRows>(a, first + id, it)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, l32 = lane & 31, half = lane >> 5;
  const int n = max(it.end - it.begin, 0), tiles = (n + KT - 1) / KT;
  auto fill = [&](int from) {  // kTabHalf entries of the row table
    for (int i = from + threadIdx.x; i < from + kTabHalf; i += 256) {
      if (i >= (n + KT - 1) / KT * KT) break;
      tab[i % (2 * kTabHalf)] = i < n ? attn_row(a, it, it.begin + i) : kNoRow;
    }
  };
  fill(0);

  const int row = it.row0 + 32 * wave + l32, tok = row / a.G, g = row - tok * a.G;
  const bool live = it.row0 + 32 * wave < it.rows;  // this wavefront has rows
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  s16x8 qf[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    uint4 u = make_uint4(0, 0, 0, 0);
    const int d = 16 * c + 8 * half;
    if (row < it.rows && d < a.D) {
      const uint16_t* qp = a.q + (int64_t)(it.token0 + tok) * a.q_t + (int64_t)(it.head * a.G + g) * a.q_h;
      __builtin_memcpy(&u, __builtin_assume_aligned(qp + d, 2), 16);
    }
    u.x ^= sign; u.y ^= sign; u.z ^= sign; u.w ^= sign;
    qf[c] = __builtin_bit_cast(s16x8, u);
  }
  const int seen = it.causal ? it.seen0 + tok : it.end;
  const int min_seen = it.causal ? it.seen0 + (it.row0 + 32 * wave) / a.G : it.end;
  const float sc = fabsf(a.scale_log2) * (FP8 ? a.ks[it.head] : 1.f);
  const uint8_t *kb = a.k + it.head * a.c_head, *vb = a.v + it.head * a.c_head;
  const int units = a.D * (FP8 ? 1 : 2) / 16, su = threadIdx.x % SU, st = threadIdx.x / SU;

  f32x16 o[DB];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  uint4 kr[PASS], vr[PASS];
  auto load = [&](int tile) {
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const uint32_t r = tab[(tile * KT + p * TP + st) % (2 * kTabHalf)];
      const bool in = r != kNoRow && su < units;
      kr[p] = in ? attn_ld16(kb, r, su) : make_uint4(0, 0, 0, 0);
      vr[p] = in ? attn_ld16(vb, r, su) : make_uint4(0, 0, 0, 0);
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int t = p * TP + st;
      if constexpr (FP8) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = (t * U + tile_unit<U>(t, 2 * su + e)) * 16;
          *reinterpret_cast<s16x8*>(lds[buf][0] + at) = e ? e4m3_to_16<BF16>(kr[p].z, kr[p].w) : e4m3_to_16<BF16>(kr[p].x, kr[p].y);
          *reinterpret_cast<s16x8*>(lds[buf][1] + at) = e ? e4m3_to_16<BF16>(vr[p].z, vr[p].w) : e4m3_to_16<BF16>(vr[p].x, vr[p].y);
        }
      } else {
        const int at = (t * U + tile_unit<U>(t, su)) * 16;
        *reinterpret_cast<uint4*>(lds[buf][0] + at) = kr[p];
        *reinterpret_cast<uint4*>(lds[buf][1] + at) = vr[p];
      }
    }
  };
  __syncthreads();
  if (tiles > 0) {
    load(0);
    store(0);
  }
  for (int i = 0; i < tiles; ++i) {
    const int t0 = i * KT, buf = i & 1;
    __syncthreads();
    if (t0 % kTabHalf == 0) fill(t0 + kTabHalf);  // read from the half's last tile on, behind other barriers
    if (i + 1 < tiles) load(i + 1);
    const uint64_t ok = __ballot(lane < KT && tab[(t0 + lane) % (2 * kTabHalf)] != kNoRow);
    if (live) {
      f32x16 s[TB];
#pragma unroll
      for (int b = 0; b < TB; ++b) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[b][j] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int t = 32 * b + l32;
          const s16x8 kf = *reinterpret_cast<const s16x8*>(lds[buf][0] + (t * U + tile_unit<U>(t, 2 * c + half)) * 16);
          s[b] = mfma32<BF16>(kf, qf[c], s[b]);
        }
      }
      if (ok != (KT == 64 ? ~0ull : 0xffffffffull) || it.begin + t0 + KT > min_seen) {
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int t = 32 * b + 8 * (j / 4) + 4 * half + j % 4;
            if (!(ok >> t & 1) || it.begin + t0 + t >= seen) s[b][j] = -__builtin_inff();
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, s[b][j]);
      top *= sc;
      if (__any(top > m + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - attn_base(mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= f;
      }
      const float base = attn_base(m);
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // 16 keys
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * e + j], sc, -base));
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * e + j + 1], sc, -base));
            sum += x + y;
            w[j / 2] = pack2<BF16>(x, y);
          }
          const s16x8 pf = __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            s16x4 v2[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // each 16 lanes read 4 keys x 16 columns
              const int t = 32 * b + 16 * e + 8 * h + 4 * half + l16 / 4, u = 4 * d + 2 * (lane >> 4 & 1) + (l16 % 4) / 2;
              v2[h] = lds_tr16(lds[buf][1] + (t * U + tile_unit<U>(t, u)) * 16 + 8 * (l16 % 2));
            }
            o[d] = mfma32<BF16>(__builtin_shufflevector(v2[0], v2[1], 0, 1, 2, 3, 4, 5, 6, 7), pf, o[d]);
          }
        }
      l += sum;
    }
    if (i + 1 < tiles) store(buf ^ 1);
  }
  l += __shfl_xor(l, 32, kWave);
  if (row >= it.rows) return;
  const int64_t t = it.token0 + tok;
  const int h = it.head * a.G + g;
  const float vs = FP8 ? a.vs[it.head] : 1.f;
  if (a.acc) {
    const int64_t at = ((int64_t)it.slot * a.T + t) * a.Hq + h;
    if (half == 0) a.ml[at] = make_float2(m, l);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const int col = 32 * d + 2 * j + 4 * half;
        if (col < a.D)
          *reinterpret_cast<f32x4*>(a.acc + at * a.D + col) = (f32x4){o[d][j] * vs, o[d][j + 1] * vs, o[d][j + 2] * vs, o[d][j + 3] * vs};
      }
  } else {
    const float f = l == 0.f ? 0.f : vs / l;
    uint16_t* op = a.out + t * a.o_t + h * a.o_h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const int col = 32 * d + 2 * j + 4 * half;
        if (col < a.D) {
          const uint2 w = make_uint2(pack2<BF16>(o[d][j] * f, o[d][j + 1] * f), pack2<BF16>(o[d][j + 2] * f, o[d][j + 3] * f));
          __builtin_memcpy(__builtin_assume_aligned(op + col, 2), &w, 8);
        }
      }
    if (a.lse && half == 0) a.lse[t * a.Hq + h] = (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
  }
}

hipError_t launch_attn_tile(const AttnArgs& a, bool bf16, bool fp8, int first, int count, hipStream_t st) {
  auto go = [&](auto b_tag, auto f_tag, auto d_tag) {
    hipLaunchKernelGGL((attn_tile_kernel<decltype(b_tag)::value, decltype(f_tag)::value, decltype(d_tag)::value>),
                       dim3((unsigned)count), dim3(256), 0, st, a, first, count);
    return hipGetLastError();
  };
  auto by_d = [&](auto b_tag, auto f_tag) {
    if (a.D <= 64) return go(b_tag, f_tag, std::integral_constant<int, 64>{});
    if (a.D <= 128) return go(b_tag, f_tag, std::integral_constant<int, 128>{});
    return go(b_tag, f_tag, std::integral_constant<int, 256>{});
  };
  auto by_f = [&](auto b_tag) { return fp8 ? by_d(b_tag, std::true_type{}) : by_d(b_tag, std::false_type{}); };
  return bf16 ? by_f(std::true_type{}) : by_f(std::false_type{});
}

}  // namespace fg
