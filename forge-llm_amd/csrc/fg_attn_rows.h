// attn_rows: work items of up to 16 rows (decoding).  What bounds them is the read of the keys and values (256 sequences of 256
// to 2048 tokens, 8 key heads of 128 in bf16: 225 us, 5.4 TB/s; a workgroup by itself reads about 34 bytes per ns), so each wavefront
// works by itself on tiles of 32 keys, without a barrier, with the loads of the next tile and the one after on their way.
//   S^T = K Q^T   (A: 16 keys x 32 columns straight from global memory, 16 bytes per lane; B: the rows, in registers)
//   O^T += V^T P^T
// S^T comes out with a row in each lane and keys 4 g + i (g the lane's group of 16) in its registers, which is the order in
// which the second product takes P^T if V^T is read in the same order: P goes from the first product to the second without
// leaving the lane.  V^T needs columns of V, so V passes through LDS and comes back through the transposing read.
#pragma once

#include "fg_attn.h"

namespace fg {

// 16-byte unit u of key t in a V tile whose rows hold U units: an exchange of units that depends on the key, so that both
// the writes (16 keys, one unit) and the transposing reads (8 keys, 32 bytes) spread over all banks.
template <int U>
__device__ __forceinline__ int rows_unit(int t, int u) {
  if constexpr (U >= 16) return u ^ ((t & 7) << 1 | ((t >> 3 ^ t >> 4) & 1));
  if constexpr (U == 8) return u ^ ((t >> 1 & 3) << 1 | ((t >> 3 ^ t >> 4) & 1));
  return u ^ ((t >> 2 & 1) << 1 | ((t >> 3 ^ t >> 4) & 1));
}

// LDS: a V tile per wavefront, later their sums; then the row table; then the wavefronts' maxima and sums.
template <bool FP8, int DP>
struct RowsLds {
  static constexpr int kV = kRowsTile * DP * (FP8 ? 1 : 2), kO = 16 * DP * 4;
  static constexpr int kTab = kRowsWaves * (kV > kO ? kV : kO), kRed = kTab + kMaxPart * 4;
  static constexpr int kBytes = kRed + 2 * kRowsWaves * 16 * 4;
};

// DP: head columns in registers (D of them are there).
template <bool BF16, bool FP8, int DP>
__device__ __forceinline__ void attn_rows(const AttnArgs& a, int id, uint8_t* lds) {
  constexpr int IT = FP8 ? 1 : 2, U = DP * IT / 16, C = DP / 32, DB = DP / 16;
  constexpr int KU = U / 4;  // 16-byte loads of a lane per key
  using L = RowsLds<FP8, DP>;
  uint32_t* tab = reinterpret_cast<uint32_t*>(lds + L::kTab);
  float* red = reinterpret_cast<float*>(lds + L::kRed);

  AttnItem it;
  if (!attn_item<16>(a, id, it)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, grp = lane >> 4;
  attn_row_table(a, it, tab, kRowsTile);

  // this lane's row: the fragment of Q, and the keys it sees
  const int row = it.row0 + l16, tok = row / a.G, g = row - tok * a.G;
  const uint16_t* qp = a.q + (int64_t)(it.token0 + tok) * a.q_t + (int64_t)(it.head * a.G + g) * a.q_h;
  const AttnFactor factor = attn_factor(a.scale_log2, FP8 ? a.ks[it.head] : 1.f);
  const uint32_t sign = factor.sign;
  s16x8 qf[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    // e4m3 keys come 16 columns per load, which makes two chunks
    const int d = FP8 ? 64 * (c / 2) + 16 * grp + 8 * (c % 2) : 32 * c + 8 * grp;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (row < it.rows && d < a.D) __builtin_memcpy(&u, __builtin_assume_aligned(qp + d, 2), 16);
    u.x ^= sign; u.y ^= sign; u.z ^= sign; u.w ^= sign;
    qf[c] = __builtin_bit_cast(s16x8, u);
  }
  const int seen = it.causal ? max(it.seen0 + tok, it.front) : it.end;
  const int min_seen = it.causal ? max(it.seen0 + it.row0 / a.G, it.front) : it.end;  // what the tile's first row sees
  const float sc = factor.value;
  const uint8_t *kb = a.k + it.head * a.c_head + grp * 16, *vb = a.v + it.head * a.c_head + grp * 16;
  const int units = a.D * IT / 16;

  f32x4 o[DB];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  __syncthreads();

  const int n = max(it.end - it.begin, 0), step = kRowsTile * kRowsWaves;
  uint8_t* vl = lds + wave * L::kV;
  // NB tiles in registers: with two, one is computed while the other is on its way (256 columns leave room for one: the next
  // is loaded behind the products that used it)
  constexpr int NB = DP > 128 ? 1 : 2;
  uint4 kr[NB][2][KU], vr[NB][2][KU];
  uint32_t ok[NB];  // bit t: key t of the tile is there
  auto fetch = [&](int b, int t0) __attribute__((always_inline)) {
    const uint32_t rows[2] = {tab[t0 + l16], tab[t0 + 16 + l16]};
    ok[b] = (uint32_t)(__ballot(rows[0] != kNoRow) & 0xffff) | (uint32_t)(__ballot(rows[1] != kNoRow) & 0xffff) << 16;
    if (ok[b] == 0xffffffffu && a.D == DP) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < KU; ++c) {
          const uint64_t at = (uint64_t)rows[h] * 16 + c * 64;
          kr[b][h][c] = *reinterpret_cast<const uint4*>(kb + at);
          vr[b][h][c] = *reinterpret_cast<const uint4*>(vb + at);
        }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < KU; ++c) {
          kr[b][h][c] = vr[b][h][c] = make_uint4(0, 0, 0, 0);
          if (rows[h] != kNoRow && 4 * c + grp < units) {
            const uint64_t at = (uint64_t)rows[h] * 16 + c * 64;
            kr[b][h][c] = *reinterpret_cast<const uint4*>(kb + at);
            vr[b][h][c] = *reinterpret_cast<const uint4*>(vb + at);
          }
        }
    }
  };
  auto turn = [&](int b, int t0) __attribute__((always_inline)) {
    const uint32_t here = ok[b];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < KU; ++c) {
        const int t = 16 * h + l16;
        *reinterpret_cast<uint4*>(vl + (t * U + rows_unit<U>(t, 4 * c + grp)) * 16) = vr[b][h][c];
      }
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        s16x8 kf;
        if constexpr (FP8) {
          const uint4& u = kr[b][h][c / 2];
          kf = c % 2 ? e4m3_to_16<BF16>(u.z, u.w) : e4m3_to_16<BF16>(u.x, u.y);
        } else {
          kf = __builtin_bit_cast(s16x8, kr[b][h][c]);
        }
        s[h] = mfma16<BF16>(kf, qf[c], c ? s[h] : (f32x4)(0.f));
      }
    if (t0 + NB * step < n) fetch(b, t0 + NB * step);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = s[j / 4][j % 4];
    if (here != 0xffffffffu || it.begin + t0 + kRowsTile > min_seen) {
      asm volatile("");  // a branch, so that whole tiles skip it
      const int left = seen - (it.begin + t0);  // keys of the tile that this lane's row sees
      const uint32_t mask = (left >= 32 ? here : (left > 0 ? here & ((1u << left) - 1) : 0u)) >> (4 * grp);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!(mask >> (16 * (j / 4) + j % 4) & 1)) x[j] = -__builtin_inff();
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
    top = attn_top<BF16>(top, sc);
    if (__any(top > m + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - attn_base(mn));
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= f;
    }
    const float base = attn_base(m);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], sc, -base));
    l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack2<BF16>(x[2 * j], x[2 * j + 1]);
    const s16x8 p = __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3]));
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      s16x8 vf;
      if constexpr (FP8) {
        // 16 lanes read 8 keys x 16 columns: keys 4 g + 0..3 of either half of the tile
        const int j = l16 / 2, t = 16 * (j / 4) + 4 * grp + j % 4;
        const i32x2 c = lds_tr8(vl + (t * U + rows_unit<U>(t, d)) * 16 + 8 * (l16 % 2));
        vf = e4m3_to_16<BF16>((uint32_t)c[0], (uint32_t)c[1]);
      } else {
        s16x4 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 16 lanes read 4 keys x 16 columns
          const int t = 16 * h + 4 * grp + l16 / 4;
          half[h] = lds_tr16(vl + (t * U + rows_unit<U>(t, 2 * d + (l16 % 4) / 2)) * 16 + 8 * (l16 % 2));
        }
        vf = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
      o[d] = mfma16<BF16>(vf, p, o[d]);
    }
    __builtin_amdgcn_wave_barrier();
  };
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (wave * kRowsTile + b * step < n) fetch(b, wave * kRowsTile + b * step);
  for (int t0 = wave * kRowsTile; t0 < n; t0 += NB * step) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (t0 + b * step < n) turn(b, t0 + b * step);
  }

  // join the wavefronts: maxima and sums first, then each adds up a quarter of the columns
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (grp == 0) {
    red[wave * 16 + l16] = m;
    red[(kRowsWaves + wave) * 16 + l16] = l;
  }
  __syncthreads();
  float top = red[l16], sum = 0.f;
#pragma unroll
  for (int w = 1; w < kRowsWaves; ++w) top = fmaxf(top, red[w * 16 + l16]);
  const float base = attn_base(top);
#pragma unroll
  for (int w = 0; w < kRowsWaves; ++w)
    sum += red[(kRowsWaves + w) * 16 + l16] * __builtin_amdgcn_exp2f(red[w * 16 + l16] - base);
  const float f = __builtin_amdgcn_exp2f(m - base);
  f32x4* ol = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int d = 0; d < DB; ++d) ol[(wave * DB + d) * 64 + lane] = o[d] * f;
  __syncthreads();
  if (row >= it.rows) return;
  const int64_t t = it.token0 + tok;
  const int h = it.head * a.G + g;
  const float vs = FP8 ? a.vs[it.head] : 1.f;
  const int64_t at = ((int64_t)it.slot * a.T + t) * a.Hq + h;
  const float inv = a.acc ? vs : (sum == 0.f ? 0.f : vs / sum);  // a row that saw no key gives zeros
#pragma unroll
  for (int e = 0; e < DB / kRowsWaves; ++e) {
    const int d = e * kRowsWaves + wave, col = 16 * d + 4 * grp;
    if (col >= a.D) continue;
    f32x4 r = ol[d * 64 + lane];
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) r += ol[(w * DB + d) * 64 + lane];
    r *= inv;
    if (a.acc) {
      *reinterpret_cast<f32x4*>(a.acc + at * a.D + col) = r;
    } else {
      const uint2 w = make_uint2(pack2<BF16>(r[0], r[1]), pack2<BF16>(r[2], r[3]));
      __builtin_memcpy(__builtin_assume_aligned(a.out + t * a.o_t + h * a.o_h + col, 2), &w, 8);
    }
  }
  if (wave == 0 && grp == 0) {
    if (a.acc) a.ml[at] = make_float2(top, sum);
    else if (a.lse) a.lse[t * a.Hq + h] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
  }
}

}  // namespace fg
