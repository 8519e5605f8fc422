// mx_tile: work items of many rows (prompts) over block-scaled keys and values.  As in attn_tile four wavefronts of 32 rows share tiles
// of 64 keys (32 for heads of more than 128 columns) of 16-bit values in two LDS buffers, with products in 32 x 32 x 16 form; a tile's
// codes pass through registers and are converted, with their scales, once per workgroup.  The loads of the next tile are on their
// way while this one is computed, its conversion stands behind the products.
#pragma once

#include "fg_attn_tile.h"
#include "fg_mx_attn.h"

namespace fg {

template <bool BF16, int BITS, bool CAP, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) mx_tile_kernel(const MxAttnArgs m_) {
  constexpr int KT = TileLds<DP>::kKeys, U = DP / 8, C = DP / 16, DB = DP / 32, TB = KT / 32, kBuf = TileLds<DP>::kBuf;
  constexpr int SU = DP * BITS / 128;                               // 16-byte units of codes per key
  constexpr int TP = 256 / SU, PASS = TP < KT ? KT / TP : 1;        // keys per pass of the workgroup, passes
  constexpr int E = 16 / BITS;                                      // 8-column units of values per unit of codes
  constexpr uint64_t kAll = KT == 64 ? ~0ull : 0xffffffffull;
  __shared__ __align__(16) uint8_t lds[TileLds<DP>::kBytes];
  uint32_t* tab = reinterpret_cast<uint32_t*>(lds + TileLds<DP>::kTab);
  const AttnArgs& a = m_.a;

  MxItem it;
  if (!mx_item<kTileRows>(m_, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, l32 = lane & 31, half = lane >> 5;
  const int n = max(it.end - it.begin, 0), tiles = (n + KT - 1) / KT;
  auto fill = [&](int from) {  // kTabHalf entries of the row table
    for (int i = from + threadIdx.x; i < from + kTabHalf; i += 256) {
      if (i >= tiles * KT) break;
      tab[i % (2 * kTabHalf)] = i < n && it.begin + i >= it.low ? attn_row(a, it, it.begin + i) : kNoRow;
    }
  };
  fill(0);

  const int row0 = it.row0 + 32 * wave, row = row0 + l32, tok = row / a.G, g = row - tok * a.G;
  const bool live = row0 < it.rows;  // this wavefront has rows
  const AttnFactor factor = attn_factor(m_.factor, 1.f);
  const uint32_t sign = CAP ? 0 : factor.sign;
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
  const int seen = it.seen0 + tok, low = seen - m_.window;                                           // keys low .. seen - 1
  const int min_seen = it.seen0 + row0 / a.G, max_low = it.seen0 + (row0 + 31) / a.G - m_.window;    // of the wavefront's rows
  const float sc = CAP ? m_.factor : factor.value, cap_in = m_.cap_in;

  f32x16 o[DB];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = (f32x16)(0.f);

  // A thread moves one unit of codes (32 or 16 columns) of PASS keys per tile; units past the head's columns stay zero in both
  // buffers.
  const int su = threadIdx.x % SU, st = threadIdx.x / SU;
  const bool mover = su * 16 < a.D * BITS / 8 && st < KT;
  const int unit = mover ? su : 0, block = unit * 128 / BITS / kMxBlock;
  const uint8_t *kb = a.k + it.head * a.c_head + unit * 16, *vb = a.v + it.head * a.c_head + unit * 16;
  const uint8_t *ksb = m_.ks + it.head * m_.s_head + block, *vsb = m_.vs + it.head * m_.s_head + block;
  // SETS tiles are on their way: one, or, where a CU has room for one workgroup only, two (heads of 256 columns, 4 prompts of up to 300
  // tokens over windows of 1024 in three parts: 87 us, one 90).  Loads stand in no branch, so that a set waits for its own only; a key
  // that is not there reads the cache's first row, a thread without a unit the row's first one.
  constexpr int SETS = DP > 128 ? 2 : 1;
  uint4 kr[SETS][PASS], vr[SETS][PASS];
  uint32_t kse[SETS][PASS], vse[SETS][PASS];
  uint64_t ok = 0, ok_next[SETS];  // which keys of the tile are there
  auto load = [&](int set, int tile) __attribute__((always_inline)) {
    tile = min(tile, tiles - 1);
    ok_next[set] = __ballot(lane < KT && tab[(tile * KT + lane) % (2 * kTabHalf)] != kNoRow);
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      uint32_t r = tab[(tile * KT + min(p * TP + st, KT - 1)) % (2 * kTabHalf)];
      r = r == kNoRow ? 0 : r;
      const uint64_t at = (uint64_t)r * 16, sat = BITS == 4 ? r : r >> 1;
      kr[set][p] = *reinterpret_cast<const uint4*>(kb + at);
      vr[set][p] = *reinterpret_cast<const uint4*>(vb + at);
      kse[set][p] = ksb[sat];
      vse[set][p] = vsb[sat];
    }
  };
  auto put = [&](uint8_t* to, int t, const uint4& w, uint32_t byte) __attribute__((always_inline)) {
    const float s = __uint_as_float(byte << 23);
    const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint4 v = BITS == 4 ? mx_eight<BF16, BITS>(c[e], 0, s) : mx_eight<BF16, BITS>(c[2 * e % 4], c[(2 * e + 1) % 4], s);
      *reinterpret_cast<uint4*>(to + (t * U + tile_unit<U>(t, E * su + e)) * 16) = v;
    }
  };
  auto store = [&](int set, uint8_t* to) __attribute__((always_inline)) {
    if (ok_next[set] != kAll) {
      asm volatile("");  // a branch, so that whole tiles skip it
#pragma unroll
      for (int p = 0; p < PASS; ++p)
        if (!(ok_next[set] >> ((p * TP + st) & 63) & 1)) {
          kr[set][p] = vr[set][p] = make_uint4(0, 0, 0, 0);
          kse[set][p] = vse[set][p] = 1;
        }
    }
    if (!mover) return;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      put(to, p * TP + st, kr[set][p], kse[set][p]);
      put(to + kBuf, p * TP + st, vr[set][p], vse[set][p]);
    }
  };
  if (a.D < DP) {
    for (int i = threadIdx.x; i < 4 * kBuf / 16; i += 256) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  if (tiles > 0) {
    load(0, 0);
    ok = ok_next[0];
    if (SETS > 1) load(SETS - 1, 1);
    store(0, lds);
  }
  // The buffer being read and the one being filled are __restrict__ pointers, so that the reads of the one do not wait for
  // the writes into the other.
  auto step = [&](int i, int set, uint8_t* __restrict__ cur, uint8_t* __restrict__ nxt) __attribute__((always_inline)) {  // set: of tile i
    const int t0 = i * KT;
    __syncthreads();
    if (t0 % kTabHalf == 0) fill(t0 + kTabHalf);  // read from the half's last tile on, behind other barriers
    if (SETS == 1) ok = ok_next[0];
    load(set, i + SETS);
    if (live) {
      f32x16 s[TB];
      s16x8 kf[3][TB];  // read two steps ahead of their products, in this order
      auto keys = [&](int c) {
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          const int t = 32 * b + l32;
          kf[c % 3][b] = *reinterpret_cast<const s16x8*>(cur + (t * U + tile_unit<U>(t, 2 * c + half)) * 16);
        }
      };
      keys(0);
      keys(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (c + 2 < C) keys(c + 2);
#pragma unroll
        for (int b = 0; b < TB; ++b) s[b] = mfma32<BF16>(kf[c % 3][b], qf[c], c ? s[b] : (f32x16)(0.f));
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (CAP) {
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[b][j] = mx_tanh(s[b][j] * cap_in);
      }
      const int first = it.begin + t0;
      if (ok != kAll || first + KT > min_seen || first < max_low) {
        // the keys that this lane's row sees, skip .. left - 1 of the tile, from its own first one on
        asm volatile("");
        const int left = seen - first, skip = low - first;
        uint64_t mask = left >= 64 ? ok : (left > 0 ? ok & ((1ull << left) - 1) : 0ull);
        if (skip > 0) mask = skip >= 64 ? 0ull : mask & ~((1ull << skip) - 1);
        mask >>= 4 * half;
        const uint32_t word[2] = {(uint32_t)mask, (uint32_t)(mask >> 32)};
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (!(word[b] >> (8 * (j / 4) + j % 4) & 1)) s[b][j] = -__builtin_inff();
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, s[b][j]);
      top = attn_top<BF16>(top, sc);
      if (__any(top > m + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - attn_base(mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= f;
      }
      const float base = attn_base(m);
      // 16 keys per step: the next step's values and weights go between the products of this one, in this order
      s16x8 vf[2][DB];
      uint32_t pw[2][4];
      auto weights = [&](int k, int j) {  // two keys
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k / 2][8 * (k % 2) + 2 * j], sc, -base));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k / 2][8 * (k % 2) + 2 * j + 1], sc, -base));
        l += x + y;
        pw[k & 1][j] = pack2<BF16>(x, y);
      };
      auto values = [&](int k, int d) {  // 32 columns
        s16x4 v2[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // each 16 lanes read 4 keys x 16 columns
          const int t = 16 * k + 8 * h + 4 * half + l16 / 4, u = 4 * d + 2 * (lane >> 4 & 1) + (l16 % 4) / 2;
          v2[h] = lds_tr16(cur + kBuf + (t * U + tile_unit<U>(t, u)) * 16 + 8 * (l16 % 2));
        }
        vf[k & 1][d] = __builtin_shufflevector(v2[0], v2[1], 0, 1, 2, 3, 4, 5, 6, 7);
      };
#pragma unroll
      for (int d = 0; d < DB; ++d) values(0, d);
#pragma unroll
      for (int j = 0; j < 4; ++j) weights(0, j);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 2 * TB; ++k) {
        const uint32_t* w = pw[k & 1];
        const s16x8 p = __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          o[d] = mfma32<BF16>(vf[k & 1][d], p, o[d]);
          if (k + 1 < 2 * TB) {
            if (d < (DB + 1) / 2) {  // early, so that they are there when the step begins
              values(k + 1, 2 * d);
              if (2 * d + 1 < DB) values(k + 1, 2 * d + 1);
            }
#pragma unroll
            for (int j = d * 4 / DB; j < (d + 1) * 4 / DB; ++j) weights(k + 1, j);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (SETS > 1) ok = ok_next[SETS - 1 - set];
    if (i + 1 < tiles) store(SETS - 1 - set, nxt);
  };
  for (int i = 0; i < tiles; i += 2) {  // the buffers' places are constants of the reads' addresses
    step(i, 0, lds, lds + 2 * kBuf);
    if (i + 1 < tiles) step(i + 1, SETS - 1, lds + 2 * kBuf, lds);
  }

  const float sum = l + __shfl_xor(l, 32, kWave);
  if (row >= it.rows) return;
  const int64_t t = it.token0 + tok;
  const int h = it.head * a.G + g;
  const int64_t at = ((int64_t)it.slot * a.T + t) * a.Hq + h;
  const float f = a.acc ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);  // a row that saw no key gives zeros
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const int col = 32 * d + 2 * j + 4 * half;
      if (col >= a.D) continue;
      const f32x4 w = {o[d][j] * f, o[d][j + 1] * f, o[d][j + 2] * f, o[d][j + 3] * f};
      if (a.acc) {
        *reinterpret_cast<f32x4*>(a.acc + at * a.D + col) = w;
      } else {
        const uint2 b = make_uint2(pack2<BF16>(w[0], w[1]), pack2<BF16>(w[2], w[3]));
        __builtin_memcpy(__builtin_assume_aligned(a.out + t * a.o_t + h * a.o_h + col, 2), &b, 8);
      }
    }
  if (half == 0) {
    if (a.acc) a.ml[at] = make_float2(m, sum);
    else if (a.lse) a.lse[t * a.Hq + h] = (m + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
  }
}

}  // namespace fg
