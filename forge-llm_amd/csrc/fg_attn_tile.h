// attn_tile: work items of many rows: the shared prefix of a batch, or prompts of several tokens.
//
// Four wavefronts of 32 rows share tiles of 64 keys (32 for heads of more than 128 columns) in LDS.  The products are those of
// attn_rows in 32 x 32 x 16 form: S^T = K Q^T leaves a row's scores in the two lanes l, l + 32, keys 8 a + 4 (l / 32) + b in
// register 4 a + b, and O^T += V^T P^T takes them as they are, V^T by transposing reads in the same key order.  The next tile
// is on its way to the other LDS buffer while this one is computed: one barrier per tile.  16-bit tiles go straight to LDS;
// e4m3 ones, and heads that do not fill DP columns, pass through registers, where e4m3 becomes 16-bit, once per workgroup.
//
// Bound by the matrix products and, beside them, by the vector instructions: per 64 keys and wavefront 32 products (1024
// cycles) and about 240 others (by the counters), 32 of them exponentials.  A fragment is read from LDS two steps before its
// product, the exponentials of 16 keys stand between the products of the 16 before, and two workgroups per CU fill each
// other's waits.
// Measured on 2048 rows x 8 key heads x 32768 keys of 128 columns: about 265 us, 1.0 PFLOP/s (a large library product: 1.2).  64
// rows per wavefront, which would halve the LDS reads, needs more than 256 registers and spends what it gains on moves to and
// from the accumulation registers; through registers instead of straight to LDS a tile costs 10% more.
#pragma once

#include "fg_attn.h"

namespace fg {

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

// LDS: two buffers of keys, then values; then the row table.
template <int DP>
struct TileLds {
  static constexpr int kKeys = DP > 128 ? 32 : 64, kBuf = kKeys * DP * 2;
  static constexpr int kTab = 4 * kBuf, kBytes = kTab + 2 * kTabHalf * 4;
};

// DIRECT (16-bit keys, all DP columns there): tiles go straight to LDS.
template <bool BF16, bool FP8, bool DIRECT, int DP>
__device__ __forceinline__ void attn_tile(const AttnArgs& a, int id, uint8_t* lds) {
  constexpr int KT = TileLds<DP>::kKeys, U = DP / 8, C = DP / 16, DB = DP / 32, TB = KT / 32, kBuf = TileLds<DP>::kBuf;
  constexpr int SU = FP8 ? DP / 16 : U;         // 16-byte units per key in memory
  constexpr int TP = 256 / SU, PASS = KT / TP;  // keys per pass of the workgroup, passes
  constexpr uint64_t kAll = KT == 64 ? ~0ull : 0xffffffffull;
  uint32_t* tab = reinterpret_cast<uint32_t*>(lds + TileLds<DP>::kTab);

  AttnItem it;
  if (!attn_item<kTileRows>(a, id, it)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, l32 = lane & 31, half = lane >> 5;
  const int n = max(it.end - it.begin, 0), tiles = (n + KT - 1) / KT;
  auto fill = [&](int from) {  // kTabHalf entries of the row table
    for (int i = from + threadIdx.x; i < from + kTabHalf; i += 256) {
      if (i >= tiles * KT) break;
      tab[i % (2 * kTabHalf)] = i < n ? attn_row(a, it, it.begin + i) : kNoRow;
    }
  };
  fill(0);

  const int row0 = it.row0 + 32 * wave, row = row0 + l32, tok = row / a.G, g = row - tok * a.G;
  const bool live = row0 < it.rows;  // this wavefront has rows
  const AttnFactor factor = attn_factor(a.scale_log2, FP8 ? a.ks[it.head] : 1.f);
  const uint32_t sign = factor.sign;
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
  const int seen = it.causal ? max(it.seen0 + tok, it.front) : it.end;
  const int min_seen = it.causal ? max(it.seen0 + row0 / a.G, it.front) : it.end;  // what the wavefront's first row sees
  const float sc = factor.value;

  f32x16 o[DB];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = (f32x16)(0.f);

  // A thread moves one unit of PASS keys per tile: straight to its place in the LDS buffer (the unit whose place that is), or
  // through registers, where units past the head's columns stay zero in both buffers.
  const int units = a.D * (FP8 ? 1 : 2) / 16, su = threadIdx.x % SU, st = threadIdx.x / SU;
  const bool mover = DIRECT || su < units;
  const uint8_t *kb = a.k + it.head * a.c_head, *vb = a.v + it.head * a.c_head;
  uint4 kr[PASS], vr[PASS];
  uint64_t ok = 0, ok_next = 0;  // which keys of the tile are there
  auto load = [&](int tile, uint8_t* to) __attribute__((always_inline)) {
    ok_next = __ballot(lane < KT && tab[(tile * KT + lane) % (2 * kTabHalf)] != kNoRow);
    if (!mover) return;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int t = p * TP + st;
      uint32_t r = tab[(tile * KT + t) % (2 * kTabHalf)];
      r = r == kNoRow ? 0 : r;
      const uint64_t at = (uint64_t)r * 16 + (DIRECT ? tile_unit<U>(t, su) : su) * 16;
      if constexpr (DIRECT) {
        __builtin_amdgcn_global_load_lds(kb + at, to + (p * 256 + wave * 64) * 16, 16, 0, 0);
        __builtin_amdgcn_global_load_lds(vb + at, to + kBuf + (p * 256 + wave * 64) * 16, 16, 0, 0);
      } else {
        kr[p] = *reinterpret_cast<const uint4*>(kb + at);
        vr[p] = *reinterpret_cast<const uint4*>(vb + at);
      }
    }
  };
  auto store = [&](uint8_t* to) __attribute__((always_inline)) {
    if constexpr (DIRECT) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      return;
    }
    if (ok_next != kAll) {
      asm volatile("");  // a branch, so that whole tiles skip it
#pragma unroll
      for (int p = 0; p < PASS; ++p)
        if (!(ok_next >> (p * TP + st) & 1)) kr[p] = vr[p] = make_uint4(0, 0, 0, 0);
    }
    if (!mover) return;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int t = p * TP + st;
      if constexpr (FP8) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = (t * U + tile_unit<U>(t, 2 * su + e)) * 16;
          *reinterpret_cast<s16x8*>(to + at) = e ? e4m3_to_16<BF16>(kr[p].z, kr[p].w) : e4m3_to_16<BF16>(kr[p].x, kr[p].y);
          *reinterpret_cast<s16x8*>(to + kBuf + at) = e ? e4m3_to_16<BF16>(vr[p].z, vr[p].w) : e4m3_to_16<BF16>(vr[p].x, vr[p].y);
        }
      } else {
        const int at = (t * U + tile_unit<U>(t, su)) * 16;
        *reinterpret_cast<uint4*>(to + at) = kr[p];
        *reinterpret_cast<uint4*>(to + kBuf + at) = vr[p];
      }
    }
  };
  if (a.D < DP) {
    for (int i = threadIdx.x; i < 4 * kBuf / 16; i += 256) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  if (tiles > 0) {
    load(0, lds);
    store(lds);
  }
  // The buffer being read and the one being filled are __restrict__ pointers, so that the reads of the one do not wait for
  // the loads into the other.
  auto step = [&](int i, uint8_t* __restrict__ cur, uint8_t* __restrict__ nxt) __attribute__((always_inline)) {
    const int t0 = i * KT;
    __syncthreads();
    if (t0 % kTabHalf == 0) fill(t0 + kTabHalf);  // read from the half's last tile on, behind other barriers
    ok = ok_next;
    if (DIRECT && ok != kAll) {  // what was loaded for keys that are not there: weights of zero do not undo a NaN
      for (int j = threadIdx.x; j < KT * U; j += 256)
        if (!(ok >> (j / U) & 1)) reinterpret_cast<uint4*>(cur + kBuf)[j] = make_uint4(0, 0, 0, 0);
      __syncthreads();
    }
    if (i + 1 < tiles) load(i + 1, nxt);
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
      if (ok != kAll || it.begin + t0 + KT > min_seen) {
        // the keys that this lane's row sees, from its own first one on
        asm volatile("");
        const int left = seen - (it.begin + t0);
        const uint64_t mask = (left >= 64 ? ok : (left > 0 ? ok & ((1ull << left) - 1) : 0ull)) >> (4 * half);
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
    if (DIRECT || i + 1 < tiles) store(nxt);  // DIRECT: its wait stands on every path to the barrier
  };
  for (int i = 0; i < tiles; i += 2) {  // the buffers' places are constants of the reads' addresses
    step(i, lds, lds + 2 * kBuf);
    if (i + 1 < tiles) step(i + 1, lds + 2 * kBuf, lds);
  }

  const float sum = l + __shfl_xor(l, 32, kWave), vs = FP8 ? a.vs[it.head] : 1.f;
  if (row >= it.rows) return;
  const int64_t t = it.token0 + tok;
  const int h = it.head * a.G + g;
  const int64_t at = ((int64_t)it.slot * a.T + t) * a.Hq + h;
  const float f = a.acc ? vs : (sum == 0.f ? 0.f : vs / sum);  // a row that saw no key gives zeros
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
