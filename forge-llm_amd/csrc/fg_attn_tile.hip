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

// DIRECT (16-bit keys, all DP columns there): tiles go straight to LDS.
template <bool BF16, bool FP8, bool DIRECT, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attn_tile_kernel(const AttnArgs a, int first, int count) {
  constexpr int KT = DP > 128 ? 32 : 64, U = DP / 8, C = DP / 16, DB = DP / 32, TB = KT / 32;
  constexpr int SU = FP8 ? DP / 16 : U;                // 16-byte units per key in memory
  constexpr int TP = 256 / SU, PASS = KT / TP;         // keys per pass of the workgroup, passes
  constexpr int kBuf = KT * DP * 2;
  constexpr int RB = 1;
  constexpr uint64_t kAll = KT == 64 ? ~0ull : 0xffffffffull;
  __shared__ __align__(16) uint8_t lds[2][2 * kBuf];   // two buffers of keys, then values
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
      if (i >= tiles * KT) break;
      tab[i % (2 * kTabHalf)] = i < n ? attn_row(a, it, it.begin + i) : kNoRow;
    }
  };
  fill(0);

  const int row0 = it.row0 + 32 * RB * wave;
  const bool live = row0 < it.rows;  // this wavefront has rows
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  s16x8 qf[RB][C];
  int seen[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + 32 * r + l32, tok = row / a.G, g = row - tok * a.G;
    seen[r] = it.causal ? it.seen0 + tok : it.end;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint4 u = make_uint4(0, 0, 0, 0);
      const int d = 16 * c + 8 * half;
      if (row < it.rows && d < a.D) {
        const uint16_t* qp = a.q + (int64_t)(it.token0 + tok) * a.q_t + (int64_t)(it.head * a.G + g) * a.q_h;
        __builtin_memcpy(&u, __builtin_assume_aligned(qp + d, 2), 16);
      }
      u.x ^= sign; u.y ^= sign; u.z ^= sign; u.w ^= sign;
      qf[r][c] = __builtin_bit_cast(s16x8, u);
    }
  }
  const int min_seen = it.causal ? it.seen0 + row0 / a.G : it.end;
  const float sc = fabsf(a.scale_log2) * (FP8 ? a.ks[it.head] : 1.f);

  f32x16 o[RB][DB];
  float m[RB], l[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = -__builtin_inff();
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[r][d] = (f32x16)(0.f);
  }

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
    load(0, lds[0]);
    store(lds[0]);
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
      f32x16 s[RB][TB];
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
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int b = 0; b < TB; ++b) s[r][b] = mfma32<BF16>(kf[c % 3][b], qf[r][c], c ? s[r][b] : (f32x16)(0.f));
        __builtin_amdgcn_sched_barrier(0);
      }
      if (ok != kAll || it.begin + t0 + KT > min_seen) {
        // the keys that this lane's rows see, from its own first one on
        asm volatile("");
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const int left = seen[r] - (it.begin + t0);
          const uint64_t mask = (left >= 64 ? ok : (left > 0 ? ok & ((1ull << left) - 1) : 0ull)) >> (4 * half);
          const uint32_t word[2] = {(uint32_t)mask, (uint32_t)(mask >> 32)};
#pragma unroll
          for (int b = 0; b < TB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (!(word[b] >> (8 * (j / 4) + j % 4) & 1)) s[r][b][j] = -__builtin_inff();
        }
      }
      float top[RB], base[RB];
      bool above = false;
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        top[r] = s[r][0][0];
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j) top[r] = fmaxf(top[r], s[r][b][j]);
        top[r] *= sc;
        above |= top[r] > m[r] + kSlack;
      }
      if (__any(above)) {
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor(top[r], 32, kWave));
          const float mn = fmaxf(m[r], top[r]), f = __builtin_amdgcn_exp2f(m[r] - attn_base(mn));
          m[r] = mn;
          l[r] *= f;
#pragma unroll
          for (int d = 0; d < DB; ++d) o[r][d] *= f;
        }
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) base[r] = attn_base(m[r]);
      // 16 keys per step: the next step's values and weights go between the products of this one, in this order
      s16x8 vf[2][DB];
      uint32_t pw[RB][2][4];
      auto weights = [&](int r, int k, int j) {  // two keys
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][k / 2][8 * (k % 2) + 2 * j], sc, -base[r]));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][k / 2][8 * (k % 2) + 2 * j + 1], sc, -base[r]));
        l[r] += x + y;
        pw[r][k & 1][j] = pack2<BF16>(x, y);
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
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) weights(r, 0, j);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 2 * TB; ++k) {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            const uint32_t* w = pw[r][k & 1];
            o[r][d] = mfma32<BF16>(vf[k & 1][d], __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3])), o[r][d]);
            if (k + 1 < 2 * TB) {
              if (r == 0 && d < (DB + 1) / 2) {  // early, so that they are there when the step begins
                values(k + 1, 2 * d);
                if (2 * d + 1 < DB) values(k + 1, 2 * d + 1);
              }
#pragma unroll
              for (int j = d * 4 / DB; j < (d + 1) * 4 / DB; ++j) weights(r, k + 1, j);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    if (i + 1 < tiles) store(nxt);
  };
  for (int i = 0; i < tiles; ++i) step(i, lds[i & 1], lds[~i & 1]);
  const float vs = FP8 ? a.vs[it.head] : 1.f;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const float sum = l[r] + __shfl_xor(l[r], 32, kWave);
    const int row = row0 + 32 * r + l32, tok = row / a.G;
    if (row >= it.rows) continue;
    const int64_t t = it.token0 + tok;
    const int h = it.head * a.G + row - tok * a.G;
    if (a.acc) {
      const int64_t at = ((int64_t)it.slot * a.T + t) * a.Hq + h;
      if (half == 0) a.ml[at] = make_float2(m[r], sum);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const int col = 32 * d + 2 * j + 4 * half;
          const f32x4 w = {o[r][d][j] * vs, o[r][d][j + 1] * vs, o[r][d][j + 2] * vs, o[r][d][j + 3] * vs};
          if (col < a.D) *reinterpret_cast<f32x4*>(a.acc + at * a.D + col) = w;
        }
    } else {
      const float f = sum == 0.f ? 0.f : vs / sum;
      uint16_t* op = a.out + t * a.o_t + h * a.o_h;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const int col = 32 * d + 2 * j + 4 * half;
          const uint2 w = make_uint2(pack2<BF16>(o[r][d][j] * f, o[r][d][j + 1] * f), pack2<BF16>(o[r][d][j + 2] * f, o[r][d][j + 3] * f));
          if (col < a.D) __builtin_memcpy(__builtin_assume_aligned(op + col, 2), &w, 8);
        }
      if (a.lse && half == 0) a.lse[t * a.Hq + h] = (m[r] + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
    }
  }
}

hipError_t launch_attn_tile(const AttnArgs& a, bool bf16, bool fp8, int first, int count, hipStream_t st) {
  auto run = [&](auto b_tag, auto f_tag, auto d_tag, auto direct_tag) {
    hipLaunchKernelGGL((attn_tile_kernel<decltype(b_tag)::value, decltype(f_tag)::value, decltype(direct_tag)::value,
                                         decltype(d_tag)::value>),
                       dim3((unsigned)count), dim3(256), 0, st, a, first, count);
    return hipGetLastError();
  };
  auto go = [&](auto b_tag, auto f_tag, auto d_tag) {
    if constexpr (!decltype(f_tag)::value) {
      if (a.D == decltype(d_tag)::value) return run(b_tag, f_tag, d_tag, std::true_type{});
    }
    return run(b_tag, f_tag, d_tag, std::false_type{});
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
