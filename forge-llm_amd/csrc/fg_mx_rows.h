// mx_rows: work items of up to 16 rows (decoding) over block-scaled keys and values.  The products are those of attn_rows: a
// wavefront by itself on tiles of 32 keys, S^T = K Q^T, then O^T += V^T P^T with P^T straight from the registers of the first.
// A lane reads one run of DP / 4 adjacent columns of a key, which is whole blocks of 32 or a part of one, so its codes become 16-bit
// floats by the conversions that take the scale along (two values an instruction, exact); the first product's columns are
// numbered as the runs lie.  Values are converted on the way to LDS and come back through the transposing read.
#pragma once

#include "fg_attn.h"
#include "fg_mx_attn.h"

namespace fg {

// A tile of values in LDS: rows of DP 16-bit columns and 32 bytes more, so that both the writes (8 keys, one unit of 16 bytes) and the
// transposing reads (4 keys, 32 bytes) spread over all banks and every place is a constant away from the lane's first.
template <int DP>
struct MxRowsLds {
  static constexpr int kRow = DP * 2 + 32, kV = kRowsTile * kRow, kO = 16 * DP * 4;
  static constexpr int kRed = kRowsWaves * (kV > kO ? kV : kO);
  static constexpr int kBytes = kRed + 2 * kRowsWaves * 16 * 4;
};

// SIXTEENS: pages hold whole sixteens of tokens, so that sixteen neighbouring keys, which a load takes, lie in one page: its id and
// the row's place are scalar.
template <bool BF16, int BITS, bool CAP, int DP, bool SIXTEENS>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) mx_rows_kernel(const MxAttnArgs m_) {
  constexpr int C = DP / 32, DB = DP / 16;
  constexpr int RUN = DP / 4, W = RUN * BITS / 32, WC = BITS / 4;  // columns of a lane's run, their words, words of 8 columns
  constexpr int SB = RUN > kMxBlock ? RUN / kMxBlock : 1;          // scales of a run
  using L = MxRowsLds<DP>;
  __shared__ __align__(16) uint8_t lds[L::kBytes];
  float* red = reinterpret_cast<float*>(lds + L::kRed);
  const AttnArgs& a = m_.a;

  MxItem it;
  if (!mx_item<16>(m_, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, grp = lane >> 4;

  // this lane's row: the fragment of Q, and the keys it sees
  const int row = it.row0 + l16, tok = row / a.G, g = row - tok * a.G;
  const uint16_t* qp = a.q + (int64_t)(it.token0 + tok) * a.q_t + (int64_t)(it.head * a.G + g) * a.q_h;
  const AttnFactor factor = attn_factor(m_.factor, 1.f);
  const uint32_t sign = CAP ? 0 : factor.sign;
  s16x8 qf[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int d = RUN * grp + 8 * c;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (row < it.rows && d < a.D) __builtin_memcpy(&u, __builtin_assume_aligned(qp + d, 2), 16);
    u.x ^= sign; u.y ^= sign; u.z ^= sign; u.w ^= sign;
    qf[c] = __builtin_bit_cast(s16x8, u);
  }
  const int seen = it.seen0 + tok, low = seen - m_.window;                              // keys low .. seen - 1
  const int min_seen = it.seen0 + it.row0 / a.G;                                        // of the tile's first row
  const int max_low = it.seen0 + min(it.rows - 1, it.row0 + 15) / a.G - m_.window;      // of its last
  const float sc = CAP ? m_.factor : factor.value, cap_in = m_.cap_in;
  // This lane's run: per block (or the part of one that it has) its bytes from the row's begin and its scale.  Columns that the head
  // lacks repeat others, against zeros of Q and for results that nobody keeps.
  constexpr int WB = W / SB;  // words of a block
  uint32_t off[SB], soff[SB];
#pragma unroll
  for (int i = 0; i < SB; ++i) {
    int col = RUN * grp + kMxBlock * i;
    if (col >= a.D) col = i ? RUN * grp : 0;
    if (col >= a.D) col = 0;
    off[i] = col * BITS / 8;
    soff[i] = col / kMxBlock;
  }
  const uint8_t *kb = a.k + it.head * a.c_head, *vb = a.v + it.head * a.c_head;
  const uint8_t *ksb = m_.ks + it.head * m_.s_head, *vsb = m_.vs + it.head * m_.s_head;

  f32x4 o[DB];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};

  const int n = max(it.end - it.begin, 0), step = kRowsTile * kRowsWaves;
  uint8_t *const vl = lds + wave * L::kV, *const vw = vl + l16 * L::kRow + C * grp * 16;
  uint8_t* const vt = vl + (4 * grp + l16 / 4) * L::kRow + 8 * (l16 % 4);
  // NB tiles in registers: while one is computed the others are on their way (a run of 64 bytes leaves room for one: the next is
  // loaded behind the products that used it)
  constexpr int NB = W >= 16 ? 1 : 2;
  uint32_t kr[NB][2][W], vr[NB][2][W], kse[NB][2][SB], vse[NB][2][SB];
  uint32_t ok[NB];  // bit t: key t of the tile is there
  auto words = [](uint32_t* to, const uint8_t* p) __attribute__((always_inline)) {
    if constexpr (WB == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      to[0] = u.x;
      to[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < WB; i += 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p + 4 * i);
        to[i] = u.x;
        to[i + 1] = u.y;
        to[i + 2] = u.z;
        to[i + 3] = u.w;
      }
    }
  };
  // Where the keys of a tile's halves are (of the first in SIXTEENS, else of this lane's): their page ids are asked for a tile ahead of
  // the loads that they are for, and vector loads of ids in front of the loads of the tile between, which then need not be waited
  // for with them.
  int32_t ids[2];
  uint32_t inside[2];  // the place in the page
  const uint32_t lane_row = SIXTEENS ? (uint32_t)l16 * a.c_token : 0;
  auto ask = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = it.begin + (SIXTEENS ? min(t0 + 16 * h, (n - 1) & ~15) : min(t0 + 16 * h + l16, n - 1));
      const int page = m_.page_shift >= 0 ? t >> m_.page_shift : t / a.page;
      inside[h] = (uint32_t)(t - page * a.page) * a.c_token;
      if constexpr (SIXTEENS)
        ids[h] = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(it.table))[page];
      else
        ids[h] = it.table[page];
    }
  };
  // No branch: loads that one goes round are waited for where it ends.  A key that is not there reads the cache's first rows; past
  // the end the last tile's keys are loaded again, which nobody uses.
  auto fetch = [&](int b, int t0, int next) __attribute__((always_inline)) {
    uint32_t row[2];
    // keys first .. last - 1 of the tile are an item's
    const int first = it.low - it.begin - t0, last = n - t0;
    uint32_t here = last >= 32 ? 0xffffffffu : (last > 0 ? (1u << last) - 1 : 0u);
    if (first > 0) here = first >= 32 ? 0u : here & ~((1u << first) - 1);
    uint32_t in_cache = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool is = ids[h] >= 0 && ids[h] < a.n_pages;
      row[h] = is ? (uint32_t)ids[h] * a.c_page + inside[h] : 0;
      if constexpr (SIXTEENS) in_cache |= is ? 0xffffu << (16 * h) : 0u;
      else in_cache |= (uint32_t)(__ballot(is) & 0xffff) << (16 * h);
    }
    ok[b] = here & in_cache;
    ask(next);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint64_t at = (uint64_t)row[h] * 16, sat = BITS == 4 ? row[h] : row[h] >> 1;
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        words(&kr[b][h][WB * i], kb + at + (lane_row * 16 + off[i]));
        words(&vr[b][h][WB * i], vb + at + (lane_row * 16 + off[i]));
        kse[b][h][i] = (ksb + sat)[lane_row / (BITS == 4 ? 1 : 2) + soff[i]];
        vse[b][h][i] = (vsb + sat)[lane_row / (BITS == 4 ? 1 : 2) + soff[i]];
      }
    }
  };
  auto turn = [&](int b, int t0, bool ahead) __attribute__((always_inline)) {
    const uint32_t here = ok[b];
    if (here != 0xffffffffu) {  // weights of zero do not undo a NaN
      asm volatile("");
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (!(here >> (16 * h + l16) & 1)) {
#pragma unroll
          for (int i = 0; i < W; ++i) vr[b][h][i] = 0;
#pragma unroll
          for (int i = 0; i < SB; ++i) vse[b][h][i] = 1;
        }
    }
    auto scale = [](uint32_t byte) { return __uint_as_float(byte << 23); };  // 255: the conversion gives NaN
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        *reinterpret_cast<uint4*>(vw + 16 * h * L::kRow + 16 * c) =
            mx_eight<BF16, BITS>(vr[b][h][c * WC], vr[b][h][c * WC + WC - 1], scale(vse[b][h][c * 8 / kMxBlock]));
      }
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint4 k8 = mx_eight<BF16, BITS>(kr[b][h][c * WC], kr[b][h][c * WC + WC - 1], scale(kse[b][h][c * 8 / kMxBlock]));
        s[h] = mfma16<BF16>(__builtin_bit_cast(s16x8, k8), qf[c], c ? s[h] : (f32x4)(0.f));
      }
    if (ahead) fetch(b, t0 + NB * step, t0 + (NB + 1) * step);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = CAP ? mx_tanh(s[j / 4][j % 4] * cap_in) : s[j / 4][j % 4];
    const int first = it.begin + t0;
    if (here != 0xffffffffu || first + kRowsTile > min_seen || first < max_low) {
      asm volatile("");  // a branch, so that whole tiles skip it
      const int left = seen - first, skip = low - first;  // keys of the tile that this lane's row sees: skip .. left - 1
      uint32_t mask = left >= 32 ? here : (left > 0 ? here & ((1u << left) - 1) : 0u);
      if (skip > 0) mask = skip >= 32 ? 0u : mask & ~((1u << skip) - 1);
      mask >>= 4 * grp;
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
    // values four blocks of columns ahead of their products
    constexpr int VB = 4;
    s16x8 vf[2][VB];
    auto values = [&](int d0) {
#pragma unroll
      for (int e = 0; e < VB; ++e) {
        s16x4 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)  // 16 lanes read 4 keys x 16 columns
          half[h] = lds_tr16(vt + 16 * h * L::kRow + 32 * (d0 + e));
        vf[d0 / VB % 2][e] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
    };
    values(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d0 = 0; d0 < DB; d0 += VB) {
      if (d0 + VB < DB) values(d0 + VB);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < VB; ++e) o[d0 + e] = mfma16<BF16>(vf[d0 / VB % 2][e], p, o[d0 + e]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_wave_barrier();
  };
  // Whole rounds of NB tiles have no branch in them that a load could be on either side of, so that a tile waits for its own loads
  // only.
  int t0 = wave * kRowsTile;
  if (t0 < n) {
    ask(t0);
#pragma unroll
    for (int b = 0; b < NB; ++b) fetch(b, t0 + b * step, t0 + (b + 1) * step);
    for (; t0 + (NB - 1) * step < n; t0 += NB * step) {
#pragma unroll
      for (int b = 0; b < NB; ++b) turn(b, t0 + b * step, true);
    }
#pragma unroll
    for (int b = 0; b + 1 < NB; ++b)
      if (t0 + b * step < n) turn(b, t0 + b * step, false);
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
  const int64_t at = ((int64_t)it.slot * a.T + t) * a.Hq + h;
  const float inv = a.acc ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);  // a row that saw no key gives zeros
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
