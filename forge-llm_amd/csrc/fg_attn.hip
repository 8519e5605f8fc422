// Attention over a paged cache for a batch whose sequences share a prefix: o = softmax(scale q K^T) V over the shared prefix's
// keys and the sequence's own.  The prefix is a product of all the batch's rows with one set of keys, read once; a
// sequence's own keys meet the rows of its query heads only.
//
// Keys are cut into parts; an item (row tile, key head, part) makes one pass over its keys with a running maximum and sum and
// leaves sum(p v), the maximum and the sum in 32 bits; attn_join_kernel weighs the parts of each row by exp2(m - max m).
//
// attn_rows_kernel, for items of up to 16 or 32 rows (decode): what bounds it is the read of the keys and values, so each
// wavefront works by itself on tiles of 32 keys, without a barrier, and loads the next tile while it computes this one.
//   S^T = K Q^T   (A: 16 keys x 32 columns straight from global memory, 16 bytes per lane; B: the rows, in registers)
//   O^T += V^T P^T
// S^T comes out with a row in each lane and keys 4 g + i (g the lane's group of 16) in its registers, which is the order in
// which the second product takes P^T if V^T is read in the same order: P goes from the first product to the second without
// leaving the lane.  V^T needs columns of V, so V passes through LDS and comes back through the transposing read.
#include <algorithm>

#include "fg_attn.h"

namespace fg {

namespace {

// 16-byte unit u of key t in a V tile whose rows hold U units: an exchange of units that depends on the key, so that both
// the writes (16 keys, one unit) and the transposing reads (8 keys, 32 bytes) spread over all banks.
template <int U>
__device__ __forceinline__ int v_unit(int t, int u) {
  if constexpr (U >= 16) return u ^ ((t & 7) << 1 | ((t >> 3 ^ t >> 4) & 1));
  if constexpr (U == 8) return u ^ ((t >> 1 & 3) << 1 | ((t >> 3 ^ t >> 4) & 1));
  return u ^ ((t >> 2 & 1) << 1 | ((t >> 3 ^ t >> 4) & 1));
}

}  // namespace

constexpr int kRowsWaves = 4;
constexpr int kRowsTile = 32;  // keys per wavefront and step

// DP: head columns in registers (D of them are there), R: row blocks of 16.
template <bool BF16, bool FP8, int DP, int R>
__global__ void __launch_bounds__(64 * kRowsWaves) attn_rows_kernel(const AttnArgs a, int first) {
  constexpr int IT = FP8 ? 1 : 2, U = DP * IT / 16, C = DP / 32, DB = DP / 16;
  constexpr int KU = U / 4;  // 16-byte loads of a lane per key
  constexpr int kVBytes = kRowsTile * DP * IT, kOBytes = 2 * 16 * R * DP * 4;
  constexpr int kLds = kRowsWaves * kVBytes > kOBytes ? kRowsWaves * kVBytes : kOBytes;
  __shared__ __align__(16) uint8_t lds[kLds];
  __shared__ uint32_t tab[kMaxPart];
  __shared__ float red[2][kRowsWaves][16 * R];

  AttnItem it;
  if (!attn_item<16 * R>(a, first + blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, grp = lane >> 4;
  const int units = a.D * IT / 16;
  attn_row_table(a, it, tab, kRowsTile);

  // this lane's row of each row block: the fragment of Q, and the keys it sees
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale turns the rows instead
  s16x8 qf[R][C];
  int seen[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = it.row0 + 16 * r + l16, tok = row / a.G, g = row - tok * a.G;
    const bool in = row < it.rows;
    const uint16_t* qp = a.q + (int64_t)(it.token0 + tok) * a.q_t + (int64_t)(it.head * a.G + g) * a.q_h;
    seen[r] = it.causal ? it.seen0 + tok : it.end;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      // e4m3 keys come 16 columns per load, which makes two chunks
      const int d = FP8 ? 64 * (c / 2) + 16 * grp + 8 * (c % 2) : 32 * c + 8 * grp;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (in && d < a.D) __builtin_memcpy(&u, __builtin_assume_aligned(qp + d, 2), 16);
      u.x ^= sign; u.y ^= sign; u.z ^= sign; u.w ^= sign;
      qf[r][c] = __builtin_bit_cast(s16x8, u);
    }
  }
  const int min_seen = it.causal ? it.seen0 + it.row0 / a.G : it.end;  // what the tile's first row sees
  const float sc = fabsf(a.scale_log2) * (FP8 ? a.ks[it.head] : 1.f);
  const uint8_t *kb = a.k + it.head * a.c_head, *vb = a.v + it.head * a.c_head;

  f32x4 o[R][DB];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -__builtin_inff();
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[r][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();

  const int n = max(it.end - it.begin, 0);
  uint8_t* vl = lds + wave * kVBytes;
  uint4 kr[2][KU], vr[2][KU];
  uint32_t rows[2];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      rows[h] = tab[t0 + 16 * h + l16];
#pragma unroll
      for (int c = 0; c < KU; ++c) {
        const int u = 4 * c + grp;
        const bool in = rows[h] != kNoRow && u < units;
        kr[h][c] = in ? attn_ld16(kb, rows[h], u) : make_uint4(0, 0, 0, 0);
        vr[h][c] = in ? attn_ld16(vb, rows[h], u) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  const int step = kRowsTile * kRowsWaves;
  if (wave * kRowsTile < n) fetch(wave * kRowsTile);
  for (int t0 = wave * kRowsTile; t0 < n; t0 += step) {
    const uint64_t ok0 = __ballot(rows[0] != kNoRow), ok1 = __ballot(rows[1] != kNoRow);
    const uint32_t ok = (uint32_t)(ok0 & 0xffff) | (uint32_t)(ok1 & 0xffff) << 16;  // bit t: key t of the tile is there
    uint4 kc[2][KU];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < KU; ++c) {
        kc[h][c] = kr[h][c];
        const int t = 16 * h + l16;
        *reinterpret_cast<uint4*>(vl + (t * U + v_unit<U>(t, 4 * c + grp)) * 16) = vr[h][c];
      }
    if (t0 + step < n) fetch(t0 + step);

    f32x4 s[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) s[r][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        s16x8 kf;
        if constexpr (FP8) {
          const uint4& u = kc[h][c / 2];
          kf = c % 2 ? e4m3_to_16<BF16>(u.z, u.w) : e4m3_to_16<BF16>(u.x, u.y);
        } else {
          kf = __builtin_bit_cast(s16x8, kc[h][c]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][h] = mfma16<BF16>(kf, qf[r][c], s[r][h]);
      }
    s16x8 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[r][j / 4][j % 4];
      if (ok != 0xffffffffu || it.begin + t0 + kRowsTile > min_seen) {
        asm volatile("");  // a branch, so that whole tiles skip it
        const int left = seen[r] - (it.begin + t0);  // keys of the tile that this lane's row sees
        const uint32_t mask = (left >= 32 ? ok : (left > 0 ? ok & ((1u << left) - 1) : 0u)) >> (4 * grp);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(mask >> (16 * (j / 4) + j % 4) & 1)) x[j] = -__builtin_inff();
      }
      float top = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
      top *= sc;
      if (__any(top > m[r] + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float mn = fmaxf(m[r], top), f = __builtin_amdgcn_exp2f(m[r] - attn_base(mn));
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[r][d] *= f;
      }
      const float base = attn_base(m[r]);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], sc, -base));
      l[r] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack2<BF16>(x[2 * j], x[2 * j + 1]);
      p[r] = __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3]));
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      s16x8 vf;
      if constexpr (FP8) {
        // 16 lanes read 8 keys x 16 columns: keys 4 g + 0..3 of either half of the tile
        const int j = l16 / 2, t = 16 * (j / 4) + 4 * grp + j % 4;
        const i32x2 c = lds_tr8(vl + (t * U + v_unit<U>(t, d)) * 16 + 8 * (l16 % 2));
        vf = e4m3_to_16<BF16>((uint32_t)c[0], (uint32_t)c[1]);
      } else {
        s16x4 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 16 lanes read 4 keys x 16 columns
          const int t = 16 * h + 4 * grp + l16 / 4;
          half[h] = lds_tr16(vl + (t * U + v_unit<U>(t, 2 * d + (l16 % 4) / 2)) * 16 + 8 * (l16 % 2));
        }
        vf = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) o[r][d] = mfma16<BF16>(vf, p[r], o[r][d]);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // join the wavefronts: their maxima and sums meet in LDS, their sums of values in a tree over the V tiles' space
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += __shfl_xor(l[r], 16, kWave);
    l[r] += __shfl_xor(l[r], 32, kWave);
    if (grp == 0) {
      red[0][wave][16 * r + l16] = m[r];
      red[1][wave][16 * r + l16] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = red[0][0][16 * r + l16], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) top = fmaxf(top, red[0][w][16 * r + l16]);
    const float base = attn_base(top);
#pragma unroll
    for (int w = 0; w < kRowsWaves; ++w)
      sum += red[1][w][16 * r + l16] * __builtin_amdgcn_exp2f(red[0][w][16 * r + l16] - base);
    const float f = __builtin_amdgcn_exp2f(m[r] - base);
#pragma unroll
    for (int d = 0; d < DB; ++d) o[r][d] *= f;
    m[r] = top;
    l[r] = sum;
  }
  f32x4* ol = reinterpret_cast<f32x4*>(lds);
  auto swap_in = [&](int from, int to) {  // wavefronts `from`, .. hand their sums to `to`, ..
    if (wave >= from && wave < 2 * from)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int d = 0; d < DB; ++d) ol[(((wave - from) * R + r) * DB + d) * 64 + lane] = o[r][d];
    __syncthreads();
    if (wave < to)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int d = 0; d < DB; ++d) o[r][d] += ol[((wave * R + r) * DB + d) * 64 + lane];
    __syncthreads();
  };
  swap_in(2, 2);
  swap_in(1, 1);
  if (wave != 0) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = it.row0 + 16 * r + l16, tok = row / a.G, g = row - tok * a.G;
    if (row >= it.rows) continue;
    const int64_t t = it.token0 + tok;
    const int h = it.head * a.G + g;
    const float vs = FP8 ? a.vs[it.head] : 1.f;
    if (a.acc) {
      const int64_t at = (int64_t)it.slot * a.T * a.Hq + t * a.Hq + h;
      if (grp == 0) a.ml[at] = make_float2(m[r], l[r]);
#pragma unroll
      for (int d = 0; d < DB; ++d)
        if (16 * d + 4 * grp < a.D) *reinterpret_cast<f32x4*>(a.acc + at * a.D + 16 * d + 4 * grp) = o[r][d] * vs;
    } else {
      const float f = l[r] == 0.f ? 0.f : vs / l[r];  // a row that saw no key gives zeros
      uint16_t* op = a.out + t * a.o_t + h * a.o_h;
#pragma unroll
      for (int d = 0; d < DB; ++d)
        if (16 * d + 4 * grp < a.D) {
          const uint2 w = make_uint2(pack2<BF16>(o[r][d][0] * f, o[r][d][1] * f), pack2<BF16>(o[r][d][2] * f, o[r][d][3] * f));
          __builtin_memcpy(__builtin_assume_aligned(op + 16 * d + 4 * grp, 2), &w, 8);
        }
      if (a.lse && grp == 0) a.lse[t * a.Hq + h] = (m[r] + __builtin_amdgcn_logf(l[r])) * 0.69314718055994531f;
    }
  }
}

// Joins the parts of each row: one wavefront per (query token, query head), four columns per lane.
template <bool BF16>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), all = (int64_t)a.T * a.Hq;
  const int lane = threadIdx.x & 63;
  if (id >= all) return;
  const int t = (int)(id / a.Hq), h = (int)(id - (int64_t)t * a.Hq);
  int seq = t;
  bool inside = true, served = true;
  if (a.starts) {  // the last sequence that starts at or before t
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    seq = lo;
    inside = a.B > 0 && a.starts[seq] <= t && t < a.starts[seq + 1];
    served = !inside || t - a.starts[seq] < a.max_q;
  }
  const int len = inside ? min(a.lens[seq], a.max_len) : 0;
  const int own = max((len + a.part_s - 1) / a.part_s, 1);
  const int n = !inside ? 0 : a.parts_p + min(own, a.parts_s);
  float top = -__builtin_inff();
  for (int i = lane; i < n; i += 64) top = fmaxf(top, a.ml[i * all + id].x);
  top = wave_max(top);
  const float base = attn_base(top);
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const bool in = 4 * lane < a.D;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 p = a.ml[i * all + id];
    const float f = __builtin_amdgcn_exp2f(p.x - base);
    sum = __builtin_fmaf(p.y, f, sum);
    if (in) o += *reinterpret_cast<const f32x4*>(a.acc + (i * all + id) * a.D + 4 * lane) * f;
  }
  // a row that saw no key gives zeros; one past max_query_len, which no item computed, shows as NaN
  const float f = !served ? __builtin_nanf("") : (sum == 0.f ? 0.f : 1.f / sum);
  if (in) {
    const uint2 w = make_uint2(pack2<BF16>(o[0] * f, o[1] * f), pack2<BF16>(o[2] * f, o[3] * f));
    __builtin_memcpy(__builtin_assume_aligned(a.out + t * a.o_t + h * a.o_h + 4 * lane, 2), &w, 8);
  }
  if (a.lse && lane == 0)
    a.lse[id] = !served ? f : (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}


// Cuts the keys of `items` row tiles into parts, a workgroup each: about `want` of them in all, whole multiples of `unit` keys
// and at most `most`.  Host lengths only: a sequence shorter than max_len leaves parts that end at once.
static int split_keys(int64_t len, int64_t items, int64_t want, int64_t unit, int64_t most, int* part) {
  const int64_t parts = std::max<int64_t>(1, want / std::max<int64_t>(items, 1));
  const int64_t p = std::min(most, std::max<int64_t>(unit, ((len + parts - 1) / parts + unit - 1) / unit * unit));
  *part = (int)p;
  return (int)std::max<int64_t>(1, (len + p - 1) / p);
}

// Rows per work item: 16 or 32 for attn_rows_kernel (32 with 256 columns would not fit its registers), 128 for attn_tile_kernel.
static int rows_tile(int64_t rows, int D) {
  if (rows <= 16) return 16;
  return rows <= 32 && D <= 128 ? 32 : 128;
}

static void plan_segment(int64_t len, int64_t rows, int64_t heads, int D, int* tile, int* tiles, int* parts, int* part) {
  *tile = rows_tile(rows, D);
  *tiles = (int)((rows + *tile - 1) / *tile);
  const int64_t items = *tiles * heads, cus = device_cus();
  *parts = *tile == 128 ? split_keys(len, items, 2 * cus, 64, 1 << 30, part)
                        : split_keys(len, items, 4 * cus, kRowsTile * kRowsWaves, kMaxPart, part);
}

// Fills in the plan; returns the partial sums' bytes.  items is -1 where the work items would pass 32 bits.
size_t attn_plan(AttnArgs& a) {
  a.parts_p = a.tiles_p = a.part_p = 0;
  a.tile_p = 16;
  if (a.prefix_len) plan_segment(a.prefix_len, (int64_t)a.T * a.G, a.Hk, a.D, &a.tile_p, &a.tiles_p, &a.parts_p, &a.part_p);
  plan_segment(a.max_len, (int64_t)a.max_q * a.G, (int64_t)a.Hk * a.B, a.D, &a.tile_s, &a.tiles_s, &a.parts_s, &a.part_s);
  const int64_t items_p = (int64_t)a.parts_p * a.tiles_p * a.Hk, items = items_p + (int64_t)a.parts_s * a.tiles_s * a.Hk * a.B;
  a.items_p = (int)items_p;
  a.items = items < (1LL << 31) ? (int)items : -1;
  if (a.parts_p + a.parts_s == 1 && !a.starts) return 0;
  return (size_t)(a.parts_p + a.parts_s) * a.T * a.Hq * ((size_t)a.D * 4 + sizeof(float2));
}

template <int R>
static hipError_t launch_attn_rows(const AttnArgs& a, bool bf16, bool fp8, int first, int count, hipStream_t st) {
  auto go = [&](auto b_tag, auto f_tag, auto d_tag) {
    hipLaunchKernelGGL((attn_rows_kernel<decltype(b_tag)::value, decltype(f_tag)::value, decltype(d_tag)::value, R>),
                       dim3((unsigned)count), dim3(64 * kRowsWaves), 0, st, a, first);
    return hipGetLastError();
  };
  auto by_d = [&](auto b_tag, auto f_tag) {
    if (a.D <= 64) return go(b_tag, f_tag, std::integral_constant<int, 64>{});
    if constexpr (R == 1) {
      if (a.D > 128) return go(b_tag, f_tag, std::integral_constant<int, 256>{});
    }
    return go(b_tag, f_tag, std::integral_constant<int, 128>{});
  };
  auto by_f = [&](auto b_tag) { return fp8 ? by_d(b_tag, std::true_type{}) : by_d(b_tag, std::false_type{}); };
  return bf16 ? by_f(std::true_type{}) : by_f(std::false_type{});
}

hipError_t launch_attn(AttnArgs& a, bool bf16, bool fp8, void* ws, hipStream_t st) {
  const size_t bytes = attn_plan(a);
  if (a.items < 0) return hipErrorInvalidValue;
  a.acc = nullptr;
  a.ml = nullptr;
  if (bytes) {
    a.acc = static_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(a.acc + (size_t)(a.parts_p + a.parts_s) * a.T * a.Hq * a.D);
  }
  auto items = [&](int tile, int first, int count) {
    if (count == 0) return hipSuccess;
    if (tile == 128) return launch_attn_tile(a, bf16, fp8, first, count, st);
    return tile == 16 ? launch_attn_rows<1>(a, bf16, fp8, first, count, st) : launch_attn_rows<2>(a, bf16, fp8, first, count, st);
  };
  // one launch for the prefix and the sequences where one kernel takes both
  const bool one = a.tile_p == a.tile_s || a.items_p == 0;
  hipError_t e = one ? hipSuccess : items(a.tile_p, 0, a.items_p);
  if (e == hipSuccess) e = one ? items(a.tile_s, 0, a.items) : items(a.tile_s, a.items_p, a.items - a.items_p);
  note_kernel("attn rows %d x %d parts + rows %d x %d parts%s", a.items_p ? a.tile_p : 0, a.parts_p, a.tile_s, a.parts_s,
              bytes ? " + attn_join_kernel" : "");
  if (e != hipSuccess || !bytes) return e;
  const unsigned grid = (unsigned)(((int64_t)a.T * a.Hq + 3) / 4);
  if (bf16) hipLaunchKernelGGL(attn_join_kernel<true>, dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(attn_join_kernel<false>, dim3(grid), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace fg
