// The join of a row's parts, shared by the attention kernels: L lanes hold a row of D columns, four each, so that a wavefront reads
// 64 / L parts at a time; W wavefronts share a row of many parts (33 parts of 256 rows: 12.8 us with one, 6.1 with four).
#pragma once

#include "fg_attn.h"

namespace fg {

// Where this thread stands: row `id`, (query token, query head), of its workgroup's 4 / W, and its first part.
template <int L, int W>
struct JoinRow {
  int wave, lane, col, first;
  int64_t id;
  __device__ __forceinline__ JoinRow()
      : wave(threadIdx.x >> 6), lane(threadIdx.x & 63), col(4 * (lane % L)), first(lane / L + (W > 1 ? wave * (64 / L) : 0)),
        id((int64_t)blockIdx.x * (4 / W) + (W > 1 ? 0 : wave)) {}
};

// n parts of row r.id joined and written to (t, h); a row that no item computed (not served) shows as NaN.
template <bool BF16, int L, int W>
__device__ __forceinline__ void attn_join(const AttnArgs& a, const JoinRow<L, W>& r, int t, int h, int n, bool served) {
  __shared__ f32x4 part_o[W > 1 ? W : 1][L];
  __shared__ float part_sum[W];
  const int64_t id = r.id, all = (int64_t)a.T * a.Hq;
  const int lane = r.lane, wave = r.wave, col = r.col;
  float top = -__builtin_inff();
  for (int i = lane; i < n; i += 64) top = fmaxf(top, a.ml[i * all + id].x);
  top = wave_max(top);
  const float base = attn_base(top);
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = r.first; i < n; i += W * 64 / L) {
    const float2 p = a.ml[i * all + id];
    const f32x4 v = col < a.D ? *reinterpret_cast<const f32x4*>(a.acc + (i * all + id) * a.D + col) : o;
    const float f = __builtin_amdgcn_exp2f(p.x - base);
    sum = __builtin_fmaf(p.y, f, sum);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(v[j], f, o[j]);
  }
#pragma unroll
  for (int off = L; off < 64; off *= 2) {
    sum += __shfl_xor(sum, off, kWave);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], off, kWave);
  }
  if constexpr (W > 1) {
    if (lane < L) part_o[wave][lane] = o;
    if (lane == 0) part_sum[wave] = sum;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      sum += part_sum[w];
      o += part_o[w][lane % L];
    }
  }
  // a row that saw no key gives zeros; one past max_query_len, which no item computed, shows as NaN
  const float f = !served ? __builtin_nanf("") : (sum == 0.f ? 0.f : 1.f / sum);
  if (lane < L && col < a.D) {
    const uint2 w = make_uint2(pack2<BF16>(o[0] * f, o[1] * f), pack2<BF16>(o[2] * f, o[3] * f));
    __builtin_memcpy(__builtin_assume_aligned(a.out + t * a.o_t + h * a.o_h + col, 2), &w, 8);
  }
  if (a.lse && lane == 0)
    a.lse[id] = !served ? f : (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}

// The last sequence that starts at or before query token t (0 where none does).
__device__ __forceinline__ int attn_sequence(const AttnArgs& a, int t) {
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace fg
