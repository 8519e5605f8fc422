// Tokens from their logits and given random numbers u.  With M the row's largest logit and T its temperature the weights are
//   w_i = 2^((l_i - M) log2(e) / T),
// kept are the first k tokens in the order of their logits (equal ones by their index), of these the shortest beginning whose weight
// reaches p times the k tokens', and of these the ones with w_i >= min_p; the token is the first, by index, at which the kept
// weights' sum passes u times their total.
//
// Weights are computed in fp64 and summed as whole numbers of 2^-bits (46 for up to 2^16 tokens, so that 2^62 holds all): sums do not hang on their
// order, so they go through atomics, and a token of less than half a unit is one that nobody draws.
//
// Nothing is sorted.  A histogram of the row over (M - l) log2(e) / T, with the weight and the number of the tokens in each
// bin, says in which bin the k-th token and the nucleus's last one lie.  Where all bins up to there hold few tokens (kList), these are
// collected and settle the row by themselves; else the border bins' tokens settle the border, and one more pass over the row sums
// up the weights in front of it, in the order of the indexes.  The border within a list is found by comparing each of a few
// tokens (kFew) with all of them, else by histograms again, each over a 2048th of the one before.
//
// One launch for each pass (extremes, histogram, collection, sums); a row is cut into chunks of a workgroup each while rows are few,
// and what follows a pass is done by the workgroup that ends last.  Bound by HBM for the first pass, for the others by
// the L2 and Infinity caches and the arithmetic of the weights; for one row by the launches (256 rows of 150001 in fp32, mixed settings
// 169 us: 32 + 47 + 50 + 41; one row of 32000 in bf16, top-k 50 and top-p 0.9 25 us).
#include <algorithm>

#include "fg_sample.h"

namespace fg {

namespace {

constexpr int kBins = 2048, kList = 4096, kThreads = 1024, kWaves = kThreads / 64, kMaxChunks = 64;

struct ChunkSum {
  float max, min;  // of the finite or infinite logits above -inf; min of those
  int arg;         // the largest one's first index, -1: none
  float sum;       // of exp(l - max)
};

struct RowState {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t list[kList];  // key << 32 | index, in any order
  uint64_t wave_mass[kMaxChunks * kWaves];
  ChunkSum part[kMaxChunks];
  uint32_t listed, ticket[2];
  uint32_t done;         // the row has its token
  uint32_t cut_key, cut_index;  // kept: a larger key, or this one up to this index
};

// A row's settings and extremes.
struct Row {
  float t, p, minp;
  int k;
  bool greedy, by_k, by_p;
  float max, min;
  int arg;
  float sum;     // of exp(l - max)
  double scale;  // log2(e) / T
};

// A logit's place in the order as an unsigned number: NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

template <int DT>
__device__ __forceinline__ float one(const void* row, int i) {
  const float l = load_f(row, DT, i);
  return __builtin_isnan(l) ? -__builtin_inff() : l;
}

typedef uint32_t u32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_by2 __attribute__((ext_vector_type(2), aligned(2)));

// Four neighbouring logits.
template <int DT>
__device__ __forceinline__ void four(const void* row, int i, float (&l)[4]) {
  if constexpr (DT == FG_F32) {
    const u32x4_by4 w = *reinterpret_cast<const u32x4_by4*>(static_cast<const float*>(row) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) l[j] = __uint_as_float(w[j]);
  } else {
    const u32x2_by2 w = *reinterpret_cast<const u32x2_by2*>(static_cast<const uint16_t*>(row) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t b = (uint16_t)(w[j / 2] >> (16 * (j % 2)));
      l[j] = DT == FG_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) l[j] = __builtin_isnan(l[j]) ? -__builtin_inff() : l[j];
}

// Calls f(i, l) for each four logits l from token i on, i = first, first + step, .. in front of end; those from end on are -inf.  U whole
// fours are loaded at a time, with no branch between the loads, which would wait for each.
template <int DT, int U, class F>
__device__ __forceinline__ void sweep(const void* row, int first, int step, int end, F f) {
  int i = first;
  for (; i + (U - 1) * step + 4 <= end; i += U * step) {
    float l[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) four<DT>(row, i + u * step, l[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) f(i + u * step, l[u]);
  }
#pragma unroll 1
  for (; i < end; i += step) {
    float l[4];
    if (i + 4 <= end) {
      four<DT>(row, i, l);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] = i + j < end ? one<DT>(row, i + j) : -__builtin_inff();
    }
    f(i, l);
  }
}

// 2^-y for the weights: 2^-(k / 64) from a table and the exponential series of the rest, |x| <= ln 2 / 128, to x^5 (the next term is
// below 2^-54).
struct Powers {
  double at[64];
  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 64) at[threadIdx.x] = exp2(-(double)threadIdx.x / 64);
  }
};
__device__ __forceinline__ double weight(const Powers& t, double y, int bits) {
  // k to the nearest by adding 3 2^51, whose last bits it then is; the power of two goes into the exponent's bits.  (Conversions and
  // ldexp run at a part of the additions' rate: 256 rows of 150001 with mixed settings 201 us against 197.)
  const double at = __builtin_fma(y, 64.0, 0x1.8p52);
  const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, at);
  const double x = __builtin_fma(at - 0x1.8p52, 0.015625, -y) * 0.6931471805599453;
  double e = __builtin_fma(x, 1.0 / 120, 1.0 / 24);
  e = __builtin_fma(x, e, 1.0 / 6);
  e = __builtin_fma(x, e, 0.5);
  e = __builtin_fma(x, e, 1.0);
  e = __builtin_fma(x, e, 1.0);
  const uint64_t w = __builtin_bit_cast(uint64_t, t.at[k & 63] * e);  // from 1/2 to 1
  return __builtin_bit_cast(double, w + ((uint64_t)(uint32_t)(bits - (k >> 6)) << 52));
}
__device__ __forceinline__ uint64_t whole(double v) {  // to the nearest whole number, of less than 2^52
  return __builtin_bit_cast(uint64_t, v + 0x1p52) & 0xfffffffffffffull;
}

// The exponent y >= 0 of logit l (infinite for one that weighs nothing).
__device__ __forceinline__ double exponent(const Row& r, float l) {
  if (l == r.max) return 0;
  return ((double)r.max - (double)l) * r.scale;
}
// A logit that no logit of an exponent of y or less is below: what is, needs no fp64.
__device__ __forceinline__ float floor_of(const Row& r, double y) {
  const double l = (double)r.max - y / r.scale;  // infinite or no number: nothing is said
  const float f = (float)(l - 1e-6 * (fabs(l) + fabs((double)r.max) + 1));
  return f == f ? f : -__builtin_inff();
}
__device__ __forceinline__ double most(int bits) { return bits + 1; }  // from here on a weight is no unit

__device__ __forceinline__ double bin_scale(const Row& r, int bits) {
  const double range = fmin(((double)r.max - (double)r.min) * r.scale, most(bits));
  return range > 0 ? kBins / range : 0;
}
__device__ __forceinline__ int bin_of(double y, double scale) { return min((int)(y * scale), kBins - 1); }

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return (uint64_t)(uint32_t)__shfl_up((int)(v >> 32), d, kWave) << 32 | (uint32_t)__shfl_up((int)v, d, kWave);
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int d) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), d, kWave) << 32 | (uint32_t)__shfl_xor((int)v, d, kWave);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += shfl_xor64(v, d);
  return v;
}

// A wavefront's own: sum of the lanes' values in front of this one; `all`: of all.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, uint64_t* all) {
  const int lane = threadIdx.x & 63;
  uint64_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = shfl_up64(s, d);
    if (lane >= d) s += o;
  }
  *all = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(s >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)s, 63);
  return s - v;
}

// Sum of the threads' values in front of this one; `all`: of all.  Two barriers.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t mine;
  const uint64_t in_front = wave_scan(v, &mine);
  __syncthreads();  // the last call's sums have been read
  if (lane == 0) part[wave] = mine;
  __syncthreads();
  uint64_t before = 0, sum = 0;
#pragma unroll 4
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? part[w] : 0;
    sum += part[w];
  }
  *all = sum;
  return before + in_front;
}

// Both at once: sums of v and of n in front of this thread, and of all.
__device__ __forceinline__ void block_scan2(uint64_t v, uint32_t n, uint64_t* part_v, uint32_t* part_n, uint64_t* v0, uint64_t* v_all, uint32_t* n0,
                                            uint32_t* n_all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t vs = v;
  uint32_t ns = n;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t vo = shfl_up64(vs, d);
    const uint32_t no = (uint32_t)__shfl_up((int)ns, d, kWave);
    if (lane >= d) {
      vs += vo;
      ns += no;
    }
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 63) {
    part_v[wave] = vs;
    part_n[wave] = ns;
  }
  __syncthreads();
  *v0 = vs - v;
  *n0 = ns - n;
  *v_all = 0;
  *n_all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    *v0 += w < wave ? part_v[w] : 0;
    *n0 += w < wave ? part_n[w] : 0;
    *v_all += part_v[w];
    *n_all += part_n[w];
  }
}

__device__ __forceinline__ void row_settings(const SampleArgs& a, int b, Row& r) {
  r.t = a.temperature ? a.temperature[b] : a.temperature_all;
  r.p = a.top_p ? a.top_p[b] : a.top_p_all;
  r.minp = a.min_p ? a.min_p[b] : a.min_p_all;
  r.k = a.top_k ? a.top_k[b] : a.top_k_all;
  r.greedy = !(r.t > 0.f);
  r.by_k = r.k > 0 && r.k < a.V;
  r.by_p = r.p < 1.f;
  r.minp = r.minp > 0.f ? fminf(r.minp, 1.f) : 0.f;
  r.scale = 1.4426950408889634 / (double)r.t;
}

// What a row's workgroups hand to the one that ends last goes past the XCDs' L2 caches both ways (a fence would write each whole
// cache back, once for every workgroup: 32 rows of 128000 357 us against 87), and is in memory when the wavefront's wait is over.
template <class T>
__device__ __forceinline__ void put_far(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T get_far(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of its row's; what the others have put far can be got.  Every thread is there.
__device__ __forceinline__ bool last_of_row(uint32_t* ticket, int chunks, int* shared) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    *shared = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)chunks - 1;
  __syncthreads();
  return *shared;
}

// The row's extremes from its chunks', a lane each; every thread has them.
static_assert(kMaxChunks <= 64, "a lane for each chunk");
__device__ __forceinline__ void row_extremes(const SampleArgs& a, const RowState& s, Row& r) {
  const int lane = threadIdx.x & 63;
  ChunkSum p = {-__builtin_inff(), __builtin_inff(), -1, 0.f};
  if (lane < a.chunks) p = s.part[lane];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    if (d >= a.chunks) break;
    const float mx = __shfl_xor(p.max, d, kWave), sum = __shfl_xor(p.sum, d, kWave);
    const int arg = __shfl_xor(p.arg, d, kWave);
    if (arg >= 0) {
      const float most = fmaxf(p.max, mx), log2e = 1.4426950408889634f;
      const float own = p.arg < 0 ? 0.f : p.sum * __builtin_amdgcn_exp2f((p.max - most) * log2e);
      p.sum = own + sum * __builtin_amdgcn_exp2f((mx - most) * log2e);
      if (p.arg < 0 || mx > p.max || (mx == p.max && arg < p.arg)) p.arg = arg;
      p.max = most;
    }
    p.min = fminf(p.min, __shfl_xor(p.min, d, kWave));
  }
  auto first = [](float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); };
  r.max = first(p.max);
  r.min = first(p.min);
  r.arg = __builtin_amdgcn_readfirstlane(p.arg);
  r.sum = first(p.sum);
}

// Token i of logit l for row b.
__device__ __forceinline__ void give(const SampleArgs& a, int b, const Row& r, int i, float l) {
  a.token[b] = i;
  if (!a.logprob) return;
  if (i < 0) {
    a.logprob[b] = -__builtin_inff();
    return;
  }
  if (r.max == __builtin_inff()) {  // the infinite ones share the row
    a.logprob[b] = __builtin_nanf("");
    return;
  }
  a.logprob[b] = (l - r.max) - __builtin_amdgcn_logf(r.sum) * 0.69314718055994531f;
}

__device__ __forceinline__ const void* row_of(const SampleArgs& a, int b, int dt) {
  return static_cast<const char*>(a.x) + (int64_t)b * a.ld * (dt == FG_F32 ? 4 : 2);
}

}  // namespace

// ------------------------------------------------------------------------------------------------ extremes
template <int DT>
__global__ void __launch_bounds__(kThreads) sample_extremes_kernel(const SampleArgs a) {
  __shared__ ChunkSum part[kWaves];
  const int b = blockIdx.x / a.chunks, c = blockIdx.x - b * a.chunks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowState& s = reinterpret_cast<RowState*>(a.ws)[b];
  if (a.cuts) {
    for (int i = c * kThreads + threadIdx.x; i < kBins; i += a.chunks * kThreads) {
      s.mass[i] = 0;
      s.count[i] = 0;
    }
  }
  if (c == 0 && threadIdx.x == 0) s.listed = s.ticket[0] = s.ticket[1] = s.done = 0;
  const void* row = row_of(a, b, DT);
  const int end = min(a.V, (c + 1) * a.chunk);
  const float inf = __builtin_inff(), log2e = 1.4426950408889634f;
  float mx = -inf, mn = inf, sum = 0.f;
  int arg = -1;
  sweep<DT, 2>(row, c * a.chunk + 4 * threadIdx.x, 4 * kThreads, end, [&](int i, const float (&l)[4]) {
    const float was = mx;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (l[j] > mx) {
        mx = l[j];
        arg = i + j;
      }
      mn = l[j] > -inf ? fminf(mn, l[j]) : mn;
    }
    if (a.logprob && mx > -inf) {
      sum *= __builtin_amdgcn_exp2f((was - mx) * log2e);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += __builtin_amdgcn_exp2f((l[j] - mx) * log2e);
    }
  });
  auto join = [&](float m2, float n2, int a2, float s2) {
    if (a2 < 0) return;
    if (arg < 0 || m2 > mx || (m2 == mx && a2 < arg)) {
      sum = s2 + (arg < 0 ? 0.f : sum * __builtin_amdgcn_exp2f((mx - m2) * log2e));
      mx = m2;
      arg = a2;
    } else {
      sum += s2 * __builtin_amdgcn_exp2f((m2 - mx) * log2e);
    }
    mn = fminf(mn, n2);
  };
  for (int d = 1; d < 64; d *= 2) {
    const float m2 = __shfl_xor(mx, d, kWave), n2 = __shfl_xor(mn, d, kWave), s2 = __shfl_xor(sum, d, kWave);
    const int a2 = __shfl_xor(arg, d, kWave);
    join(m2, n2, a2, s2);
  }
  if (lane == 0) part[wave] = {mx, mn, arg, sum};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) join(part[w].max, part[w].min, part[w].arg, part[w].sum);
    s.part[c] = {mx, mn, arg, sum};
  }
}

// ------------------------------------------------------------------------------------------------ histogram
template <int DT>
__global__ void __launch_bounds__(kThreads) sample_histogram_kernel(const SampleArgs a) {
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ Powers powers;
  const int b = blockIdx.x / a.chunks, c = blockIdx.x - b * a.chunks;
  RowState& s = reinterpret_cast<RowState*>(a.ws)[b];
  Row r;
  row_settings(a, b, r);
  if (r.greedy || !(r.by_k || r.by_p)) return;
  row_extremes(a, s, r);
  if (r.arg < 0) return;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  powers.fill();
  __syncthreads();
  const void* row = row_of(a, b, DT);
  const int end = min(a.V, (c + 1) * a.chunk);
  const double scale = bin_scale(r, a.bits), top = most(a.bits);
  sweep<DT, 2>(row, c * a.chunk + 4 * threadIdx.x, 4 * kThreads, end, [&](int, const float (&l)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double y = exponent(r, l[j]);
      if (!(y < top)) continue;
      const int bin = bin_of(y, scale);
      // without top-p nobody asks what the bins weigh
      if (r.by_p) atomicAdd(reinterpret_cast<unsigned long long*>(&mass[bin]), (unsigned long long)whole(weight(powers, y, a.bits)));
      atomicAdd(&count[bin], 1u);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    if (a.chunks == 1) {
      s.mass[i] = mass[i];
      s.count[i] = count[i];
    } else if (count[i]) {
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[i]), (unsigned long long)mass[i]);
      atomicAdd(&s.count[i], count[i]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ borders
namespace {

struct Shared {
  uint64_t mass[kBins];
  uint64_t list[kList];
  uint64_t part[kWaves];
  Powers powers;
  uint64_t found[3];
  uint32_t lo[kWaves], hi[kWaves], tokens[kWaves];
  uint64_t kept, total;
  uint32_t edges, cut_key, cut_index;
  int last;
  // the borders' bins, the tokens and the weight in front of them and in them
  int bin_k, bin_lo, bin_hi;
  uint64_t k_mass, k_full, lo_mass;
  uint32_t k_count, k_tokens, lo_count, hi_count;
  uint32_t listed, place;
};

// The smallest coordinate at which the sum of the values of the elements up to there reaches `target`; the sum in front of it, and what
// it has itself: by histograms, each over a bin of the one before.  each(f) calls f(coordinate, value) for the elements, whose
// coordinates are lo .. hi, or where lo > hi looked for first; false: the sum of all of them does not reach it.
struct Border {
  uint32_t at;
  uint64_t before, here;
};
template <class Each>
__device__ __forceinline__ bool border(Shared& m, uint64_t target, uint32_t lo, uint32_t hi, const Each& each, Border* found) {
  constexpr int kPer = kBins / kThreads, kLog = 11;  // bins of a thread, of all
  static_assert(kBins == 1 << kLog, "");
  const int me = threadIdx.x;
  __syncthreads();  // what an earlier call left in m has been read
  if (lo > hi) {
    each([&](uint32_t c, uint64_t) {
      lo = min(lo, c);
      hi = max(hi, c);
    });
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, d, kWave));
      hi = max(hi, (uint32_t)__shfl_xor((int)hi, d, kWave));
    }
    if ((threadIdx.x & 63) == 0) {
      m.lo[threadIdx.x >> 6] = lo;
      m.hi[threadIdx.x >> 6] = hi;
    }
    __syncthreads();
#pragma unroll 4  // a sixteenth at once takes the registers of the second workgroup on a CU
    for (int w = 0; w < kWaves; ++w) {
      lo = min(lo, m.lo[w]);
      hi = max(hi, m.hi[w]);
    }
  }
  uint64_t base = 0;
  if (lo > hi) return false;
  for (;;) {
    const int width = 32 - __clz((int)(hi - lo)), shift = width > kLog ? width - kLog : 0;  // (hi - lo) >> shift < 2^kLog
#pragma unroll
    for (int j = 0; j < kPer; ++j) m.mass[me * kPer + j] = 0;
    if (me == 0) m.found[0] = ~0ull;
    __syncthreads();
    each([&](uint32_t c, uint64_t v) {
      if (c >= lo && c <= hi) atomicAdd(reinterpret_cast<unsigned long long*>(&m.mass[(c - lo) >> shift]), (unsigned long long)v);
    });
    __syncthreads();
    uint64_t v[kPer], sum = 0, all;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      v[j] = m.mass[me * kPer + j];
      sum += v[j];
    }
    sum = base + block_scan(sum, m.part, &all);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (sum < target && target <= sum + v[j]) {
        m.found[0] = me * kPer + j;
        m.found[1] = sum;
        m.found[2] = v[j];
      }
      sum += v[j];
    }
    __syncthreads();
    const uint64_t bin = m.found[0], here = m.found[2];
    if (bin == ~0ull) return false;
    base = m.found[1];
    lo += (uint32_t)bin << shift;
    if (shift == 0) {
      *found = {lo, base, here};
      return true;
    }
    hi = (uint32_t)min((uint64_t)hi, (uint64_t)lo + ((1u << shift) - 1));
    __syncthreads();
  }
}

// The smallest whole number that is p times s or more, and not less than one.
__device__ __forceinline__ uint64_t share(float p, uint64_t s) {
  const double v = ceil((double)p * (double)s);
  return v > 1 ? min((uint64_t)v, s) : 1;
}
// Whether a token weighs min_p of the largest.
__device__ __forceinline__ bool weighs(const Row& r, const Powers& t, double y, int bits) {
  return !(r.minp > 0.f) || weight(t, y, bits) >= (double)r.minp * (double)(1ull << bits);
}
// What the kept weights' sum has to reach: the first whole number past u times the total.
__device__ __forceinline__ uint64_t drawn(float u, uint64_t total) {
  const double v = floor((double)u * (double)total);
  return v > 0 ? min((uint64_t)v, total - 1) + 1 : 1;  // NaN counts as 0
}

constexpr int kFew = 256;  // tokens that are settled by comparing each with all

// What the histogram says of a row: its border bins (bin_lo .. bin_hi of top-p, bin_k of top-k) and what is collected.
struct Edges {
  bool by_k, by_p, whole_row, fits;
  int bin_k, bin_lo, bin_hi;
  uint64_t mass;  // of all tokens
  double scale;
  __device__ __forceinline__ bool border_bin(int bin) const { return (by_k && bin == bin_k) || (bin >= bin_lo && bin <= bin_hi); }
};

// Where the kept tokens end, from the tokens of the border bins: m.cut_key, m.cut_index.  each(f) calls f(key, index, weight, bin) for
// them (and maybe others).
template <class Each>
__device__ __forceinline__ void cut_by_bins(const SampleArgs& a, Shared& m, const Row& r, const Edges& q, const Each& each) {
  constexpr uint32_t kAny = 0xffffffffu;
  // the k-th token's key, and how many of that key are among the k
  Border at;
  uint32_t cut = 0;
  uint64_t ties = ~0ull, equals = 0, kept = q.mass;
  if (q.by_k) {
    const uint64_t need = (uint64_t)r.k - m.k_count;
    border(m, need, kAny, 0, [&](auto f) {
      each([&](uint32_t key, uint32_t, uint64_t, int bin) {
        if (bin == q.bin_k) f(~key, 1);
      });
    }, &at);
    cut = ~at.at;
    ties = need - at.before;
    equals = at.here;
    if (r.by_p) {  // what the k tokens weigh
      uint64_t above = 0;
      each([&](uint32_t key, uint32_t, uint64_t w, int bin) {
        if (bin == q.bin_k && key > cut) above += w;
      });
      block_scan(above, m.part, &kept);
      kept += m.k_mass + ties * whole(weight(m.powers, exponent(r, of_key(cut)), a.bits));
    }
  }
  if (r.by_p) {
    const uint64_t need = share(r.p, kept), lo_mass = m.lo_mass;
    if (need > lo_mass && border(m, need - lo_mass, kAny, 0, [&](auto f) {
          each([&](uint32_t key, uint32_t, uint64_t w, int bin) {
            if (bin >= q.bin_lo && bin <= q.bin_hi) f(~key, w);
          });
        }, &at)) {
      const uint32_t key = ~at.at;
      const uint64_t one_of = max(whole(weight(m.powers, exponent(r, of_key(key)), a.bits)), (uint64_t)1);
      const uint64_t some = (need - lo_mass - at.before + one_of - 1) / one_of;
      if (key > cut || (key == cut && some < ties)) {
        cut = key;
        ties = some;
        equals = at.here / one_of;
      }
    }
  }
  // the last one of the border's equals that is kept, if not all are
  uint32_t cut_index = kAny;
  if (ties < equals && border(m, ties, 0, (uint32_t)a.V - 1, [&](auto f) {
        each([&](uint32_t key, uint32_t i, uint64_t, int) {
          if (key == cut) f(i, 1);
        });
      }, &at))
    cut_index = at.at;
  if (threadIdx.x == 0) {
    m.cut_key = cut;
    m.cut_index = cut_index;
  }
}

// The same for few tokens: four threads each, which go over a quarter of all of them for what stands in front of their own.  m.mass
// holds a pair for each token, its place in the order (the key, then the index backwards) and its weight.
__device__ __forceinline__ void cut_by_places(const SampleArgs& a, Shared& m, const Row& r, const Edges& q, int listed) {
  ulonglong2* const pairs = reinterpret_cast<ulonglong2*>(m.mass);
  static_assert(kFew * sizeof(ulonglong2) <= sizeof(m.mass) && kFew * 4 == kThreads, "");
  for (int i = threadIdx.x; i < listed; i += kThreads) {
    const uint64_t item = m.list[i];
    const uint32_t key = (uint32_t)(item >> 32);
    const double y = exponent(r, of_key(key));
    if (!q.border_bin(bin_of(y, q.scale))) continue;
    const uint32_t at = atomicAdd(&m.edges, 1u);
    if (at < kFew) pairs[at] = make_ulonglong2((uint64_t)key << 32 | (uint32_t)~(uint32_t)item, whole(weight(m.powers, y, a.bits)));
  }
  __syncthreads();
  const int count = min((int)m.edges, kFew), i = threadIdx.x / 4, quarter = threadIdx.x % 4;
  const bool is = i < count;
  uint64_t place = 0, w = 0, w_front = 0;
  uint32_t n_front = 0;
  if (is) {
    place = pairs[i].x;
    w = pairs[i].y;
#pragma unroll 4
    for (int j = quarter; j < count; j += 4) {
      const ulonglong2 p = pairs[j];
      const bool front = p.x > place;
      n_front += front;
      w_front += front ? p.y : 0;
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    n_front += (uint32_t)__shfl_xor((int)n_front, d, kWave);
    w_front += shfl_xor64(w_front, d);
  }
  // The bins of top-p (tokens that weigh up to its mark lie in these alone), then bin_k.
  bool keep = is;
  uint64_t mass = q.mass;
  if (q.by_k) {
    const uint32_t in_front = !q.by_p ? 0 : (q.bin_k > q.bin_hi ? m.hi_count : m.k_count) - m.lo_count;
    const bool in_k = is && n_front >= in_front;
    keep = is && (!in_k || n_front + (m.k_count - in_front) < (uint32_t)r.k);
    if (q.by_p) {  // what the k tokens weigh
      if (keep && in_k && quarter == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&m.kept), (unsigned long long)w);
      __syncthreads();
      mass = m.k_mass + m.kept;
    }
  }
  if (q.by_p) keep = keep && w_front + m.lo_mass < share(r.p, mass);
  const int kept = __syncthreads_count(keep && quarter == 0);
  if (keep && quarter == 0 && (int)n_front == kept - 1) {  // the last one
    m.cut_key = (uint32_t)(place >> 32);
    m.cut_index = ~(uint32_t)place;
  }
}

// The row's border from its collected tokens and, where these are the whole row that matters, its token.
template <int DT>
__device__ __forceinline__ void settle(const SampleArgs& a, Shared& m, RowState& s, int b, const Row& r, const void* row, const Edges& q, int count,
                                       int edge) {
  const double scale = q.scale, top = most(a.bits);
  const int me = threadIdx.x, all = q.fits ? count : a.V;
  if (q.fits && a.chunks > 1)
    for (int i = me; i < count; i += kThreads) m.list[i] = get_far(&s.list[i]);
  if (me == 0) {
    m.kept = m.total = 0;
    m.edges = m.cut_key = 0;
    m.cut_index = 0xffffffffu;
  }
  __syncthreads();
  // Calls f(key, index, weight, bin) for the collected tokens or, where they are too many for the list, for the border bins'.  (Nothing
  // of them stays in registers: the kernel's 64 let a CU hold two workgroups.)
  auto each = [&](auto f) {
#pragma unroll 1
    for (int i = me; i < all; i += kThreads) {
      const uint64_t item = q.fits ? m.list[i] : (uint64_t)key_of(one<DT>(row, i)) << 32 | (uint32_t)i;
      const uint32_t key = (uint32_t)(item >> 32);
      const double y = exponent(r, of_key(key));
      if (!(y < top)) continue;
      const int bin = bin_of(y, scale);
      if (q.fits || q.border_bin(bin)) f(key, (uint32_t)item, whole(weight(m.powers, y, a.bits)), bin);
    }
  };
  if (q.by_k || q.by_p) {
    if (q.fits && edge <= kFew) cut_by_places(a, m, r, q, count);
    else cut_by_bins(a, m, r, q, each);
    __syncthreads();
  }
  const uint32_t cut = m.cut_key, cut_index = m.cut_index;
  if (!q.whole_row) {
    if (me == 0) {
      s.cut_key = cut;
      s.cut_index = cut_index;
    }
    return;
  }
  auto keeps = [&](uint32_t key, uint32_t i) {
    return (key > cut || (key == cut && i <= cut_index)) && weighs(r, m.powers, exponent(r, of_key(key)), a.bits);
  };
  int token = -1;  // of the one thread that has it
  if (count <= kFew) {
    // four threads a token, for the sum of what is kept in front of it
    ulonglong2* const pairs = reinterpret_cast<ulonglong2*>(m.mass);  // index, weight
    const int i = me / 4, quarter = me % 4;
    uint32_t index = 0;
    uint64_t w = 0, before = 0;
    if (i < count) {
      const uint64_t item = m.list[i];
      const uint32_t key = (uint32_t)(item >> 32);
      index = (uint32_t)item;
      if (keeps(key, index)) w = whole(weight(m.powers, exponent(r, of_key(key)), a.bits));
    }
    if (quarter == 0) {
      pairs[i] = make_ulonglong2(index, w);
      if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&m.total), (unsigned long long)w);
    }
    __syncthreads();
    if (w) {
#pragma unroll 4
      for (int j = quarter; j < count; j += 4) {
        const ulonglong2 p = pairs[j];
        before += p.x < index ? p.y : 0;
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d *= 2) before += shfl_xor64(before, d);
    const uint64_t target = drawn(a.u[b], m.total);
    if (quarter == 0 && before < target && target <= before + w) token = (int)index;
  } else {
    uint64_t mine = 0, total = 0;
    each([&](uint32_t key, uint32_t i, uint64_t w, int) { mine += keeps(key, i) ? w : 0; });
    block_scan(mine, m.part, &total);
    Border at;
    border(m, drawn(a.u[b], total), 0, (uint32_t)a.V - 1, [&](auto f) {
      each([&](uint32_t key, uint32_t i, uint64_t w, int) {
        if (keeps(key, i)) f(i, w);
      });
    }, &at);
    if (me == 0) token = (int)at.at;
  }
  if (token >= 0) {
    give(a, b, r, token, one<DT>(row, token));
    s.done = 1;
  }
}

}  // namespace

template <int DT>
__global__ void __launch_bounds__(kThreads, 8) sample_borders_kernel(const SampleArgs a) {
  __shared__ Shared m;
  const int b = blockIdx.x / a.chunks, c = blockIdx.x - b * a.chunks;
  RowState& s = reinterpret_cast<RowState*>(a.ws)[b];
  Row r;
  row_settings(a, b, r);
  if (r.greedy || !(r.by_k || r.by_p)) return;
  uint64_t v[2];
  uint32_t n[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    v[j] = r.by_p ? s.mass[2 * threadIdx.x + j] : 0;
    n[j] = s.count[2 * threadIdx.x + j];
  }
  row_extremes(a, s, r);
  if (r.arg < 0) return;
  const void* row = row_of(a, b, DT);
  const double scale = bin_scale(r, a.bits), top = most(a.bits);
  m.powers.fill();
  if (threadIdx.x == 0) {
    m.bin_k = kBins;
    m.k_mass = m.k_full = m.lo_mass = 0;
    m.listed = 0;
  }

  // Where the borders are: sums in front of each thread's two bins.
  uint64_t mass, v0;
  uint32_t tokens, n0;
  block_scan2(v[0] + v[1], n[0] + n[1], m.part, m.tokens, &v0, &mass, &n0, &tokens);
  auto find = [&](auto f) {  // calls f(bin, weight in front, tokens in front, weight, tokens)
    uint64_t vs = v0;
    uint32_t ns = n0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f(2 * (int)threadIdx.x + j, vs, ns, v[j], n[j]);
      vs += v[j];
      ns += n[j];
    }
  };
  const bool by_k = r.by_k && (uint32_t)r.k < tokens;
  if (by_k)
    find([&](int bin, uint64_t vs, uint32_t ns, uint64_t vb, uint32_t nb) {
      if (ns < (uint32_t)r.k && (uint32_t)r.k <= ns + nb) {
        m.bin_k = bin;
        m.k_mass = vs;
        m.k_full = vs + vb;
        m.k_count = ns;
        m.k_tokens = nb;
      }
    });
  __syncthreads();
  const int bin_k = m.bin_k;
  if (r.by_p) {
    // the k tokens weigh k_mass at least and k_full at most
    const uint64_t t0 = share(r.p, by_k ? m.k_mass : mass), t1 = share(r.p, by_k ? m.k_full : mass);
    find([&](int bin, uint64_t vs, uint32_t ns, uint64_t vb, uint32_t nb) {
      if (bin > bin_k) return;
      if (vs < t0 && t0 <= vs + vb) {
        m.bin_lo = bin;
        m.lo_mass = vs;
        m.lo_count = ns;
      }
      if (vs < t1 && t1 <= vs + vb) {
        m.bin_hi = bin;
        m.hi_count = ns + nb;
      }
    });
  }
  __syncthreads();
  // All tokens up to the last border, where they are few; else the border bins' own: from bin_lo to bin_hi, and bin_k.
  const int bin_lo = r.by_p ? m.bin_lo : kBins, bin_hi = r.by_p ? m.bin_hi : -1;
  const uint32_t upto = by_k ? m.k_count + m.k_tokens : (r.by_p ? m.hi_count : tokens);
  const bool whole_row = upto <= kList;
  if (!whole_row && !by_k && !r.by_p) {  // fewer than k tokens weigh anything
    if (c == 0 && threadIdx.x == 0) s.cut_key = s.cut_index = 0;
    return;
  }
  const uint32_t edge = (r.by_p ? m.hi_count - m.lo_count : 0) + (by_k && bin_k > bin_hi ? m.k_tokens : 0);
  const bool fits = whole_row || edge <= kList;
  const int last = whole_row ? (by_k ? bin_k : (r.by_p ? bin_hi : kBins - 1)) : max(by_k ? bin_k : 0, bin_hi);
  const Edges q = {by_k, r.by_p, whole_row, fits, bin_k, bin_lo, bin_hi, mass, scale};
  if (fits) {
    const int end = min(a.V, (c + 1) * a.chunk);
    const float least = floor_of(r, (last + 1.0) / scale);
    sweep<DT, 2>(row, c * a.chunk + 4 * threadIdx.x, 4 * kThreads, end, [&](int i, const float (&l)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(l[j] >= least)) continue;
        const double y = exponent(r, l[j]);
        if (!(y < top)) continue;
        const int bin = bin_of(y, scale);
        if (whole_row ? bin <= last : q.border_bin(bin)) {
          const uint32_t at = atomicAdd(&m.listed, 1u);  // the histogram has counted them: below kList
          if (at < kList) m.list[at] = (uint64_t)key_of(l[j]) << 32 | (uint32_t)(i + j);
        }
      }
    });
  }
  if (a.chunks > 1) {
    __syncthreads();
    const uint32_t n = min(m.listed, (uint32_t)kList);
    if (threadIdx.x == 0 && n) m.place = atomicAdd(&s.listed, n);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads)
      if (m.place + i < kList) put_far(&s.list[m.place + i], m.list[i]);
    if (!last_of_row(&s.ticket[0], a.chunks, &m.last)) return;
  } else {
    __syncthreads();
  }

  const int count = fits ? (int)(whole_row ? upto : edge) : 0;
  settle<DT>(a, m, s, b, r, row, q, count, (int)edge);
}

// ------------------------------------------------------------------------------------------------ sums in the order of the indexes
template <int DT>
__global__ void __launch_bounds__(kThreads, 8) sample_sums_kernel(const SampleArgs a) {
  __shared__ Powers powers;
  __shared__ uint64_t part[kWaves];
  __shared__ int is_last, found;
  __shared__ uint64_t found_before;
  const int b = blockIdx.x / a.sum_chunks, c = blockIdx.x - b * a.sum_chunks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowState& s = reinterpret_cast<RowState*>(a.ws)[b];
  Row r;
  row_settings(a, b, r);
  const void* row = row_of(a, b, DT);
  const bool cuts = r.by_k || r.by_p;
  if (!r.greedy && cuts && s.done) return;
  row_extremes(a, s, r);
  if (r.greedy || r.arg < 0) {  // the first of the largest, or none
    if (c == 0 && threadIdx.x == 0) give(a, b, r, r.arg, r.max);
    return;
  }
  powers.fill();
  __syncthreads();
  const uint32_t cut = cuts ? s.cut_key : 0, cut_index = cuts ? s.cut_index : 0;
  const double top = most(a.bits), least = (double)r.minp * (double)(1ull << a.bits);
  auto value = [&](float l, int i) -> uint64_t {  // what token i adds to the sum
    const uint32_t key = key_of(l);
    if (key < cut || (key == cut && (uint32_t)i > cut_index)) return 0;
    const double y = exponent(r, l);
    if (!(y < top)) return 0;
    const double w = weight(powers, y, a.bits);
    return w >= least ? whole(w) : 0;
  };
  // a wavefront sums up a stretch of its own
  const int stretch = a.sum_chunk / kWaves;
  auto first_of = [&](int piece) { return piece * stretch; };
  const int begin = first_of(c * kWaves + wave), end = min(a.V, begin + stretch);
  uint64_t sum = 0;
  sweep<DT, 4>(row, begin + 4 * lane, 256, end, [&](int i, const float (&l)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += value(l[j], i + j);
  });
  sum = wave_sum64(sum);
  if (lane == 0) put_far(&s.wave_mass[c * kWaves + wave], sum);
  if (!last_of_row(&s.ticket[1], a.sum_chunks, &is_last)) return;
  // the stretch in which the sum passes its mark, then the token: a thread takes some neighbours each
  auto pick = [&](uint64_t v, uint64_t base, uint64_t target, int id) {  // the thread whose values reach it
    uint64_t all;
    const uint64_t before = base + block_scan(v, part, &all);
    if (before < target && target <= before + v) {
      found = id;
      found_before = before;
    }
    __syncthreads();
  };
  const int pieces = a.sum_chunks * kWaves;  // 1024 at most
  const uint64_t mine = (int)threadIdx.x < pieces ? get_far(&s.wave_mass[threadIdx.x]) : 0;
  uint64_t total;
  block_scan(mine, part, &total);
  const uint64_t target = drawn(a.u[b], total);
  pick(mine, 0, target, threadIdx.x);
  const int from = first_of(found), to = min(a.V, from + stretch), per = (stretch + kThreads - 1) / kThreads;
  const uint64_t base = found_before;
  const int i0 = from + (int)threadIdx.x * per, i1 = min(to, i0 + per);
  uint64_t few = 0;
  for (int i = i0; i < i1; ++i) few += value(one<DT>(row, i), i);
  __syncthreads();
  pick(few, base, target, threadIdx.x);
  if (found == (int)threadIdx.x) {
    uint64_t at = found_before;
    for (int i = i0; i < i1; ++i) {
      const float l = one<DT>(row, i);
      at += value(l, i);
      if (at >= target) {
        give(a, b, r, i, l);
        break;
      }
    }
  }
}

// Chunks of whole 4096 columns, so that the rows fill the CUs about twice.
size_t sample_plan(SampleArgs& a) {
  const int64_t unit = 4 * kThreads, most_chunks = std::min<int64_t>(kMaxChunks, (a.V + unit - 1) / unit);
  const int64_t chunks = std::min<int64_t>(most_chunks, std::max<int64_t>(1, 2 * (int64_t)device_cus() / std::max(a.B, 1)));
  a.chunk = (int)(((a.V + chunks - 1) / chunks + unit - 1) / unit * unit);
  a.chunks = (a.V + a.chunk - 1) / a.chunk;
  // The sums in pieces of half that, where it is 32768 columns or more (and a row's stretches stay as many as a workgroup's threads): rows that are settled before leave their CUs to the others (256 rows of 150001: mixed settings 192 us, now 169,
  // top-p 0.95 for all 185, now 192).
  a.sum_chunk = a.chunk >= 8 * unit && a.chunks <= kMaxChunks / 2 ? (int)((a.chunk / 2 + unit - 1) / unit * unit) : a.chunk;
  a.sum_chunks = (a.V + a.sum_chunk - 1) / a.sum_chunk;
  int log = 0;
  while ((1LL << log) < a.V) ++log;
  a.bits = std::min(46, 62 - log);  // the sum of all weights stays below 2^63
  return (size_t)a.B * sizeof(RowState);
}

hipError_t launch_sample(const SampleArgs& a, int dt, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.B * a.chunks)), block(kThreads);
  auto go = [&](auto dt_tag) {
    constexpr int DT = decltype(dt_tag)::value;
    hipLaunchKernelGGL((sample_extremes_kernel<DT>), grid, block, 0, st, a);
    if (a.cuts) {
      hipLaunchKernelGGL((sample_histogram_kernel<DT>), grid, block, 0, st, a);
      hipLaunchKernelGGL((sample_borders_kernel<DT>), grid, block, 0, st, a);
    }
    hipLaunchKernelGGL((sample_sums_kernel<DT>), dim3((unsigned)((int64_t)a.B * a.sum_chunks)), block, 0, st, a);
    note_kernel("sample_extremes_kernel%s + sample_sums_kernel chunks=%d",
                a.cuts ? " + sample_histogram_kernel + sample_borders_kernel" : "", a.chunks);
    return hipGetLastError();
  };
  if (dt == FG_F32) return go(std::integral_constant<int, FG_F32>{});
  if (dt == FG_BF16) return go(std::integral_constant<int, FG_BF16>{});
  return go(std::integral_constant<int, FG_F16>{});
}

}  // namespace fg
