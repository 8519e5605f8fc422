// Rotary position embedding of a qkv projection's queries and keys, and the keys' and values' way into a paged cache, in one
// launch.  Columns a, b of a pair turn by the position's angle: a' = a cos - b sin, b' = b cos + a sin in fp32, rounded once,
// to the queries' type or to the cache's (e4m3 of the IEEE quotient by the key head's scale).  A pair is columns
// (i, i + rot / 2), or (2 i, 2 i + 1) interleaved; columns from rot on pass through.
//
// One token per workgroup row of the grid: a thread keeps the cosines and sines of one item (V pairs) and walks the token's
// heads with it, so the table is read once per token and not once per head.  Bound by one read and one write of the token
// for a prompt (8192 tokens of 32 + 2 x 8 heads of 128, bf16: 38.6 us, 5.3 TB/s), by the latency of position -> table ->
// store for few tokens (one: 2.7 us).
#include <algorithm>

#include "fg_codes.h"
#include "fg_decoder.h"

namespace fg {

// Threads per workgroup: a token's heads are walked in equal turns (us, up to 128 / 256 / 512 threads: 8192 tokens of 32 + 2 x 8
// heads of 128 in bf16 38.6 / 43.2 / 58.6, into an e4m3 cache 37.3 / 40.1 / 60.1, 64 tokens 4.2 / 5.1 / 4.4; a fixed 256
// threads, the last turn partly empty: 48.2, 45.2, 4.2).
constexpr int kRopeThreads = 128;

namespace {

template <int V>
struct Vec16;
template <>
struct Vec16<8> {
  typedef uint16_t t __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Vec16<4> {
  typedef uint16_t t __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Vec16<1> {
  typedef uint16_t t __attribute__((ext_vector_type(1), aligned(2)));
};

template <bool BF16>
__device__ __forceinline__ float bits_f(uint16_t b) {
  return BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}
template <bool BF16>
__device__ __forceinline__ uint16_t f_bits(float f) {
  return BF16 ? f32_to_bf16_bits_hw(f) : f32_to_f16_bits(f);
}

template <bool BF16, int V>
__device__ __forceinline__ void load_v(const uint16_t* p, float (&f)[V]) {
  const auto r = *reinterpret_cast<const typename Vec16<V>::t*>(p);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = bits_f<BF16>(r[j]);
}

template <bool BF16, int V>
__device__ __forceinline__ void store_v(uint16_t* p, const float (&f)[V]) {
  typename Vec16<V>::t r;
#pragma unroll
  for (int j = 0; j < V; ++j) r[j] = f_bits<BF16>(f[j]);
  *reinterpret_cast<typename Vec16<V>::t*>(p) = r;
}

// V columns of a cache row at column `col`: 16-bit values, or e4m3 codes of f / scale.
template <bool BF16, bool FP8, int V>
__device__ __forceinline__ void store_cache(uint8_t* row, int col, const float (&f)[V], float scale) {
  if constexpr (!FP8) {
    store_v<BF16, V>(reinterpret_cast<uint16_t*>(row) + col, f);
  } else {
    uint32_t w[(V + 3) / 4] = {};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float c = __fdiv_rn(f[j], scale);
      w[j / 4] |= (uint32_t)f32_to_e4m3(__builtin_isnan(c) ? c : fminf(fmaxf(c, -448.f), 448.f)) << (8 * (j % 4));
    }
    if constexpr (V == 8) *reinterpret_cast<uint2*>(row + col) = make_uint2(w[0], w[1]);
    else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(row + col) = w[0];
    else row[col] = (uint8_t)w[0];
  }
}

}  // namespace

template <bool BF16, bool FP8, bool INTER, int V>
__global__ void __launch_bounds__(256) rope_append_kernel(const RopeAppendArgs a, int rows) {
  const int64_t t = blockIdx.x;
  const int pairs = a.rot / 2 / V, items = pairs + (a.D - a.rot) / V;
  const int item = threadIdx.x % items, row = threadIdx.x / items;
  if (row >= rows) return;
  const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
  const int64_t slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[t] : static_cast<const int32_t*>(a.slots)[t];
  const bool keep = slot >= 0 && slot < a.n_slots;  // any other slot is padding
  const int64_t page = keep ? slot / a.page : 0, off = keep ? slot - page * a.page : 0;
  float cs[V], sn[V];
  if (item < pairs) {
    const bool in = pos >= 0 && pos < a.max_pos;  // a position that the table lacks shows as NaN
#pragma unroll
    for (int j = 0; j < V; ++j) {
      cs[j] = in ? a.table[pos * a.ld_table + item * V + j] : __builtin_nanf("");
      sn[j] = in ? a.table[pos * a.ld_table + a.rot / 2 + item * V + j] : __builtin_nanf("");
    }
  }
  const int H = a.Hq + 2 * a.Hk;
  for (int h = blockIdx.y * rows + row; h < H; h += gridDim.y * rows) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
    const int hk = is_v ? h - a.Hq - a.Hk : h - a.Hq;
    if (!is_q && !keep) continue;
    const uint16_t* src = is_q ? a.q + t * a.q_t + h * a.q_h : (is_v ? a.v + t * a.v_t + hk * a.v_h : a.k + t * a.k_t + hk * a.k_h);
    uint8_t* cache = (is_v ? a.vc : a.kc) + page * a.c_page + hk * a.c_head + off * a.c_token;
    uint16_t* qo = a.qo + t * a.qo_t + h * a.qo_h;
    const float scale = FP8 && !is_q ? (is_v ? a.vs : a.ks)[hk] : 1.f;
    auto put = [&](int col, const float(&f)[V]) {
      if (is_q) store_v<BF16, V>(qo + col, f);
      else store_cache<BF16, FP8, V>(cache, col, f, scale);
    };
    float x[V], y[V];
    if (is_v) {  // two units of V columns per item
      if (item >= a.D / 2 / V) continue;
      load_v<BF16, V>(src + 2 * item * V, x);
      load_v<BF16, V>(src + 2 * item * V + V, y);
      put(2 * item * V, x);
      put(2 * item * V + V, y);
    } else if (item >= pairs) {
      const int col = a.rot + (item - pairs) * V;
      load_v<BF16, V>(src + col, x);
      put(col, x);
    } else {
      const int c0 = INTER ? 2 * item * V : item * V, c1 = INTER ? c0 + V : c0 + a.rot / 2;
      load_v<BF16, V>(src + c0, x);
      load_v<BF16, V>(src + c1, y);
      float u[2 * V], o[V], p[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // pair j: neighbours of the 2 V columns, or column j of either half
        const float f0 = INTER ? (2 * j < V ? x[2 * j % V] : y[2 * j % V]) : x[j];
        const float f1 = INTER ? (2 * j + 1 < V ? x[(2 * j + 1) % V] : y[(2 * j + 1) % V]) : y[j];
        const float r0 = f0 * cs[j] - f1 * sn[j], r1 = f1 * cs[j] + f0 * sn[j];
        u[INTER ? 2 * j : j] = r0;
        u[INTER ? 2 * j + 1 : V + j] = r1;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        o[j] = u[j];
        p[j] = u[V + j];
      }
      put(c0, o);
      put(c1, p);
    }
  }
}

hipError_t launch_rope_append(const RopeAppendArgs& a, int64_t T, bool bf16, bool fp8, bool inter, hipStream_t st) {
  // V: the widest unit that the halves, the columns that pass through and the values' halves are whole multiples of
  auto fits = [&](int v) { return (a.rot / 2) % v == 0 && (a.D - a.rot) % v == 0 && (a.D / 2) % v == 0; };
  const int V = fits(8) ? 8 : (fits(4) ? 4 : 1);
  // few tokens: the turns are workgroups.  A head has at most 255 items (256 columns, one at a time)
  const int items = a.rot / 2 / V + (a.D - a.rot) / V, H = a.Hq + 2 * a.Hk;
  const int turns = (H * items + kRopeThreads - 1) / kRopeThreads, rows = std::max(1, std::min((H + turns - 1) / turns, kRopeThreads / items));
  const unsigned threads = (unsigned)(items * rows + 63) / 64 * 64;
  const unsigned gy = T <= 2 * device_cus() ? (unsigned)((H + rows - 1) / rows) : 1u;
  if (!launchable(T * gy, (int)threads)) return hipErrorInvalidConfiguration;
  auto go = [&](auto b_tag, auto f_tag, auto i_tag, auto v_tag) {
    note_kernel("rope_append_kernel<V=%d> heads/%u", V, gy);
    hipLaunchKernelGGL((rope_append_kernel<decltype(b_tag)::value, decltype(f_tag)::value, decltype(i_tag)::value,
                                           decltype(v_tag)::value>),
                       dim3((unsigned)T, gy), dim3(threads), 0, st, a, rows);
    return hipGetLastError();
  };
  auto by_v = [&](auto b_tag, auto f_tag, auto i_tag) {
    if (V == 8) return go(b_tag, f_tag, i_tag, std::integral_constant<int, 8>{});
    if (V == 4) return go(b_tag, f_tag, i_tag, std::integral_constant<int, 4>{});
    return go(b_tag, f_tag, i_tag, std::integral_constant<int, 1>{});
  };
  auto by_i = [&](auto b_tag, auto f_tag) {
    return inter ? by_v(b_tag, f_tag, std::true_type{}) : by_v(b_tag, f_tag, std::false_type{});
  };
  auto by_f = [&](auto b_tag) { return fp8 ? by_i(b_tag, std::true_type{}) : by_i(b_tag, std::false_type{}); };
  return bf16 ? by_f(std::true_type{}) : by_f(std::false_type{});
}

}  // namespace fg
