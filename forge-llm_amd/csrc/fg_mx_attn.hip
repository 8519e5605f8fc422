// Attention over a block-scaled cache: o = softmax(s) V over the keys in a query token's window, s = scale q k or, capped,
// cap tanh(scale q k / cap).  Keys are cut into parts, an item (row tile, key head, part) makes one pass over its keys with a running
// maximum and sum (mx_rows, mx_tile), and the parts of a row are joined as in attention over 16-bit pages.  Here: the join and the
// plan.
#include <algorithm>

#include "fg_attn_join.h"
#include "fg_mx_attn.h"

namespace fg {

template <bool BF16, int L, int W>
__global__ void __launch_bounds__(256) mx_join_kernel(const MxAttnArgs m) {
  const AttnArgs& a = m.a;
  const JoinRow<L, W> r;
  if (r.id >= (int64_t)a.T * a.Hq) return;
  const int t = (int)(r.id / a.Hq), h = (int)(r.id - (int64_t)t * a.Hq);
  int seq = t, tok = 0, count = 1;
  bool inside = true;
  if (a.starts) {
    seq = attn_sequence(a, t);
    inside = a.B > 0 && a.starts[seq] <= t && t < a.starts[seq + 1];
    if (inside) {
      const int first = attn_start(a, seq);
      tok = t - first;
      count = attn_start(a, seq + 1) - first;
    }
  }
  const bool served = !inside || tok < a.max_q;
  int n = 0;
  if (inside && served) {  // the parts of the row's tile
    const int len = max(min(a.lens[seq], a.max_len), 0), rows = min(count, a.max_q) * a.G, tile = m.tile ? kTileRows : 16;
    const int row0 = (tok * a.G + h % a.G) / tile * tile;
    const MxRange all = mx_range(m, len, len - count + 1, row0 / a.G, min(rows - 1, row0 + tile - 1) / a.G);
    n = max((all.end - all.begin + a.part_s - 1) / a.part_s, 1);
  }
  attn_join<BF16, L, W>(a, r, t, h, n, served);
}

static int join_waves(const MxAttnArgs& m) { return m.a.parts_s >= 8 ? 4 : 1; }

// Fills in the plan; returns the partial sums' bytes.  items is -1 where the threads of a launch would pass 32 bits.
size_t mx_attn_plan(MxAttnArgs& m) {
  AttnArgs& a = m.a;
  const int64_t rows = (int64_t)a.max_q * a.G, cus = device_cus();
  m.tile = rows > 16;
  const int64_t tile = m.tile ? kTileRows : 16, tokens = std::min<int64_t>(a.max_q, tile / a.G + 2);
  // keys that a tile's rows see at most, from a whole tile of 32 on
  const int64_t span = std::min<int64_t>(a.max_len, (int64_t)m.window + tokens + 30);
  a.tiles_s = (int)((rows + tile - 1) / tile);
  const int64_t sets = (int64_t)a.Hk * a.B, items = std::max<int64_t>(sets * a.tiles_s, 1), unit = m.tile ? 64 : kRowsTile * kRowsWaves;
  int64_t parts = 1;
  if (m.tile) {
    // The cheapest number by rounds of the CUs times keys of a part, and 96 keys' worth for each part's begin, end and share of the join.
    // Row tiles are those that the number of query tokens suggests, as prompts of a batch have other lengths than the longest.  us with 1 /
    // 2 / 3 / 4 parts: 16 + 2 x 8 heads of 256, one workgroup on a CU, windows of 1024, prompts of 75 to 300 (2) 84 / 63 / 79 / 76, of 300
    // (3) 86 / 109 / 88 / 108, 512 queries on 4096 keys (4) 251 / 145 / 108 / 87; 32 + 2 x 8 heads of 128, two on a CU, 300 queries
    // each on 4 x 4000 (3) 156 / 148 / 135 / 137; of 64, 200 on 8 x 2000 (1) 51 / 80 / 79 / 79.
    const int64_t slots = (a.D > 128 ? 1 : 2) * cus;
    const int64_t real = std::max<int64_t>(1, std::min(items, a.Hk * ((int64_t)a.T * a.G / tile + (a.B + 1) / 2)));
    int64_t best = INT64_MAX;
    for (int p = 1; p <= 16; ++p) {
      const int64_t cost = (real * p + slots - 1) / slots * ((span + p - 1) / p) + 96 * p;
      if (cost < best) {
        best = cost;
        parts = p;
      }
    }
  } else {
    // About two workgroups per CU: us by keys per part, 32 + 2 x 8 heads of 128 in 4 bits, 1 sequence of 5000 128 / 256 / 512: 11.6 /
    // 10.9 / 12.0, 4 of 16000 512 / 1024: 20.0 / 19.6, 16 of 4000 with 4 queries each 512 / 1024: 21.2 / 20.5.  Where the sequences fill
    // the CUs by themselves one part does, but for long ones, which would outlast the others: parts of 2048 keys (64 of 2048 to 16384,
    // 64 + 2 x 8 heads, 16384 / 4096 / 2048: 170 / 148 / 150; 64 of up to 8000 x 64 columns 8000 / 4096 / 2048: 58 / 66 / 56; 64 of up
    // to 4000 x 256 columns 4000 / 2048: 108 / 129).
    parts = std::max<int64_t>(1, 2 * cus / items);
    if (span > 8192) parts = std::max<int64_t>(parts, (span + 2047) / 2048);
  }
  const int64_t part = std::max<int64_t>(m.tile ? 64 : 256, ((span + parts - 1) / parts + unit - 1) / unit * unit);
  a.part_s = (int)part;
  a.parts_s = (int)std::max<int64_t>(1, (span + part - 1) / part);
  const int64_t all = attn_count(a.parts_s * sets, a.tiles_s);
  a.items = all < (1LL << 24) - 64 ? (int)all : -1;
  if (a.parts_s == 1 && a.B > 0) return 0;  // nothing to join
  if ((int64_t)a.T * a.Hq * join_waves(m) >= 1LL << 26) a.items = -1;
  return (size_t)a.parts_s * a.T * a.Hq * ((size_t)a.D * 4 + sizeof(float2));
}

hipError_t launch_mx_attn_bf16(const MxAttnArgs& m, hipStream_t st);
hipError_t launch_mx_attn_fp16(const MxAttnArgs& m, hipStream_t st);

// A planned call; `bytes`: what mx_attn_plan returned for it.
hipError_t launch_mx_attn(MxAttnArgs& m, bool bf16, void* ws, size_t bytes, hipStream_t st) {
  AttnArgs& a = m.a;
  m.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz((unsigned)a.page) : -1;
  a.acc = nullptr;
  a.ml = nullptr;
  if (bytes) {
    a.acc = static_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(a.acc + (size_t)a.parts_s * a.T * a.Hq * a.D);
  }
  if (a.items) {
    const hipError_t e = bf16 ? launch_mx_attn_bf16(m, st) : launch_mx_attn_fp16(m, st);
    if (e != hipSuccess) return e;
  }
  note_kernel("%s<%d> parts=%d%s", m.tile ? "mx_tile_kernel" : "mx_rows_kernel", m.bits, a.parts_s, bytes ? " + mx_join_kernel" : "");
  if (!bytes) return hipSuccess;
  const int many = join_waves(m);
  auto join = [&](auto b_tag, auto l_tag) {
    constexpr bool B = decltype(b_tag)::value;
    constexpr int L = decltype(l_tag)::value;
    const dim3 grid((unsigned)(((int64_t)a.T * a.Hq * many + 3) / 4));
    if (many == 1) hipLaunchKernelGGL((mx_join_kernel<B, L, 1>), grid, dim3(256), 0, st, m);
    else hipLaunchKernelGGL((mx_join_kernel<B, L, 4>), grid, dim3(256), 0, st, m);
    return hipGetLastError();
  };
  auto by_d = [&](auto b_tag) {
    if (a.D <= 64) return join(b_tag, std::integral_constant<int, 16>{});
    if (a.D <= 128) return join(b_tag, std::integral_constant<int, 32>{});
    return join(b_tag, std::integral_constant<int, 64>{});
  };
  return bf16 ? by_d(std::true_type{}) : by_d(std::false_type{});
}

}  // namespace fg
