// Attention over a paged cache for a batch whose sequences share a prefix: o = softmax(scale q K^T) V over the shared prefix's
// keys and the sequence's own.  The prefix is a product of all the batch's rows with one set of keys, read once; a
// sequence's own keys meet the rows of its query heads only.
//
// Keys are cut into parts; an item (row tile, key head, part) makes one pass over its keys with a running maximum and sum and
// leaves sum(p v), the maximum and the sum in 32 bits (attn_rows, attn_tile); attn_join_kernel weighs the parts of each row by
// exp2(m - max m).  Here: the join, and the plan that cuts the work.
#include <algorithm>

#include "fg_attn_join.h"

namespace fg {

template <bool BF16, int L, int W>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  const JoinRow<L, W> r;
  if (r.id >= (int64_t)a.T * a.Hq) return;
  const int t = (int)(r.id / a.Hq), h = (int)(r.id - (int64_t)t * a.Hq);
  int seq = t;
  bool inside = true, served = true;
  if (a.starts) {
    seq = attn_sequence(a, t);
    inside = a.B > 0 && a.starts[seq] <= t && t < a.starts[seq + 1];
    served = !inside || t - attn_start(a, seq) < a.max_q;
  }
  const int len = inside ? (a.joined ? a.prefix_len : 0) + max(min(a.lens[seq], a.max_len), 0) : 0;
  const int own = max((len + a.part_s - 1) / a.part_s, 1), n = inside ? a.parts_p + own : 0;
  attn_join<BF16, L, W>(a, r, t, h, n, served);
}

// Parts of whole tiles of `unit` keys for `items` row tiles and key heads, a workgroup each.  Host lengths only: a sequence
// shorter than max_len leaves parts that end at once.
static int cut(int64_t len, int64_t parts, int64_t unit, int* part) {
  const int64_t p = std::max<int64_t>(unit, ((len + parts - 1) / parts + unit - 1) / unit * unit);
  *part = (int)p;
  return (int)std::max<int64_t>(1, (len + p - 1) / p);
}

// attn_rows: about `want` workgroups per CU (one; four among a prefix's items of many rows, where the sequences' lengths
// should even out), parts as long as the row table at most.  Where nothing is joined to them (`alone`), up to kOnePart keys are
// one part, which needs no second launch (250 keys: 8.7 us against 9.4 in two parts; 500: 12.1 against 9.5).
constexpr int kOnePart = 256;
static int cut_rows(int64_t len, int64_t items, bool alone, int64_t want, int* part) {
  if (alone && len <= kOnePart) return cut(len, 1, kOnePart, part);
  const int64_t parts = std::max<int64_t>(want * device_cus() / std::max<int64_t>(items, 1), (len + kMaxPart - 1) / kMaxPart);
  return cut(len, std::max<int64_t>(parts, 1), kRowsTile * kRowsWaves, part);
}

// attn_tile: the number of parts with the least time in us, where a tile of 64 keys takes 1.6 alone on a CU and 1.2 by each
// workgroup there beside others, and a part's sums (`sums` values in all) are written and read back at 4 TB/s, with 4 for the
// second launch where one part would need none.  (Graph replays, us, by parts of the prefix: 64 sequences behind 8192 tokens 8 /
// 16 / 32: 68 / 60 / 64; 16 sequences 16 / 64: 20.8 / 23.6; 256 behind 32768 2 / 4 / 8: 400 / 350 / 370.)
static int cut_tile(int64_t len, int64_t items, int64_t sums, bool alone, int* part) {
  const int64_t tiles = std::max<int64_t>((len + 63) / 64, 1), cus = device_cus();
  const int64_t most = std::min(tiles, std::max<int64_t>(1, 4 * cus / std::max<int64_t>(items, 1)));
  double best = 0;
  int64_t parts = 1;
  for (int64_t p = 1; p <= most; p += std::max<int64_t>(1, p / 8)) {
    const int64_t per_cu = (items * p + cus - 1) / cus, each = (tiles + p - 1) / p;
    const double t = each * (per_cu <= 1 ? 1.6 : 1.2 * per_cu) + (p == 1 && alone ? 0 : 4 + p * (double)sums * 8 / 4e6);
    if (p == 1 || t < best) {
      best = t;
      parts = p;
    }
  }
  return cut(len, parts, 64, part);
}

// Wavefronts that join a row.
static int join_waves(const AttnArgs& a) { return a.parts_p + a.parts_s >= 8 ? 4 : 1; }

// Fills in the plan; returns the partial sums' bytes.  items is -1 where the threads of a launch would pass 32 bits.  Rows past
// 16 go to attn_tile, which is ahead even where most of its 128 rows are empty (16 sequences of 2000 tokens with 8 queries of 4
// heads: 23.2 us against 35.6 in two row tiles), but for 17 to 32 rows of a prefix in e4m3, which attn_rows converts as it
// computes and attn_tile in front of that (8 sequences of one query behind 8192 tokens: 15.4 us against 19.1; 16-bit 18.1
// against 16.2).
size_t attn_plan(AttnArgs& a) {
  const int64_t rows_p = (int64_t)a.T * a.G, rows_s = (int64_t)a.max_q * a.G;
  a.tile_s = rows_s > 16;
  a.tile_p = a.tile_s || rows_p > (a.item == 1 ? 32 : 16);
  // Sequences that fill two row tiles each on average take the prefix along with their own keys: the rows that packing the
  // whole batch's into tiles would save cost less than the parts' sums (4 prompts of up to 500 tokens,
  // 32 + 2 x 8 heads, behind 4000: 139 us, 159 apart).
  a.joined = a.tile_s && a.prefix_len && rows_p >= 2 * kTileRows * (int64_t)a.B;
  if (!a.tile_s && a.prefix_len) {
    // So do single queries where all keys make one part, or where the sequences fill the CUs by themselves and reading the
    // prefix again for each (at 8 TB/s, from L2) takes less than a second launch and two parts' sums.  (us, graph replays,
    // 32 + 2 x 8 heads of 128, apart / along: 4 sequences, 100 + 130 tokens 9.3 / 8.4, 64 sequences 19.8 / 12.9, 64 x (250 +
    // 130) 20.0 / 16.5, 64 x (500 + 130) 22.2 / 23.2, 4 x (500 + 130), which does not fill the CUs, 9.5 / 13.7.)
    const double again = (double)a.B * a.prefix_len * a.Hk * a.D * 2 * a.item / 8e6, sums = 4 + 2.0 * a.T * a.Hq * a.D * 8 / 4e6;
    a.joined = a.prefix_len + a.max_len <= kOnePart || ((int64_t)a.B * a.Hk >= device_cus() && again < sums);
  }
  // The prefix's items go first where their products (1.2 us per tile of 64 keys) outlast the reads of the sequences' keys at
  // 4 TB/s (256 sequences behind 32768 tokens: 350 us, 450 spread); else they spread among the sequences' items (64 behind 8192:
  // 61 us, 68 first).
  const int64_t per_p = a.tile_p ? kTileRows : 16, per_s = a.tile_s ? kTileRows : 16, sums = (int64_t)a.T * a.Hq * a.D;
  a.tiles_p = (int)((rows_p + per_p - 1) / per_p);
  a.tiles_s = (int)((rows_s + per_s - 1) / per_s);
  const double products = (double)a.tiles_p * a.Hk * ((a.prefix_len + 63) / 64) * 1.2 / device_cus();
  a.lead = products > (double)a.B * a.max_len * a.Hk * a.D * 2 * a.item / 4e6;
  const bool apart = a.prefix_len && !a.joined;
  const int64_t sets = (int64_t)a.Hk * a.B, own = (a.joined ? (int64_t)a.prefix_len : 0) + a.max_len;
  a.parts_p = a.part_p = 0;
  if (apart) {
    const int64_t n = (int64_t)a.tiles_p * a.Hk;
    a.parts_p = a.tile_p ? cut_tile(a.prefix_len, n, sums, false, &a.part_p) : cut_rows(a.prefix_len, n, false, 1, &a.part_p);
  }
  a.parts_s = a.tile_s ? cut_tile(own, a.tiles_s * sets, sums, !apart, &a.part_s)
                       : cut_rows(own, a.tiles_s * sets, !apart, apart && a.tile_p ? 4 : 1, &a.part_s);
  const int64_t items_p = apart ? attn_count((int64_t)a.parts_p * a.Hk, a.tiles_p) : 0;
  const int64_t items = items_p + attn_count(a.parts_s * sets, a.tiles_s);
  a.items_p = (int)items_p;
  a.items = items < (1LL << 24) - 64 ? (int)items : -1;
  if (a.parts_p + a.parts_s == 1 && a.B > 0) return 0;  // nothing to join
  if ((int64_t)a.T * a.Hq * join_waves(a) >= 1LL << 26) a.items = -1;
  return (size_t)(a.parts_p + a.parts_s) * a.T * a.Hq * ((size_t)a.D * 4 + sizeof(float2));
}

hipError_t launch_attn_bf16(const AttnArgs& a, bool fp8, int kind, hipStream_t st);
hipError_t launch_attn_fp16(const AttnArgs& a, bool fp8, int kind, hipStream_t st);

// A planned call; `bytes`: what attn_plan returned for it.
hipError_t launch_attn(AttnArgs& a, bool bf16, bool fp8, void* ws, size_t bytes, hipStream_t st) {
  a.acc = nullptr;
  a.ml = nullptr;
  if (bytes) {
    a.acc = static_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(a.acc + (size_t)(a.parts_p + a.parts_s) * a.T * a.Hq * a.D);
  }
  const int kind = a.tile_s || a.items == a.items_p ? (a.tile_p ? kAttnTile : kAttnRows)
                                                    : (a.tile_p && a.items_p ? kAttnMixed : kAttnRows);
  static const char* const names[] = {"attn_rows_kernel", "attn_tile_kernel", "attn_mixed_kernel"};
  if (a.items) {
    const hipError_t e = bf16 ? launch_attn_bf16(a, fp8, kind, st) : launch_attn_fp16(a, fp8, kind, st);
    if (e != hipSuccess) return e;
  }
  note_kernel("%s parts=%d+%d%s", names[kind], a.parts_p, a.parts_s, bytes ? " + attn_join_kernel" : "");
  if (!bytes) return hipSuccess;
  const int many = join_waves(a);
  auto join = [&](auto b_tag, auto l_tag) {
    constexpr bool B = decltype(b_tag)::value;
    constexpr int L = decltype(l_tag)::value;
    const dim3 grid((unsigned)(((int64_t)a.T * a.Hq * many + 3) / 4));
    if (many == 1) hipLaunchKernelGGL((attn_join_kernel<B, L, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_join_kernel<B, L, 4>), grid, dim3(256), 0, st, a);
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
