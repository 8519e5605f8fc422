// What the attention kernels over a block-scaled cache share: arguments, a work item's rows and keys, scores under a cap.
#pragma once

#include "fg_attn.h"
#include "fg_mx.h"

namespace fg {

// The keys and values of AttnArgs are codes here (k, v; c_head in bytes, c_page and c_token in 16-byte units), there is no prefix,
// and an item's keys begin where its first row's window does.
struct MxAttnArgs {
  AttnArgs a;
  const uint8_t *ks, *vs;  // scale bytes
  int64_t s_head;          // byte stride of key heads among them
  int bits;
  int window;              // keys that a query token sees, its own included; kNoWindow: all
  float cap_in;            // CAP: a score s becomes tanh(s cap_in), in units of the cap
  float factor;            // what makes that, or a score, an exponent of 2
  bool tile;               // whether mx_tile takes the rows, or mx_rows
  int page_shift;          // log2 of the page size, -1: no power of two
};

constexpr int kNoWindow = 1 << 30;

size_t mx_attn_plan(MxAttnArgs& m);
hipError_t launch_mx_attn(MxAttnArgs& m, bool bf16, void* ws, size_t bytes, hipStream_t st);

// The keys [low, end) that some of a tile's rows see: the tokens a0 .. a1 of the sequence's, of which token i sees seen0 + i keys from
// the front, but the last `window` of them.  begin: low down to a whole tile, so that tiles do not cross the pages' sixteens.
struct MxRange {
  int begin, low, end;
};
__device__ __forceinline__ MxRange mx_range(const MxAttnArgs& m, int len, int seen0, int a0, int a1) {
  const int low = max(seen0 + a0 - m.window, 0);
  return {low & ~31, low, max(min(seen0 + a1, len), 0)};
}

struct MxItem : AttnItem {
  int low;  // keys in front of it are nobody's
};

// Item `id` of the grid; false: nothing to do.  TILE rows per item.
template <int TILE>
__device__ __forceinline__ bool mx_item(const MxAttnArgs& m, int id, MxItem& it) {
  const AttnArgs& a = m.a;
  const int tiles = a.tiles_s, pairs = a.parts_s * a.Hk * a.B;
  int pair, tile;
  if (attn_by_xcd(pairs)) {
    pair = (id / 8) / tiles * 8 + id % 8;
    tile = (id / 8) % tiles;
    if (pair >= pairs) return false;
  } else {
    pair = id / tiles;
    tile = id % tiles;
  }
  // Workgroups go to the shader engines in turn and wait for theirs: sequences begin with another part each, so that the parts that
  // short ones lack do not always fall to the same engine (64 sequences of 2048 to 16384 tokens in 8 parts: 2 to 15 items per CU).
  const int rest = pair / a.Hk, seq = rest / a.parts_s, part = (rest - seq * a.parts_s + seq) % a.parts_s;
  tile = tiles - 1 - tile;  // the tiles that see the most first
  int t0 = seq, n = 1;      // the sequence's query tokens
  if (a.starts) {
    t0 = attn_start(a, seq);
    n = attn_start(a, seq + 1) - t0;
  }
  it.head = pair - rest * a.Hk;
  if (a.starts && !a.acc && tile == 0 && part == 0) attn_uncovered(a, seq, it.head);
  const int len = max(min(a.lens[seq], a.max_len), 0);
  it.front = 0;
  it.row0 = tile * TILE;
  it.rows = min(n, a.max_q) * a.G;
  if (it.row0 >= it.rows) return false;
  it.token0 = t0;
  it.seen0 = len - n + 1;
  const MxRange all = mx_range(m, len, it.seen0, it.row0 / a.G, min(it.rows - 1, it.row0 + TILE - 1) / a.G);
  it.begin = all.begin + part * a.part_s;
  it.end = min(it.begin + a.part_s, all.end);
  it.low = all.low;
  it.causal = true;
  it.table = a.pages + seq * a.ld_pages;
  it.slot = part;
  // a part past the keys is not asked for by the join; the first one always is
  return part == 0 || it.begin < all.end;
}

// tanh(z): by the exponential, and below 1/8, where 1 - 2 / (e^2z + 1) would lose what it subtracts, by the series' first four
// terms (the next is below 2^-22 of the sum).
__device__ __forceinline__ float mx_tanh(float z) {
  const float e = __builtin_amdgcn_exp2f(z * 2.8853900817779268f);  // 2 log2 e
  const float far = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f), q = z * z;
  const float near = __builtin_fmaf(z * q, __builtin_fmaf(q, __builtin_fmaf(q, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), z);
  return fabsf(z) < 0.125f ? near : far;
}

}  // namespace fg
