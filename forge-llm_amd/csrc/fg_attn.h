// What the attention kernels over a paged cache share: arguments, a work item's rows and keys, the pieces of one softmax pass.
#pragma once

#include "fg_device.h"

namespace fg {

// A call's rows are (query token, query head); the g = Hq / Hk query heads of one key head lie next to each other, so the
// tokens of a sequence (of the whole batch, for the shared prefix) make count * g rows for each key head.
struct AttnArgs {
  const uint16_t* q;
  int64_t q_t, q_h;  // element strides
  uint16_t* out;
  int64_t o_t, o_h;
  float* lse;  // [T][Hq] or null
  const uint8_t *k, *v;
  int64_t c_head;             // byte stride of key heads
  uint32_t c_page, c_token;   // strides of pages and tokens in 16-byte units
  const float *ks, *vs;       // e4m3 caches: a scale per key head
  const int32_t* prefix_pages;
  const int32_t* pages;  // [B][ld_pages]
  int64_t ld_pages;
  const int32_t *lens, *starts;  // starts: [B + 1] or null (one query token per sequence)
  int T, B, Hq, Hk, G, D, page, n_pages;
  int item;  // bytes of a cached value
  int prefix_len, max_len, max_q;
  float scale_log2;  // softmax scale * log2(e)
  // keys are split into parts of whole tiles, one workgroup each; parts_p of the prefix, parts_s of each sequence's own tokens
  int parts_p, parts_s, part_p, part_s;  // counts and tokens per part
  bool tile_p, tile_s;                   // whether attn_tile takes the segment, or attn_rows
  bool joined;                           // a sequence's items take the prefix's keys too
  bool lead;                             // the prefix's items go first, not spread among the sequences'
  int tiles_p, tiles_s;                  // row tiles
  int items_p, items;                    // workgroups for the prefix, and in all
  float* acc;  // partial sums [parts_p + parts_s][T * Hq][D], null: one part, written to out
  float2* ml;  // their maxima (in log2) and sums [parts_p + parts_s][T * Hq]
};

size_t attn_plan(AttnArgs& a);
hipError_t launch_attn(AttnArgs& a, bool bf16, bool fp8, void* ws, size_t bytes, hipStream_t st);

constexpr uint32_t kNoRow = 0xffffffffu;  // an entry of the row table that stands for no key
constexpr int kMaxPart = 2048;            // attn_rows: tokens per part, entries of its row table
constexpr int kRowsWaves = 4, kRowsTile = 32;  // wavefronts, keys per wavefront and step
constexpr int kTileRows = 128;            // attn_tile: rows per item
enum { kAttnRows = 0, kAttnTile = 1, kAttnMixed = 2 };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// What one work item computes.
struct AttnItem {
  int head;         // key head
  int row0, rows;   // first row of the tile among the segment's rows, and the segment's rows
  int token0;       // first query token of the segment
  int begin, end;   // its keys
  int front;        // keys in front that are the prefix's (an item of a sequence that takes both)
  int seen0;        // keys that the segment's first query token sees, each further one sees one more, and none fewer than
                    // the front (not causal: all see all)
  bool causal;
  const int32_t* table;
  int slot;  // part index
};

// Work item `id` of `pairs` sets of keys (key head, part, sequence) times `tiles` row tiles: consecutive workgroups go to the
// eight XCDs in turn, so every eighth one takes the next row tile of the same keys and finds them in its L2.  Needs sets
// enough for all XCDs: else row tiles go round in turn.
__host__ __device__ __forceinline__ bool attn_by_xcd(int pairs) { return pairs % 8 == 0 || pairs >= 64; }
__host__ __device__ __forceinline__ int64_t attn_count(int64_t pairs, int64_t tiles) {
  return (pairs < (1 << 30) && attn_by_xcd((int)pairs) ? (pairs + 7) / 8 * 8 : pairs) * tiles;
}

// Where sequence i's query tokens start: offsets outside the queries count as their begin or end.
__device__ __forceinline__ int attn_start(const AttnArgs& a, int i) { return min(max(a.starts[i], 0), a.T); }

// Rows of query tokens that no item computes, written where no join follows: tokens of no sequence give zeros (the first
// sequence's workgroup takes those in front of it, the last one's those behind it), tokens past max_query_len NaN.
__device__ __forceinline__ void attn_uncovered(const AttnArgs& a, int seq, int head) {
  auto fill = [&](int from, int to, float out, float lse) {
    for (int64_t i = (int64_t)from * a.G * a.D + threadIdx.x; i < (int64_t)to * a.G * a.D; i += blockDim.x) {
      const int col = (int)(i % a.D), h = head * a.G + (int)(i / a.D % a.G);
      const int64_t t = i / a.D / a.G;
      a.out[t * a.o_t + h * a.o_h + col] = out == 0.f ? 0 : 0x7fff;  // a NaN of either type
      if (a.lse && col == 0) a.lse[t * a.Hq + h] = lse;
    }
  };
  const float nan = __builtin_nanf(""), inf = __builtin_inff();
  const int first = attn_start(a, seq), next = attn_start(a, seq + 1);
  if (next - first > a.max_q) fill(first + a.max_q, next, nan, nan);
  if (seq == 0) fill(0, first, 0.f, -inf);
  if (seq == a.B - 1) fill(next, a.T, 0.f, -inf);
}

// Item `id` of the grid; false: nothing to do.  TILE rows per item.
template <int TILE>
__device__ __forceinline__ bool attn_item(const AttnArgs& a, int id, AttnItem& it) {
  const bool prefix = id < a.items_p;
  if (!prefix) id -= a.items_p;
  const int tiles = prefix ? a.tiles_p : a.tiles_s, pairs = prefix ? a.parts_p * a.Hk : a.parts_s * a.Hk * a.B;
  int pair, tile;
  if (attn_by_xcd(pairs)) {
    pair = (id / 8) / tiles * 8 + id % 8;
    tile = (id / 8) % tiles;
    if (pair >= pairs) return false;
  } else {
    pair = id / tiles;
    tile = id % tiles;
  }
  it.front = 0;
  if (prefix) {
    const int part = pair / a.Hk;  // neighbours read the heads of one page, which lie next to each other
    it.head = pair - part * a.Hk;
    it.row0 = tile * TILE;
    it.rows = a.T * a.G;
    it.token0 = 0;
    it.begin = part * a.part_p;
    it.end = min(it.begin + a.part_p, a.prefix_len);
    it.seen0 = a.prefix_len;
    it.causal = false;
    it.table = a.prefix_pages;
    it.slot = part;
    return it.row0 < it.rows;
  }
  const int rest = pair / a.Hk, seq = rest / a.parts_s, part = rest - seq * a.parts_s;
  tile = a.tiles_s - 1 - tile;  // the tiles that see the most first
  int t0 = seq, n = 1;  // the sequence's query tokens
  if (a.starts) {
    t0 = attn_start(a, seq);
    n = attn_start(a, seq + 1) - t0;
  }
  it.head = pair - rest * a.Hk;
  if (a.starts && !a.acc && tile == 0 && part == 0) attn_uncovered(a, seq, it.head);
  if (a.joined) it.front = a.prefix_len;
  const int len = it.front + max(min(a.lens[seq], a.max_len), 0);
  it.row0 = tile * TILE;
  it.rows = min(n, a.max_q) * a.G;
  it.token0 = t0;
  it.begin = part * a.part_s;
  it.causal = n > 1;
  it.seen0 = len - n + 1;
  // the tile's last token sees the most; what precedes the sequence's first token sees the prefix
  const int last = min(it.rows - 1, it.row0 + TILE - 1);
  it.end = min(min(it.begin + a.part_s, len), max(it.seen0 + last / a.G, it.front));
  it.table = a.pages + seq * a.ld_pages;
  it.slot = a.parts_p + part;
  // a part past the sequence is not asked for by the join; the first one always is
  return it.row0 < it.rows && (part == 0 || it.begin < len);
}

// Key t's row in 16-byte units from the first page; kNoRow for a page outside the cache.
__device__ __forceinline__ uint32_t attn_row(const AttnArgs& a, const AttnItem& it, int t) {
  const int32_t* table = t < it.front ? a.prefix_pages : it.table;
  if (t >= it.front) t -= it.front;
  const int page = t / a.page, off = t - page * a.page, id = table[page];
  return id >= 0 && id < a.n_pages ? (uint32_t)id * a.c_page + (uint32_t)off * a.c_token : kNoRow;
}

// Table of the item's keys in LDS: each key's row in 16-byte units from the first page, up to a whole number of tiles of
// `tile` keys; kNoRow past the end and for pages outside the cache.
__device__ __forceinline__ void attn_row_table(const AttnArgs& a, const AttnItem& it, uint32_t* tab, int tile) {
  const int n = max(it.end - it.begin, 0), padded = (n + tile - 1) / tile * tile;
  for (int i = threadIdx.x; i < padded; i += blockDim.x) tab[i] = i < n ? attn_row(a, it, it.begin + i) : kNoRow;
}

// The transposing LDS reads: 16 lanes read 4 keys x 16 columns of 16 bits (8 keys of 8 bits), lanes 4 j .. 4 j + 3 (2 j, 2 j + 1)
// 8 bytes each of key j, and get one column each.
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ s16x4 lds_tr16(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      reinterpret_cast<__attribute__((address_space(3))) s16x4*>((__attribute__((address_space(3))) uint8_t*)(p)));
}
__device__ __forceinline__ i32x2 lds_tr8(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      reinterpret_cast<__attribute__((address_space(3))) i32x2*>((__attribute__((address_space(3))) uint8_t*)(p)));
}

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(const s16x8& x, const s16x8& y, const f32x4& c) {
  if constexpr (BF16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, x), __builtin_bit_cast(v8, y), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, x), __builtin_bit_cast(v8, y), c, 0, 0, 0);
  }
}

// Eight e4m3 codes as 16-bit floats: exact in both types.
template <bool BF16>
__device__ __forceinline__ s16x8 e4m3_to_16(uint32_t lo, uint32_t hi) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int src = (int)(i < 2 ? lo : hi);
    if constexpr (BF16) {
      w[i] = __builtin_bit_cast(uint32_t, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.f, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.f, false));
    } else {
      w[i] = __builtin_bit_cast(uint32_t, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(src, 1.f, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(src, 1.f, false));
    }
  }
  return __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

// Two fp32 values rounded to nearest even as one packed pair.  The weights of the second product go through it, since the
// matrix cores take 16-bit operands: each is off by half a unit in its last place, their sum is of the fp32 values.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, b2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, h2));
  }
}

// What makes a score an exponent of 2: the softmax's scale and, in e4m3, the key head's.  Masked scores are -inf, which a factor
// of zero would make NaN and one below zero +inf: the rows change their sign instead, and the smallest normal number, which
// leaves all weights equal, stands for anything under it.
struct AttnFactor {
  float value;
  uint32_t sign;  // of two 16-bit values of a row
};
__device__ __forceinline__ AttnFactor attn_factor(float scale_log2, float key_scale) {
  const float f = scale_log2 * key_scale, size = fabsf(f);
  return {size < 0x1p-126f ? 0x1p-126f : size, f < 0.f ? 0x80008000u : 0u};
}

// A row whose running maximum is still -inf has seen no key: its exponents count from 0, so that they are exp2(-inf) = 0.
__device__ __forceinline__ float attn_base(float m) { return m == -__builtin_inff() ? 0.f : m; }

// The maximum that exponents count from moves only when a score is more than 2^kSlack times above it: most tiles then need
// neither an exchange between lanes nor a rescaling of the sums.  fp16 has weights from 2^-24 to 2^16 only: there exponents
// count from 2^-kLift below the maximum, so that the largest weight is 2^15 and what is lost of a key that a later one
// dominates is 2^-32 of that one's weight (2^-25 without: 131072 keys were lost behind one 2^25 above them, 0.4% of the
// result).  A slack of 2^4 would leave 2^-36 and costs 1% (prompts of up to 500 tokens behind 4000: 140.3 us, 141.7).  bf16
// has fp32's range.  The lift is part of the running maximum that is kept, so sums, joins and logarithms need nothing else.
constexpr float kSlack = 8.f;
template <bool BF16>
__device__ __forceinline__ float attn_top(float score, float factor) {
  constexpr float kLift = 15.f - kSlack;
  return BF16 ? score * factor : __builtin_fmaf(score, factor, -kLift);
}

}  // namespace fg
