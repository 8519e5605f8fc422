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
  int prefix_len, max_len, max_q;
  float scale_log2;  // softmax scale * log2(e)
  // keys are split into parts of whole tiles, one workgroup each; parts_p of the prefix, parts_s of each sequence's own tokens
  int parts_p, parts_s, part_p, part_s;  // counts and tokens per part
  int tile_p, tile_s, tiles_p, tiles_s;  // rows per tile, row tiles
  int items_p, items;                    // work items of the prefix, and in all
  float* acc;  // partial sums [parts_p + parts_s][T * Hq][D], null: one part, written to out
  float2* ml;  // their maxima (in log2) and sums [parts_p + parts_s][T * Hq]
};

size_t attn_plan(AttnArgs& a);
hipError_t launch_attn(AttnArgs& a, bool bf16, bool fp8, void* ws, hipStream_t st);
hipError_t launch_attn_tile(const AttnArgs& a, bool bf16, bool fp8, int first, int count, hipStream_t st);

constexpr uint32_t kNoRow = 0xffffffffu;  // an entry of the row table that stands for no key
constexpr int kMaxPart = 2048;            // tokens per part: entries of the row table

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
  int len;          // keys of the segment
  int seen0;        // keys that the segment's first query token sees; each further one sees one more (prefix: all see all)
  bool causal;
  const int32_t* table;
  int slot;  // part index
};

// Item `id` of the grid; false: nothing to do.  TILE rows per item.
template <int TILE>
__device__ __forceinline__ bool attn_item(const AttnArgs& a, int id, AttnItem& it) {
  if (id < a.items_p) {
    // neighbours share keys: row tiles innermost
    const int tile = id % a.tiles_p, rest = id / a.tiles_p, part = rest % a.parts_p;
    it.head = rest / a.parts_p;
    it.row0 = tile * TILE;
    it.rows = a.T * a.G;
    it.token0 = 0;
    it.begin = part * a.part_p;
    it.end = min(it.begin + a.part_p, a.prefix_len);
    it.len = it.seen0 = a.prefix_len;
    it.causal = false;
    it.table = a.prefix_pages;
    it.slot = part;
    return it.row0 < it.rows;
  }
  id -= a.items_p;
  const int tile = id % a.tiles_s, rest = id / a.tiles_s, head = rest % a.Hk, rest2 = rest / a.Hk;
  const int part = rest2 % a.parts_s, seq = rest2 / a.parts_s;
  int t0 = seq, n = 1;  // the sequence's query tokens
  if (a.starts) {
    t0 = max(a.starts[seq], 0);
    n = min(a.starts[seq + 1], a.T) - t0;
  }
  const int len = min(a.lens[seq], a.max_len);
  it.head = head;
  it.row0 = tile * TILE;
  it.rows = min(n, a.max_q) * a.G;
  it.token0 = t0;
  it.begin = part * a.part_s;
  it.len = len;
  it.causal = n > 1;
  it.seen0 = len - n + 1;
  // the tile's last token sees the most
  const int last = min(it.rows - 1, it.row0 + TILE - 1);
  it.end = min(min(it.begin + a.part_s, len), it.seen0 + last / a.G);
  it.table = a.pages + seq * a.ld_pages;
  it.slot = a.parts_p + part;
  // a part past the sequence is not asked for by the join; the first one always is
  return it.row0 < it.rows && (part == 0 || it.begin < len);
}

// Key t's row in 16-byte units from the first page; kNoRow for a page outside the cache.
__device__ __forceinline__ uint32_t attn_row(const AttnArgs& a, const AttnItem& it, int t) {
  const int page = t / a.page, off = t - page * a.page, id = it.table[page];
  return id >= 0 && id < a.n_pages ? (uint32_t)id * a.c_page + (uint32_t)off * a.c_token : kNoRow;
}

// Table of the item's keys in LDS: each key's row in 16-byte units from the first page, up to a whole number of tiles of
// `tile` keys; kNoRow past the end and for pages outside the cache.
__device__ __forceinline__ void attn_row_table(const AttnArgs& a, const AttnItem& it, uint32_t* tab, int tile) {
  const int n = max(it.end - it.begin, 0), padded = (n + tile - 1) / tile * tile;
  for (int i = threadIdx.x; i < padded; i += blockDim.x) tab[i] = i < n ? attn_row(a, it, it.begin + i) : kNoRow;
}

__device__ __forceinline__ uint4 attn_ld16(const uint8_t* base, uint32_t row, int unit) {
  return *reinterpret_cast<const uint4*>(base + ((uint64_t)row + (uint32_t)unit) * 16);
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

// Two fp32 values rounded to nearest even as one packed pair.
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

// A row whose running maximum is still -inf has seen no key: its exponents count from 0, so that they are exp2(-inf) = 0.
__device__ __forceinline__ float attn_base(float m) { return m == -__builtin_inff() ? 0.f : m; }

// The maximum that exponents count from moves only when a score is more than 2^kSlack times above it: most tiles then need
// neither an exchange between lanes nor a rescaling of the sums.  Probabilities up to 2^8 are as exact in 16 bits as those up
// to 1, and fp16 holds them.
constexpr float kSlack = 8.f;

}  // namespace fg
