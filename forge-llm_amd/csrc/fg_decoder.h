// Arguments and launchers of the operators between a decoder layer's linears.
#pragma once

#include "fg_device.h"

namespace fg {

constexpr int kNormMaxK = 32768;  // four units for each of 1024 threads

// A launch has fewer than 2^32 threads.
inline bool launchable(int64_t blocks, int threads) { return blocks * threads < (1LL << 32); }

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* r;
  int64_t ldr;
  void* ro;
  int64_t ldro;
  const void* w;
  int wdt;
  float eps;
  void* y;
  int64_t ldy;
  int ydt;  // FG_I8, FG_E4M3, or x's type
  float* s;
  int64_t s_row, s_block;
  int log_l;  // lanes per block of scales (a block is 8 << log_l columns), -1: one scale per row
  int K;
};

struct RopeAppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;  // element strides of tokens and heads
  uint16_t* qo;
  int64_t qo_t, qo_h;
  const void* pos;
  int pos64;
  const float* table;  // [max_pos][rot]: cosines of the pairs, then sines
  int64_t ld_table, max_pos;
  const void* slots;
  int slots64;
  uint8_t *kc, *vc;
  int64_t c_page, c_head, c_token;  // byte strides
  int64_t n_slots;
  int page;
  const float *ks, *vs;  // e4m3 caches: a scale per key head
  int Hq, Hk, D, rot;
};

bool norm_fits(int64_t M, int64_t K);  // whether one launch takes M rows of K columns
hipError_t launch_add_rmsnorm(const NormArgs& a, int xdt, int rdt, int64_t M, hipStream_t st);
hipError_t launch_rope_append(const RopeAppendArgs& a, int64_t T, bool bf16, bool fp8, bool inter, hipStream_t st);

}  // namespace fg
