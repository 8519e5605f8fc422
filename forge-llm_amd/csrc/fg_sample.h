// Arguments of the sampling of tokens.
#pragma once

#include "fg_device.h"

namespace fg {

struct SampleArgs {
  const void* x;  // logits [B][V]
  int64_t ld;
  int B, V;
  const float* u;
  // one value for each row, or (null) one for all
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* token;
  float* logprob;  // or null
  int bits;           // a weight of one is 2^bits
  int chunks, chunk;  // workgroups per row, and their columns
  int sum_chunks, sum_chunk;  // of the sums
  bool cuts;          // some row may have top-k or top-p
  uint8_t* ws;
};

size_t sample_plan(SampleArgs& a);
hipError_t launch_sample(const SampleArgs& a, int dt, hipStream_t st);

}  // namespace fg
