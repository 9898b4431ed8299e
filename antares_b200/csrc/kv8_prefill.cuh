// The prompt kernel of the 8-bit cache's attention (kv8_prefill.cu), as its caller (kv8_attention.cu) sees it.
#pragma once
#include "kv8.cuh"

namespace ab200 {

struct Kv8PrefillParams {
  Kv8Cache c;
  Kv8Rows r;
  const void *q;
  long q_stride;
  void *out;
  int Hq, group;
  float scale;        // times log2(e)
  int few;            // sequences of up to this many rows (times group) are another kernel's
  float *partial;     // splits > 1: [slot][kv head][split][tile][128][128], and the rows' maximum and sum
  float2 *partial_ml;
  int *status;
  int slots, slots_per_seq, splits;  // set by kv8_prefill: tiles of rows, those of a sequence (cu == nullptr), shares of the keys
};
int kv8_prefill(Kv8PrefillParams p, int dtype, cudaStream_t stream);

}  // namespace ab200
