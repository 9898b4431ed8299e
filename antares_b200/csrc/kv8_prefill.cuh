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
  int *status;
  // set by kv8_prefill_plan: tiles of rows, those of a sequence (cu == nullptr), shares of the keys
  int slots, slots_per_seq, splits;
  // splits > 1: [slot][kv head][split][row of the slot][128], and the rows' maximum and sum
  float *partial;
  float2 *partial_ml;
};
int kv8_prefill_plan(Kv8PrefillParams *p, int dtype, long capacity, size_t *bytes);
int kv8_prefill(Kv8PrefillParams p, int dtype, void *workspace, cudaStream_t stream);
int kv8_prefill_join(Kv8PrefillParams p, int dtype, void *workspace, cudaStream_t stream);  // after every launch that may run beside the one above

}  // namespace ab200
