// What the two kernels of the attention over the 8-bit cache share.
#pragma once

#include "common.cuh"
#include "documents.cuh"

namespace nob200 {

struct CacheParams {
  const __nv_bfloat16* query;
  const float* key_scales;
  const float* value_scales;
  const int* table;
  const int* lengths;
  const int* bounds;
  const int* prefix;    // or NULL
  const float* slopes;  // BIAS form
  __nv_bfloat16* output;
  float* partial;  // of KeyShares, when the keys are divided
  float* lse;
  uint32_t* status;
  int rows, sequences, max_blocks, num_blocks, heads, kv_heads, group, total_heads, head_offset;
  int slots, splits, causal, joined;  // joined: the shares of a unit are a cluster, which joins them itself
  float scale;    // of a raw score; CAP form: divided by the cap
  float to_log2;  // from a (capped) scaled score to log2 units
};

// Units of 128 rows on the tensor cores' own instructions; slots counts such units.  Defined beside that kernel.
int launch_cache_tiles(const CacheParams& params, const void* key, const void* value, bool capped, void* stream);

}  // namespace nob200
