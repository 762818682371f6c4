// What the two kernels of the attention over the 8-bit cache share.
#pragma once

#include "common.cuh"
#include "documents.cuh"

namespace nob200 {

// Probabilities are rounded to f16, whose range they use from above: relative to 2^-kLift of a row's running maximum, which they
// outgrow by 2^8 at most before it is raised, they stay below 2^15, and a weight counts down to 2^-32 of the largest (2^-25
// without the lift: 131071 keys of 2^-26 each, 0.2 % together, were lost).
constexpr float kLift = 7.0f;  // log2 units

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
  float near;     // tiles, CAP form: the largest share of the cap for cap_scores' first way
};

// Units of 128 rows on the tensor cores' own instructions; slots counts such units.  Defined beside that kernel.
int launch_cache_tiles(const CacheParams& params, const void* key, const void* value, bool capped, void* stream);

}  // namespace nob200
