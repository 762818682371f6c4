// Ragged batches: which document and which of its rows a CTA works on.
//
// Documents (or the sequences of a cache) are packed row behind row; `bounds` [count + 1] on the device holds where each
// begins and the last one ends.  The host sizes a grid by what all rows and one partly filled unit per document can come to;
// a CTA looks its unit up and leaves when there is none.  Bounds are clamped to the tensors, so whatever they hold nothing
// outside is touched.
#pragma once

#include <climits>

#include "common.cuh"

namespace nob200 {

// Units of `unit` items that `rows` items in up to `documents` documents can come to.
inline long long most_units(long long rows, long long documents, int unit) {
  const long long most = (rows + documents * (unit - 1)) / unit;
  return most < rows ? most : rows;
}

// Scores are multiplied by scale / cap, which fp32 has to hold with all of its bits.
inline bool cap_fits(float scale, float cap) { return cap == 0.f || (scale / cap >= 1e-35f && scale / cap <= 1e35f); }

// For cap_scores: with c between 1e-7 and 1e5 and f up to 1e10 its coefficients stay in fp32; below, those past the first vanish, which
// changes nothing for x up to 1e-3.
constexpr float kLeastNear = 1e-7f, kMostNear = 1e5f, kMostNearFactor = 1e10f;
inline float near_scores(float c, float f) {  // the largest score for the first way
  if (c > kMostNear || f > kMostNearFactor) return -1.f;
  const float top = (c >= kLeastNear ? 0.3f : 1e-3f) / c;
  return top < 1e18f ? top : 1e18f;
}

#ifdef __CUDACC__

__device__ __forceinline__ int clamped(int x, int low, int high) { return min(max(x, low), high); }

// Rows [begin, end) of document `d`, inside [0, rows].  `behind` of them, if given, are rows that it claims past the last one.
__device__ __forceinline__ int2 document_rows(const int* bounds, int d, int rows, int* behind = nullptr) {
  const int begin = clamped(bounds[d], 0, rows), end = clamped(bounds[d + 1], begin, rows);
  if (behind) *behind = max(bounds[d + 1], end) - end;
  return make_int2(begin, end);
}

// Whether document `d` begins and ends inside [0, rows], in this order.  Both bounds are under way at once.
__device__ __forceinline__ bool bounds_fit(const int* bounds, int d, int rows) {
  const int begin = bounds[d], end = bounds[d + 1];
  return (begin >= 0) & (begin <= end) & (end <= rows);
}

// Sets bit 6 of the status word if one of the documents first, first + step, .. is not right.  For a single CTA or warp of a launch,
// beside its own work: noted by every CTA as it looks for its unit, one token of 1021 x 14 heads took 9.1 us instead of 8.95.
template <typename Right>
__device__ __forceinline__ void note_documents(int first, int count, int step, uint32_t* status, const Right& right) {
  bool all = true;
#pragma unroll 4
  for (int d = first; d < count; d += step) all &= right(d);
  if (!all) atomicOr(status, kBadIndex);
}

// Finds the `slot`-th unit of `count` documents with all THREADS threads of a CTA, a document each, so that what is to be known of
// THREADS documents is one load's latency away: load(d, live) brings a document's record to its thread, with its `units` and
// their `weight`, and found(record, document, unit) is called by the thread of the document that the unit is in, before the last
// barrier.
// LONGEST_FIRST: up to THREADS documents are taken by falling weight (the longest key ranges), and a document's units from its
// last one backwards (under a causal mask the longest again), so that short ones are left for the end of a launch; else, and
// among more documents, they come in order.
template <int THREADS>
struct FindScratch {
  int totals[THREADS / 32];
  __align__(16) int weight[THREADS];
  int order[THREADS], units[THREADS], hit[2];
};
template <int THREADS, bool LONGEST_FIRST, typename Load, typename Found>
__device__ __forceinline__ void find_unit(int count, int slot, FindScratch<THREADS>& S, const Load& load, const Found& found) {
  const int thread = static_cast<int>(threadIdx.x), warp = thread >> 5, lane = thread & 31;
  const bool sorted = LONGEST_FIRST && count > 1 && count <= THREADS;
  for (int base = 0; base < count; base += THREADS) {
    const int d = base + thread;
    const auto record = load(d, d < count);
    int units = record.units, document = d;
    if (sorted) {
      S.weight[thread] = d < count ? record.weight : INT_MIN;
      __syncthreads();
      if (d < count) {
        int rank = 0;
        for (int e = 0; e < count; e += 4) {  // what lies behind the last document weighs less than any
          const int4 four = *reinterpret_cast<const int4*>(&S.weight[e]);
          const int w[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) rank += w[i] > record.weight || (w[i] == record.weight && e + i < d);
        }
        S.order[rank] = d, S.units[rank] = units;
      }
      __syncthreads();
      units = d < count ? S.units[thread] : 0, document = d < count ? S.order[thread] : 0;
    }
    int through = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, through, o);
      if (lane >= o) through += other;
    }
    if (lane == 31) S.totals[warp] = through;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w == warp) through += total;
      total += S.totals[w];
    }
    if (slot < through && slot >= through - units) {
      const int index = LONGEST_FIRST ? through - 1 - slot : slot - (through - units);
      if (sorted)
        S.hit[0] = document, S.hit[1] = index;
      else
        found(record, d, index);
    }
    __syncthreads();
    if (sorted && slot < total) {
      if (thread == S.hit[0]) found(record, d, S.hit[1]);
      __syncthreads();
    }
    if (slot < total) return;
    slot -= total;
  }
}

// What the queries of a document see: query i of `queries` stands at position i + keys - queries and sees the first
// visible(i) of its keys - all of them, or under a causal mask those up to its own position and the document's prefix.
struct Sight {
  int keys, ahead, prefix;  // ahead: position of query 0
  bool causal;
  __device__ __forceinline__ int visible(int query) const {
    return causal ? clamped(max(prefix, ahead + query + 1), 0, keys) : keys;
  }
};

#endif  // __CUDACC__

// Key ranges that were divided over several CTAs: share z of row r of head h is at [z][h][r].
struct KeyShares {
  const int* bounds;  // rows outside [bounds[0], bounds[documents]) are left as they are
  float* partial;     // normalised rows of 128
  float* lse;         // log2 units; -inf: a share without weight
  __nv_bfloat16* output;
  int documents, rows, heads, total_heads, head_offset, splits;
};
inline size_t key_shares_bytes(long long rows, long long heads, int splits) {
  return splits <= 1 ? 0 : static_cast<size_t>(splits) * heads * rows * (512 + 4);
}
// Joins them into the output; defined beside the masked attention kernel.
int launch_join_shares(const KeyShares& shares, void* stream);

}  // namespace nob200
