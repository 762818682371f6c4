// Attention of a few queries per sequence over the 8-bit cache of kv_cache.cu, head_dim 128, sm_100a; of many in
// cache_attention_tiles.cu.
//
//   s = scale * q . (code_k * scale_k[block]);  o = sum_j softmax_j(s) code_v * scale_v[block], masks, cap and distance bias as
// in fa_fwd_masked_bf16.cu.  No counterpart in the reference.
//
// One token reads every cached byte once and computes 2 x 128 multiply-adds per 256 bytes and head, so the call is bound by
// HBM, and the kernel by the bytes it keeps in flight and the instructions it spends on a byte (an SM has some 700 cycles for
// the 16 KiB of a block).  Keys are the 16 rows of the matrix instructions (mma.sync m16n8k16) and queries their 8 columns: the
// query heads that share a key head, of all new tokens of a sequence, are 8 or 16 columns of a CTA.  (Queries as 16 rows took
// twice the instructions for one token of up to eight heads, and 242 registers: 64 contexts x 32 heads 253 us.)  Eight columns
// spill 4 to 28 bytes of registers a thread, sixteen 36 to 116, which have three CTAs to an SM at 168 registers.
//
// A CTA's four warps take steps of 32 keys in turn from its share of the sequence, each with a running maximum, sum and
// accumulator of its own, joined at the end.  A warp feeds itself: its lane 0 issues TMA loads of K and V (32 x 128 bytes,
// 128-byte swizzle) into a ring of three, two of which are in flight while one is worked on; sixteen warps per SM make
// 128 KiB in flight, well over the 45 KiB that latency x bandwidth asks for.  One token against 131072 x 14 heads 84-90 us (5.2-5.6
// TB/s), 64 ragged contexts x 8 key heads 5.5-6.2 TB/s, of the 6.55 of a copy; the schedulers issue in 59 % of the cycles.
//  * scores: A = codes, which f16 holds exactly (byte -> f16 by a permute onto 1024 + (code + 128) and a subtraction); B = the
//    queries as f16, scaled by a power of two to a row maximum in [1, 2): exact down to 2^-17 of it, what is smaller off by 2^-25
//    of it at most.  The channels of an instruction's k index are chosen so that a lane reads 32 consecutive bytes of a key.
//  * values: A = V transposed by ldmatrix.trans, which delivers two channels of two keys per register; a permute puts the even
//    channels in rows 0-7 and the odd ones in rows 8-15.  B = the probabilities, from the scores' layout by movmatrix,
//    rounded to f16 (2^-11, and 2^-32 of the largest: kLift; their sum is taken before); the block's scale of V multiplies the
//    step's product as it joins the accumulator.
#include <cuda.h>
#include <cuda_fp16.h>

#include "cache_attention.cuh"
#include "common.cuh"
#include "documents.cuh"
#include "fa_common.cuh"
#include "tensor_map.cuh"
#include "../../include/nano_omni_b200.h"

namespace nob200 {
namespace {

constexpr int kBlock = 64, kDim = 128, kStep = 32, kStepBytes = kStep * kDim;
constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 3;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: the running maximum is raised, and what is there rescaled, past this growth
constexpr int kMaxCluster = 8;            // shares that a cluster can hold
constexpr float kLowestMaximum = -1e38f;  // relative to it a key of score -inf weighs 0

struct Unit {
  int sequence, index;   // -1: none; which group of columns of it
  int row0, tokens;      // its new tokens that are there
  int behind;            // new tokens whose rows would lie past the last one
  int length, prefix;
};

struct __align__(1024) Shared {
  uint8_t ring[kWarps][kStages][kStepBytes];  // after the last step: the warps' accumulators [columns][128] f32
  uint64_t full[kWarps][kStages];
  float top[kWarps][16], sum[kWarps][16];
  float share_top[16], share_sum[16];  // of the CTA, for the other CTAs of its cluster
  Unit unit;
  FindScratch<kThreads> find;
  uint32_t abort;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two of a word's four signed bytes (already offset by 128) as f16: a byte u under the exponent of 1024 is 1024 + u.
template <uint32_t SELECT>
__device__ __forceinline__ uint32_t widen(uint32_t offset_word) {
  const uint32_t with_exponent = __byte_perm(offset_word, 0x64646464u, SELECT);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&with_exponent), __float2half2_rn(1152.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// An 8 x 8 matrix of f16 transposed: a lane's two elements of a row become two elements of a column.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ---- clusters: a float of another CTA's shared memory, at this CTA's address of it
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote_address(uint32_t mine, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(mine), "r"(rank));
  return r;
}
__device__ __forceinline__ float remote_float(uint32_t mine, int rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(remote_address(mine, rank)) : "memory");
  return x;
}
__device__ __forceinline__ float4 remote_float4(uint32_t mine, int rank) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(remote_address(mine, rank))
               : "memory");
  return x;
}

// NT: columns of a CTA in eights.
template <bool CAP, bool BIAS, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3)
cache_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const CacheParams P) {
  constexpr int kColumns = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  Shared& S = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, part = lane & 3;  // of a fragment: row of A, column of B; and which pair of the other index
  volatile uint32_t* abort_flag = &S.abort;
  if (threadIdx.x >= 32 && threadIdx.x < 34) tma_prefetch_desc(threadIdx.x == 32 ? &map_k : &map_v);
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) mbar_init(&S.full[w][s], 1);
    S.unit.sequence = -1;
    S.abort = 0;
    mbar_fence_init();
  }
  __syncthreads();
  // all key heads of a unit are neighbours in the grid, the longest sequences' units first
  const int piece = static_cast<int>(blockIdx.x) % P.splits, place = static_cast<int>(blockIdx.x) / P.splits;
  const int key_head = place % P.kv_heads, slot = place / P.kv_heads;
  pdl_wait();
  struct Sequence {
    int2 rows;
    int behind, length, prefix, units, weight;
  };
  find_unit<kThreads, true>(
      P.sequences, slot, S.find,
      [&](int d, bool live) {
        Sequence r = {};
        if (live) {
          r.length = r.weight = P.lengths[d];
          r.prefix = P.prefix ? P.prefix[d] : 0;
          r.rows = document_rows(P.bounds, d, P.rows, &r.behind);
          r.units = ((r.rows.y - r.rows.x) * P.group + kColumns - 1) / kColumns;
        }
        return r;
      },
      [&](const Sequence& r, int d, int index) { S.unit = {d, index, r.rows.x, r.rows.y - r.rows.x, r.behind, r.length, r.prefix}; });
  pdl_release();
  const Unit unit = S.unit;
  const int sequence = unit.sequence;
  auto note_bounds = [&] {
    if (blockIdx.x == 0)
      note_documents(threadIdx.x, P.sequences, kThreads, P.status, [&](int d) { return bounds_fit(P.bounds, d, P.rows); });
  };
  if (sequence < 0) {  // the whole cluster
    note_bounds();
    return;
  }

  Sight sight;
  sight.keys = clamped(unit.length, 0, P.max_blocks * kBlock);
  if (unit.length != sight.keys && threadIdx.x == 0) atomicOr(P.status, kBadIndex);
  sight.ahead = sight.keys - unit.tokens - unit.behind;
  sight.prefix = unit.prefix;
  sight.causal = P.causal != 0;
  const int items = unit.tokens * P.group;  // (token, head of the group) pairs
  const int item0 = unit.index * kColumns;
  const int steps = (sight.visible((min(items, item0 + kColumns) - 1) / P.group) + kStep - 1) / kStep;
  const int begin = static_cast<int>(static_cast<long long>(steps) * piece / P.splits);
  const int end = static_cast<int>(static_cast<long long>(steps) * (piece + 1) / P.splits);
  const int first_step = begin + warp, mine = (end - first_step + kWarps - 1) / kWarps;
  // first_step, + kWarps, ...; under a distance bias from the last, and so nearest and largest, one backwards
  auto step_at = [&](int i) { return first_step + (BIAS ? mine - 1 - i : i) * kWarps; };

  // ---- the table two steps ahead of the loads, the scales one step ahead of their use
  const int* table = P.table + static_cast<size_t>(sequence) * P.max_blocks;
  auto entry = [&](int i) {
    int block = i < mine ? table[step_at(i) / 2] : 0;
    if (block < 0 || block >= P.num_blocks) {
      if (lane == 0) atomicOr(P.status, kBadIndex);
      block = -1;
    }
    return block;
  };
  uint8_t(*ring)[kStepBytes] = S.ring[warp];
  uint64_t* full = S.full[warp];
  auto load = [&](int i, int which, int block) {  // K (0) or V (1) of this warp's i-th step
    const int n = 2 * i + which;
    if (i < mine && lane == 0) {
      mbar_expect_tx(&full[n % kStages], kStepBytes);
      // a block that is not there: any block, whose scores are masked
      tma_load_3d(ring[n % kStages], which ? &map_v : &map_k, &full[n % kStages], 0,
                  (max(block, 0) * P.kv_heads + key_head) * kBlock + (step_at(i) & 1) * kStep, 0);
    }
  };
  int e0 = entry(0), e1 = entry(1), e2 = entry(2);
  load(0, 0, e0);
  load(0, 1, e0);
  load(1, 0, e1);

  // ---- the columns: a lane reads a quarter of column quad of each eight and works on columns 2 part and 2 part + 1
  uint32_t q[NT][kDim / 16][2];
  float factor[NT][2];  // raw product of a column's f16 form with a key's codes, without the key's scale -> scaled score
  int visible[NT][2], position[NT][2];
  float slope[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int item = item0 + 8 * n + quad;
    const bool live = item < items;
    const int token = live ? item / P.group : 0, head = key_head * P.group + (live ? item - token * P.group : 0);
    uint32_t w[16];
    const uint4* src = reinterpret_cast<const uint4*>(P.query + (static_cast<size_t>(unit.row0 + token) * P.heads + head) * kDim + 32 * part);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 x = live ? src[i] : make_uint4(0, 0, 0, 0);
      w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t exponent = min(max(__float_as_uint(top) >> 23, 1u), 253u);
    const float down = __uint_as_float((254u - exponent) << 23);
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = w[2 * t + h];
        q[n][t][h] = pack_f16(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xffff0000u) * down);
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int from = 4 * (2 * part + c);  // a lane that read the column
      factor[n][c] = __shfl_sync(0xffffffffu, __uint_as_float(exponent << 23) * P.scale, from);
      if (CAP) factor[n][c] = fminf(factor[n][c], 1e30f);  // past the cap at any scale of K, and a score of 0 is not 0 x inf
      visible[n][c] = __shfl_sync(0xffffffffu, live ? sight.visible(token) : 0, from);
      position[n][c] = BIAS ? __shfl_sync(0xffffffffu, sight.ahead + token, from) : 0;
      slope[n][c] = BIAS ? __shfl_sync(0xffffffffu, P.slopes[head] * 1.4426950408889634f, from) : 0.f;
    }
  }
  int fewest = visible[0][0];
#pragma unroll
  for (int n = 0; n < NT; ++n) fewest = min(fewest, min(visible[n][0], visible[n][1]));
  fewest = __reduce_min_sync(0xffffffffu, fewest);

  float o[kDim / 16][NT][4];  // channels 16 m + 2 quad (+ 1: the second two), columns 2 part and 2 part + 1
#pragma unroll
  for (int m = 0; m < kDim / 16; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[m][n][c] = 0.f;
  float top[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = kLowestMaximum, sum[n][0] = sum[n][1] = 0.f;
  auto scale_of = [&](const float* scales, int block) { return scales[static_cast<size_t>(max(block, 0)) * P.kv_heads + key_head]; };
  float key_scale = mine > 0 ? scale_of(P.key_scales, e0) : 0.f, value_scale = mine > 0 ? scale_of(P.value_scales, e0) : 0.f;
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int e3 = entry(i + 3);
    float next_key_scale = 0.f, next_value_scale = 0.f;
    if (i + 1 < mine) next_key_scale = scale_of(P.key_scales, e1), next_value_scale = scale_of(P.value_scales, e1);

    // ---- scores
    const int nk = 2 * i, nv = 2 * i + 1;
    ok = warp_rest(&full[nk % kStages], (nk / kStages) & 1, abort_flag, P.status, kWaitTimeoutLoad);
    if (!ok) break;
    float s[kStep / 16][NT][4];  // keys 16 m + quad (+ 8: the second two), columns 2 part and 2 part + 1
    const uint8_t* k_at = ring[nk % kStages] + quad * kDim;
#pragma unroll
    for (int m = 0; m < kStep / 16; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[m][n][c] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 16 of the lane's 32 channels; the swizzle puts the lanes of a phase on different banks
        const int at = ((2 * part + h) ^ quad) << 4;
        const uint4 x = *reinterpret_cast<const uint4*>(k_at + (16 * m) * kDim + at);
        const uint4 y = *reinterpret_cast<const uint4*>(k_at + (16 * m + 8) * kDim + at);
        const uint32_t w[2][4] = {{x.x, x.y, x.z, x.w}, {y.x, y.y, y.z, y.w}};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t u = w[0][t] ^ 0x80808080u, v = w[1][t] ^ 0x80808080u;
          const uint32_t a[4] = {widen<0x4140>(u), widen<0x4140>(v), widen<0x4342>(u), widen<0x4342>(v)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[m][n], a, q[n][4 * h + t][0], q[n][4 * h + t][1]);
        }
      }
    }
    __syncwarp();  // all lanes have read K
    load(i + 1, 1, e1);

    const int key0 = step_at(i) * kStep;
    const bool whole = e0 >= 0 && fewest >= key0 + kStep;
    uint32_t p[kStep / 16][NT][2];
    float mx[NT][2];
    bool grown = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float f = factor[n][c] * key_scale * (CAP ? 1.f : P.to_log2);
#pragma unroll
        for (int m = 0; m < kStep / 16; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) s[m][n][2 * h + c] *= f;
      }
    if constexpr (CAP) {
      float most = 0.f;
      auto each = [&](auto function) {
#pragma unroll
        for (int m = 0; m < kStep / 16; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) function(s[m][n][c]);
      };
      each([&](float& x) { most = fmaxf(most, fabsf(x)); });
      if (__all_sync(0xffffffffu, most <= 0.3f))
        each([&](float& x) { x = tanh_near(x) * P.to_log2; });
      else
        each([&](float& x) { x = tanh_any(x) * P.to_log2; });
    }
    if constexpr (BIAS) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int m = 0; m < kStep / 16; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              s[m][n][2 * h + c] -= slope[n][c] * static_cast<float>(abs(position[n][c] - (key0 + quad + 16 * m + 8 * h)));
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int seen = e0 < 0 ? 0 : visible[n][c] - key0 - quad;
#pragma unroll
          for (int m = 0; m < kStep / 16; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (16 * m + 8 * h >= seen) s[m][n][2 * h + c] = -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[n][c] = fmaxf(fmaxf(s[0][n][c], s[0][n][2 + c]), fmaxf(s[1][n][c], s[1][n][2 + c]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx[n][c] = fmaxf(mx[n][c], __shfl_xor_sync(0xffffffffu, mx[n][c], d));
        grown |= mx[n][c] - top[n][c] > kLift + kRescaleThreshold;  // a difference of neighbours is exact, the sum would be rounded
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float alpha[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float now = fmaxf(top[n][c], mx[n][c] - kLift);
          alpha[c] = ex2(top[n][c] - now);
          top[n][c] = now;
          sum[n][c] *= alpha[c];
        }
#pragma unroll
        for (int m = 0; m < kDim / 16; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[m][n][c] *= alpha[c & 1];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < kStep / 16; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = ex2(s[m][n][2 * h] - top[n][0]), b = ex2(s[m][n][2 * h + 1] - top[n][1]);
          sum[n][0] += a, sum[n][1] += b;
          p[m][n][h] = transposed(pack_f16(a, b));
        }

    // ---- values
    ok = warp_rest(&full[nv % kStages], (nv / kStages) & 1, abort_flag, P.status, kWaitTimeoutLoad);
    if (!ok) break;
    float take[NT][2];  // a column that sees nothing of the step has probabilities of 0 and takes 0 of it, whatever its scale is
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) take[n][c] = e0 >= 0 && visible[n][c] > key0 ? value_scale : 0.f;
    const uint32_t v_at = smem_u32(ring[nv % kStages]);
    const int v_key = ((lane >> 3) & 1) * 8 + (lane & 7);  // ldmatrix: the row whose address this lane gives
#pragma unroll
    for (int mm = 0; mm < kDim / 32; ++mm) {  // 32 channels
      float d[2][NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) d[0][n][c] = d[1][n][c] = 0.f;
#pragma unroll
      for (int kt = 0; kt < kStep / 16; ++kt) {
        const int key = kt * 16 + v_key;
        uint32_t w[4];
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(v_at + key * kDim + (((2 * mm + (lane >> 4)) ^ (key & 7)) << 4))
                     : "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u = w[2 * h] ^ 0x80808080u, v = w[2 * h + 1] ^ 0x80808080u;
          const uint32_t a[4] = {widen<0x4240>(u), widen<0x4341>(u), widen<0x4240>(v), widen<0x4341>(v)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(d[h][n], a, p[kt][n][0], p[kt][n][1]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[2 * mm + h][n][c] = fmaf(d[h][n][c], take[n][c & 1], o[2 * mm + h][n][c]);
    }
    __syncwarp();  // all lanes have read V
    load(i + 2, 0, e2);
    e0 = e1, e1 = e2, e2 = e3;
    key_scale = next_key_scale, value_scale = next_value_scale;
  }
  if (!ok) {  // gave up: let the copies in flight land before the CTA exits (one millisecond)
    for (const uint64_t start = global_timer_ns(); global_timer_ns() - start < 1000000ull;) {
    }
  }

  note_bounds();

  // ---- join of the four warps
  float* joined = reinterpret_cast<float*>(ring[0]);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int column = 8 * n + 2 * part + c;
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], d);
      if (quad == 0) S.top[warp][column] = top[n][c], S.sum[warp][column] = sum[n][c];
#pragma unroll
      for (int m = 0; m < kDim / 16; ++m)
        *reinterpret_cast<float2*>(joined + column * kDim + 16 * m + 2 * quad) = make_float2(o[m][n][c], o[m][n][2 + c]);
    }
  __syncthreads();
  constexpr int kLanes = kThreads / kColumns, kEach = kDim / kLanes;  // threads of a column, channels of each
  const int column = threadIdx.x / kLanes, channel = (threadIdx.x % kLanes) * kEach;
  float most = S.top[0][column];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) most = fmaxf(most, S.top[w][column]);
  float total = 0.f, acc[kEach] = {};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float weight = ex2(S.top[w][column] - most);
    total += weight * S.sum[w][column];
    const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(S.ring[w][0]) + column * kDim + channel);
#pragma unroll
    for (int c = 0; c < kEach / 4; ++c) {
      const float4 x = src[c];
      acc[4 * c] = fmaf(weight, x.x, acc[4 * c]), acc[4 * c + 1] = fmaf(weight, x.y, acc[4 * c + 1]);
      acc[4 * c + 2] = fmaf(weight, x.z, acc[4 * c + 2]), acc[4 * c + 3] = fmaf(weight, x.w, acc[4 * c + 3]);
    }
  }
  // where a column's output goes; nullptr for a column that is none, or after a wait that gave up
  auto output_of = [&](int column) -> __nv_bfloat16* {
    const int item = item0 + column;
    if (item >= items) return nullptr;
    const int token = item / P.group, head = key_head * P.group + item - token * P.group, row = unit.row0 + token;
    if (!NOB_CHECK(row < P.rows && head + P.head_offset < P.total_heads, P.status)) return nullptr;
    return P.output + (static_cast<size_t>(row) * P.total_heads + head + P.head_offset) * kDim;
  };
  if (P.joined) {
    // every CTA of the cluster leaves its result in its shared memory and joins some channels of all of them
    float* share = reinterpret_cast<float*>(S.ring[column >> 3][2]) + (column & 7) * kDim + channel;
#pragma unroll
    for (int c = 0; c < kEach / 4; ++c)
      *reinterpret_cast<float4*>(share + 4 * c) = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    if (channel == 0) S.share_top[column] = most, S.share_sum[column] = *abort_flag ? __uint_as_float(0x7fffffffu) : total;
    cluster_sync();
    for (int at = piece * kThreads + threadIdx.x; at < kColumns * (kDim / 4); at += P.splits * kThreads) {
      const int column = at / (kDim / 4), channel = at % (kDim / 4) * 4;
      const uint32_t tops = smem_u32(&S.share_top[column]), sums = smem_u32(&S.share_sum[column]);
      const uint32_t from = smem_u32(reinterpret_cast<const float*>(S.ring[column >> 3][2]) + (column & 7) * kDim + channel);
      float most = kLowestMaximum;
      for (int z = 0; z < P.splits; ++z) most = fmaxf(most, remote_float(tops, z));
      float total = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int z = 0; z < P.splits; ++z) {
        const float weight = ex2(remote_float(tops, z) - most);
        const float4 x = remote_float4(from, z);
        total = fmaf(weight, remote_float(sums, z), total);
        acc.x = fmaf(weight, x.x, acc.x), acc.y = fmaf(weight, x.y, acc.y), acc.z = fmaf(weight, x.z, acc.z), acc.w = fmaf(weight, x.w, acc.w);
      }
      const float inv = total == 0.f ? 0.f : 1.0f / total;
      if (__nv_bfloat16* dst = output_of(column))
        *reinterpret_cast<uint2*>(dst + channel) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    }
    cluster_sync();  // nobody reads this CTA's shared memory any more
    return;
  }
  __nv_bfloat16* out = output_of(column);
  if (!out || *abort_flag) return;
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  if (P.splits > 1) {
    const int item = item0 + column, token = item / P.group, head = key_head * P.group + item - token * P.group;
    const size_t at = (static_cast<size_t>(piece) * P.heads + head) * P.rows + unit.row0 + token;
    float4* dst = reinterpret_cast<float4*>(P.partial + at * kDim + channel);
#pragma unroll
    for (int c = 0; c < kEach / 4; ++c) dst[c] = make_float4(acc[4 * c] * inv, acc[4 * c + 1] * inv, acc[4 * c + 2] * inv, acc[4 * c + 3] * inv);
    if (channel == 0) P.lse[at] = most + log2f(total);
  } else {
    uint4* dst = reinterpret_cast<uint4*>(out + channel);
#pragma unroll
    for (int c = 0; c < kEach / 8; ++c)
      dst[c] = make_uint4(pack_bf16(acc[8 * c] * inv, acc[8 * c + 1] * inv), pack_bf16(acc[8 * c + 2] * inv, acc[8 * c + 3] * inv),
                          pack_bf16(acc[8 * c + 4] * inv, acc[8 * c + 5] * inv), pack_bf16(acc[8 * c + 6] * inv, acc[8 * c + 7] * inv));
  }
}

}  // namespace
}  // namespace nob200

extern "C" size_t nob200_int8_cache_attention_d128_workspace_bytes(int num_rows, int heads, int kv_splits) {
  return num_rows <= 0 || heads <= 0 ? 0 : nob200::key_shares_bytes(num_rows, heads, kv_splits);
}

extern "C" int nob200_int8_cache_attention_d128(int num_rows, int sequences, int max_blocks, int num_blocks, int head_offset,
                                                const void* query, const void* key, const void* value,
                                                const void* key_scales, const void* value_scales, const void* table,
                                                const void* lengths, const void* bounds, const void* prefix,
                                                const void* slopes, void* output, int heads, int kv_heads, int total_heads,
                                                int causal, float scale, float cap, int columns, int kv_splits, void* workspace,
                                                size_t workspace_bytes, void* stream) {
  using namespace nob200;
  const char* name = "int8_cache_attention_d128";
  NOB_REQUIRE(num_rows > 0 && sequences > 0 && max_blocks > 0 && num_blocks > 0 && heads > 0 && kv_heads > 0 && total_heads > 0,
              "%s: sizes must be positive", name);
  NOB_REQUIRE(heads % kv_heads == 0, "%s: %d heads cannot share %d key heads evenly", name, heads, kv_heads);
  NOB_REQUIRE(head_offset >= 0 && head_offset <= total_heads - heads, "%s: head_offset %d outside [0, %d]", name,
              head_offset, total_heads - heads);
  NOB_REQUIRE(max_blocks <= 0x7fffffff / kBlock, "%s: %d blocks of a sequence exceed the limit of %d", name, max_blocks, 0x7fffffff / kBlock);
  NOB_REQUIRE(static_cast<long long>(num_blocks) * kv_heads <= 0x7fffffffll / kBlock, "%s: %d blocks x %d key heads exceed the limit of %d",
              name, num_blocks, kv_heads, 0x7fffffff / kBlock);
  NOB_REQUIRE(query && key && value && key_scales && value_scales && table && lengths && bounds && output, "%s: NULL tensor", name);
  NOB_REQUIRE(reinterpret_cast<uintptr_t>(query) % 16 == 0 && reinterpret_cast<uintptr_t>(output) % 16 == 0,
              "%s: a tensor is not 16-byte aligned", name);
  NOB_REQUIRE(scale > 0.f && scale <= 1e30f, "%s: scale %g must be positive and finite", name, scale);
  NOB_REQUIRE(cap >= 0.f && cap <= 1e30f, "%s: cap %g must be finite, 0 for none", name, cap);
  NOB_REQUIRE(cap_fits(scale, cap), "%s: scale / cap must lie between 1e-35 and 1e35 (got %g / %g)", name, scale, cap);
  NOB_REQUIRE(columns == 8 || columns == 16 || columns == 128, "%s: columns must be 8, 16 or 128 (got %d)", name, columns);
  NOB_REQUIRE(kv_splits >= 1 && kv_splits <= 64, "%s: kv_splits %d outside [1, 64]", name, kv_splits);
  const int group = heads / kv_heads;
  const long long items = static_cast<long long>(num_rows) * group;
  NOB_REQUIRE(items + columns <= 0x7fffffffll, "%s: %d rows x %d heads a key head exceed the limit of 2^31", name, num_rows, group);
  const long long slots = most_units(items, sequences, columns);
  const long long grid = slots * kv_heads * kv_splits;
  NOB_REQUIRE(grid <= 0x7fffffffll, "%s: %lld units x %d key heads x %d key shares exceed the grid limit", name, slots, kv_heads, kv_splits);
  const bool joined = kv_splits > 1 && kv_splits <= kMaxCluster && columns < 128 && !workspace;
  const size_t need = joined ? 0 : key_shares_bytes(num_rows, heads, kv_splits);
  NOB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
              "%s: %zu B of 16-byte aligned workspace required for %d key shares, %zu B given", name, need, kv_splits, workspace_bytes);

  CacheParams P = {};
  P.status = status_word_device_ptr();
  if (!P.status) return fail(kCudaError, "%s: no current CUDA device", name);
  P.query = static_cast<const __nv_bfloat16*>(query), P.output = static_cast<__nv_bfloat16*>(output);
  P.key_scales = static_cast<const float*>(key_scales), P.value_scales = static_cast<const float*>(value_scales);
  P.table = static_cast<const int*>(table), P.lengths = static_cast<const int*>(lengths);
  P.bounds = static_cast<const int*>(bounds), P.prefix = static_cast<const int*>(prefix);
  P.slopes = static_cast<const float*>(slopes);
  P.rows = num_rows, P.sequences = sequences, P.max_blocks = max_blocks, P.num_blocks = num_blocks;
  P.heads = heads, P.kv_heads = kv_heads, P.group = group, P.total_heads = total_heads, P.head_offset = head_offset;
  P.slots = static_cast<int>(slots), P.splits = kv_splits, P.causal = causal != 0, P.joined = joined;
  const float log2e = 1.4426950408889634f;
  P.scale = cap > 0.f ? scale / cap : scale;
  P.to_log2 = cap > 0.f ? cap * log2e : log2e;
  P.near = P.to_log2 <= kMostNearFactor ? 0.3f : -1.f;
  if (need) {
    P.partial = static_cast<float*>(workspace);
    P.lse = P.partial + static_cast<size_t>(kv_splits) * heads * num_rows * kDim;
  }

  int rc;
  if (columns == 128) {
    rc = launch_cache_tiles(P, key, value, cap > 0.f, stream);
    if (rc || !need) return rc;
    return launch_join_shares({P.bounds, P.partial, P.lse, P.output, sequences, num_rows, heads, total_heads, head_offset, kv_splits}, stream);
  }
  CUtensorMap mk, mv;
  const uint64_t lines = static_cast<uint64_t>(num_blocks) * kv_heads * kBlock;
  if ((rc = make_tensor_map_3d(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, key, kDim, lines, 1, kDim, kDim * lines, kDim, kStep, 1))) return rc;
  if ((rc = make_tensor_map_3d(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, value, kDim, lines, 1, kDim, kDim * lines, kDim, kStep, 1))) return rc;
  const bool capped = cap > 0.f;
  auto kernel = columns == 8 ? (capped ? (slopes ? cache_attention_kernel<true, true, 1> : cache_attention_kernel<true, false, 1>)
                                       : (slopes ? cache_attention_kernel<false, true, 1> : cache_attention_kernel<false, false, 1>))
                             : (capped ? (slopes ? cache_attention_kernel<true, true, 2> : cache_attention_kernel<true, false, 2>)
                                       : (slopes ? cache_attention_kernel<false, true, 2> : cache_attention_kernel<false, false, 2>));
  const size_t smem = sizeof(Shared) + 1024;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess)
    return fail(kCudaError, "%s: cannot reserve %zu B of shared memory: %s", name, smem, cudaGetErrorString(err));
  if ((rc = launch_pdl_clusters(name, kernel, static_cast<unsigned>(grid), joined ? kv_splits : 1, kThreads, smem, stream, mk, mv, P)))
    return rc;
  if (!need) return kOk;
  return launch_join_shares({P.bounds, P.partial, P.lse, P.output, sequences, num_rows, heads, total_heads, head_offset, kv_splits}, stream);
}
