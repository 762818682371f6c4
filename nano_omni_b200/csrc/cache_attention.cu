// Attention of a few queries per sequence over the 8-bit cache of kv_cache.cu, head_dim 128, sm_100a.
//
//   s = scale * q . (code_k * scale_k[block]);  o = sum_j softmax_j(s) code_v * scale_v[block], masks, cap and distance bias as
// in fa_fwd_masked_bf16.cu.  No counterpart in the reference.
//
// One token reads every cached byte once and computes 2 x 128 multiply-adds per 256 bytes and head, so the call is bound by
// HBM and the kernel by how many bytes it keeps in flight.  The query heads that share a key head, of all new tokens of a
// sequence, are rows of one 16-row matrix instruction (mma.sync: a tcgen05 tile of 128 rows would stand empty, and its
// operands would have to go through shared memory once more after they are widened).
//
// A CTA owns 16 such rows of one sequence and key head and a contiguous share of its blocks; its four warps take blocks in turn,
// each with a running maximum, sum and 16 x 128 accumulator of its own, joined at the end.  A warp feeds itself: its lane 0
// issues TMA loads of K and V blocks (64 x 128 bytes, 128-byte swizzle) into a ring of three, two of which are in flight while
// one is worked on; two CTAs per SM make 128 KiB in flight, well over the 45 KiB that latency x bandwidth asks for.
//  * scores: A = the queries as f16, scaled by a power of two to a row maximum in [1, 2) (exact down to 2^-24 of it);
//    B = codes, which f16 holds exactly: byte -> f16 by a permute onto 1024 + (code + 128) and a subtraction.  The channels
//    of an instruction's k index are chosen so that a lane reads 32 consecutive bytes of a key.
//  * values: V's bytes come through ldmatrix.trans, which delivers two channels of two keys per register; a permute
//    separates the channels into two n tiles.  The probabilities are rounded to f16 (2^-11), their sum is taken before;
//    the block's scale of V multiplies the block's product as it joins the accumulator.
#include <cuda.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "documents.cuh"
#include "fa_common.cuh"
#include "tensor_map.cuh"
#include "../../include/nano_omni_b200.h"

namespace nob200 {
namespace {

constexpr int kBlock = 64, kDim = 128, kBlockBytes = kBlock * kDim;
constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16, kStages = 3;
constexpr float kLowestMaximum = -1e38f;  // relative to it a key of score -inf weighs 0

struct __align__(1024) Shared {
  uint8_t ring[kWarps][kStages][kBlockBytes];  // after the last block: the warps' accumulators [16][128] f32
  uint64_t full[kWarps][kStages];
  float top[kWarps][kRows], sum[kWarps][kRows];
  int unit[2];
  uint32_t abort;
};

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
  int slots, splits, causal;
  float scale;    // of a raw score; CAP form: divided by the cap
  float to_log2;  // from a (capped) scaled score to log2 units
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
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 - 2 / (1 + e^2x): absolute error some 2^-22 for any x
__device__ __forceinline__ float tanh_any(float x) { return fmaf(-2.f, rcp(1.f + ex2(x * 2.885390081777927f)), 1.f); }

template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 2)
cache_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const CacheParams P) {
  extern __shared__ uint8_t smem_raw[];
  Shared& S = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, part = lane & 3;  // row (and key / channel) of a fragment, quarter of its columns
  volatile uint32_t* abort_flag = &S.abort;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) mbar_init(&S.full[w][s], 1);
    S.abort = 0;
    mbar_fence_init();
  }
  const int piece = static_cast<int>(blockIdx.x) % P.splits;
  const int slot = static_cast<int>(blockIdx.x) / P.splits % P.slots;
  const int key_head = static_cast<int>(blockIdx.x) / P.splits / P.slots;
  pdl_wait();
  if (warp == 0) {
    const int2 found = find_unit(P.sequences, slot, [&](int s) {
      const int2 r = document_rows(P.bounds, s, P.rows);
      return ((r.y - r.x) * P.group + kRows - 1) / kRows;
    });
    if (lane == 0) S.unit[0] = found.x, S.unit[1] = found.y;
  }
  __syncthreads();
  pdl_release();
  const int sequence = S.unit[0];
  if (sequence < 0) return;

  const int2 rows = document_rows(P.bounds, sequence, P.rows);
  const int given = P.lengths[sequence];
  Sight sight;
  sight.keys = clamped(given, 0, P.max_blocks * kBlock);
  if (given != sight.keys && threadIdx.x == 0) atomicOr(P.status, kBadIndex);
  sight.ahead = sight.keys - (rows.y - rows.x);
  sight.prefix = P.prefix ? P.prefix[sequence] : 0;
  sight.causal = P.causal != 0;
  const int items = (rows.y - rows.x) * P.group;  // (token, head of the group) pairs
  const int item0 = S.unit[1] * kRows;
  const int blocks = (sight.visible((min(items, item0 + kRows) - 1) / P.group) + kBlock - 1) / kBlock;
  const int begin = static_cast<int>(static_cast<long long>(blocks) * piece / P.splits);
  const int end = static_cast<int>(static_cast<long long>(blocks) * (piece + 1) / P.splits);
  const int mine = (end - begin - warp + kWarps - 1) / kWarps;  // blocks of this warp: begin + warp, + kWarps, ...

  // ---- the table two blocks ahead of the loads, the scales one block ahead of their use
  const int* table = P.table + static_cast<size_t>(sequence) * P.max_blocks + begin + warp;
  auto entry = [&](int i) {
    int block = i < mine ? table[i * kWarps] : 0;
    if (block < 0 || block >= P.num_blocks) {
      if (lane == 0) atomicOr(P.status, kBadIndex);
      block = -1;
    }
    return block;
  };
  uint8_t(*ring)[kBlockBytes] = S.ring[warp];
  uint64_t* full = S.full[warp];
  auto load = [&](int i, int which, int block) {  // K (0) or V (1) of this warp's i-th block
    const int n = 2 * i + which;
    if (i < mine && lane == 0) {
      mbar_expect_tx(&full[n % kStages], kBlockBytes);
      // a block that is not there: any block, whose scores are masked
      tma_load_3d(ring[n % kStages], which ? &map_v : &map_k, &full[n % kStages], 0, (max(block, 0) * P.kv_heads + key_head) * kBlock, 0);
    }
  };
  int e0 = entry(0), e1 = entry(1), e2 = entry(2);
  load(0, 0, e0);
  load(0, 1, e0);
  load(1, 0, e1);

  // ---- the 16 rows
  uint32_t q[kDim / 16][4];
  float factor[2];  // raw score of the row's f16 form and a key's codes, without the key's scale -> scaled score
  int visible[2], position[2];
  float slope[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int item = item0 + quad + 8 * r;
    const bool live = item < items;
    const int token = live ? item / P.group : 0, head = key_head * P.group + (live ? item - token * P.group : 0);
    visible[r] = live ? sight.visible(token) : 0;
    position[r] = sight.ahead + token;
    slope[r] = BIAS ? P.slopes[head] * 1.4426950408889634f : 0.f;
    uint32_t w[16];
    const uint4* src = reinterpret_cast<const uint4*>(P.query + (static_cast<size_t>(rows.x + token) * P.heads + head) * kDim + 32 * part);
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
    factor[r] = __uint_as_float(exponent << 23) * P.scale;
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = w[2 * t + h];
        q[t][2 * h + r] = pack_f16(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xffff0000u) * down);
      }
  }

  float o[kDim / 8][4];
#pragma unroll
  for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
  float top[2] = {kLowestMaximum, kLowestMaximum}, sum[2] = {0.f, 0.f};
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
    float s[kBlock / 8][4];
    const uint8_t* k_at = ring[nk % kStages] + quad * kDim;
#pragma unroll
    for (int n = 0; n < kBlock / 8; ++n) {
#pragma unroll
      for (int c = 0; c < 4; ++c) s[n][c] = 0.f;
      uint32_t w[8];  // 32 channels of key 8 n + quad; the swizzle leaves the eight lanes of a phase on different banks
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(k_at + n * 8 * kDim + (((2 * part + h) ^ quad) << 4));
        w[4 * h] = x.x, w[4 * h + 1] = x.y, w[4 * h + 2] = x.z, w[4 * h + 3] = x.w;
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t u = w[t] ^ 0x80808080u;
        mma_f16(s[n], q[t], widen<0x4140>(u), widen<0x4342>(u));
      }
    }
    __syncwarp();  // all lanes have read the K block
    load(i + 1, 1, e1);

    const int key0 = (begin + warp + i * kWarps) * kBlock;
    const int first = key0 + 2 * part;  // the lane's keys: first + 8 n, first + 8 n + 1
    float mx[2] = {kLowestMaximum, kLowestMaximum};
    float alpha[2];
    const bool whole = e0 >= 0 && __all_sync(0xffffffffu, min(visible[0], visible[1]) >= key0 + kBlock);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float f = factor[r] * key_scale * (CAP ? 1.f : P.to_log2);
      const int seen = e0 < 0 ? 0 : visible[r] - first;
#pragma unroll
      for (int n = 0; n < kBlock / 8; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = s[n][2 * r + c] * f;
          if constexpr (CAP) x = tanh_any(x) * P.to_log2;
          if constexpr (BIAS) x -= slope[r] * static_cast<float>(abs(position[r] - (first + 8 * n + c)));
          if (!whole && 8 * n + c >= seen) x = -INFINITY;
          s[n][2 * r + c] = x;
          mx[r] = fmaxf(mx[r], x);
        }
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float now = fmaxf(top[r], mx[r]);
      alpha[r] = ex2(top[r] - now);
      top[r] = now;
      sum[r] *= alpha[r];
    }
    uint32_t p[kBlock / 16][4];
#pragma unroll
    for (int n = 0; n < kBlock / 8; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float a = ex2(s[n][2 * r] - top[r]), b = ex2(s[n][2 * r + 1] - top[r]);
        sum[r] += a + b;
        p[n >> 1][2 * (n & 1) + r] = pack_f16(a, b);
      }

    // ---- values
    ok = warp_rest(&full[nv % kStages], (nv / kStages) & 1, abort_flag, P.status, kWaitTimeoutLoad);
    if (!ok) break;
    // rows that see nothing of the block take nothing of it, whatever its scale is
    const float take[2] = {e0 >= 0 && visible[0] > key0 ? value_scale : 0.f, e0 >= 0 && visible[1] > key0 ? value_scale : 0.f};
    const uint32_t v_at = smem_u32(ring[nv % kStages]);
    const int v_key = ((lane >> 3) & 1) * 8 + (lane & 7);  // ldmatrix: the row whose address this lane gives
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {  // 32 channels
      float d[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) d[n][c] = 0.f;
#pragma unroll
      for (int kt = 0; kt < kBlock / 16; ++kt) {
        const int key = kt * 16 + v_key;
        uint32_t w[4];
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(v_at + key * kDim + (((2 * cc + (lane >> 4)) ^ (key & 7)) << 4))
                     : "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u0 = w[2 * h] ^ 0x80808080u, u1 = w[2 * h + 1] ^ 0x80808080u;
          mma_f16(d[2 * h], p[kt], widen<0x4240>(u0), widen<0x4240>(u1));      // even channels
          mma_f16(d[2 * h + 1], p[kt], widen<0x4341>(u0), widen<0x4341>(u1));  // odd channels
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = c >> 1;
          const float kept = o[4 * cc + n][c] * alpha[r];
          o[4 * cc + n][c] = take[r] != 0.f ? fmaf(d[n][c], take[r], kept) : kept;
        }
    }
    __syncwarp();  // all lanes have read the V block
    load(i + 2, 0, e2);
    e0 = e1, e1 = e2, e2 = e3;
    key_scale = next_key_scale, value_scale = next_value_scale;
  }
  if (!ok) {  // gave up: let the copies in flight land before the CTA exits (one millisecond)
    for (const uint64_t start = global_timer_ns(); global_timer_ns() - start < 1000000ull;) {
    }
  }

  // ---- join of the four warps
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    if (part == 0) S.top[warp][quad + 8 * r] = top[r], S.sum[warp][quad + 8 * r] = sum[r];
  }
  float* joined = reinterpret_cast<float*>(ring[0]);
#pragma unroll
  for (int n = 0; n < 8; ++n)  // a lane's columns of an even / odd pair of n tiles are four consecutive channels
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float4*>(joined + (quad + 8 * r) * kDim + 16 * n + 4 * part) =
          make_float4(o[2 * n][2 * r], o[2 * n + 1][2 * r], o[2 * n][2 * r + 1], o[2 * n + 1][2 * r + 1]);
  __syncthreads();
  if (*abort_flag) return;
  const int row = threadIdx.x >> 3, channel = (threadIdx.x & 7) * 16;
  const int item = item0 + row;
  if (item >= items) return;
  float most = S.top[0][row];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) most = fmaxf(most, S.top[w][row]);
  float total = 0.f, acc[16] = {};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float weight = ex2(S.top[w][row] - most);
    total += weight * S.sum[w][row];
    const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(S.ring[w][0]) + row * kDim + channel);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 x = src[c];
      acc[4 * c] = fmaf(weight, x.x, acc[4 * c]), acc[4 * c + 1] = fmaf(weight, x.y, acc[4 * c + 1]);
      acc[4 * c + 2] = fmaf(weight, x.z, acc[4 * c + 2]), acc[4 * c + 3] = fmaf(weight, x.w, acc[4 * c + 3]);
    }
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  const int token = item / P.group, head = key_head * P.group + item - token * P.group;
  const size_t out_row = rows.x + token;
  if (!NOB_CHECK(static_cast<int>(out_row) < P.rows && head + P.head_offset < P.total_heads, P.status)) return;
  if (P.splits > 1) {
    const size_t at = (static_cast<size_t>(piece) * P.heads + head) * P.rows + out_row;
    float4* dst = reinterpret_cast<float4*>(P.partial + at * kDim + channel);
#pragma unroll
    for (int c = 0; c < 4; ++c) dst[c] = make_float4(acc[4 * c] * inv, acc[4 * c + 1] * inv, acc[4 * c + 2] * inv, acc[4 * c + 3] * inv);
    if (channel == 0) P.lse[at] = most + log2f(total);
  } else {
    uint4* dst = reinterpret_cast<uint4*>(P.output + (out_row * P.total_heads + head + P.head_offset) * kDim + channel);
#pragma unroll
    for (int c = 0; c < 2; ++c)
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
                                                int causal, float scale, float cap, int kv_splits, void* workspace,
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
  NOB_REQUIRE(kv_splits >= 1 && kv_splits <= 64, "%s: kv_splits %d outside [1, 64]", name, kv_splits);
  const int group = heads / kv_heads;
  const long long items = static_cast<long long>(num_rows) * group;
  NOB_REQUIRE(items + kRows <= 0x7fffffffll, "%s: %d rows x %d heads a key head exceed the limit of 2^31", name, num_rows, group);
  const long long slots = most_units(items, sequences, kRows);
  const long long grid = slots * kv_heads * kv_splits;
  NOB_REQUIRE(grid <= 0x7fffffffll, "%s: %lld units x %d key heads x %d key shares exceed the grid limit", name, slots, kv_heads, kv_splits);
  const size_t need = key_shares_bytes(num_rows, heads, kv_splits);
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
  P.slots = static_cast<int>(slots), P.splits = kv_splits, P.causal = causal != 0;
  const float log2e = 1.4426950408889634f;
  P.scale = cap > 0.f ? scale / cap : scale;
  P.to_log2 = cap > 0.f ? cap * log2e : log2e;
  if (need) {
    P.partial = static_cast<float*>(workspace);
    P.lse = P.partial + static_cast<size_t>(kv_splits) * heads * num_rows * kDim;
  }

  CUtensorMap mk, mv;
  int rc;
  const uint64_t lines = static_cast<uint64_t>(num_blocks) * kv_heads * kBlock;
  if ((rc = make_tensor_map_3d(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, key, kDim, lines, 1, kDim, kDim * lines, kDim, kBlock, 1))) return rc;
  if ((rc = make_tensor_map_3d(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, value, kDim, lines, 1, kDim, kDim * lines, kDim, kBlock, 1))) return rc;
  auto kernel = cap > 0.f ? (slopes ? cache_attention_kernel<true, true> : cache_attention_kernel<true, false>)
                          : (slopes ? cache_attention_kernel<false, true> : cache_attention_kernel<false, false>);
  const size_t smem = sizeof(Shared) + 1024;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess)
    return fail(kCudaError, "%s: cannot reserve %zu B of shared memory: %s", name, smem, cudaGetErrorString(err));
  if ((rc = launch_pdl(name, kernel, static_cast<unsigned>(grid), kThreads, smem, stream, mk, mv, P))) return rc;
  if (kv_splits == 1) return kOk;
  return launch_join_shares({P.bounds, P.partial, P.lse, P.output, sequences, num_rows, heads, total_heads, head_offset, kv_splits}, stream);
}
