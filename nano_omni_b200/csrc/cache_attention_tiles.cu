// Attention over the 8-bit cache of kv_cache.cu for many rows per sequence and key head: a chunk of new tokens, or a few drafted
// ones whose query heads share a key head.  head_dim 128, sm_100a; the definition is cache_attention.cu's.
//
// A unit is 128 rows - (new token, head of the group) pairs of a sequence and key head - against 128 keys, two blocks, at a
// time.  The scores and values are tcgen05 products of f16 operands, which hold an 8-bit code exactly (and take five instructions
// for four codes, bf16 eight); queries are scaled by a power of two to a row maximum in [1, 2) (exact down to 2^-24 of it).  The
// scales of K multiply the scores as they leave TMEM, those of V the probabilities before these are rounded to f16, so
// nothing of K and V is rounded.  (Sixteen columns at a time by mma.sync widen every code once per sixteen rows: 1200 warp instructions per 32 keys,
// 28 rows against 4000 keys x 8 heads x 16 sequences 102 us.)
//   warps 16, 19  TMA producers: the blocks of K and of V as they are, 8 bits, into a ring of five blocks each (one producer for both,
//                 whose K waited for V's places, held the kernel at 1.8 us a tile)
//   warps 8-11    widen the blocks of K to f16 in the 128-byte-swizzled layout of the MMAs, warps 12-15 those of V, into a ring of
//                 four 32 KiB tiles; first of all warps 12-15 bring the queries, a row per thread, into TMEM
//   warps 17, 18  issue the score and the value MMAs
//   warps 0-3     softmax of the even blocks, a thread per row; warps 4-7 of the odd ones.  Each half has a running maximum, sum
//                 and accumulator of its own, so that they need not meet before the end, where they join through shared
//                 memory and put out half of the channels each.  (One warp per 32 rows for both halves had its scheduler to
//                 itself and waited for its own instructions: 3500 cycles a tile, so .... )
// TMEM columns: S 0-127, P 128-191 (f16, two keys per column), O of the even blocks 192-319, of the odd ones 320-447,
// Q 448-511 (f16, two channels per column).
#include <cuda.h>
#include <cuda_fp16.h>

#include "cache_attention.cuh"
#include "common.cuh"
#include "documents.cuh"
#include "fa_common.cuh"
#include "tensor_map.cuh"

namespace nob200 {
namespace {

constexpr int kTile = 128, kBlock = 64, kDim = 128;
constexpr int kHalfBytes = kTile * 64 * 2, kTileBytes = 2 * kHalfBytes;  // f16
constexpr int kRawBytes = kBlock * kDim;
constexpr int kStages = 4, kRawStages = 5;
constexpr int kThreads = 640;
constexpr int kWidenWarp = 8, kKeyWarp = 16, kMmaWarp = 17, kValueWarp = 19;  // warp 18 issues the value MMAs
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr float kLowestMaximum = -1e38f;   // relative to it a key of score -inf weighs 0
constexpr int kSoftmaxRegs = 152, kWidenRegs = 64, kServiceRegs = 48;
static_assert(128 * (2 * kSoftmaxRegs + 2 * kWidenRegs + kServiceRegs) <= kThreads * 96, "setmaxnreg split exceeds the registers the CTA owns");
// A block's scales are overwritten sixteen blocks later, when V's block eleven or more later has left the ring of blocks: its
// tile, five later, is widened into a place that the value MMAs of a later tile than this one have left.
constexpr int kScaleSlots = 16;
constexpr float kNotThere = -1e30f;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192, kColQ = 448;

struct Unit {
  int sequence, item0, items;  // items: of the sequence from this unit's first on (0: no unit)
  int row0, kv_begin, kv_end;  // first new row of the sequence; key tiles of this CTA
  Sight sight;
};

struct __align__(1024) Shared {
  uint8_t kv[kStages][kTileBytes];
  uint8_t raw[2][kRawStages][kRawBytes];  // of K, of V
  __align__(16) float2 scales[kScaleSlots];  // (K's, log2 of V's) of a block; NaN, kNotThere for one that is not there
  uint64_t q_full;
  uint64_t raw_full[2][kRawStages], raw_empty[2][kRawStages];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t s_full, s_taken, p_full[2], pv_done[2];
  uint64_t scales_full[kScaleSlots];  // a block's scales are there
  uint64_t joined[8];               // a softmax warp has left what its partner needs
  float top[2][kTile], sum[2][kTile];
  float factor[kTile];  // of a row's f16 form
  Unit unit;
  FindScratch<kThreads> find;
  uint32_t tmem_base;
  uint32_t abort;
  uint32_t qk_issued;
};
static_assert(sizeof(Shared) + 1024 <= 227 * 1024, "shared memory of an SM");

// The unit of this CTA, into shared memory.
__device__ __forceinline__ void find_own_unit(const CacheParams& P, Shared& S, int slot, int piece) {
  struct Sequence {
    int2 rows;
    int length, prefix, units, weight;
  };
  find_unit<kThreads, true>(
      P.sequences, slot, S.find,
      [&](int d, bool live) {
        Sequence r = {};
        if (live) {
          r.length = r.weight = P.lengths[d];
          r.prefix = P.prefix ? P.prefix[d] : 0;
          r.rows = document_rows(P.bounds, d, P.rows);
          r.units = ((r.rows.y - r.rows.x) * P.group + kTile - 1) / kTile;
        }
        return r;
      },
      [&](const Sequence& r, int d, int index) {
        Unit u;
        const int tokens = r.rows.y - r.rows.x;
        u.sequence = d;
        u.item0 = index * kTile;
        u.items = tokens * P.group - u.item0;
        u.row0 = r.rows.x;
        u.sight.keys = clamped(r.length, 0, P.max_blocks * kBlock);
        if (u.sight.keys != r.length) atomicOr(P.status, kBadIndex);
        u.sight.ahead = u.sight.keys - tokens;
        u.sight.prefix = r.prefix;
        u.sight.causal = P.causal != 0;
        const int seen = u.sight.visible((u.item0 + min(u.items, kTile) - 1) / P.group);
        const int tiles = (seen + kTile - 1) / kTile;
        u.kv_begin = static_cast<int>(static_cast<long long>(tiles) * piece / P.splits);
        u.kv_end = static_cast<int>(static_cast<long long>(tiles) * (piece + 1) / P.splits);
        S.unit = u;
      });
}

// The block of keys 64 b .. 64 b + 63; -1 and a note for one that is not there, -1 without past the table.
__device__ __forceinline__ int block_of(const CacheParams& P, const int* table, int b) {
  if (b >= P.max_blocks) return -1;
  const int block = table[b];
  return block >= 0 && block < P.num_blocks ? block : -1;
}

// Four signed bytes as f16: offset by 128, a byte u under the exponent of 1024 is 1024 + u.
__device__ __forceinline__ uint2 widen(uint32_t w) {
  const uint32_t offset = w ^ 0x80808080u;
  auto two = [&](uint32_t select) {
    const uint32_t a = __byte_perm(offset, 0x64646464u, select);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), __float2half2_rn(1152.f));
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  return make_uint2(two(0x4140), two(0x4342));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
cache_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const CacheParams P) {
  extern __shared__ uint8_t smem_raw[];
  Shared& S = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* abort_flag = &S.abort;
  uint32_t* status = P.status;

  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 4);
    for (int s = 0; s < kRawStages; ++s)
      for (int v = 0; v < 2; ++v) {
        mbar_init(&S.raw_full[v][s], 1);
        mbar_init(&S.raw_empty[v][s], 4);
      }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&S.kv_full[s], 4);
      mbar_init(&S.kv_empty[s], 1);
    }
    mbar_init(&S.s_full, 1);
    mbar_init(&S.s_taken, 8);
    for (int h = 0; h < 2; ++h) {
      mbar_init(&S.p_full[h], 4);
      mbar_init(&S.pv_done[h], 1);
    }
    for (int w = 0; w < 8; ++w) mbar_init(&S.joined[w], 1);
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&S.scales_full[i], 1);
    S.unit = Unit{};
    S.abort = 0;
    S.qk_issued = 0;
    mbar_fence_init();
  }
  if (warp == kKeyWarp) {
    tmem_alloc(&S.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();  // launched as a programmatic dependent: the set-up above overlaps the kernel before
  // all key heads of a unit are neighbours in the grid, a sequence's units with the longest key ranges first
  const int piece = static_cast<int>(blockIdx.x % P.splits), place = static_cast<int>(blockIdx.x / P.splits);
  const int key_head = place % P.kv_heads;
  find_own_unit(P, S, place / P.kv_heads, piece);
  const uint32_t tmem = S.tmem_base;
  pdl_release();

  const int items = S.unit.items;  // 0: no unit
  const int kv_begin = S.unit.kv_begin, n_kv = S.unit.kv_end - kv_begin;
  const int* table = P.table + static_cast<size_t>(S.unit.sequence) * P.max_blocks;
  // the order of the key tiles: under a distance bias from the last, and so nearest and largest, one backwards
  auto tile_at = [&](int j) { return BIAS ? n_kv - 1 - j : j; };
  auto spin = [&](uint64_t* bar, uint32_t parity, uint32_t bit) { return warp_poll(bar, parity, abort_flag, status, bit); };
  auto rest = [&](uint64_t* bar, uint32_t parity, uint32_t bit) { return warp_rest(bar, parity, abort_flag, status, bit); };

  if (warp >= kKeyWarp) {
    reg_dealloc<kServiceRegs>();
    if (n_kv == 0) {
    } else if (warp == kKeyWarp || warp == kValueWarp) {
      // ------------------------------------------------------------ TMA producers, a block at a time
      const int v = warp == kValueWarp;
      const CUtensorMap* map = v ? &map_v : &map_k;
      if (lane == 0) tma_prefetch_desc(map);
      // A lane holds the number and scales of one block in 32, those of the next 32 on their way: one after the other they
      // would take two loads' latency each.
      struct Blocks {
        int number;
        float key, value_log2;
      };
      auto blocks_from = [&](int i) {
        Blocks r = {-1, 0.f, kNotThere};
        if (i + lane < 2 * n_kv) {
          const int at = 2 * (kv_begin + tile_at((i + lane) >> 1)) + ((i + lane) & 1);
          r.number = block_of(P, table, at);
          if (r.number < 0 && at * kBlock < S.unit.sight.keys) atomicOr(status, kBadIndex);
          if (v && r.number >= 0) {
            const size_t place = static_cast<size_t>(r.number) * P.kv_heads + key_head;
            const float value = P.value_scales[place];
            r.key = P.key_scales[place];
            // a summand of the exponent; of a block whose scale is 0 (or less) next to nothing is taken
            r.value_log2 = log2f(value > 0.f ? value : value != value ? value : 1e-30f);
          }
        }
        return r;
      };
      bool ok = true;
      Blocks some = {}, next = blocks_from(0);
      for (int i = 0; ok && i < 2 * n_kv; ++i) {
        const int st = i % kRawStages;
        if (i % 32 == 0) some = next, next = blocks_from(i + 32);
        const int block = __shfl_sync(0xffffffffu, some.number, i % 32);
        if (i >= kRawStages) ok = rest(&S.raw_empty[v][st], ((i / kRawStages) - 1) & 1, kWaitTimeoutRing);
        if (!ok) break;
        if (v) {
          const float key = __shfl_sync(0xffffffffu, some.key, i % 32), value_log2 = __shfl_sync(0xffffffffu, some.value_log2, i % 32);
          if (lane == 0) S.scales[i % kScaleSlots] = make_float2(key, value_log2);
        }
        if (lane == 0) {
          mbar_expect_tx(&S.raw_full[v][st], kRawBytes);
          // a block that is not there: any block, whose scores are masked
          tma_load_3d(S.raw[v][st], map, &S.raw_full[v][st], 0, (max(block, 0) * P.kv_heads + key_head) * kBlock, 0);
          if (v) mbar_arrive(&S.scales_full[i % kScaleSlots]);
        }
        __syncwarp();
      }
    } else if (warp == kMmaWarp) {
      // --------------------------------------------------------- score MMAs: S = Q K_j^T
      constexpr uint32_t idesc_qk = umma_idesc(kDF32, kFmtF16, kFmtF16, 0, 0, kTile, kTile);
      const uint64_t kv_k_desc = umma_smem_desc(0, 16, 1024, kSwizzle128B) + (smem_u32(S.kv[0]) >> 4);
      bool ok = rest(&S.q_full, 0, kWaitTimeoutLoad);
      for (int j = 0; ok && j < n_kv; ++j) {
        const int ik = 2 * j, sk = ik % kStages;
        const uint64_t b0 = kv_k_desc + sk * (kTileBytes >> 4);
        ok = rest(&S.kv_full[sk], (ik / kStages) & 1, kWaitTimeoutLoad) && (j == 0 || spin(&S.s_taken, (j - 1) & 1, kWaitTimeoutSoftmax));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          // 16 channels: 8 columns of Q, 32 bytes inside a 64-channel half of K
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_ts<0>(tmem + kColS, tmem + kColQ + 8 * k, b0 + (k >> 2) * (kHalfBytes >> 4) + 2 * (k & 3), idesc_qk, k > 0);
          tc_commit(&S.s_full);
          tc_commit(&S.kv_empty[sk]);
          *reinterpret_cast<volatile uint32_t*>(&S.qk_issued) = j + 1;
        }
        __syncwarp();
      }
    } else {
      // --------------------------------------------------------- value MMAs of either half, behind the next score group
      constexpr uint32_t idesc_pv = umma_idesc(kDF32, kFmtF16, kFmtF16, 0, 1, kTile, kDim);
      const uint64_t kv_n_desc = umma_smem_desc(0, kHalfBytes, 1024, kSwizzle128B) + (smem_u32(S.kv[0]) >> 4);
      bool ok = true;
      for (int j = 0; ok && j < n_kv; ++j) {
        const int iv = 2 * j + 1, sv = iv % kStages;
        for (int half = 0; ok && half < 2; ++half) {
          ok = (half > 0 || rest(&S.kv_full[sv], (iv / kStages) & 1, kWaitTimeoutLoad)) && spin(&S.p_full[half], j & 1, kWaitTimeoutSoftmax) &&
               warp_wait_counter(&S.qk_issued, min(j + 2, n_kv), abort_flag, status, kWaitTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            // 16 keys = 16 rows of 128 B = 2048 B; P holds two keys per 32-bit column
            const uint64_t b0 = kv_n_desc + sv * (kTileBytes >> 4) + half * (4 * 2048 >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_ts<0>(tmem + kColO + half * kDim, tmem + kColP + half * 32 + 8 * k, b0 + k * (2048 >> 4), idesc_pv, j > 0 || k > 0);
            tc_commit(&S.pv_done[half]);
            if (half == 1) tc_commit(&S.kv_empty[sv]);
          }
          __syncwarp();
        }
      }
    }
  } else if (warp >= kWidenWarp) {
    // ------------------------------------------------- queries, then codes to bf16 tiles
    reg_dealloc<kWidenRegs>();
    const int v = warp >= kWidenWarp + 4, quarter = warp & 3;  // of K or V; which 32 rows of a tile
    if (v && n_kv > 0) {
      // row `thread` of the unit
      const int thread = threadIdx.x - 32 * (kWidenWarp + 4);
      const bool live = thread < items;
      const int item = S.unit.item0 + (live ? thread : 0), token = item / P.group, head = key_head * P.group + item - token * P.group;
      const uint4* src = reinterpret_cast<const uint4*>(P.query + (static_cast<size_t>(S.unit.row0 + token) * P.heads + head) * kDim);
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint4 x = live ? src[c] : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
      }
      const uint32_t exponent = min(max(__float_as_uint(top) >> 23, 1u), 253u);
      const float down = __uint_as_float((254u - exponent) << 23);
      S.factor[thread] = __uint_as_float(exponent << 23);
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {
        uint32_t h[32];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 x = live ? src[8 * g + c] : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) h[4 * c + i] = pack_f16(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i] & 0xffff0000u) * down);
        }
        tmem_st32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + kColQ + 32 * g, h);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.q_full);
    }
    // a lane's 16 bytes of a row become two pieces of one half; which of the two goes first keeps the eight lanes of a row apart
    const int piece16 = lane & 7, swap = piece16 >> 2, first = 2 * (piece16 & 3);
    bool ok = true;
    for (int j = 0; ok && j < n_kv; ++j) {  // a tile of K is in ring stage 0 or 2, of V in 1 or 3
      const int st = (2 * j + v) % kStages;
      ok = j < 2 || rest(&S.kv_empty[st], ((j >> 1) - 1) & 1, kWaitTimeoutMma);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 2 * j + half, raw = i % kRawStages;
        ok = ok && rest(&S.raw_full[v][raw], (i / kRawStages) & 1, kWaitTimeoutLoad);
        if (!ok) break;
        const uint8_t* from = S.raw[v][raw] + quarter * 16 * kDim + lane * 16;
        uint4 x[4];  // rows 4 k + lane / 8 of the warp's 16
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const uint4*>(from + k * 512);
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.raw_empty[v][raw]);
        uint8_t* to = S.kv[st] + swap * kHalfBytes + (half * kBlock + quarter * 16 + (lane >> 3)) * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint2 a = widen(x[k].x), b = widen(x[k].y), c = widen(x[k].z), d = widen(x[k].w);
          const uint4 low = make_uint4(a.x, a.y, b.x, b.y), high = make_uint4(c.x, c.y, d.x, d.y);
          const int row = 4 * k + (lane >> 3);
          *reinterpret_cast<uint4*>(to + k * 512 + (((first + swap) ^ (row & 7)) << 4)) = swap ? high : low;
          *reinterpret_cast<uint4*>(to + k * 512 + (((first + 1 - swap) ^ (row & 7)) << 4)) = swap ? low : high;
        }
      }
      if (!ok) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.kv_full[st]);
    }
  } else {
    // ------------------------------------------------- softmax + epilogue warps
    reg_alloc<kSoftmaxRegs>();
    if (items > 0) {
      const int half = warp >> 2, in_unit = static_cast<int>(threadIdx.x & 127);
      const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + lane_base + kColS + 64 * half, p_addr = tmem + lane_base + kColP + 32 * half;
      const uint32_t o_addr = tmem + lane_base + kColO + kDim * half;
      const bool live = in_unit < items;
      const int item = S.unit.item0 + (live ? in_unit : 0), token = item / P.group, head = key_head * P.group + item - token * P.group;
      const int visible = S.unit.sight.visible(token) - kv_begin * kTile - 64 * half;  // keys from this half's first block on
      const int partly = max(0, S.unit.sight.visible(S.unit.item0 / P.group) / kTile - kv_begin);
      const float slope = BIAS ? P.slopes[head] * 1.4426950408889634f : 0.f;
      // relative to this half's first key
      const int position = BIAS ? S.unit.sight.ahead + token - kv_begin * kTile - 64 * half : 0;
      // a warp without live rows only keeps the others' pace: what its rows of P and O hold goes nowhere
      const bool idle = (warp & 3) * 32 >= items;
      // The maximum is that of the probabilities times V's scale, which are what is rounded; the sum is relative to it too.
      float m_used = kLowestMaximum, sum = 0.f, row_scale = 0.f;
      bool ok = true;
      for (int j = 0; j < n_kv; ++j) {
        ok = rest(&S.s_full, j & 1, kWaitTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        if (idle) {
          // no further ahead than the others: a second arrival in one phase would stand for theirs
          if (j > 0 && !(ok = rest(&S.pv_done[half], (j - 1) & 1, kWaitTimeoutMma))) break;
          if (lane == 0) mbar_arrive(&S.s_taken), mbar_arrive(&S.p_full[half]);
          continue;
        }
        uint32_t s[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.s_taken);
        if (j == 0) row_scale = *const_cast<const volatile float*>(&S.factor[in_unit]) * P.scale;
        const int block = 2 * j + half;
        ok = rest(&S.scales_full[block % kScaleSlots], (block / kScaleSlots) & 1, kWaitTimeoutLoad);
        if (!ok) break;
        const volatile float* kept = &S.scales[block % kScaleSlots].x;
        const float key_scale = kept[0] * row_scale, value_scale = kept[1];
        const bool there = value_scale != kNotThere;
        const int valid = visible - tile_at(j) * kTile;
        // from a raw score to log2 units; a capped or biased one is turned into them at once
        const float unit = CAP || BIAS ? 1.f : key_scale * P.to_log2;
        if constexpr (CAP) cap_scores(s, key_scale, P.to_log2);
        if constexpr (BIAS) {
          const float from = static_cast<float>(position - tile_at(j) * kTile), f = CAP ? 1.f : key_scale * P.to_log2;
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] = __float_as_uint(fmaf(__uint_as_float(s[i]), f, -slope * fabsf(from - static_cast<float>(i))));
        }
        if (tile_at(j) >= partly || !there) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= valid || !there) s[i] = 0xff800000u;  // -inf
        }
        float a = __uint_as_float(s[0]), b = __uint_as_float(s[1]);
#pragma unroll
        for (int i = 2; i < 62; i += 4) {
          a = max3(a, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          b = max3(b, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
        }
        const bool sees = there && valid > 0;  // a row that sees nothing of the block takes nothing of it, whatever its scales are
        const float value_log2 = sees ? value_scale : 0.f;
        const float mx = sees ? fmaf(max3(a, b, fmaxf(__uint_as_float(s[62]), __uint_as_float(s[63]))), unit, value_log2) : kLowestMaximum;
        if (__any_sync(0xffffffffu, mx > m_used + kRescaleThreshold)) {
          const float m_new = fmaxf(m_used, mx);
          const float alpha = ex2(m_used - m_new);
          m_used = m_new;
          if (j > 0) {  // P and O are untouched by the tensor core before the first PV
            sum *= alpha;
            ok = spin(&S.pv_done[half], (j - 1) & 1, kWaitTimeoutMma);
            if (!ok) break;
            tc_fence_after();
            tmem_scale_rows(o_addr, alpha);
          }
        }
        // Probabilities times V's scale at once: 2^(x + log2 scale - m), rounded to f16 for the value MMAs; the row sum is taken
        // before, and divided by the scale.
        const float offset = value_log2 - m_used, f = sees ? unit : 1.f;
        const uint64_t unit2 = pack2(f, f), offset2 = pack2(offset, offset);
        uint64_t la = 0ull, lb = 0ull;
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          float x0, x1, x2, x3;
          unpack2(fma2(pack2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), unit2, offset2), x0, x1);
          unpack2(fma2(pack2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), unit2, offset2), x2, x3);
          const float c = ex2(x0), d = ex2(x1), e = ex2(x2), g = ex2(x3);
          la = add2(la, pack2(c, d));
          lb = add2(lb, pack2(e, g));
          p[i / 2] = pack_f16(c, d);
          p[i / 2 + 1] = pack_f16(e, g);
        }
        float l0, l1, l2, l3;
        unpack2(la, l0, l1);
        unpack2(lb, l2, l3);
        sum = fmaf((l0 + l1) + (l2 + l3), ex2(-value_log2), sum);
        if (j > 0) {
          ok = spin(&S.pv_done[half], (j - 1) & 1, kWaitTimeoutMma);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_st32(p_addr, p);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full[half]);
      }
      if (ok && n_kv > 0) ok = spin(&S.pv_done[half], (n_kv - 1) & 1, kWaitTimeoutMma);
      if (ok) {
        // ---- join of the halves: each leaves the 64 channels that the other puts out in a K tile (whose last reader is done)
        tc_fence_after();
        float4* leave = reinterpret_cast<float4*>(S.kv[2 * half]) + in_unit;  // [16 pieces of 4 channels][128 rows]
        const float4* take = reinterpret_cast<const float4*>(S.kv[2 - 2 * half]) + in_unit;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t o[32];
          if (n_kv > 0) {
            tmem_ld32(o_addr + 64 * (1 - half) + 32 * c, o);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
#pragma unroll
          for (int g = 0; g < 8; ++g)
            leave[(8 * c + g) * kTile] = make_float4(__uint_as_float(o[4 * g]), __uint_as_float(o[4 * g + 1]), __uint_as_float(o[4 * g + 2]),
                                                     __uint_as_float(o[4 * g + 3]));
        }
        S.top[half][in_unit] = m_used, S.sum[half][in_unit] = sum;
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.joined[warp]);
        ok = spin(&S.joined[warp ^ 4], 0, kWaitTimeoutSoftmax);
        if (ok) {
          const float other_top = S.top[1 - half][in_unit], other_sum = S.sum[1 - half][in_unit], top = fmaxf(m_used, other_top);
          const float mine_weight = ex2(m_used - top), other_weight = ex2(other_top - top);
          const float l = fmaf(sum, mine_weight, other_sum * other_weight);
          const float inv = l == 0.f ? 0.f : 1.0f / l, mine_inv = mine_weight * inv, other_inv = other_weight * inv;
          const int row = S.unit.row0 + token;
          const bool store = NOB_CHECK(!live || (row >= 0 && row < P.rows && head + P.head_offset < P.total_heads), status) && live;
          const size_t share = static_cast<size_t>(piece) * P.heads * P.rows;  // of divided keys
          if (P.splits > 1 && store && half == 0) P.lse[share + static_cast<size_t>(head) * P.rows + row] = top + log2f(l);
          // rows leave through shared memory, 64 bytes of each at a time, so that four lanes write one row's piece
          const int to = P.splits > 1 ? head * P.rows + row : row * P.total_heads + head + P.head_offset;  // the host checks the range
          uint8_t* mine = S.raw[0][0] + warp * 2048;  // all blocks have been widened
          const uint32_t rows_live = __ballot_sync(0xffffffffu, store);
          uint4 part[4];
          auto flush = [&](int byte) {  // `part`, the bytes from `byte` on of every lane's row
            __syncwarp();
#pragma unroll
            for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(mine + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4)) = part[g];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 8 * i + (lane >> 2);
              const size_t at = __shfl_sync(0xffffffffu, to, r);
              if (!(rows_live >> r & 1)) continue;
              const uint4 x = *reinterpret_cast<const uint4*>(mine + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
              char* dst = P.splits > 1 ? reinterpret_cast<char*>(P.partial) + (share + at) * 512 : reinterpret_cast<char*>(P.output) + at * 256;
              *reinterpret_cast<uint4*>(dst + byte + 16 * (lane & 3)) = x;
            }
          };
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            if (n_kv > 0) {
              tmem_ld32(o_addr + 64 * half + 32 * c, o);
              tc_wait_ld();
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0;
            }
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              const float4 x = take[(8 * c + g) * kTile];
              const float other[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[4 * g + i] = __float_as_uint(fmaf(__uint_as_float(o[4 * g + i]), mine_inv, other[i] * other_inv));
            }
            if (P.splits > 1) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int g = 0; g < 4; ++g) part[g] = make_uint4(o[16 * k + 4 * g], o[16 * k + 4 * g + 1], o[16 * k + 4 * g + 2], o[16 * k + 4 * g + 3]);
                flush(256 * half + 128 * c + 64 * k);
              }
            } else {
              auto two = [&](int i) { return pack_bf16(__uint_as_float(o[i]), __uint_as_float(o[i + 1])); };
#pragma unroll
              for (int g = 0; g < 4; ++g) part[g] = make_uint4(two(8 * g), two(8 * g + 2), two(8 * g + 4), two(8 * g + 6));
              flush(128 * half + 64 * c);
            }
          }
        }
      }
    }
  }

  if (*abort_flag) {  // gave up: let the copies in flight land before the CTA exits (a microsecond; one millisecond)
    for (const uint64_t start = global_timer_ns(); global_timer_ns() - start < 1000000ull;) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kKeyWarp) tmem_dealloc(tmem, kTmemCols);
}

}  // namespace

int launch_cache_tiles(const CacheParams& params, const void* key, const void* value, bool capped, void* stream) {
  const char* name = "int8_cache_attention_d128";
  CUtensorMap mk, mv;
  int rc;
  const uint64_t lines = static_cast<uint64_t>(params.num_blocks) * params.kv_heads * kBlock;
  for (int i = 0; i < 2; ++i)
    if ((rc = make_tensor_map_3d(i ? &mv : &mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, i ? value : key, kDim, lines, 1, kDim, kDim * lines, kDim,
                                 kBlock, 1, CU_TENSOR_MAP_SWIZZLE_NONE)))
      return rc;
  auto kernel = capped ? (params.slopes ? cache_tiles_kernel<true, true> : cache_tiles_kernel<true, false>)
                       : (params.slopes ? cache_tiles_kernel<false, true> : cache_tiles_kernel<false, false>);
  const size_t smem = sizeof(Shared) + 1024;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess)
    return fail(kCudaError, "%s: cannot reserve %zu B of shared memory: %s", name, smem, cudaGetErrorString(err));
  const long long grid = static_cast<long long>(params.slots) * params.kv_heads * params.splits;
  return launch_pdl(name, kernel, static_cast<unsigned>(grid), kThreads, smem, stream, mk, mv, params);
}

}  // namespace nob200
