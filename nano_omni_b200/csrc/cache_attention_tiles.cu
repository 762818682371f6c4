// Attention over the 8-bit cache of kv_cache.cu for many rows per sequence and key head: a chunk of new tokens, or a few drafted
// ones whose query heads share a key head.  head_dim 128, sm_100a; the definition is cache_attention.cu's.
//
// A unit is up to 128 rows - (new token, head of the group) pairs of a sequence and key head - against 128 keys, two blocks, at a
// time.  The scores and values are tcgen05 products of f16 operands, which hold an 8-bit code exactly (and take five instructions
// for four codes, bf16 eight); queries are scaled by a power of two to a row maximum in [1, 2) (exact down to 2^-17 of it).  The
// scales of K multiply the scores as they leave TMEM, those of V the probabilities before these are rounded to f16, and their
// signs the codes, in the fused multiply-add that widens them, so nothing of K and V is rounded.  (Sixteen columns at a time by
// mma.sync widen every code once per sixteen rows: 1200 warp instructions per 32 keys, 28 rows against 4000 keys x 8 heads x 16
// sequences 102 us, here 60.)
//   warps 16, 19  TMA producers: the blocks of K and of V as they are, 8 bits, into a ring of five blocks each (one producer for both,
//                 whose K waited for V's places, held the kernel at 1.8 us a tile)
//   warps 8-11    widen the blocks of K to f16 in the 128-byte-swizzled layout of the MMAs, warps 12-15 those of V, into a ring of
//                 four 32 KiB tiles; first of all warps 12-15 bring the queries, a row per thread, into TMEM
//   warps 17, 18  issue the score and the value MMAs
//   warps 0-3     softmax of the even blocks, a thread per row; warps 4-7 of the odd ones.  Each half has a running maximum, sum
//                 and accumulator of its own, so that they need not meet before the end, where they join through shared memory.
//                 The two warps of a scheduler take turns at the exponentials, whose unit one of them keeps busy (1560 rows
//                 against 31560 keys x 14 heads 511 us, 527 at once).
// Up to 64 (32) rows stand twice (four times) in the 128 of the MMAs, and each copy's warps take their half (quarter) of the keys of a
// block; the probabilities of the others' are zero, and the copies join like the halves.  A warp reaches only its own 32 lanes of
// TMEM, so without copies one scheduler of four did all of the softmax (60 drafted tokens of 16 sequences x 56 heads 78 us, 60).
// What bounds it: a softmax warp's chain of waits, loads, maximum, exponentials (512 cycles of the MUFU a tile for each of two warps)
// and store, 2700 cycles a tile of 128 full rows; the widening (1300) and the MMAs (1024) run beside it and with half of the
// exponentials left out the time falls by 13 %, without the widening not at all.
// TMEM columns: S 0-127, P 128-191 (f16, two keys per column), O of the even blocks 192-319, of the odd ones 320-447,
// Q 448-511 (f16, two channels per column).
#include <cuda.h>
#include <cuda_fp16.h>

#include <type_traits>

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
  __align__(16) float2 scales[kScaleSlots];  // (K's, log2 of V's) magnitude for a block; NaN, kNotThere for one that is not there
  __half2 sign[2][kRawStages];               // and their signs, for the codes of K and of V; 0 for a V whose scale counts as 0
  uint64_t q_full;
  uint64_t raw_full[2][kRawStages], raw_empty[2][kRawStages];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t s_full, s_taken, p_full[2], pv_done[2];
  uint64_t values_done;  // after the last value MMA
  uint64_t scales_full[kScaleSlots];  // a block's scales are there
  uint64_t turn[2][4];                // a half's warp of a quarter of the rows is through with a tile's exponentials
  uint64_t joined;                    // the softmax warps have left their rows
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
        u.sight.ahead = u.sight.keys - tokens - r.behind;
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

// Four signed bytes times 1, -1 or 0 as f16: offset by 128, a byte u under the exponent of 1024 is 1024 + u; base is -1152 sign.
__device__ __forceinline__ uint2 widen(uint32_t w, __half2 sign, __half2 base) {
  const uint32_t offset = w ^ 0x80808080u;
  auto two = [&](uint32_t select) {
    const uint32_t a = __byte_perm(offset, 0x64646464u, select);
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), sign, base);
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
    mbar_init(&S.values_done, 1);
    mbar_init(&S.joined, 8);
    for (int q = 0; q < 8; ++q) mbar_init(&S.turn[q >> 2][q & 3], 1);
    for (int h = 0; h < 2; ++h) {
      mbar_init(&S.p_full[h], 4);
      mbar_init(&S.pv_done[h], 1);
    }
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&S.scales_full[i], 1);
    S.unit = Unit{};
    S.abort = 0;
    S.qk_issued = 0;
    mbar_fence_init();
  }
  if (warp == kKeyWarp) {
    if (lane < 2) tma_prefetch_desc(lane ? &map_v : &map_k);
    __syncwarp();
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
  // Few rows stand four or two times in the MMAs' 128, and the warps of either copy take their own part of the keys.
  const int unit_rows = items <= 32 ? 32 : items <= 64 ? 64 : kTile;
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
      // A lane holds the number and scales of one block in 32; those of the next 32 are asked for eight blocks earlier: one after
      // the other they would take two loads' latency each.
      struct Blocks {
        int number;
        float key, value;
        __half2 sign;
      };
      auto blocks_from = [&](int i) {
        Blocks r = {-1, 0.f, 0.f, __float2half2_rn(1.f)};
        if (i + lane < 2 * n_kv) {
          const int at = 2 * (kv_begin + tile_at((i + lane) >> 1)) + ((i + lane) & 1);
          r.number = block_of(P, table, at);
          if (r.number < 0 && at * kBlock < S.unit.sight.keys) atomicOr(status, kBadIndex);
          if (r.number >= 0) {
            const size_t place = static_cast<size_t>(r.number) * P.kv_heads + key_head;
            r.key = P.key_scales[place];
            if (v) r.value = P.value_scales[place];
            r.sign = __float2half2_rn(v && fabsf(r.value) < 1e-30f ? 0.f : (v ? r.value : r.key) < 0.f ? -1.f : 1.f);
          }
        }
        return r;
      };
      bool ok = true;
      Blocks some = {}, next = blocks_from(0);
      for (int i = 0; ok && i < 2 * n_kv; ++i) {
        const int st = i % kRawStages;
        if (i % 32 == 0) some = next;
        const int block = __shfl_sync(0xffffffffu, some.number, i % 32);
        const __half2 sign = __shfl_sync(0xffffffffu, some.sign, i % 32);
        if (i >= kRawStages) ok = rest(&S.raw_empty[v][st], ((i / kRawStages) - 1) & 1, kWaitTimeoutRing);
        if (!ok) break;
        if (lane == 0) {
          S.sign[v][st] = sign;
          mbar_expect_tx(&S.raw_full[v][st], kRawBytes);
          // a block that is not there: any block, whose scores are masked
          tma_load_3d(S.raw[v][st], map, &S.raw_full[v][st], 0, (max(block, 0) * P.kv_heads + key_head) * kBlock, 0);
        }
        if (v) {
          const float key = __shfl_sync(0xffffffffu, some.key, i % 32), value = __shfl_sync(0xffffffffu, some.value, i % 32);
          // V's is a summand of the exponent; of a block whose scale counts as 0 next to nothing is taken, of zeros
          const float value_log2 = block < 0 ? kNotThere : log2f(fabsf(value) < 1e-30f ? 1e-24f : fabsf(value));
          if (lane == 0) {
            S.scales[i % kScaleSlots] = make_float2(fabsf(key), value_log2);
            mbar_arrive(&S.scales_full[i % kScaleSlots]);
          }
        }
        if (i % 32 == 24) next = blocks_from(i + 8);
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
        ok = rest(&S.kv_full[sk], (ik / kStages) & 1, kWaitTimeoutLoad) && (j == 0 || rest(&S.s_taken, (j - 1) & 1, kWaitTimeoutSoftmax));
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
          ok = (half > 0 || rest(&S.kv_full[sv], (iv / kStages) & 1, kWaitTimeoutLoad)) && rest(&S.p_full[half], j & 1, kWaitTimeoutSoftmax) &&
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
            if (half == 1 && j == n_kv - 1) tc_commit(&S.values_done);
          }
          __syncwarp();
        }
      }
    }
    if (warp == kMmaWarp && blockIdx.x == 0)  // through before the others
      note_documents(lane, P.sequences, 32, status, [&](int d) { return bounds_fit(P.bounds, d, P.rows); });
  } else if (warp >= kWidenWarp) {
    // ------------------------------------------------- queries, then codes to f16 tiles
    reg_dealloc<kWidenRegs>();
    const int v = warp >= kWidenWarp + 4, quarter = warp & 3;  // of K or V; which 32 rows of a tile
    if (v && n_kv > 0) {
      // a thread per row of the MMAs
      const int thread = threadIdx.x - 32 * (kWidenWarp + 4), in_unit = thread & (unit_rows - 1);
      const bool live = in_unit < items;
      const int item = S.unit.item0 + (live ? in_unit : 0), token = item / P.group, head = key_head * P.group + item - token * P.group;
      const uint4* src = reinterpret_cast<const uint4*>(P.query + (static_cast<size_t>(S.unit.row0 + token) * P.heads + head) * kDim);
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint4 x = live ? src[c] : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
      }
      // of a row that is none, or nothing, any; one that leaves cap_scores its shortest way
      const uint32_t exponent = top == 0.f ? 127u : min(max(__float_as_uint(top) >> 23, 1u), 253u);
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
    // A lane's 16 bytes become two pieces of 16; eight lanes take as many rows, whose swizzles keep loads and stores apart.
    const int row = quarter * 16 + (lane & 7), piece = lane >> 3;  // and row + 8; piece and piece + 4
    const int from[2] = {row * kDim + ((piece ^ (lane & 7)) << 4), row * kDim + (((piece + 4) ^ (lane & 7)) << 4)};
    const int to[2] = {row * 128 + (((2 * piece) ^ (lane & 7)) << 4), row * 128 + (((2 * piece + 1) ^ (lane & 7)) << 4)};
    bool ok = true;
    for (int j = 0; ok && j < n_kv; ++j) {  // a tile of K is in ring stage 0 or 2, of V in 1 or 3
      const int st = (2 * j + v) % kStages;
      ok = j < 2 || rest(&S.kv_empty[st], ((j >> 1) - 1) & 1, kWaitTimeoutMma);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 2 * j + half, raw = i % kRawStages;
        ok = ok && rest(&S.raw_full[v][raw], (i / kRawStages) & 1, kWaitTimeoutLoad);
        if (!ok) break;
        uint4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const uint4*>(S.raw[v][raw] + from[k >> 1] + (k & 1) * 8 * kDim);
        const __half2 sign = S.sign[v][raw], base = __hmul2(sign, __float2half2_rn(-1152.f));
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.raw_empty[v][raw]);
        uint8_t* tile = S.kv[st] + half * kBlock * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint2 a = widen(x[k].x, sign, base), b = widen(x[k].y, sign, base), c = widen(x[k].z, sign, base), d = widen(x[k].w, sign, base);
          uint8_t* at = tile + (k >> 1) * kHalfBytes + (k & 1) * 8 * 128;
          *reinterpret_cast<uint4*>(at + to[0]) = make_uint4(a.x, a.y, b.x, b.y);
          *reinterpret_cast<uint4*>(at + to[1]) = make_uint4(c.x, c.y, d.x, d.y);
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
    auto softmax = [&](auto copies_constant) {
      constexpr int kCopies = decltype(copies_constant)::value, kRows = kTile / kCopies, kKeys = kBlock / kCopies;
      const int half = warp >> 2, quarter = warp & 3, in_unit = static_cast<int>(threadIdx.x) & (kRows - 1);
      const int part = quarter / (4 / kCopies) * kKeys;  // the first of this warp's keys in a block
      const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t s_addr = tmem + lane_base + kColS + kBlock * half + part, p_addr = tmem + lane_base + kColP + 32 * half;
      const uint32_t o_addr = tmem + lane_base + kColO + kDim * half;
      const bool live = in_unit < items;
      const int item = S.unit.item0 + (live ? in_unit : 0), token = item / P.group, head = key_head * P.group + item - token * P.group;
      const int first_key = kv_begin * kTile + kBlock * half + part;
      const int visible = S.unit.sight.visible(token) - first_key;
      const int partly = max(0, S.unit.sight.visible(S.unit.item0 / P.group) / kTile - kv_begin);
      [[maybe_unused]] const float slope = BIAS ? P.slopes[head] * 1.4426950408889634f : 0.f;
      [[maybe_unused]] const int position = BIAS ? S.unit.sight.ahead + token - first_key : 0;
      // a warp without live rows only keeps the others' pace: what its rows of P and O hold goes nowhere
      const bool idle = (quarter * 32 & (kRows - 1)) >= items;
      // The maximum is that of the probabilities times V's scale, which are what is rounded; the sum is relative to it too.
      float m_used = kLowestMaximum, sum = 0.f, row_scale = 0.f;
      bool ok = true;
      if constexpr (kCopies > 1) {  // the other copies' keys weigh nothing in this one
        uint32_t none[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) none[i] = 0;
        if (n_kv > 0) tmem_st32(p_addr, none), tc_wait_st();
      }
      for (int j = 0; j < n_kv; ++j) {
        const int block = 2 * j + half;
        ok = spin(&S.scales_full[block % kScaleSlots], (block / kScaleSlots) & 1, kWaitTimeoutLoad) && rest(&S.s_full, j & 1, kWaitTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        if (idle) {
          // no further ahead than the others: a second arrival in one phase would stand for theirs
          if (j > 0 && !(ok = rest(&S.pv_done[half], (j - 1) & 1, kWaitTimeoutMma))) break;
          if (lane == 0) mbar_arrive(&S.s_taken), mbar_arrive(&S.p_full[half]);
          continue;
        }
        uint32_t s[kKeys];
        if constexpr (kKeys == 16) {
          tmem_ld16(s_addr, s);
        } else {
#pragma unroll
          for (int c = 0; c < kKeys / 32; ++c) tmem_ld32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
        }
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.s_taken);
        if (j == 0) {
          row_scale = *const_cast<const volatile float*>(&S.factor[threadIdx.x & 127]) * P.scale;
          if (CAP) row_scale = fminf(row_scale, 1e30f);  // past the cap at any scale of K, and a score of 0 is not 0 x inf
        }
        const volatile float* kept = &S.scales[block % kScaleSlots].x;
        const float key_scale = kept[0] * row_scale, value_scale = kept[1];
        const bool there = value_scale != kNotThere;
        const int valid = visible - tile_at(j) * kTile;
        // from a raw score to log2 units; a capped or biased one is turned into them at once
        const float unit = CAP || BIAS ? 1.f : key_scale * P.to_log2;
        if constexpr (CAP) {
          const uint32_t least = __float_as_uint(kLeastNear);  // of positive numbers the order is that of their bits
          const bool ordinary = __float_as_uint(key_scale) - least <= __float_as_uint(kMostNear) - least;
          cap_scores(s, key_scale, P.to_log2, [&](float, float x) { return ordinary && x <= P.near; });
        }
        if constexpr (BIAS) {
          const float from = static_cast<float>(position - tile_at(j) * kTile), f = CAP ? 1.f : key_scale * P.to_log2;
#pragma unroll
          for (int i = 0; i < kKeys; ++i) s[i] = __float_as_uint(fmaf(__uint_as_float(s[i]), f, -slope * fabsf(from - static_cast<float>(i))));
        }
        if (tile_at(j) >= partly || !there) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (i >= valid || !there) s[i] = 0xff800000u;  // -inf
        }
        float a = __uint_as_float(s[0]), b = __uint_as_float(s[1]);
#pragma unroll
        for (int i = 2; i < kKeys - 2; i += 4) {
          a = max3(a, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          b = max3(b, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
        }
        const bool sees = there && valid > 0;  // a row that sees nothing of the keys takes nothing of them, whatever their scales are
        const float value_log2 = sees ? value_scale : 0.f;
        const float most = max3(a, b, fmaxf(__uint_as_float(s[kKeys - 2]), __uint_as_float(s[kKeys - 1])));
        // The largest exponent as the probabilities' are computed below: large scores and maxima are rounded by more than a unit.  Of a
        // row that sees nothing it is -inf, or NaN under a scale that is: neither raises the maximum.
        float offset = value_log2 - m_used;
        if (__any_sync(0xffffffffu, fmaf(most, unit, offset) > kLift + kRescaleThreshold)) {
          const float m_new = fmaxf(m_used, fmaf(most, unit, value_log2) - kLift);
          const float alpha = ex2(m_used - m_new);
          m_used = m_new;
          offset = value_log2 - m_used;
          if (j > 0) {  // P and O are untouched by the tensor core before the first PV
            sum *= alpha;
            ok = spin(&S.pv_done[half], (j - 1) & 1, kWaitTimeoutMma);
            if (!ok) break;
            tc_fence_after();
            tmem_scale_rows(o_addr, alpha);
          }
        }
        if (kCopies == 1 && j >= 1 - half && !(ok = rest(&S.turn[1 - half][quarter], (j - 1 + half) & 1, kWaitTimeoutSoftmax))) break;
        // Probabilities times V's scale at once: 2^(x + log2 scale - m), rounded to f16 for the value MMAs; the row sum is taken
        // before, and divided by the scale.
        const float f = sees ? unit : 1.f;
        const uint64_t unit2 = pack2(f, f), offset2 = pack2(offset, offset);
        uint64_t la = 0ull, lb = 0ull;
        uint32_t p[kKeys / 2];
#pragma unroll
        for (int i = 0; i < kKeys; i += 4) {
          float x0, x1, x2, x3;
          unpack2(fma2(pack2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), unit2, offset2), x0, x1);
          unpack2(fma2(pack2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), unit2, offset2), x2, x3);
          const float c = ex2(x0), d = ex2(x1), e = ex2(x2), g = ex2(x3);
          la = add2(la, pack2(c, d));
          lb = add2(lb, pack2(e, g));
          p[i / 2] = pack_f16(c, d);
          p[i / 2 + 1] = pack_f16(e, g);
        }
        if (kCopies == 1 && lane == 0) mbar_arrive(&S.turn[half][quarter]);
        float l0, l1, l2, l3;
        unpack2(la, l0, l1);
        unpack2(lb, l2, l3);
        sum = fmaf((l0 + l1) + (l2 + l3), ex2(-value_log2), sum);
        if (j > 0) {
          ok = spin(&S.pv_done[half], (j - 1) & 1, kWaitTimeoutMma);
          if (!ok) break;
          tc_fence_after();
        }
        if constexpr (kKeys == 64)
          tmem_st32(p_addr, p);
        else if constexpr (kKeys == 32)
          tmem_st16(p_addr + part / 2, p);
        else
          tmem_st8(p_addr + part / 2, p);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full[half]);
      }
      if (ok && n_kv > 0) ok = spin(&S.values_done, 0, kWaitTimeoutMma);
      if (!ok) return;
      // ---- join of the 2 kCopies parts of a row: every warp leaves its rows in the place of the tiles, whose last reader is done,
      // a row in 32 pieces of four channels, and puts out every eighth row of the unit
      if (n_kv > 0 && !idle) {
        tc_fence_after();
        float4* leave = reinterpret_cast<float4*>(S.kv[0]) + (warp * 32 + lane) * 32;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tc_wait_ld();
#pragma unroll
          for (int g = 0; g < 8; ++g)
            leave[8 * c + (g ^ (lane & 7))] = make_float4(__uint_as_float(o[4 * g]), __uint_as_float(o[4 * g + 1]),
                                                          __uint_as_float(o[4 * g + 2]), __uint_as_float(o[4 * g + 3]));
        }
        S.top[half][threadIdx.x & 127] = m_used, S.sum[half][threadIdx.x & 127] = sum;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.joined);
      if (!spin(&S.joined, 0, kWaitTimeoutSoftmax)) return;
      const size_t share = static_cast<size_t>(piece) * P.heads * P.rows;  // of divided keys
#pragma unroll 2
      for (int r = warp; r < min(items, kRows); r += 8) {
        float top = kLowestMaximum, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n_kv > 0) {
#pragma unroll
          for (int i = 0; i < 2 * kCopies; ++i) top = fmaxf(top, S.top[i & 1][r + (i >> 1) * kRows]);
#pragma unroll
          for (int i = 0; i < 2 * kCopies; ++i) {
            const int from = r + (i >> 1) * kRows;
            const float weight = ex2(S.top[i & 1][from] - top);
            const float4 x = (reinterpret_cast<const float4*>(S.kv[0]) + ((i & 1) * kTile + from) * 32)[lane ^ (r & 7)];
            l = fmaf(S.sum[i & 1][from], weight, l);
            o.x = fmaf(x.x, weight, o.x), o.y = fmaf(x.y, weight, o.y), o.z = fmaf(x.z, weight, o.z), o.w = fmaf(x.w, weight, o.w);
          }
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int at = S.unit.item0 + r, of = at / P.group, row = S.unit.row0 + of, own_head = key_head * P.group + at - of * P.group;
        if (!NOB_CHECK(row >= 0 && row < P.rows && own_head + P.head_offset < P.total_heads, status)) continue;
        if (P.splits > 1) {
          const size_t to = share + static_cast<size_t>(own_head) * P.rows + row;
          reinterpret_cast<float4*>(P.partial + to * kDim)[lane] = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
          if (lane == 0) P.lse[to] = top + log2f(l);
        } else {
          const size_t to = static_cast<size_t>(row) * P.total_heads + own_head + P.head_offset;
          reinterpret_cast<uint2*>(P.output + to * kDim)[lane] = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
        }
      }
    };
    if (items > 64)
      softmax(std::integral_constant<int, 1>());
    else if (items > 32)
      softmax(std::integral_constant<int, 2>());
    else if (items > 0)
      softmax(std::integral_constant<int, 4>());
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
                                 kBlock, 1, CU_TENSOR_MAP_SWIZZLE_128B)))
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
