// bf16 attention over packed documents for head_dim 128 on sm_100a: document, causal and prefix masks, scores capped by a
// tanh, a bias that grows with distance, query heads that share key heads.
//
//   s(i, j) = scale * q_i . k_j ;  capped: s = cap * tanh(s / cap) ;  biased: s -= slope[head] * |p_i - j|
//   o_i = sum_{j < visible(i)} softmax_j(s(i, j)) v_j,   p_i = i + keys - queries of the document
// Every mask leaves a row the first visible(i) keys of its document, so a row carries one number; a row that sees none gets
// zeros.  No counterpart in the reference, whose attention of this head width is neither masked nor ragged.
//
// One CTA owns a unit of 256 (or 128) query rows of one document and head and walks the key tiles of 128 that its last row
// sees; warps, TMEM columns, hand-overs and issue order are those of the dense kernel (fa_fwd_bf16.cu): two query tiles
// take turns at one score buffer, softmax with a thread per row, probabilities to the value MMAs through TMEM.  What the
// masks add:
//  * tiles that some row of the unit does not see whole are masked in registers, a compare and a select per score;
//  * rows of V behind the document's end (another document's, or anything at all) and rows of it that are not finite would
//    spoil rows that do not see them: 0 x NaN.  A warp walks the V tiles that are not seen whole before their value
//    MMAs start, zeroes such rows and notes the non-finite ones; a query row that does see one of those becomes NaN.
//  * capped scores: tanh by odd polynomials while all of a warp's rows stay within a third of the cap, or within the cap, else
//    by 1 - 2 / (1 + e^2x) on the MUFU (cap_scores).
// Bound by the softmax warps like the dense kernel, 3500 cycles per 256 rows x 128 keys of which the MMAs and the MUFU have 2048
// each, and under long loads by the power cap: 32768 causal rows x 14 heads 3.44-3.57 ms (1.08-1.12 PFLOP/s), 15104 with a distance
// bias 800-857 us, 9461 rows of nine documents 114-125 us (0.70-0.77), 4096 capped rows of three, 32 heads over 4, 136-137 us
// (107 without the cap).  Short documents pay a CTA's start and end, two to three tiles' time.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "documents.cuh"
#include "fa_common.cuh"
#include "tensor_map.cuh"
#include "../../include/nano_omni_b200.h"

namespace nob200 {
namespace {

constexpr int kTile = 128;
constexpr int kHalfBytes = kTile * 64 * 2;
constexpr int kTileBytes = 2 * kHalfBytes;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr float kLowestMaximum = -1e38f;   // relative to it a key of score -inf weighs 0
// SMALL: a CTA of one query tile, half of an SM's shared memory, TMEM and registers: two of them overlap one's start and end with
// the other's tiles (148 documents of 100 rows x 4 heads 44 us, one CTA to an SM 57; 592 of 4 rows 23, 38), which long key ranges
// pay for with 15 to 25 % (8192 rows x 14 heads 582 us, 491).  Its probabilities take the place of its scores, so a tile's scores wait
// for the value MMAs of the one before (those of the 64 keys whose columns are free issued at once: 2 % more, not less).
template <bool SMALL>
struct Form {
  static constexpr int kSoftmaxWarps = SMALL ? 4 : 8, kThreads = 32 * (kSoftmaxWarps + 4), kStages = SMALL ? 2 : 4;
  static constexpr int kProducerWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1, kCleanWarp = kSoftmaxWarps + 3;  // between: value MMAs
  static constexpr int kLaunchRegs = SMALL ? 128 : 168, kServiceRegs = SMALL ? 56 : 88;
  static constexpr int kSoftmaxRegs = (kThreads * kLaunchRegs - 128 * kServiceRegs) / (32 * kSoftmaxWarps) / 8 * 8;
  static_assert(32 * kSoftmaxWarps * kSoftmaxRegs + 128 * kServiceRegs <= kThreads * kLaunchRegs, "setmaxnreg split exceeds the registers the CTA owns");
  static constexpr uint32_t kTmemCols = SMALL ? 256 : 512;
  static constexpr uint32_t kColS = 0, kColP = SMALL ? 0 : 128, kColO = SMALL ? 128 : 256;  // P_t at kColP + 64 t, O_t at kColO + 128 t
};

struct Unit {
  int row0, rows;        // first row, rows of the document from there on (0: no unit)
  int key0, query0;      // first key row of the document, first row of the unit within the document
  int kv_begin, kv_end;  // key tiles of this CTA
  Sight sight;
};

template <bool SMALL>
struct __align__(1024) Shared {
  using F = Form<SMALL>;
  uint8_t q[SMALL ? 1 : 2][kTileBytes];
  uint8_t kv[F::kStages][kTileBytes];
  uint64_t q_full;
  uint64_t kv_full[F::kStages];
  uint64_t kv_empty[F::kStages];
  uint64_t s_full[2];
  uint64_t s_taken[2];
  uint64_t p_full[2][2];
  uint64_t pv_done[2];
  uint64_t v_clean[2];  // an even / odd V tile has been looked through
  uint32_t bad[2][4];   // and these of its rows were not finite
  Unit unit;
  FindScratch<F::kThreads> find;
  __align__(16) uint8_t staging[F::kSoftmaxWarps][32 * 64];  // of the softmax warps: 64 bytes of each of their rows
  uint32_t tmem_base;
  uint32_t abort;
  uint32_t qk_issued;
};

struct MaskedParams {
  const int* bounds;
  const int* key_bounds;
  const int* prefix;    // or NULL
  const float* slopes;  // BIAS form
  __nv_bfloat16* output;
  float* partial;  // of KeyShares, when the keys are divided
  float* lse;
  uint32_t* status;
  int rows, key_rows, documents, heads, group, total_heads, head_offset;
  int unit_rows, splits, causal;
  float scale;    // of a raw score; CAP form: divided by the cap
  float to_log2;  // from a raw or capped score to log2 units
  float near;     // near_scores
};

// The unit of this CTA, into shared memory.
template <bool SMALL>
__device__ __forceinline__ void find_own_unit(const MaskedParams& P, Shared<SMALL>& S, int slot, int piece) {
  struct Document {
    int2 rows, keys;
    int prefix, units, weight;
  };
  find_unit<Form<SMALL>::kThreads, true>(
      P.documents, slot, S.find,
      [&](int d, bool live) {
        Document r = {};
        if (live) {
          r.keys = document_rows(P.key_bounds, d, P.key_rows);
          r.prefix = P.prefix ? P.prefix[d] : 0;
          r.rows = document_rows(P.bounds, d, P.rows);
          r.units = (r.rows.y - r.rows.x + P.unit_rows - 1) / P.unit_rows;
          r.weight = r.keys.y - r.keys.x;
        }
        return r;
      },
      [&](const Document& r, int, int index) {
        Unit u;
        u.query0 = index * P.unit_rows;
        u.row0 = r.rows.x + u.query0;
        u.rows = r.rows.y - u.row0;
        u.key0 = r.keys.x;
        u.sight.keys = r.keys.y - r.keys.x;
        u.sight.ahead = u.sight.keys - (r.rows.y - r.rows.x);
        u.sight.prefix = r.prefix;
        u.sight.causal = P.causal != 0;
        const int seen = u.sight.visible(u.query0 + min(u.rows, P.unit_rows) - 1);
        const int tiles = (seen + kTile - 1) / kTile;
        u.kv_begin = static_cast<int>(static_cast<long long>(tiles) * piece / P.splits);
        u.kv_end = static_cast<int>(static_cast<long long>(tiles) * (piece + 1) / P.splits);
        S.unit = u;
      });
}

template <bool CAP, bool BIAS, bool SMALL>
__global__ void __launch_bounds__(Form<SMALL>::kThreads, SMALL ? 2 : 1)
fa_fwd_masked_bf16_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const MaskedParams P) {
  extern __shared__ uint8_t smem_raw[];
  using F = Form<SMALL>;
  constexpr int kStages = F::kStages, kProducerWarp = F::kProducerWarp, kMmaWarp = F::kMmaWarp, kCleanWarp = F::kCleanWarp;
  constexpr uint32_t kColS = F::kColS, kColP = F::kColP, kColO = F::kColO;
  Shared<SMALL>& S = *reinterpret_cast<Shared<SMALL>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  volatile uint32_t* abort_flag = &S.abort;
  uint32_t* status = P.status;

  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&S.kv_full[s], 1);
      mbar_init(&S.kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&S.s_full[t], 1);
      mbar_init(&S.s_taken[t], 4);
      mbar_init(&S.p_full[t][0], 4);
      mbar_init(&S.p_full[t][1], 4);
      mbar_init(&S.pv_done[t], 1);
      mbar_init(&S.v_clean[t], 1);
    }
    S.unit = Unit{};
    S.abort = 0;
    S.qk_issued = 0;
    mbar_fence_init();
  }
  if (warp == kProducerWarp) {
    tmem_alloc(&S.tmem_base, F::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();  // launched as a programmatic dependent: the set-up above overlaps the kernel before
  // All heads of a unit are neighbours in the grid, and the units with the longest key ranges come first: the short ones are
  // left for its end (8192 causal rows x 14 heads 341 us head by head, so 270).
  const int piece = static_cast<int>(blockIdx.x % P.splits), place = static_cast<int>(blockIdx.x / P.splits);
  const int head = place % P.heads;
  find_own_unit(P, S, place / P.heads, piece);
  const uint32_t tmem = S.tmem_base;
  pdl_release();

  const int unit_rows = min(S.unit.rows, P.unit_rows);  // 0: no unit
  const int n_kv = S.unit.kv_end - S.unit.kv_begin;
  const int kv_begin = S.unit.kv_begin;
  const bool two = !SMALL && unit_rows > kTile;
  // The order of the key tiles: a distance bias makes the nearest ones the largest, so they come first, from the last row's own
  // backwards, then the ones ahead.  (From the first key on, steep slopes raised the maximum with every tile: 15104 causal rows x
  // 14 heads 1065 us, so 821.)
  const int nearest = BIAS ? clamped((S.unit.sight.ahead + S.unit.query0 + unit_rows - 1) / kTile - kv_begin, 0, n_kv - 1) : -1;
  auto tile_at = [&](int j) { return j <= nearest ? nearest - j : j; };
  // key tiles from this one on (of this CTA's) are not seen whole by the unit's first row
  const int partly = max(0, S.unit.sight.visible(S.unit.query0) / kTile - kv_begin);

  if (warp >= F::kSoftmaxWarps) {
    reg_dealloc<F::kServiceRegs>();
    auto note_bounds = [&] {  // beside the others' work; at the start or at the end as the form's registers like it (1 to 2 %)
      if (warp == kCleanWarp && blockIdx.x == 0)
        note_documents(lane, P.documents, 32, status,
                       [&](int d) { return (P.bounds[d] <= P.bounds[d + 1]) & (P.key_bounds[d] <= P.key_bounds[d + 1]); });
    };
    if (SMALL) note_bounds();
    if (n_kv == 0) {
    } else if (warp == kProducerWarp) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        const int key_head = head / P.group, row0 = S.unit.row0, key0 = S.unit.key0;
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
        mbar_expect_tx(&S.q_full, two ? 2 * kTileBytes : kTileBytes);
        tma_load_3d(S.q[0], &map_q, &S.q_full, 0, head, row0);
        tma_load_3d(S.q[0] + kHalfBytes, &map_q, &S.q_full, 64, head, row0);
        if (two) {
          tma_load_3d(S.q[SMALL ? 0 : 1], &map_q, &S.q_full, 0, head, row0 + kTile);
          tma_load_3d(S.q[SMALL ? 0 : 1] + kHalfBytes, &map_q, &S.q_full, 64, head, row0 + kTile);
        }
        const int loads = 2 * n_kv;  // K_j at 2j, V_j at 2j+1
        int issued = 0;
        for (int i = 0; i < loads; ++i) {
          const int st = i % kStages;
          if (i >= kStages) {
            if (!mbar_wait(&S.kv_empty[st], ((i / kStages) - 1) & 1, abort_flag, status, kWaitTimeoutRing)) break;
          }
          mbar_expect_tx(&S.kv_full[st], kTileBytes);
          const CUtensorMap* map = (i & 1) ? &map_v : &map_k;
          const int token = key0 + (kv_begin + tile_at(i >> 1)) * kTile;
          tma_load_3d(S.kv[st], map, &S.kv_full[st], 0, key_head, token);
          tma_load_3d(S.kv[st] + kHalfBytes, map, &S.kv_full[st], 64, key_head, token);
          issued = i + 1;
        }
        if (*abort_flag) {
          // Gave up: let the copies already in flight land before the CTA exits.
          for (int i = (issued > kStages ? issued - kStages : 0); i < issued; ++i) {
            uint64_t* bar = &S.kv_full[i % kStages];
            const uint32_t parity = (i / kStages) & 1;
            for (int spin = 0; spin < (1 << 16) && !mbar_try_wait(bar, parity); ++spin) {
            }
          }
        }
      }
    } else if (warp == kCleanWarp) {
      // ---------------------------------------------- V rows that must not reach the value MMAs
      // Every tile in turn, and the value MMAs wait for it: a wait that skipped some phases of a barrier could not tell them apart.
      for (int j = 0; j < n_kv; ++j) {
        const int st = (2 * j + 1) % kStages, which = j & 1;
        if (!warp_rest(&S.kv_full[st], ((2 * j + 1) / kStages) & 1, abort_flag, status, kWaitTimeoutLoad)) break;
        const int tile = tile_at(j), left = S.unit.sight.keys - (kv_begin + tile) * kTile;  // rows of the tile that belong to the document
        bool wrote = false;
#pragma unroll 1
        for (int k = 0; k < 4 && tile >= partly; ++k) {
          const int row = 32 * k + lane;
          uint8_t* at[2] = {S.kv[st] + row * 128, S.kv[st] + kHalfBytes + row * 128};
          // x * 0 is NaN for a value that is not finite, else 0
          __nv_bfloat162 seen[4];
          const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) seen[i] = zero;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(at[c >> 3] + (((c + lane) & 7) << 4));
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) seen[i] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), zero, seen[i]);
          }
          const __nv_bfloat162 all = __hadd2(__hadd2(seen[0], seen[1]), __hadd2(seen[2], seen[3]));
          const bool finite = __low2float(all) == 0.f && __high2float(all) == 0.f;
          const bool outside = row >= left;
          const uint32_t bad = __ballot_sync(0xffffffffu, !finite && !outside);
          if (lane == 0) S.bad[which][k] = bad;
          if (outside || !finite) {
            wrote = true;
#pragma unroll
            for (int c = 0; c < 16; ++c)
              *reinterpret_cast<uint4*>(at[c >> 3] + (((c + lane) & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
        }
        if (__any_sync(0xffffffffu, wrote)) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.v_clean[which]);
      }
    } else {
      // --------------------------------------------------------- tcgen05 issuers, as in the dense kernel
      constexpr uint32_t idesc_qk = umma_idesc(kDF32, kFmtBF16, kFmtBF16, 0, 0, kTile, kTile);
      constexpr uint32_t idesc_pv = umma_idesc(kDF32, kFmtBF16, kFmtBF16, 0, 1, kTile, 128);
      auto full_parity = [](int i) { return (uint32_t)((i / kStages) & 1); };
      auto spin = [&](uint64_t* bar, uint32_t parity, uint32_t bit) { return warp_poll(bar, parity, abort_flag, status, bit); };
      auto rest = [&](uint64_t* bar, uint32_t parity, uint32_t bit) { return warp_rest(bar, parity, abort_flag, status, bit); };
      if (warp == kMmaWarp) {
        const uint64_t desc_k_major = umma_smem_desc(0, 16, 1024, kSwizzle128B);
        const uint64_t q_desc[2] = {desc_k_major + (smem_u32(S.q[0]) >> 4), desc_k_major + (smem_u32(S.q[SMALL ? 0 : 1]) >> 4)};
        const uint64_t kv_k_desc = desc_k_major + (smem_u32(S.kv[0]) >> 4);
        const uint32_t d = tmem + kColS;
        uint32_t issued = 0;
        auto qk = [&](int t, int j, uint64_t* taken, uint32_t taken_parity) -> bool {  // S = Q_t K_j^T
          const int ik = 2 * j, sk = ik % kStages;
          const uint64_t a0 = t ? q_desc[1] : q_desc[0], b0 = kv_k_desc + sk * (kTileBytes >> 4);
          const uint64_t a1 = a0 + 2, a2 = a0 + 4, a3 = a0 + 6, a4 = a0 + (kHalfBytes >> 4), a5 = a4 + 2, a6 = a4 + 4, a7 = a4 + 6;
          const uint64_t b1 = b0 + 2, b2 = b0 + 4, b3 = b0 + 6, b4 = b0 + (kHalfBytes >> 4), b5 = b4 + 2, b6 = b4 + 4, b7 = b4 + 6;
          if (t == 0 && !rest(&S.kv_full[sk], full_parity(ik), kWaitTimeoutLoad)) return false;
          if (taken && !spin(taken, taken_parity, kWaitTimeoutSoftmax)) return false;
          tc_fence_after();
          if (elect_one()) {
            asm volatile(
                "{\n\t.reg .pred p0, p1;\n\t"
                "setp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %2, %10, %1, p0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %3, %11, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %4, %12, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %5, %13, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %6, %14, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %7, %15, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %8, %16, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], %9, %17, %1, p1;\n\t}" ::"r"(d),
                "r"(idesc_qk), "l"(a0), "l"(a1), "l"(a2), "l"(a3), "l"(a4), "l"(a5), "l"(a6), "l"(a7), "l"(b0), "l"(b1),
                "l"(b2), "l"(b3), "l"(b4), "l"(b5), "l"(b6), "l"(b7)
                : "memory");
            tc_commit(&S.s_full[t]);
            if (t == 1 || !two) tc_commit(&S.kv_empty[sk]);  // last reader of K_j
            *reinterpret_cast<volatile uint32_t*>(&S.qk_issued) = issued + 1;
          }
          ++issued;
          return true;
        };
        bool ok = rest(&S.q_full, 0, kWaitTimeoutLoad) && qk(0, 0, nullptr, 0);
        for (int j = 0; ok && j < n_kv; ++j) {
          if (two && !(ok = qk(1, j, &S.s_taken[0], j & 1))) break;
          if (j + 1 < n_kv && !(ok = qk(0, j + 1, SMALL ? &S.pv_done[0] : &S.s_taken[two ? 1 : 0], j & 1))) break;
        }
      } else {
        const uint64_t desc_n_major = umma_smem_desc(0, kHalfBytes, 1024, kSwizzle128B);
        const uint64_t kv_n_desc = desc_n_major + (smem_u32(S.kv[0]) >> 4);
        const uint32_t total_qk = (two ? 2 : 1) * n_kv;
        // O_t += P_t(j)[:, 64 half : 64 half + 64] V_j[64 half : 64 half + 64, :], after `gate` score groups
        auto pv_half = [&](int t, int j, int half, uint32_t gate) -> bool {
          const int iv = 2 * j + 1, sv = iv % kStages;
          const uint64_t b0 = kv_n_desc + sv * (kTileBytes >> 4) + half * (4 * 2048 >> 4);
          const uint64_t b1 = b0 + (2048 >> 4), b2 = b0 + 2 * (2048 >> 4), b3 = b0 + 3 * (2048 >> 4);
          const uint32_t d = tmem + kColO + t * kTile, a0 = tmem + kColP + t * 64 + half * 32;
          const uint32_t accumulate = (j > 0 || half > 0) ? 1u : 0u;
          if (gate > total_qk) gate = total_qk;
          if (half == 0 && !rest(&S.kv_full[sv], full_parity(iv), kWaitTimeoutLoad)) return false;
          if (half == 0 && !rest(&S.v_clean[j & 1], (j >> 1) & 1, kWaitTimeoutLoad)) return false;
          if (!spin(&S.p_full[t][half], j & 1, kWaitTimeoutSoftmax)) return false;
          if (!warp_wait_counter(&S.qk_issued, gate, abort_flag, status, kWaitTimeoutMma)) return false;
          tc_fence_after();
          if (elect_one()) {
            asm volatile(
                "{\n\t.reg .pred p0, p1;\n\t"
                "setp.ne.b32 p0, %2, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], [%3], %7, %1, p0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], [%4], %8, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], [%5], %9, %1, p1;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], [%6], %10, %1, p1;\n\t}" ::"r"(d),
                "r"(idesc_pv), "r"(accumulate), "r"(a0), "r"(a0 + 8), "r"(a0 + 16), "r"(a0 + 24), "l"(b0), "l"(b1), "l"(b2),
                "l"(b3)
                : "memory");
            if (half == 1) {
              tc_commit(&S.pv_done[t]);
              if (t == 1 || !two) tc_commit(&S.kv_empty[sv]);  // last reader of V_j
            }
          }
          return true;
        };
        bool ok = true;
        if (two) {
          for (int j = 0; ok && j < n_kv; ++j) {
            ok = pv_half(0, j, 0, 2 * j + 3) && pv_half(0, j, 1, 2 * j + 4) && pv_half(1, j, 0, 2 * j + 4) &&
                 pv_half(1, j, 1, 2 * j + 5);
          }
        } else {
          for (int j = 0; ok && j < n_kv; ++j) ok = pv_half(0, j, 0, SMALL ? 0 : j + 2) && pv_half(0, j, 1, SMALL ? 0 : j + 2);
        }
      }
    }
    if (!SMALL) note_bounds();
  } else {
    // ------------------------------------------------- softmax + epilogue warps
    reg_alloc<F::kSoftmaxRegs>();
    auto poll = [&](uint64_t* bar, uint32_t parity, uint32_t bit) { return warp_poll(bar, parity, abort_flag, status, bit); };
    const int t = warp >> 2;
    if (unit_rows > 0 && (t == 0 || two)) {
      const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + lane_base + kColS;
      const uint32_t p_addr = tmem + lane_base + kColP + t * 64;
      const uint32_t o_addr = tmem + lane_base + kColO + t * kTile;
      const int query = S.unit.query0 + t * kTile + (warp & 3) * 32 + lane;
      const int visible = S.unit.sight.visible(query) - kv_begin * kTile;  // keys of this CTA's that the row sees
      const float unit_log2 = CAP ? 1.f : P.to_log2;  // from a raw score to log2 units; capped ones are turned into them at once
      const float slope = !BIAS ? 0.f : CAP ? P.slopes[head] * 1.4426950408889634f : P.slopes[head] / P.scale;  // in units of a score
      const int position = BIAS ? S.unit.sight.ahead + query - kv_begin * kTile : 0;  // relative to this CTA's first key
      float m_used = 0.f;
      uint64_t la = 0ull, lb = 0ull;  // four partial row sums as two fp32 pairs
      bool ok = true;
      for (int j = 0; j < n_kv; ++j) {
        ok = warp_rest(&S.s_full[t], j & 1, abort_flag, status, kWaitTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.s_taken[t]);
        if constexpr (CAP) cap_scores(s, P.scale, P.to_log2, [&](float top, float) { return top <= P.near; });
        [[maybe_unused]] float row_base = 0.f;
        if constexpr (BIAS) {
          const int key = tile_at(j) * kTile;
          const int first = __shfl_sync(0xffffffffu, position, 0);  // of the warp's rows
          const bool below = key + kTile - 1 <= first, above = key >= first + 31;
          if (below || above) {
            // All keys on one side of all rows: the distance is linear in the key, and the same for all rows but for a summand,
            // which joins the maximum; the slope is in units of a raw score, so that a key costs one fma with its number as an
            // immediate (821 us of the 15104 rows above with packed pairs of keys, so 761).
            const float step = below ? slope : -slope;
            row_base = step * static_cast<float>(key - position);
#pragma unroll
            for (int i = 0; i < 128; ++i) s[i] = __float_as_uint(fmaf(step, static_cast<float>(i), __uint_as_float(s[i])));
          } else {
            const float from = static_cast<float>(position - key);
#pragma unroll
            for (int i = 0; i < 128; ++i) s[i] = __float_as_uint(fmaf(-slope, fabsf(from - static_cast<float>(i)), __uint_as_float(s[i])));
          }
          row_base *= unit_log2;
        }
        if (tile_at(j) >= partly && __any_sync(0xffffffffu, visible < (tile_at(j) + 1) * kTile)) {
          const int valid = visible - tile_at(j) * kTile;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= valid) s[i] = 0xff800000u;  // -inf
        }
        float mx0 = __uint_as_float(s[0]), mx1 = __uint_as_float(s[1]);
        float mx2 = __uint_as_float(s[2]), mx3 = __uint_as_float(s[3]);
#pragma unroll
        for (int i = 4; i < 124; i += 8) {
          mx0 = max3(mx0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          mx1 = max3(mx1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
          mx2 = max3(mx2, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
          mx3 = max3(mx3, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
        }
        mx0 = max3(mx0, __uint_as_float(s[124]), __uint_as_float(s[125]));
        mx1 = max3(mx1, __uint_as_float(s[126]), __uint_as_float(s[127]));
        const float mx = BIAS ? fmaf(fmaxf(max3(mx0, mx1, mx2), mx3), unit_log2, row_base) : fmaxf(max3(mx0, mx1, mx2), mx3) * unit_log2;
        bool pv_waited = j == 0;  // P_t and O_t are untouched by the tensor core before the first PV
        if (j == 0) {
          m_used = fmaxf(mx, kLowestMaximum);
        } else if (__any_sync(0xffffffffu, mx > m_used + kRescaleThreshold)) {
          const float m_new = fmaxf(m_used, mx);
          const float alpha = ex2(m_used - m_new);
          const uint64_t alpha2 = pack2(alpha, alpha);
          la = fma2(la, alpha2, 0ull);
          lb = fma2(lb, alpha2, 0ull);
          // O_t += P_t V_{j-1} must have completed; the next PV waits for our arrival on p_full.
          ok = poll(&S.pv_done[t], (j - 1) & 1, kWaitTimeoutMma);
          if (!ok) break;
          pv_waited = true;
          tc_fence_after();
          tmem_scale_rows(o_addr, alpha);
          m_used = m_new;
        }
        if (tile_at(j) >= partly) {
          // which of the tile's rows of V were not finite; before the probabilities go, as the note is overwritten after them
          ok = poll(&S.v_clean[j & 1], (j >> 1) & 1, kWaitTimeoutLoad);
          if (!ok) break;
          const int valid = visible - tile_at(j) * kTile;
          uint32_t bad = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int seen = clamped(valid - 32 * k, 0, 32);
            bad |= *const_cast<const volatile uint32_t*>(&S.bad[j & 1][k]) & (seen == 32 ? ~0u : (1u << seen) - 1u);
          }
          if (bad) la = ~0ull;  // the row sees one: its sum, and with it the row, is not a number
        }
        const uint64_t scale2 = pack2(unit_log2, unit_log2);
        const float neg_m = BIAS ? row_base - m_used : -m_used;
        const uint64_t neg_m2 = pack2(neg_m, neg_m);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            const int e = half * 64 + i;
            float x0, x1, x2, x3;
            unpack2(fma2(pack2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, neg_m2), x0, x1);
            unpack2(fma2(pack2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), scale2, neg_m2), x2, x3);
            const float a = ex2(x0), b = ex2(x1), c = ex2(x2), d = ex2(x3);
            la = add2(la, pack2(a, b));
            lb = add2(lb, pack2(c, d));
            // probabilities go to bf16 for the value MMAs, as V is; the row sum is taken before the rounding
            p[i / 2] = pack_bf16(a, b);
            p[i / 2 + 1] = pack_bf16(c, d);
          }
          if (half == 0 && !pv_waited) {
            // the previous tile's PV still reads P_t until this completes (normally long ago)
            ok = poll(&S.pv_done[t], (j - 1) & 1, kWaitTimeoutMma);
            if (!ok) break;
            tc_fence_after();
          }
          tmem_st32(p_addr + 32 * half, p);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&S.p_full[t][half]);
        }
        if (!ok) break;
      }
      if (ok && n_kv > 0) ok = poll(&S.pv_done[t], (n_kv - 1) & 1, kWaitTimeoutMma);
      if (ok) {
        tc_fence_after();
        float l0, l1, l2, l3;
        unpack2(la, l0, l1);
        unpack2(lb, l2, l3);
        const float l = (l0 + l1) + (l2 + l3);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int in_unit = t * kTile + (warp & 3) * 32 + lane, row = S.unit.row0 + in_unit;
        const bool live = NOB_CHECK(in_unit >= S.unit.rows || (row >= 0 && row < P.rows && head + P.head_offset < P.total_heads), status) &&
                          in_unit < S.unit.rows;
        const size_t share = static_cast<size_t>(piece) * P.heads + head;  // of divided keys
        if (P.splits > 1 && live) P.lse[share * P.rows + row] = m_used + log2f(l);
        // Rows leave through shared memory, 64 bytes of each at a time, so that four lanes write one row's piece: a lane per row
        // touches 32 lines with every store (packed documents 140 us, so 128).
        uint8_t* mine = S.staging[warp];
        const uint32_t rows_live = __ballot_sync(0xffffffffu, live);
        uint4 part[4];
        auto flush = [&](int byte) {  // `part`, the bytes from `byte` on of every lane's row
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(mine + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4)) = part[g];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + (lane >> 2);
            if (!(rows_live >> r & 1)) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(mine + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
            const size_t to = row - lane + r;
            char* dst = P.splits > 1 ? reinterpret_cast<char*>(P.partial) + (share * P.rows + to) * 512
                                     : reinterpret_cast<char*>(P.output) + (to * P.total_heads + head + P.head_offset) * 256;
            *reinterpret_cast<uint4*>(dst + byte + 16 * (lane & 3)) = x;
          }
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          if (n_kv > 0) {
            tmem_ld32(o_addr + 32 * c, o);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          auto value = [&](int i) { return __uint_as_float(o[i]) * inv; };
          if (P.splits > 1) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const int i = 16 * k + 4 * g;
                part[g] = make_uint4(__float_as_uint(value(i)), __float_as_uint(value(i + 1)), __float_as_uint(value(i + 2)),
                                     __float_as_uint(value(i + 3)));
              }
              flush(128 * c + 64 * k);
            }
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int i = 8 * g;
              part[g] = make_uint4(pack_bf16(value(i), value(i + 1)), pack_bf16(value(i + 2), value(i + 3)),
                                   pack_bf16(value(i + 4), value(i + 5)), pack_bf16(value(i + 6), value(i + 7)));
            }
            flush(64 * c);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) tmem_dealloc(tmem, F::kTmemCols);
}

// o = sum_z 2^(lse_z - max) o_z / sum_z 2^(lse_z - max).  A thread owns eight channels of a row and every LANES-th share of it, so
// that many shares of few rows are not read one after the other (42 shares of 14 rows: 12 us by one thread each).  A row that
// no share gave any weight gets zeros.
template <int LANES>
__global__ void __launch_bounds__(256)
join_shares_kernel(const KeyShares P) {
  __shared__ float tops[16], sums[16];
  __shared__ float parts[LANES > 1 ? 256 : 1][8];
  pdl_wait();
  const int group = threadIdx.x >> 4, piece = threadIdx.x & 15, lane = group % LANES;  // a group: one row, one set of shares
  const long long all = static_cast<long long>(P.heads) * P.rows;
  const long long place = blockIdx.x * static_cast<long long>(16 / LANES) + group / LANES;
  const int head = static_cast<int>(place / P.rows), row = static_cast<int>(place - static_cast<long long>(head) * P.rows);
  const bool live = place < all && row >= P.bounds[0] && row < P.bounds[P.documents];
  float top = -INFINITY;
  if (live)
    for (int z = lane; z < P.splits; z += LANES) top = fmaxf(top, P.lse[z * all + place]);
  if (LANES > 1) {
    if (piece == 0) tops[group] = top;
    __syncthreads();
#pragma unroll
    for (int l = 0; l < LANES; ++l) top = fmaxf(top, tops[group - lane + l]);
  }
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  float sum = 0.f;
  if (live)
    for (int z = lane; z < P.splits; z += LANES) {
      const long long at = z * all + place;
      const float4* src = reinterpret_cast<const float4*>(P.partial + at * 128 + piece * 8);
      const float4 x = src[0], y = src[1];
      const float lse = P.lse[at];
      if (lse == -INFINITY) continue;
      const float w = exp2f(lse - top);
      sum += w;
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += w * v[i];
    }
  if (LANES > 1) {
    if (piece == 0) sums[group] = sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) parts[threadIdx.x][i] = acc[i];
    __syncthreads();
    if (lane > 0) return;
#pragma unroll
    for (int l = 1; l < LANES; ++l) {
      sum += sums[group + l];
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += parts[threadIdx.x + 16 * l][i];
    }
  }
  if (!live) return;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  uint4 v;
  v.x = pack_bf16(acc[0] * inv, acc[1] * inv);
  v.y = pack_bf16(acc[2] * inv, acc[3] * inv);
  v.z = pack_bf16(acc[4] * inv, acc[5] * inv);
  v.w = pack_bf16(acc[6] * inv, acc[7] * inv);
  *reinterpret_cast<uint4*>(P.output + (static_cast<size_t>(row) * P.total_heads + head + P.head_offset) * 128 + piece * 8) = v;
}

}  // namespace

int launch_join_shares(const KeyShares& shares, void* stream) {
  const int lanes = shares.splits <= 4 ? 1 : shares.splits <= 16 ? 4 : 16;
  const long long rows = static_cast<long long>(shares.rows) * shares.heads;
  auto kernel = lanes == 1 ? join_shares_kernel<1> : lanes == 4 ? join_shares_kernel<4> : join_shares_kernel<16>;
  return launch_pdl("attention (join of key shares)", kernel, static_cast<unsigned>((rows * lanes + 15) / 16), 256, 0, stream, shares);
}

}  // namespace nob200

extern "C" size_t nob200_masked_bf16_attention_d128_workspace_bytes(int num_rows, int heads, int kv_splits) {
  return num_rows <= 0 || heads <= 0 ? 0 : nob200::key_shares_bytes(num_rows, heads, kv_splits);
}

extern "C" int nob200_masked_bf16_attention_d128(int num_rows, int num_key_rows, int documents, int head_offset,
                                                 const void* query, const void* key, const void* value, const void* bounds,
                                                 const void* key_bounds, const void* prefix, const void* slopes,
                                                 void* output, int heads, int kv_heads, int total_heads, int causal,
                                                 float scale, float cap, int unit_rows, int kv_splits, void* workspace,
                                                 size_t workspace_bytes, void* stream) {
  using namespace nob200;
  const char* name = "masked_bf16_attention_d128";
  NOB_REQUIRE(num_rows > 0 && num_key_rows > 0 && documents > 0 && heads > 0 && kv_heads > 0 && total_heads > 0,
              "%s: sizes must be positive", name);
  NOB_REQUIRE(heads % kv_heads == 0, "%s: %d heads cannot share %d key heads evenly", name, heads, kv_heads);
  NOB_REQUIRE(head_offset >= 0 && head_offset <= total_heads - heads, "%s: head_offset %d outside [0, %d]", name,
              head_offset, total_heads - heads);
  NOB_REQUIRE(query && key && value && bounds && key_bounds && output, "%s: NULL tensor", name);
  NOB_REQUIRE(reinterpret_cast<uintptr_t>(output) % 16 == 0, "%s: output %p is not 16-byte aligned", name, output);
  NOB_REQUIRE(scale > 0.f && scale <= 1e30f, "%s: scale %g must be positive and finite", name, scale);
  NOB_REQUIRE(cap >= 0.f && cap <= 1e30f, "%s: cap %g must be finite, 0 for none", name, cap);
  NOB_REQUIRE(cap_fits(scale, cap), "%s: scale / cap must lie between 1e-35 and 1e35 (got %g / %g)", name, scale, cap);
  NOB_REQUIRE(!slopes || cap > 0.f || scale >= 1e-12f, "%s: slopes, which are divided by it, need a scale of 1e-12 or more (got %g)", name, scale);
  NOB_REQUIRE(unit_rows == kTile || unit_rows == 2 * kTile, "%s: unit_rows must be 128 or 256 (got %d)", name, unit_rows);
  NOB_REQUIRE(kv_splits >= 1 && kv_splits <= 64, "%s: kv_splits %d outside [1, 64]", name, kv_splits);
  const long long slots = most_units(num_rows, documents, unit_rows);
  const long long blocks = slots * heads * kv_splits;
  NOB_REQUIRE(blocks <= 0x7fffffffll, "%s: %lld units x %d heads x %d key shares exceed the grid limit", name, slots, heads, kv_splits);
  const size_t need = key_shares_bytes(num_rows, heads, kv_splits);
  NOB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
              "%s: %zu B of 16-byte aligned workspace required for %d key shares, %zu B given", name, need, kv_splits, workspace_bytes);

  MaskedParams P = {};
  P.status = status_word_device_ptr();
  if (!P.status) return fail(kCudaError, "%s: no current CUDA device", name);
  P.bounds = static_cast<const int*>(bounds), P.key_bounds = static_cast<const int*>(key_bounds);
  P.prefix = static_cast<const int*>(prefix), P.slopes = static_cast<const float*>(slopes);
  P.output = static_cast<__nv_bfloat16*>(output);
  P.rows = num_rows, P.key_rows = num_key_rows, P.documents = documents;
  P.heads = heads, P.group = heads / kv_heads, P.total_heads = total_heads, P.head_offset = head_offset;
  P.unit_rows = unit_rows, P.splits = kv_splits, P.causal = causal != 0;
  const float log2e = 1.4426950408889634f;
  P.scale = cap > 0.f ? scale / cap : scale;
  P.to_log2 = cap > 0.f ? cap * log2e : scale * log2e;
  P.near = near_scores(P.scale, P.to_log2);
  if (need) {
    P.partial = static_cast<float*>(workspace);
    P.lse = P.partial + static_cast<size_t>(kv_splits) * heads * num_rows * 128;
  }

  CUtensorMap mq, mk, mv;
  int rc;
  const uint64_t pitch = static_cast<uint64_t>(heads) * 256, key_pitch = static_cast<uint64_t>(kv_heads) * 256;
  if ((rc = make_tensor_map_3d(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, query, 128, heads, num_rows, 256, pitch, 64, 1, kTile)))
    return rc;
  if ((rc = make_tensor_map_3d(&mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, key, 128, kv_heads, num_key_rows, 256, key_pitch, 64, 1, kTile)))
    return rc;
  if ((rc = make_tensor_map_3d(&mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, value, 128, kv_heads, num_key_rows, 256, key_pitch, 64, 1, kTile)))
    return rc;

  // CTAs of one query tile share an SM once there are more of them than SMs (148, as the planner counts them); alone on it a tile's
  // scores need not wait
  const bool small = unit_rows == kTile && blocks > 148;
  auto launch = [&](auto small_form) -> int {
    constexpr bool kSmall = decltype(small_form)::value;
    auto kernel = cap > 0.f ? (slopes ? fa_fwd_masked_bf16_kernel<true, true, kSmall> : fa_fwd_masked_bf16_kernel<true, false, kSmall>)
                            : (slopes ? fa_fwd_masked_bf16_kernel<false, true, kSmall> : fa_fwd_masked_bf16_kernel<false, false, kSmall>);
    const size_t smem = sizeof(Shared<kSmall>) + 1024;
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess)
      return fail(kCudaError, "%s: cannot reserve %zu B of shared memory: %s", name, smem, cudaGetErrorString(err));
    return launch_pdl(name, kernel, static_cast<unsigned>(blocks), Form<kSmall>::kThreads, smem, stream, mq, mk, mv, P);
  };
  if ((rc = small ? launch(std::true_type()) : launch(std::false_type()))) return rc;
  if (kv_splits == 1) return kOk;
  return launch_join_shares({P.bounds, P.partial, P.lse, P.output, documents, num_rows, heads, total_heads, head_offset, kv_splits}, stream);
}
