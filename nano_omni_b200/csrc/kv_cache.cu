// A cache of keys and values in 8 bits: blocks of 64 tokens, int8 codes, one fp32 scale per block and head for each of K and V.
//
//   codes int8 [blocks, heads, 64, 128], scales f32 [blocks, heads]: value = code * scale
//   table int32 [sequences, max_blocks]: the block that holds tokens 64 b .. 64 b + 63 of a sequence; lengths int32 [sequences]
// No counterpart in the reference, whose quantised K and V are written once per attention (one scale per 64 keys as here).
//
// Append.  A block's scale is the largest magnitude it has seen times fp32(1 / 127).  A token that exceeds it raises the scale and what
// the block held is rounded again on the new grid: half a step more per raise, and of 64 tokens in random order only about
// ln 64 = 4 raise it.  The arithmetic (IEEE division and products, rounding to even) is fixed, so that codes do not depend on
// the launch.  A CTA owns one touched block of one head of K or of V: the new rows are read once into registers, their maximum
// is taken across the CTA, and their codes leave from the registers.
// Read.  The sequences' tokens as bf16 rows one behind the other, for kernels that take bf16 operands; a CTA per block and head.
// Both are bound by HBM: 15104 tokens x 14 heads appended in 31.7 us and read back in 31.0 (5.4 TB/s of the 6.55 of a copy); one
// token of 64 sequences x 8 heads by the latency of a launch and four dependent loads, 17 us for the two.
#include "common.cuh"
#include "documents.cuh"
#include "fa_common.cuh"
#include "../../include/nano_omni_b200.h"

namespace nob200 {
namespace {

constexpr int kBlock = 64, kDim = 128, kThreads = 256;
constexpr int kPieces = kBlock * kDim / 8 / kThreads;  // pieces of eight channels that a thread owns
constexpr int kAppendThreads = 128, kAppendRows = kAppendThreads / 16, kAppendPieces = kBlock / kAppendRows;
constexpr int kHeads = 4;                              // heads that a CTA of the read has under way

struct AppendParams {
  const __nv_bfloat16* source[2];  // new rows of K, V [rows, heads * 128]
  int8_t* codes[2];
  float* scales[2];
  const int* bounds;   // [sequences + 1] of the new rows
  const int* table;
  const int* lengths;  // with the new tokens
  uint32_t* status;
  int rows, sequences, max_blocks, num_blocks, heads, slots, each;  // each: heads of a CTA
};

// The codes of eight values, round(x / scale) to even of the correctly rounded quotient, as two words of four.  The quotient
// follows Markstein (IBM Journal of Research and Development 34, 1990): with y = 1 / b correctly rounded, q = a y,
// r = a - q b exact in an fma, q + r y is correctly rounded unless b's significand is all ones, for which the caller takes
// EXACT.  Half of a block's largest value is exactly between two codes, and common, so that quotients near the middle could
// not be left to a rare division (59 us for 15104 tokens x 14 heads with every value divided, 55 with those).  Adding
// 1.5 * 2^23 rounds to an integer, which is then the low byte.
template <bool EXACT>
__device__ __forceinline__ uint2 codes_of(const uint4& x, float scale, float inverse) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    float q;
    if (EXACT) {
      q = __fdiv_rn(a, scale);
    } else {
      q = __fmul_rn(a, inverse);
      q = __fmaf_rn(__fmaf_rn(-q, scale, a), inverse, q);
    }
    t[i] = __float_as_uint(__fadd_rn(q, 12582912.f));
  }
  auto four = [&](int i) { return __byte_perm(__byte_perm(t[i], t[i + 1], 0x0040), __byte_perm(t[i + 2], t[i + 3], 0x0040), 0x5410); };
  return make_uint2(four(0), four(4));
}
// Of two bf16 each, the larger magnitude; NaN if either is.
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  b &= 0x7fff7fffu;
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint2 pack_codes(const int8_t (&c)[8]) {
  uint2 r;
  r.x = static_cast<uint8_t>(c[0]) | static_cast<uint8_t>(c[1]) << 8 | static_cast<uint8_t>(c[2]) << 16 | static_cast<uint32_t>(static_cast<uint8_t>(c[3])) << 24;
  r.y = static_cast<uint8_t>(c[4]) | static_cast<uint8_t>(c[5]) << 8 | static_cast<uint8_t>(c[6]) << 16 | static_cast<uint32_t>(static_cast<uint8_t>(c[7])) << 24;
  return r;
}
// A code on the grid of another scale; of the magnitudes only 128 can leave the codes, on a grid that has turned.
__device__ __forceinline__ int8_t again(int code, float ratio) {
  return static_cast<int8_t>(__float2int_rn(fminf(__fmul_rn(static_cast<float>(code), ratio), 127.f)));
}
__device__ __forceinline__ int code_at(uint32_t word, int i) { return static_cast<int8_t>(word >> (8 * i)); }

__global__ void __launch_bounds__(kAppendThreads)
cache_append_kernel(const AppendParams P) {
  struct Sequence {
    int first, before, end, units, weight;  // first new row; tokens held before; with the new ones
  };
  __shared__ Sequence own;
  __shared__ int own_index[2];  // sequence, which of the blocks that it touches
  __shared__ FindScratch<kAppendThreads> scratch;
  __shared__ float most[2][kAppendThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = static_cast<int>(blockIdx.x) % P.slots, which = static_cast<int>(blockIdx.x) / P.slots;
  const int head0 = (which >> 1) * P.each, tensor = which & 1;
  if (threadIdx.x == 0) own_index[0] = -1;
  __syncthreads();
  pdl_wait();
  pdl_release();
  find_unit<kAppendThreads, false>(
      P.sequences, slot, scratch,
      [&](int d, bool live) {
        Sequence r = {};
        if (live) {
          r.end = P.lengths[d];
          const bool fit = bounds_fit(P.bounds, d, P.rows);
          r.first = P.bounds[d];
          const int fresh = P.bounds[d + 1] - r.first;  // of bounds that fit
          r.before = r.end - fresh;
          const bool right = fit && (fresh == 0 || (r.end >= fresh && r.end <= P.max_blocks * kBlock));
          r.units = right && fresh > 0 ? (r.end + kBlock - 1) / kBlock - r.before / kBlock : 0;
          if (!right) atomicOr(P.status, kBadIndex);  // bounds or a length that cannot be right: no rows of it are appended
        }
        return r;
      },
      [&](const Sequence& r, int d, int index) { own = r, own_index[0] = d, own_index[1] = index; });
  if (blockIdx.x == 0)  // sequences that no CTA may come to as it looks for its block
    note_documents(kAppendThreads + static_cast<int>(threadIdx.x), P.sequences, kAppendThreads, P.status,
                   [&](int d) { return bounds_fit(P.bounds, d, P.rows); });
  const int sequence = own_index[0];
  if (sequence < 0) return;
  const int place = own.before / kBlock + own_index[1], token0 = place * kBlock;
  const int row_of_token0 = own.first - own.before;  // row of the sequence's token 0, if it were among the new ones
  const int kept = clamped(own.before - token0, 0, kBlock);  // tokens that the block holds
  const int end = min(own.end - token0, kBlock);             // and will hold
  const int block = P.table[static_cast<size_t>(sequence) * P.max_blocks + place];
  if (block < 0 || block >= P.num_blocks) {
    if (threadIdx.x == 0) atomicOr(P.status, kBadIndex);
    return;
  }
  const int channel = (threadIdx.x & 15) * 8, first = threadIdx.x >> 4, last = min(head0 + P.each, P.heads);
  const __nv_bfloat16* source = (tensor ? P.source[1] : P.source[0]) + channel;
  int8_t* codes = (tensor ? P.codes[1] : P.codes[0]) + static_cast<size_t>(block) * P.heads * kBlock * kDim + channel;
  float* scales = (tensor ? P.scales[1] : P.scales[0]) + static_cast<size_t>(block) * P.heads;
  for (int head = head0; head < last; ++head) {
    uint4 x[kAppendPieces];  // eight new values, or in .x and .y the codes that are there
    const float old = kept ? scales[head] : 0.f;
    int8_t* mine = codes + (static_cast<size_t>(head) * kBlock + first) * kDim;
    const __nv_bfloat16* fresh = source + (static_cast<size_t>(row_of_token0 + token0 + first) * P.heads + head) * kDim;
    const size_t pitch = static_cast<size_t>(P.heads) * kDim * kAppendRows;
#pragma unroll
    for (int i = 0; i < kAppendPieces; ++i) {
      const int token = first + kAppendRows * i;
      x[i] = make_uint4(0, 0, 0, 0);
      if (token < kept) {
        const uint2 was = *reinterpret_cast<const uint2*>(mine + kAppendRows * kDim * i);
        x[i].x = was.x, x[i].y = was.y;
      } else if (token < end) {
        x[i] = *reinterpret_cast<const uint4*>(fresh + pitch * i);
      }
    }
    uint32_t pair = 0;
#pragma unroll
    for (int i = 0; i < kAppendPieces; ++i)
      if (first + kAppendRows * i >= kept) pair = larger(larger(larger(larger(pair, x[i].x), x[i].y), x[i].z), x[i].w);
    float top = max_nan(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));  // a value that is not a number shows
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    float* maxima = most[head & 1];  // the other half is still read by warps behind
    if (lane == 0) maxima[warp] = top;
    __syncthreads();  // also: everyone has read the old scale
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) top = max_nan(top, maxima[w]);
    const float scale = max_nan(fabsf(old), max_nan(__fmul_rn(top, 1.0f / 127.0f), 1e-10f));
    if (threadIdx.x == 0) scales[head] = scale;
    const float inverse = __frcp_rn(scale);
    const bool finite = scale <= 3.4e38f;  // else codes of 0, whose values are not numbers
    if ((__float_as_uint(scale) & 0x7fffffu) != 0x7fffffu) {
#pragma unroll
      for (int i = 0; i < kAppendPieces; ++i) {
        const int token = first + kAppendRows * i;
        if (token >= kept && token < end)
          *reinterpret_cast<uint2*>(mine + kAppendRows * kDim * i) = finite ? codes_of<false>(x[i], scale, inverse) : make_uint2(0, 0);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kAppendPieces; ++i) {
        const int token = first + kAppendRows * i;
        if (token >= kept && token < end)  // read once more: the copies are not to be indexed at run time
          *reinterpret_cast<uint2*>(mine + kAppendRows * kDim * i) =
              finite ? codes_of<true>(*reinterpret_cast<const uint4*>(fresh + pitch * i), scale, inverse) : make_uint2(0, 0);
      }
    }
    if (kept > 0 && scale != old) {  // the grid has grown, or turned from a negative one: what was there is rounded again
      const float ratio = __fdiv_rn(old, scale);
#pragma unroll
      for (int i = 0; i < kAppendPieces; ++i) {
        if (first + kAppendRows * i >= kept) continue;
        int8_t c[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          c[k] = again(code_at(x[i].x, k), ratio);
          c[4 + k] = again(code_at(x[i].y, k), ratio);
        }
        *reinterpret_cast<uint2*>(mine + kAppendRows * kDim * i) = pack_codes(c);
      }
    }
  }
}

struct ReadParams {
  const int8_t* codes[2];
  const float* scales[2];
  const int* table;
  const int* lengths;
  __nv_bfloat16* rows[2];  // [capacity, heads * 128]
  int* bounds;             // [sequences + 1]
  uint32_t* status;
  int capacity, sequences, max_blocks, num_blocks, heads, slots, each;  // each: heads of a CTA
};

__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const ReadParams P) {
  __shared__ int unit[4];  // sequence, block in it, output row of its first token, tokens of it to write
  __shared__ int blocks_of[kThreads / 32];
  __shared__ long long tokens_of[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = static_cast<int>(blockIdx.x) % P.slots, which = static_cast<int>(blockIdx.x) / P.slots;
  const int head0 = (which >> 1) * P.each, tensor = which & 1;
  if (threadIdx.x == 0) unit[0] = -1;
  __syncthreads();
  pdl_wait();
  pdl_release();
  // A sequence per thread, as in find_unit, with the rows before each as well; the first CTA walks all of them and notes where
  // each begins.
  const bool notes = blockIdx.x == 0;
  long long row = 0;
  int before = 0;
  for (int base = 0; base < P.sequences && (notes || before <= slot); base += kThreads) {
    const int s = base + static_cast<int>(threadIdx.x);
    const int given = s < P.sequences ? P.lengths[s] : 0;
    const int length = clamped(given, 0, P.max_blocks * kBlock), blocks = (length + kBlock - 1) / kBlock;
    int through = blocks;
    long long rows = length;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int b = __shfl_up_sync(0xffffffffu, through, o);
      const long long r = __shfl_up_sync(0xffffffffu, rows, o);
      if (lane >= o) through += b, rows += r;
    }
    if (lane == 31) blocks_of[warp] = through, tokens_of[warp] = rows;
    __syncthreads();
    int all_blocks = 0;
    long long all_rows = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) through += all_blocks, rows += all_rows;
      all_blocks += blocks_of[w], all_rows += tokens_of[w];
    }
    const long long until = row + rows;
    if (notes && s < P.sequences) {
      P.bounds[s + 1] = static_cast<int>(until < P.capacity ? until : P.capacity);
      if (s == 0) P.bounds[0] = 0;
      if (until > P.capacity || given != length) atomicOr(P.status, kBadIndex);
    }
    const int mine = slot - before;  // of this group's blocks
    if (mine >= through - blocks && mine < through) {
      const int b = mine - (through - blocks);
      const long long at = until - length + static_cast<long long>(b) * kBlock;
      if (at < P.capacity) {
        unit[0] = s, unit[1] = b, unit[2] = static_cast<int>(at);
        unit[3] = static_cast<int>(min(static_cast<long long>(min(length - b * kBlock, kBlock)), P.capacity - at));
      }
    }
    before += all_blocks, row += all_rows;
    __syncthreads();
  }
  const int sequence = unit[0];
  if (sequence < 0) return;
  const int end = unit[3];
  const int block = P.table[static_cast<size_t>(sequence) * P.max_blocks + unit[1]];
  const bool known = block >= 0 && block < P.num_blocks;
  if (!known && threadIdx.x == 0) atomicOr(P.status, kBadIndex);
  const int channel = (threadIdx.x & 15) * 8, first = threadIdx.x >> 4;
  const size_t from = known ? static_cast<size_t>(block) * P.heads : 0;
  const int8_t* codes = (tensor ? P.codes[1] : P.codes[0]) + from * (kBlock * kDim) + first * kDim + channel;
  const float* scales = (tensor ? P.scales[1] : P.scales[0]) + from;
  __nv_bfloat16* rows = (tensor ? P.rows[1] : P.rows[0]) + (static_cast<size_t>(unit[2]) + first) * P.heads * kDim + channel;
  const int last = min(head0 + P.each, P.heads);
  for (int some = head0; some < last; some += kHeads) {
    uint2 c[kHeads][kPieces];  // of a few heads, so that their loads are under way together
    float scale[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int head = min(some + h, last - 1);
      scale[h] = known ? scales[head] : 0.f;  // of a block that is not there: zeros
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        c[h][i] = first + 16 * i < end && some + h < last ? *reinterpret_cast<const uint2*>(codes + (static_cast<size_t>(head) * kBlock + 16 * i) * kDim)
                                                          : make_uint2(0, 0);
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        if (first + 16 * i >= end || some + h >= last) continue;
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // the product of 7 and 24 bits is rounded to fp32, then to bf16
          o[k] = pack_bf16(code_at(c[h][i].x, 2 * k) * scale[h], code_at(c[h][i].x, 2 * k + 1) * scale[h]);
          o[2 + k] = pack_bf16(code_at(c[h][i].y, 2 * k) * scale[h], code_at(c[h][i].y, 2 * k + 1) * scale[h]);
        }
        *reinterpret_cast<uint4*>(rows + (static_cast<size_t>(16 * i) * P.heads + some + h) * kDim) = make_uint4(o[0], o[1], o[2], o[3]);
      }
  }
}

// Heads of a CTA: finding the block is two loads' latency, so that a launch has some 1184 CTAs where heads can make it so (64
// short sequences x 8 heads read back in 12.9 us with a head each).  An SM holds seven of the append's (72 registers) and four of
// the read's (256 threads x 64); the last CTA of a block may have fewer heads than the others.
int heads_each(int heads, long long all) {
  const long long each = (all + 8 * 148 - 1) / (8 * 148);
  return static_cast<int>(each > heads ? heads : each);
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace nob200

extern "C" int nob200_int8_cache_append_d128(int num_rows, int sequences, int max_blocks, int num_blocks, const void* key,
                                             const void* value, const void* bounds, const void* table, const void* lengths,
                                             void* key_codes, void* key_scales, void* value_codes, void* value_scales,
                                             int heads, void* stream) {
  using namespace nob200;
  const char* name = "int8_cache_append_d128";
  NOB_REQUIRE(num_rows > 0 && sequences > 0 && max_blocks > 0 && num_blocks > 0 && heads > 0, "%s: sizes must be positive", name);
  NOB_REQUIRE(max_blocks <= 0x7fffffff / kBlock, "%s: %d blocks of a sequence exceed the limit of %d", name, max_blocks, 0x7fffffff / kBlock);
  NOB_REQUIRE(key && value && bounds && table && lengths && key_codes && key_scales && value_codes && value_scales,
              "%s: NULL tensor", name);
  NOB_REQUIRE(aligned16(key) && aligned16(value) && aligned16(key_codes) && aligned16(value_codes),
              "%s: a tensor is not 16-byte aligned", name);
  AppendParams P = {};
  P.status = status_word_device_ptr();
  if (!P.status) return fail(kCudaError, "%s: no current CUDA device", name);
  P.source[0] = static_cast<const __nv_bfloat16*>(key), P.source[1] = static_cast<const __nv_bfloat16*>(value);
  P.codes[0] = static_cast<int8_t*>(key_codes), P.codes[1] = static_cast<int8_t*>(value_codes);
  P.scales[0] = static_cast<float*>(key_scales), P.scales[1] = static_cast<float*>(value_scales);
  P.bounds = static_cast<const int*>(bounds), P.table = static_cast<const int*>(table), P.lengths = static_cast<const int*>(lengths);
  P.rows = num_rows, P.sequences = sequences, P.max_blocks = max_blocks, P.num_blocks = num_blocks, P.heads = heads;
  // new rows of a sequence touch at most (rows + 126) / 64 blocks, the first and the last of them perhaps in part
  const long long slots = most_units(num_rows + 63ll * sequences, sequences, kBlock);
  P.slots = static_cast<int>(slots < num_rows ? slots : num_rows);
  P.each = heads_each(heads, 2ll * heads * P.slots);
  const long long blocks = 2ll * ((heads + P.each - 1) / P.each) * P.slots;
  NOB_REQUIRE(blocks <= 0x7fffffffll, "%s: %d blocks x %d heads exceed the grid limit", name, P.slots, heads);
  return launch_pdl(name, cache_append_kernel, static_cast<unsigned>(blocks), kAppendThreads, 0, stream, P);
}

extern "C" int nob200_int8_cache_read_d128(int capacity, int sequences, int max_blocks, int num_blocks, const void* key_codes,
                                           const void* value_codes, const void* key_scales, const void* value_scales,
                                           const void* table, const void* lengths, void* key, void* value, void* bounds,
                                           int heads, void* stream) {
  using namespace nob200;
  const char* name = "int8_cache_read_d128";
  NOB_REQUIRE(capacity > 0 && sequences > 0 && max_blocks > 0 && num_blocks > 0 && heads > 0, "%s: sizes must be positive", name);
  NOB_REQUIRE(max_blocks <= 0x7fffffff / kBlock, "%s: %d blocks of a sequence exceed the limit of %d", name, max_blocks, 0x7fffffff / kBlock);
  NOB_REQUIRE(key_codes && value_codes && key_scales && value_scales && table && lengths && key && value && bounds,
              "%s: NULL tensor", name);
  NOB_REQUIRE(aligned16(key) && aligned16(value) && aligned16(key_codes) && aligned16(value_codes),
              "%s: a tensor is not 16-byte aligned", name);
  ReadParams P = {};
  P.status = status_word_device_ptr();
  if (!P.status) return fail(kCudaError, "%s: no current CUDA device", name);
  P.codes[0] = static_cast<const int8_t*>(key_codes), P.codes[1] = static_cast<const int8_t*>(value_codes);
  P.scales[0] = static_cast<const float*>(key_scales), P.scales[1] = static_cast<const float*>(value_scales);
  P.table = static_cast<const int*>(table), P.lengths = static_cast<const int*>(lengths);
  P.rows[0] = static_cast<__nv_bfloat16*>(key), P.rows[1] = static_cast<__nv_bfloat16*>(value);
  P.bounds = static_cast<int*>(bounds);
  P.capacity = capacity, P.sequences = sequences, P.max_blocks = max_blocks, P.num_blocks = num_blocks, P.heads = heads;
  const long long slots = most_units(capacity, sequences, kBlock);
  P.slots = static_cast<int>(slots);
  P.each = heads_each(heads, 2ll * heads * slots);
  const long long blocks = 2ll * ((heads + P.each - 1) / P.each) * slots;
  NOB_REQUIRE(blocks <= 0x7fffffffll, "%s: %lld blocks x %d heads exceed the grid limit", name, slots, heads);
  return launch_pdl(name, cache_read_kernel, static_cast<unsigned>(blocks), kThreads, 0, stream, P);
}
