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
// Both are bound by HBM.
#include "common.cuh"
#include "documents.cuh"
#include "fa_common.cuh"
#include "../../include/nano_omni_b200.h"

namespace nob200 {
namespace {

constexpr int kBlock = 64, kDim = 128, kThreads = 256;
constexpr int kPieces = kBlock * kDim / 8 / kThreads;  // pieces of eight channels that a thread owns

struct AppendParams {
  const __nv_bfloat16* source[2];  // new rows of K, V [rows, heads * 128]
  int8_t* codes[2];
  float* scales[2];
  const int* bounds;   // [sequences + 1] of the new rows
  const int* table;
  const int* lengths;  // with the new tokens
  uint32_t* status;
  int rows, sequences, max_blocks, num_blocks, heads, slots;
};

// Tokens that a sequence held before, or -1 where its length cannot be right.
__device__ __forceinline__ int held_before(const AppendParams& P, int s, int fresh) {
  const int length = P.lengths[s];
  return length >= fresh && length <= P.max_blocks * kBlock ? length - fresh : -1;
}

__device__ __forceinline__ int8_t code_of(float x, float scale) {
  return static_cast<int8_t>(__float2int_rn(fminf(fmaxf(__fdiv_rn(x, scale), -127.f), 127.f)));
}
__device__ __forceinline__ uint2 pack_codes(const int8_t (&c)[8]) {
  uint2 r;
  r.x = static_cast<uint8_t>(c[0]) | static_cast<uint8_t>(c[1]) << 8 | static_cast<uint8_t>(c[2]) << 16 | static_cast<uint32_t>(static_cast<uint8_t>(c[3])) << 24;
  r.y = static_cast<uint8_t>(c[4]) | static_cast<uint8_t>(c[5]) << 8 | static_cast<uint8_t>(c[6]) << 16 | static_cast<uint32_t>(static_cast<uint8_t>(c[7])) << 24;
  return r;
}
__device__ __forceinline__ int code_at(uint32_t word, int i) { return static_cast<int8_t>(word >> (8 * i)); }

__global__ void __launch_bounds__(kThreads)
cache_append_kernel(const AppendParams P) {
  __shared__ int unit[4];  // sequence, block in it, first new row, tokens held before
  __shared__ float most[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = static_cast<int>(blockIdx.x) % P.slots, which = static_cast<int>(blockIdx.x) / P.slots;
  const int head = which >> 1, tensor = which & 1;
  pdl_wait();
  pdl_release();
  if (warp == 0) {
    const int2 found = find_unit(P.sequences, slot, [&](int s) {
      const int2 r = document_rows(P.bounds, s, P.rows);
      const int before = held_before(P, s, r.y - r.x);
      if (before < 0 && r.y > r.x) atomicOr(P.status, kBadIndex);
      return before < 0 || r.y == r.x ? 0 : (before + r.y - r.x + kBlock - 1) / kBlock - before / kBlock;
    });
    if (lane == 0) {
      unit[0] = found.x;
      if (found.x >= 0) {
        const int2 r = document_rows(P.bounds, found.x, P.rows);
        const int before = held_before(P, found.x, r.y - r.x);
        unit[1] = before / kBlock + found.y;
        unit[2] = r.x - before;  // row of the sequence's token 0, if it were among the new ones
        unit[3] = before;
      }
    }
  }
  __syncthreads();
  const int sequence = unit[0];
  if (sequence < 0) return;
  const int token0 = unit[1] * kBlock, row_of_token0 = unit[2];
  const int kept = clamped(unit[3] - token0, 0, kBlock);                       // tokens that the block holds
  const int end = min(P.lengths[sequence] - token0, kBlock);                   // and will hold
  const int block = P.table[static_cast<size_t>(sequence) * P.max_blocks + unit[1]];
  if (block < 0 || block >= P.num_blocks) {
    if (threadIdx.x == 0) atomicOr(P.status, kBadIndex);
    return;
  }
  const __nv_bfloat16* source = tensor ? P.source[1] : P.source[0];
  int8_t* codes = (tensor ? P.codes[1] : P.codes[0]) + (static_cast<size_t>(block) * P.heads + head) * kBlock * kDim;
  float* scale_at = (tensor ? P.scales[1] : P.scales[0]) + static_cast<size_t>(block) * P.heads + head;
  const int channel = (threadIdx.x & 15) * 8, first = threadIdx.x >> 4;

  uint4 x[kPieces];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int token = first + 16 * i;
    x[i] = make_uint4(0, 0, 0, 0);
    if (token >= kept && token < end)
      x[i] = *reinterpret_cast<const uint4*>(source + (static_cast<size_t>(row_of_token0 + token0 + token) * P.heads + head) * kDim + channel);
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k)  // a value that is not a number shows in the scale
      top = max_nan(top, max_nan(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u))));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) most[warp] = top;
  const float old = kept ? *scale_at : 0.f;
  __syncthreads();  // also: everyone has read the old scale
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = max_nan(top, most[w]);
  const float scale = max_nan(old, max_nan(__fmul_rn(top, 1.0f / 127.0f), 1e-10f));
  if (threadIdx.x == 0) *scale_at = scale;
  const float ratio = __fdiv_rn(old, scale);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int token = first + 16 * i;
    uint2* at = reinterpret_cast<uint2*>(codes + token * kDim + channel);
    int8_t c[8];
    if (token >= kept && token < end) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        c[2 * k] = code_of(__uint_as_float(w[k] << 16), scale);
        c[2 * k + 1] = code_of(__uint_as_float(w[k] & 0xffff0000u), scale);
      }
      *at = pack_codes(c);
    } else if (token < kept && scale != old) {  // the grid has grown: what was there is rounded again
      const uint2 was = *at;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        c[k] = static_cast<int8_t>(__float2int_rn(__fmul_rn(static_cast<float>(code_at(was.x, k)), ratio)));
        c[4 + k] = static_cast<int8_t>(__float2int_rn(__fmul_rn(static_cast<float>(code_at(was.y, k)), ratio)));
      }
      *at = pack_codes(c);
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
  int capacity, sequences, max_blocks, num_blocks, heads, slots;
};

__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const ReadParams P) {
  __shared__ int unit[3];  // sequence, block in it, output row of its first token
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = static_cast<int>(blockIdx.x) % P.slots, which = static_cast<int>(blockIdx.x) / P.slots;
  const int head = which >> 1, tensor = which & 1;
  pdl_wait();
  pdl_release();
  if (warp == 0) {
    if (lane == 0) unit[0] = -1;
    __syncwarp();
    long long row = 0;
    int before = 0;
    const bool notes = blockIdx.x == 0;  // this CTA walks all sequences and writes where each begins
    for (int base = 0; base < P.sequences && (notes || before <= slot); base += 32) {
      const int s = base + lane;
      const int given = s < P.sequences ? P.lengths[s] : 0;
      const int length = clamped(given, 0, P.max_blocks * kBlock);
      if (notes && given != length) atomicOr(P.status, kBadIndex);
      const int blocks = (length + kBlock - 1) / kBlock;
      int through = blocks;
      long long rows = length;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int b = __shfl_up_sync(0xffffffffu, through, o);
        const long long r = __shfl_up_sync(0xffffffffu, rows, o);
        if (lane >= o) through += b, rows += r;
      }
      if (notes && s < P.sequences) {
        const long long until = row + rows;
        P.bounds[s + 1] = static_cast<int>(until < P.capacity ? until : P.capacity);
        if (s == 0) P.bounds[0] = 0;
        if (until > P.capacity) atomicOr(P.status, kBadIndex);
      }
      const int mine = slot - before;  // of this group's blocks
      if (mine >= through - blocks && mine < through) {
        const int b = mine - (through - blocks);
        const long long at = row + rows - length + static_cast<long long>(b) * kBlock;
        if (at < P.capacity) unit[0] = s, unit[1] = b, unit[2] = static_cast<int>(at);
      }
      before += __shfl_sync(0xffffffffu, through, 31);
      row += __shfl_sync(0xffffffffu, rows, 31);
    }
  }
  __syncthreads();
  const int sequence = unit[0];
  if (sequence < 0) return;
  const int end = min(min(P.lengths[sequence], P.max_blocks * kBlock) - unit[1] * kBlock, P.capacity - unit[2]);
  const int block = P.table[static_cast<size_t>(sequence) * P.max_blocks + unit[1]];
  const bool known = block >= 0 && block < P.num_blocks;
  if (!known && threadIdx.x == 0) atomicOr(P.status, kBadIndex);
  const size_t from = known ? static_cast<size_t>(block) * P.heads + head : 0;
  const float scale = known ? (tensor ? P.scales[1] : P.scales[0])[from] : 0.f;  // of a block that is not there: zeros
  const int channel = (threadIdx.x & 15) * 8, first = threadIdx.x >> 4;
  const int8_t* codes = (tensor ? P.codes[1] : P.codes[0]) + from * (kBlock * kDim) + channel;
  __nv_bfloat16* rows = (tensor ? P.rows[1] : P.rows[0]) + channel;
  uint2 c[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    c[i] = first + 16 * i < end ? *reinterpret_cast<const uint2*>(codes + (first + 16 * i) * kDim) : make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int token = first + 16 * i;
    if (token >= end) continue;
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // one rounding to bf16, of the exact product in fp32
      o[k] = pack_bf16(code_at(c[i].x, 2 * k) * scale, code_at(c[i].x, 2 * k + 1) * scale);
      o[2 + k] = pack_bf16(code_at(c[i].y, 2 * k) * scale, code_at(c[i].y, 2 * k + 1) * scale);
    }
    *reinterpret_cast<uint4*>(rows + (static_cast<size_t>(unit[2] + token) * P.heads + head) * kDim) =
        make_uint4(o[0], o[1], o[2], o[3]);
  }
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
  const long long blocks = 2ll * heads * P.slots;
  NOB_REQUIRE(blocks <= 0x7fffffffll, "%s: %d blocks x %d heads exceed the grid limit", name, P.slots, heads);
  return launch_pdl(name, cache_append_kernel, static_cast<unsigned>(blocks), kThreads, 0, stream, P);
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
  const long long blocks = 2ll * heads * slots;
  NOB_REQUIRE(blocks <= 0x7fffffffll, "%s: %lld blocks x %d heads exceed the grid limit", name, slots, heads);
  return launch_pdl(name, cache_read_kernel, static_cast<unsigned>(blocks), kThreads, 0, stream, P);
}
