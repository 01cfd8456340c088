// The 8-bit KV pool: format constants and device helpers.
//
// 16 tokens of one (block, KV head) make a unit of 4128 contiguous bytes, and
// a layer's pool is [num_blocks, kv_heads, block_size / 16, 4128]:
//   [0, 2048)     K codes, e4m3: token r's 128 dims at 128 r, the 16-byte
//                 chunk c (dims 16 c .. 16 c + 15) at place c ^ (r & 7)
//   [2048, 4096)  V codes, the same
//   [4096, 4104)  the exponents of K and of V, int32
//   [4104, 4128)  zeros: a unit is a whole number of 32-byte sectors
// A value is code * 2^exponent. The exponent is the unit's, K's or V's: the
// least e with amax <= 448 * 2^e over the finite values of the rows it was
// made for, held to [kLeastExp, kMostExp]. A power of two costs an e4m3 code
// nothing inside its range and keeps every value exact in bf16 (4 significant
// bits), so the attention kernels multiply exactly what is stored, and bringing
// a row to a larger exponent moves its codes' exponents (and rounds once more
// what becomes subnormal). +-40 is what the decode kernel's weights take
// without leaving fp32 (fp8_decode.cu).
// The order of the chunks lets eight lanes read eight tokens' chunks of the
// same dims, or one chunk each of four tokens' two halves, without a bank
// conflict, and costs the copies nothing.
// A row with a NaN is held as NaN throughout (the prefill kernel looks at one
// byte of a row); infinities saturate.
#pragma once

#include <cuda_fp16.h>

#include "fp4_kv.cuh"
#include "host_common.h"
#include "nvk_common.cuh"

namespace nvk {
namespace fp8 {

using fp4::e4m3_to_half2;
using fp4::f32_to_pair;
using fp4::floats_to_e4m3x2;
using fp4::pair_to_f32;
using fp4::units_log2;

constexpr int kD = 128;
constexpr int kUnitTokens = NVK_FP8_UNIT_TOKENS;
constexpr int kUnitBytes = NVK_FP8_UNIT_BYTES;
constexpr int kOffV = 2048;
constexpr int kOffExp = 4096;
constexpr int kLeastExp = -40, kMostExp = 40;

// Byte offset of chunk c of token r in K's or V's part of a unit.
__device__ __forceinline__ int chunk_at(int r, int c) { return 128 * r + ((c ^ (r & 7)) << 4); }

// 2^e for e in the range of fp32's normal numbers.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }

// An exponent as the pool holds it; whatever else the bytes are, one in range.
__device__ __forceinline__ int held_exp(int e) { return min(max(e, kLeastExp), kMostExp); }

// The least e with amax <= 448 * 2^e = 1.75 * 2^(e + 8): adding to the fraction
// carries where it is above 0.75.
__device__ __forceinline__ int exponent_for(float amax) {
  return held_exp(static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8);
}

// Byte address of unit `unit` (slot / 16) of a head.
__device__ __forceinline__ uint8_t* unit_at(uint8_t* pool, int64_t unit, int head, int kvh, int upb_log2) {
  const int64_t block = unit >> upb_log2, in_block = unit & ((1 << upb_log2) - 1);
  return pool + ((((block * kvh + head) << upb_log2) + in_block) * kUnitBytes);
}

// Checks that every entry point over an 8-bit pool shares; 0 or an error code.
inline int check_pool(const void* kv_cache, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                      const char* who) {
  if (head_dim != kD) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", who, head_dim);
  if (units_log2(block_size) < 0)
    return fail(NVK_ERR_UNSUPPORTED, "%s: block_size %d unsupported (a power of two in [16, 256])", who, block_size);
  if (num_blocks <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad pool (blocks=%d kv_heads=%d)", who, num_blocks, num_kv_heads);
  if (!kv_cache) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(kv_cache)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: the pool must be 16-byte aligned", who);
  return NVK_OK;
}

}  // namespace fp8
}  // namespace nvk
