// The 4-bit KV pool: format constants and device helpers.
//
// A row (128 dims of one token and KV head) is held as 8 groups of 16
// neighbouring dims. A group has one e4m3 scale s = rn(amax / 6) and 16 e2m1
// codes c = rn(x / s) (both round to nearest, ties to even, and saturate); it
// stands for g * s * c with g a power of two that the whole layer shares.
// e2m1 has two significant bits and e4m3 four, so s * c is exact in bf16 and
// fp16: what the attention kernels multiply is exactly what is stored.
//
// 16 tokens of one (block, KV head) make a unit of 2304 contiguous bytes, and
// a layer's pool is [num_blocks, kv_heads, block_size / 16, 2304]: any run of
// units inside a block is one contiguous copy. The order inside a unit is the
// one in which the decode kernel's matrix fragments take the data, so that a
// lane reads whole 16-byte words and no code moves between lanes:
//   [0, 1024)     K codes, byte 64 i + 16 t + 2 j + h of token i: dims
//                 16 j + 4 t + 2 h (low nibble) and + 1 (high nibble)
//   [1024, 1152)  K scales, byte 8 i + j: token i, group j
//   [1152, 2176)  V codes, byte 256 (i / 4) + 32 g + 8 (i % 4) + j of token i:
//                 dims 16 j + 2 g (low nibble) and + 1 (high nibble)
//   [2176, 2304)  V scales, byte 32 (i / 4) + 4 j + i % 4
// No byte is shared by two tokens, so appends of different tokens never touch
// the same byte.
#pragma once

#include <cuda_fp16.h>

#include <cstring>

#include "host_common.h"
#include "nvk_common.cuh"

namespace nvk {
namespace fp4 {

constexpr int kD = 128;
constexpr int kGroups = kD / 16;
constexpr int kUnitTokens = NVK_FP4_UNIT_TOKENS;
constexpr int kUnitBytes = NVK_FP4_UNIT_BYTES;
constexpr int kOffKScale = 1024;
constexpr int kOffV = 1152;
constexpr int kOffVScale = 2176;

// Byte address of the unit that holds `slot` of KV head `head`; upb_log2 is
// log2 of the units of a block.
__device__ __forceinline__ uint8_t* unit_of(uint8_t* pool, int64_t slot, int head, int kvh, int upb_log2) {
  const int64_t unit = slot >> 4;  // units before it in one head's [block, unit] order
  const int64_t block = unit >> upb_log2;
  const int64_t in_block = unit & ((1 << upb_log2) - 1);
  return pool + ((((block * kvh + head) << upb_log2) + in_block) * kUnitBytes);
}

// Four bytes, each two e2m1 codes, to four half2 (low nibble in the low half).
__device__ __forceinline__ void e2m1_to_half2(uint32_t w, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
      : "r"(w));
}

// Two e4m3 values of each half of a word to half2.
__device__ __forceinline__ void e4m3_to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t floats_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ uint32_t floats_to_e2m1x2(float lo, float hi) {
  uint16_t r;
  asm("{\n\t.reg .b8 a;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.u16.u8 %0, a;\n\t}"
      : "=h"(r)
      : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Rounds a quotient computed as a product with a reciprocal (relative error
// below 2^-21) to 18 significant bits. The rows are bf16 or fp16 (at most 11
// significant bits) and every rounding border of e2m1 and e4m3, times s or 6,
// has at most 7: a quotient that is not exactly on a border is at least 2^-12
// of it away, and one that is on it lands on it again. So the code that
// follows is the one that an exact division would give.
__device__ __forceinline__ float snap18(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x20u) & ~0x3fu);  // not for NaN
}

// One row by eight lanes: lane g holds x[j] = dims {16 j + 2 g, 16 j + 2 g +
// 1} of group j, already divided by the layer's constant. Returns this lane's
// codes (byte j of w0 | w1) and the row's eight scales (e4m3 bytes).
// A group with a NaN gets a NaN scale (and so reads back as NaN); infinities
// saturate to 6 * 448; a group whose scale rounds to 0 gets codes of 0.
__device__ __forceinline__ void quantise_row(const float2 (&x)[kGroups], uint32_t& w0, uint32_t& w1, uint32_t& s0,
                                             uint32_t& s1) {
  float amax[kGroups];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) amax[j] = fmax_nan(fabsf(x[j].x), fabsf(x[j].y));
#pragma unroll
  for (int off = 1; off < 8; off <<= 1)
#pragma unroll
    for (int j = 0; j < kGroups; ++j) amax[j] = fmax_nan(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], off));
  uint32_t sc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    auto sixth = [](float m) { return m == m ? snap18(m * (1.f / 6.f)) : m; };
    sc[j] = floats_to_e4m3x2(sixth(amax[2 * j]), sixth(amax[2 * j + 1]));
  }
  s0 = sc[0] | (sc[1] << 16);
  s1 = sc[2] | (sc[3] << 16);
  uint32_t h[4];
  e4m3_to_half2(s0, h[0], h[1]);
  e4m3_to_half2(s1, h[2], h[3]);
  uint32_t code[kGroups];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    const __half2 hs = *reinterpret_cast<const __half2*>(&h[j >> 1]);
    const float s = (j & 1) ? __high2float(hs) : __low2float(hs);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    r = s > 0.f ? r : 0.f;  // also for a NaN scale: its codes do not matter
    // an infinity times a zero reciprocal cannot happen: its scale is 448
    code[j] = floats_to_e2m1x2(snap18(x[j].x * r), snap18(x[j].y * r));
  }
  w0 = code[0] | (code[1] << 8) | (code[2] << 16) | (code[3] << 24);
  w1 = code[4] | (code[5] << 8) | (code[6] << 16) | (code[7] << 24);
}

// Stores the codes and scales of one row (see quantise_row) as token i of a
// unit: eight bytes of codes a lane. All lanes of the warp call it (the K
// order exchanges words between neighbouring lanes); `store` is false for
// rows that are not written.
__device__ __forceinline__ void store_row(uint8_t* unit, int i, bool is_v, bool store, int g, uint32_t w0,
                                          uint32_t w1, uint32_t s0, uint32_t s1) {
  // K: byte 2 j + h of a lane pair's 16: the even lane stores groups 0-3 of both lanes, the odd one 4-7
  const bool odd = g & 1;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? w0 : w1, 1);
  const uint32_t e = odd ? other : w0, o = odd ? w1 : other;
  if (!store) return;
  if (is_v) {
    *reinterpret_cast<uint2*>(unit + kOffV + 256 * (i >> 2) + 32 * g + 8 * (i & 3)) = make_uint2(w0, w1);
    unit[kOffVScale + 32 * (i >> 2) + 4 * g + (i & 3)] = static_cast<uint8_t>((g < 4 ? s0 : s1) >> (8 * (g & 3)));
  } else {
    *reinterpret_cast<uint2*>(unit + 64 * i + 8 * g) =
        make_uint2(__byte_perm(e, o, 0x5140), __byte_perm(e, o, 0x7362));
    if (g == 0) *reinterpret_cast<uint2*>(unit + kOffKScale + 8 * i) = make_uint2(s0, s1);
  }
}

// A power of two that fp32 products with row values and scales stay finite and exact under.
inline bool good_constant(float g) {
  uint32_t u;
  memcpy(&u, &g, 4);
  const int e = static_cast<int>(u >> 23) - 127;
  return (u & 0x807fffffu) == 0 && e >= -60 && e <= 60;
}

// log2 of the units of a block, or -1 for a block size outside what the pool takes.
inline int units_log2(int block_size) {
  for (int l = 0; l <= 4; ++l)
    if (block_size == (kUnitTokens << l)) return l;
  return -1;
}

// Checks that every entry point over a 4-bit pool shares; 0 or an error code.
inline int check_pool(const void* kv_cache, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                      float k_scale, float v_scale, const char* who) {
  if (head_dim != kD) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", who, head_dim);
  if (units_log2(block_size) < 0)
    return fail(NVK_ERR_UNSUPPORTED, "%s: block_size %d unsupported (a power of two in [16, 256])", who, block_size);
  if (num_blocks <= 0 || num_kv_heads <= 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad pool (blocks=%d kv_heads=%d)", who, num_blocks, num_kv_heads);
  if (!kv_cache) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(kv_cache)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: the pool must be 16-byte aligned", who);
  if (!good_constant(k_scale) || !good_constant(v_scale))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: k_scale %g and v_scale %g must be powers of two in [2^-60, 2^60]", who,
                double(k_scale), double(v_scale));
  return NVK_OK;
}

}  // namespace fp4
}  // namespace nvk
