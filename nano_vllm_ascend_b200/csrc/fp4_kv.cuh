// The 4-bit KV pool: format constants and device helpers.
//
// A row (128 dims of one token and KV head) is held as 8 groups of 16
// neighbouring dims. A group has one e4m3 scale s = rn(amax / 6) and 16 e2m1
// codes c = rn(x / s) (both round to nearest, ties to even, and saturate); it
// stands for g * s * c with g a power of two that the whole layer shares. The
// sign of a value that rounds to 0 is not kept.
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

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Q for the tensor cores: a row from bf16 to fp16, scaled by a power of two.
// fp16's exponent field is bf16's less f, such that the row's largest entry
// gets 30, and 10 fraction bits hold bf16's 7. Entries 2^29 below the largest
// become 0 or a wrong subnormal, which a sum of 128 terms does not show.
__device__ __forceinline__ uint32_t bf16x2_abs_max(uint32_t a, uint32_t b) {  // (signs mixed; NaN wins)
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
struct HalfRow {
  uint32_t base;  // f in both exponent fields
  float up;       // what the row's scores have to be multiplied by: 2^(f - 112), or NaN for a row with a
                  // NaN or an infinity (whose softmax is NaN everywhere)
};
__device__ __forceinline__ HalfRow half_row(uint32_t largest) {  // the bf16x2_abs_max of the row's pairs
  const uint32_t top = max(largest & 0x7fffu, (largest >> 16) & 0x7fffu) >> 7;
  const uint32_t f = max(top, 30u) - 30u;
  return HalfRow{f * 0x00800080u, __uint_as_float(top == 255u ? 0x7fffffffu : (127u - 112u + f) << 23)};
}
// The factor from a row's products, which are below 2^35, to its scores in log2
// units, kept where both ends stay numbers. At least the smallest normal, so
// that a masked product, -inf, stays -inf under it (a row of zeros has the
// smallest `up`, and times a small scale and constant it would be 0): such
// scores are 0 to fp32 anyway. At most 2^90, so that scores stay finite:
// products that differ do so by 2^-34 or more, whose weights are 1 and 0 anyway.
__device__ __forceinline__ float score_factor(float up, float scale_log2) {
  constexpr float kLeast = 1.17549435e-38f, kMost = 1.2379400392853803e27f;
  const float f = up * scale_log2;
  return f < kLeast ? kLeast : f > kMost ? kMost : f;  // NaN stays
}
__device__ __forceinline__ uint32_t bf16x2_to_half2(uint32_t w, uint32_t base) {
  uint32_t m;  // of magnitudes
  asm("max.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(w & 0x7fff7fffu), "r"(base));
  return ((m - base) << 3) | (w & 0x80008000u);
}

// A pair of 16-bit floats to fp32, and back.
template <typename T>
__device__ __forceinline__ float2 pair_to_f32(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_to_f32<__nv_bfloat16>(uint32_t w) {
  return make_float2(bf16lo_to_f32(w), bf16hi_to_f32(w));
}
template <>
__device__ __forceinline__ float2 pair_to_f32<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t f32_to_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t f32_to_pair<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t f32_to_pair<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Quotients are computed as products with a reciprocal (relative error below
// 2^-21) and moved onto a grid that holds every rounding border before they
// are rounded, so that the codes are those of an exact division: the rows have
// at most 11 significant bits and a border times s (or 6) at most 7, so a
// quotient that is not on a border is at least 2^-11 of it away.
// The scale: to 18 significant bits, 2^-18 of it.
__device__ __forceinline__ float snap18(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x20u) & ~0x3fu);  // not for NaN
}
// The codes: borders are multiples of 1/4 from 1/4 to 5, so to multiples of
// 2^-14, by adding and subtracting 768 (its step in fp32).
constexpr float kGrid = 768.f;

// One row by eight lanes: word j of lane g holds dims 16 j + 2 g and + 1 of
// group j as 16-bit floats of type T; `inv` is the reciprocal of the layer's
// constant. Returns this lane's codes (byte j of w0 | w1) and the e4m3 byte of
// group g. A group with a NaN gets a NaN scale (and so reads back as NaN);
// infinities saturate to 6 * 448; a group whose scale rounds to 0 gets zeros.
template <typename T>
__device__ __forceinline__ void quantise_row(const uint32_t (&x)[kGroups], float inv, int g, uint32_t& w0,
                                             uint32_t& w1, uint32_t& scale) {
  // Magnitudes of 16-bit floats order as integers (NaN above infinity). The
  // maxima of the eight groups are reduced and scattered: three exchanges,
  // after which lane g has group g's.
  uint32_t m[4];  // groups 2 k and 2 k + 1
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t a = x[2 * k] & 0x7fff7fffu, b = x[2 * k + 1] & 0x7fff7fffu;
    m[k] = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
  }
  const bool up4 = g & 4, up2 = g & 2, up1 = g & 1;
  const uint32_t r0 = __shfl_xor_sync(0xffffffffu, up4 ? m[0] : m[2], 4);
  const uint32_t r1 = __shfl_xor_sync(0xffffffffu, up4 ? m[1] : m[3], 4);
  const uint32_t n0 = __vmaxu2(up4 ? m[2] : m[0], r0), n1 = __vmaxu2(up4 ? m[3] : m[1], r1);
  const uint32_t r2 = __shfl_xor_sync(0xffffffffu, up2 ? n0 : n1, 2);
  const uint32_t o = __vmaxu2(up2 ? n1 : n0, r2);
  const uint32_t both = __vmaxu2(o, __shfl_xor_sync(0xffffffffu, o, 1));
  const float2 pair = pair_to_f32<T>(both);
  const float amax = (up1 ? pair.y : pair.x) * inv;
  scale = floats_to_e4m3x2(amax == amax ? snap18(amax * (1.f / 6.f)) : amax, 0.f);
  uint32_t lo, hi;
  e4m3_to_half2(scale, lo, hi);
  const float s = __low2float(*reinterpret_cast<const __half2*>(&lo));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  r = s > 0.f ? r * inv : 0.f;  // also for a NaN scale: its codes do not matter
  const uint64_t grid = f32x2_pack(kGrid, kGrid), back = f32x2_pack(-kGrid, -kGrid);
  uint32_t code[kGroups];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    const float rj = __shfl_sync(0xffffffffu, r, j, 8);
    const float2 f = pair_to_f32<T>(x[j]);
    float u, v;
    f32x2_unpack(f32x2_add(f32x2_fma(f32x2_pack(f.x, f.y), f32x2_pack(rj, rj), grid), back), u, v);
    code[j] = floats_to_e2m1x2(u, v);
  }
  w0 = code[0] | (code[1] << 8) | (code[2] << 16) | (code[3] << 24);
  w1 = code[4] | (code[5] << 8) | (code[6] << 16) | (code[7] << 24);
}

// Stores the codes and scales of one row (see quantise_row) as token i of a
// unit: eight bytes of codes and one scale a lane. All lanes of the warp call
// it (the K order exchanges words between neighbouring lanes); `store` is
// false for rows that are not written.
__device__ __forceinline__ void store_row(uint8_t* unit, int i, bool is_v, bool store, int g, uint32_t w0,
                                          uint32_t w1, uint32_t scale) {
  // K: byte 2 j + h of a lane pair's 16: the even lane stores groups 0-3 of both lanes, the odd one 4-7
  const bool odd = g & 1;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? w0 : w1, 1);
  const uint32_t e = odd ? other : w0, o = odd ? w1 : other;
  if (!store) return;
  if (is_v) {
    *reinterpret_cast<uint2*>(unit + kOffV + 256 * (i >> 2) + 32 * g + 8 * (i & 3)) = make_uint2(w0, w1);
    unit[kOffVScale + 32 * (i >> 2) + 4 * g + (i & 3)] = static_cast<uint8_t>(scale);
  } else {
    *reinterpret_cast<uint2*>(unit + 64 * i + 8 * g) =
        make_uint2(__byte_perm(e, o, 0x5140), __byte_perm(e, o, 0x7362));
    unit[kOffKScale + 8 * i + g] = static_cast<uint8_t>(scale);
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
  if (num_blocks <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535)
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
