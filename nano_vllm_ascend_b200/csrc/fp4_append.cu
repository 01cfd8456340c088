// Rows into and out of the 4-bit KV pool: the quantising append, the read of
// rows back, and the attention prologue (per-head RMSNorm of q and k, rotary
// embedding, append) that writes the pool. The format is in fp4_kv.cuh.
//
// HBM-bound byte movement with some arithmetic: per (token, KV head) the
// append reads 512 B and writes 144 B, the read the other way round. Eight
// lanes take a row, lane g its dims {16 j + 2 g, 16 j + 2 g + 1}: a group's
// maximum is three shuffles, each 4-byte load of the eight lanes is one whole
// 32-byte sector, a lane's eight code bytes are what it stores, and the
// rotation pairs (i, i + 64) sit in one lane.
#include <type_traits>

#include "fp4_kv.cuh"

namespace nvk {
namespace fp4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// n / d for n < 2^31 as a multiplication: m = ceil(2^(31 + l) / d) with l the
// least such that 2^l >= d; n * (m * d - 2^(31 + l)) < 2^(31 + l), so the
// product's excess never reaches the next quotient.
struct Divisor {
  uint32_t m, shift;
  int d;
};
inline Divisor divisor(int d) {  // d of 1 is for the caller
  uint32_t l = 1;
  while ((int64_t(1) << l) < d) ++l;
  return Divisor{static_cast<uint32_t>(((uint64_t(1) << (31 + l)) + d - 1) / d), l - 1, d};
}
__device__ __forceinline__ int quotient(int n, const Divisor& v) {
  return static_cast<int>(__umulhi(static_cast<uint32_t>(n), v.m) >> v.shift);
}
constexpr int64_t kMostItems = int64_t(1) << 30;  // of a launch (more go in several)

// A warp's item is the K (or V) rows of one head of four tokens, eight lanes a
// row: where their slots follow each other, as in a prefill, the four rows'
// 8-byte stores (and a read's loads) of V make whole sectors, 256 bytes in all.

struct AppendArgs {
  const uint8_t* key;
  const uint8_t* value;
  int64_t key_stride, value_stride;  // bytes between tokens
  uint8_t* pool;
  const int64_t* slots;
  int64_t num_slots;
  int num_tokens, items;  // items: ceil(tokens / 4) * 2 kvh
  int kvh, upb_log2;
  Divisor per_token;  // 2 kvh
  float k_inv, v_inv;
  int* err;
};

// 32 registers: eight blocks an SM (8192 tokens: 12.2 us against 14.2 with six).
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) append_kernel(const AppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int g = threadIdx.x & 7, sub = (threadIdx.x >> 3) & 3;
  for (int w = blockIdx.x * kWarps + (threadIdx.x >> 5); w < a.items; w += gridDim.x * kWarps) {
    const int group = quotient(w, a.per_token);
    const int kr = w - group * a.per_token.d, t = 4 * group + sub;
    const bool is_v = kr >= a.kvh;
    const int head = is_v ? kr - a.kvh : kr;
    const bool live = t < a.num_tokens;
    const int64_t slot = live ? a.slots[t] : -1;
    const bool ok = slot >= 0 && slot < a.num_slots;
    if (live && !ok && kr == 0 && g == 0 && a.err) atomicOr(a.err, kErrBadSlot);
    const uint8_t* src = (is_v ? a.value + t * a.value_stride : a.key + t * a.key_stride) +
                         head * (kD * 2) + 4 * g;
    const float inv = is_v ? a.v_inv : a.k_inv;
    uint32_t raw[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) raw[j] = ok ? *reinterpret_cast<const uint32_t*>(src + 32 * j) : 0u;
    uint32_t w0, w1, scale;
    quantise_row<T>(raw, inv, g, w0, w1, scale);
    store_row(ok ? unit_of(a.pool, slot, head, a.kvh, a.upb_log2) : a.pool, static_cast<int>(slot & 15), is_v, ok, g,
              w0, w1, scale);
  }
}

struct ReadArgs {
  uint8_t* key;  // [tokens, kvh, 128] contiguous
  uint8_t* value;
  uint8_t* pool;
  const int64_t* slots;
  int64_t num_slots;
  int num_tokens, items;  // items: ceil(tokens / 4) * 2 kvh
  int kvh, upb_log2;
  Divisor per_token;  // 2 kvh
  float k_scale, v_scale;
  int* err;
};

// One row a group of eight lanes; the rows of a bad slot come out as zeros.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int g = threadIdx.x & 7, sub = (threadIdx.x >> 3) & 3;
  for (int item = blockIdx.x * kWarps + (threadIdx.x >> 5); item < a.items; item += gridDim.x * kWarps) {
    const int group = quotient(item, a.per_token);
    const int kr = item - group * a.per_token.d, t = 4 * group + sub;
    const bool is_v = kr >= a.kvh;
    const int head = is_v ? kr - a.kvh : kr;
    if (t >= a.num_tokens) continue;
    const int64_t slot = a.slots[t];
    const bool ok = slot >= 0 && slot < a.num_slots;
    if (!ok && kr == 0 && g == 0 && a.err) atomicOr(a.err, kErrBadSlot);
    uint2 w = make_uint2(0, 0), sw = make_uint2(0, 0);
    const int i = static_cast<int>(slot & 15);
    if (ok) {
      const uint8_t* unit = unit_of(a.pool, slot, head, a.kvh, a.upb_log2);
      if (is_v) {
        w = *reinterpret_cast<const uint2*>(unit + kOffV + 256 * (i >> 2) + 32 * g + 8 * (i & 3));
        // byte i % 4 of the eight words of its quad
        const uint4 s0 = *reinterpret_cast<const uint4*>(unit + kOffVScale + 32 * (i >> 2));
        const uint4 s1 = *reinterpret_cast<const uint4*>(unit + kOffVScale + 32 * (i >> 2) + 16);
        const uint32_t pick = (i & 3) | ((4 + (i & 3)) << 4);
        sw.x = __byte_perm(__byte_perm(s0.x, s0.y, pick), __byte_perm(s0.z, s0.w, pick), 0x5410);
        sw.y = __byte_perm(__byte_perm(s1.x, s1.y, pick), __byte_perm(s1.z, s1.w, pick), 0x5410);
      } else {
        w = *reinterpret_cast<const uint2*>(unit + 64 * i + 8 * g);
        sw = *reinterpret_cast<const uint2*>(unit + kOffKScale + 8 * i);
      }
    }
    uint32_t c[8], s[4];
    e2m1_to_half2(w.x, c[0], c[1], c[2], c[3]);
    e2m1_to_half2(w.y, c[4], c[5], c[6], c[7]);
    e4m3_to_half2(sw.x, s[0], s[1]);
    e4m3_to_half2(sw.y, s[2], s[3]);
    const float mul = is_v ? a.v_scale : a.k_scale;
    auto scale_of = [&](int j) {
      const __half2 h = *reinterpret_cast<const __half2*>(&s[j >> 1]);
      return ((j & 1) ? __high2float(h) : __low2float(h)) * mul;
    };
    auto value = [&](int k, float sc) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&c[k]));
      return f32_to_pair<T>(f.x * sc, f.y * sc);
    };
    uint8_t* dst = (is_v ? a.value : a.key) + (static_cast<int64_t>(t) * a.kvh + head) * (kD * 2);
    if (is_v) {  // byte j: dims 16 j + 2 g and + 1
#pragma unroll
      for (int j = 0; j < kGroups; ++j) *reinterpret_cast<uint32_t*>(dst + 32 * j + 4 * g) = value(j, scale_of(j));
    } else {  // bytes 2 k and 2 k + 1: dims 16 j + 4 t .. + 3 of group j = 4 (g % 2) + k, t = g / 2
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float sc = (g & 1) ? scale_of(4 + k) : scale_of(k);
        *reinterpret_cast<uint2*>(dst + 32 * (4 * (g & 1) + k) + 8 * (g >> 1)) =
            make_uint2(value(2 * k, sc), value(2 * k + 1, sc));
      }
    }
  }
}

struct NormArgs {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  int64_t q_stride, k_stride, v_stride;  // bytes between tokens
  const uint8_t* q_weight;
  const uint8_t* k_weight;
  const float* cos_table;  // [max_pos, 128]
  const float* sin_table;
  int max_pos;
  const int64_t* positions;
  const int64_t* slots;
  uint8_t* q_out;  // [T, H, 128] contiguous
  uint8_t* pool;
  int64_t num_slots;
  int num_heads, kvh, upb_log2;
  int items;            // num_tokens * chunks
  int chunk, chunks;    // rounds of four head rows per warp item, items per token
  Divisor per_token;    // chunks, where it is not 1
  float eps, k_inv, v_inv;
  int* err;
};

__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t bf16x2_to_f32x2(uint32_t w) { return f32x2_pack(bf16lo_to_f32(w), bf16hi_to_f32(w)); }
__device__ __forceinline__ uint32_t f32x2_to_bf16x2(uint64_t v) {
  float lo, hi;
  f32x2_unpack(v, lo, hi);
  return pack_bf16x2(lo, hi);
}

// Rows of one token in rounds of four (eight lanes a row): the q heads, then
// the k heads, then the v heads; a warp takes `chunk` rounds of a token. The
// rows' arithmetic is the separate operators':
//   y   = bf16(x * rsqrt(mean(x^2) + eps) * w)
//   out = bf16(y * cos + rotate_half(y) * sin),  cos and sin cast to bf16.
// The mean square is summed in 64 bits and its root is correctly rounded, so
// the bf16 row does not hang on the order of the sum: a row that differed in
// one bf16 bit could be stored one whole e2m1 step away.
// HBM-bound once enough is in flight: each warp copies its rounds ahead, kDepth
// at a time, into a ring in shared memory (cp.async; with the cos and sin rows
// of a new token), across the borders of its items: 64 KB an SM. One round
// ahead in registers, 16 KB an SM, took 37.5 us for 8192 tokens of 16 + 2 * 8
// heads.
constexpr int kDepth = 4;
constexpr int kRowPitch = 256 + 32;  // the four rows of a round lie eight banks apart
struct NormSmem {
  alignas(16) uint8_t rows[kWarps][kDepth][4 * kRowPitch];
  alignas(16) float table[kWarps][kDepth + 1][2][kD];  // cos and sin of the items that have rounds in the ring
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// kWide: rows and tables are 16-byte aligned; else they are copied 4 bytes at a time.
template <bool kWide>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_kernel(const NormArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  NormSmem& sm = *reinterpret_cast<NormSmem*>(smem_raw);
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane & 7, sub = lane >> 3;
  const int rq = (a.num_heads + 3) / 4, rk = (a.kvh + 3) / 4, rounds = rq + 2 * rk;
  const int nw = gridDim.x * kWarps;
  const int64_t unit_step = static_cast<int64_t>(4 * kUnitBytes) << a.upb_log2;  // to the unit of four heads on
  const uint32_t ring = smem_u32(sm.rows[warp]), tables = smem_u32(sm.table[warp]);
  auto token_of = [&](int w) { return a.chunks == 1 ? w : quotient(w, a.per_token); };

  // ---- copies ahead: the next round to copy, its item, and the one after that one's position ----
  int cw = blockIdx.x * kWarps + warp, cr = 0, chi = 0, citem = -1, cstage = 0;
  int64_t cpos = cw < a.items ? a.positions[token_of(cw)] : 0;
  int ct = 0, crows = 0;  // rows from the round's first one to the end of its q, k or v heads
  const uint8_t* csrc = nullptr;  // where this lane's first copy of the round starts
  bool cnew = true;  // at an item's first round
  const int crow = kWide ? lane >> 4 : sub, ccol = kWide ? 16 * (lane & 15) : 4 * g;  // of that copy
  auto at_round = [&] {  // csrc and crows of round cr
    const bool q = cr < rq, k = cr < rq + rk;
    const int i = q ? cr : k ? cr - rq : cr - rq - rk;
    csrc = (q ? a.q + ct * a.q_stride : k ? a.k + ct * a.k_stride : a.v + ct * a.v_stride) + (4 * i + crow) * 256 + ccol;
    crows = (q ? a.num_heads : a.kvh) - 4 * i;
  };
  auto copy_round = [&] {
    if (cw < a.items) {
      if (cnew) {
        ct = token_of(cw);
        cr = (cw - ct * a.chunks) * a.chunk;
        chi = min(cr + a.chunk, rounds);
        ++citem;
        at_round();
        if (cr < rq + rk) {
          int64_t p = cpos;
          if (p < 0 || p >= a.max_pos) {
            if (lane == 0 && cr == 0 && a.err) atomicOr(a.err, kErrContextTooLong);
            p = p < 0 ? 0 : a.max_pos - 1;
          }
          const uint32_t to = tables + (citem % (kDepth + 1)) * (2 * kD * 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* row = (h ? a.sin_table : a.cos_table) + p * kD;
            if (kWide) {
              cp_async16(to + h * kD * 4 + 16 * lane, row + 4 * lane);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) cp_async4(to + h * kD * 4 + 4 * (lane + 32 * k), row + lane + 32 * k);
            }
          }
        }
        if (cw + nw < a.items) cpos = a.positions[token_of(cw + nw)];
      }
      const uint32_t to = ring + cstage * (4 * kRowPitch) + crow * kRowPitch + ccol;
      if (kWide) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (crow + 2 * h < crows) cp_async16(to + 2 * h * kRowPitch, csrc + 512 * h);
      } else if (crow < crows) {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) cp_async4(to + 32 * j, csrc + 32 * j);
      }
      csrc += 1024;
      crows -= 4;
      cnew = ++cr == chi;
      if (cnew) cw += nw;
      else if (cr == rq || cr == rq + rk) at_round();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // empty behind the last round: the waits count groups
    cstage = cstage + 1 == kDepth ? 0 : cstage + 1;
  };
#pragma unroll 1  // (one copy of the code: 0.3 us of 36, 0.13 of 2.8)
  for (int k = 0; k < kDepth; ++k) copy_round();

  int stage = 0, item = 0;
  int64_t next_slot = blockIdx.x * kWarps + warp < a.items ? a.slots[token_of(blockIdx.x * kWarps + warp)] : 0;
  for (int w = blockIdx.x * kWarps + warp; w < a.items; w += nw, ++item) {
    const int64_t t = token_of(w);
    const int lo = (w - static_cast<int>(t) * a.chunks) * a.chunk, hi = min(lo + a.chunk, rounds);
    const int64_t slot = next_slot;
    if (w + nw < a.items) next_slot = a.slots[token_of(w + nw)];
    const bool slot_ok = slot >= 0 && slot < a.num_slots;
    if (!slot_ok && lane == 0 && lo == 0 && a.err) atomicOr(a.err, kErrBadSlot);
    uint8_t* unit = unit_of(a.pool, slot_ok ? slot : 0, sub, a.kvh, a.upb_log2);  // of KV head sub
    const int token = static_cast<int>(slot & 15);
    uint8_t* q_dst = a.q_out + (t * a.num_heads + sub) * 256 + 4 * g;
    uint64_t cs[kGroups], sn[kGroups], wt[kGroups];  // sn of the lower half negated
    // Round i of the q (kind 0), k (1) or v heads (2).
    auto round = [&](auto kind, int i, bool first) {
      constexpr int kKind = decltype(kind)::value;
      const bool live = 4 * i + sub < (kKind == 0 ? a.num_heads : a.kvh);
      if (kKind < 2 && (first || i == 0)) {
        const uint8_t* weight = (kKind == 0 ? a.q_weight : a.k_weight) + 4 * g;
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
          wt[j] = bf16x2_to_f32x2(*reinterpret_cast<const uint32_t*>(weight + 32 * j));
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      __syncwarp();  // the round's rows, copied by all lanes
      uint32_t x[kGroups];
      const uint32_t from = ring + stage * (4 * kRowPitch) + sub * kRowPitch + 4 * g;
#pragma unroll
      for (int j = 0; j < kGroups; ++j) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x[j]) : "r"(from + 32 * j));
      if (kKind < 2 && first) {
        const float* row = &sm.table[warp][item % (kDepth + 1)][0][2 * g];
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          const float2 c = *reinterpret_cast<const float2*>(row + 16 * j);
          const float2 s = *reinterpret_cast<const float2*>(row + kD + 16 * j);
          cs[j] = bf16x2_to_f32x2(pack_bf16x2(c.x, c.y));
          sn[j] = bf16x2_to_f32x2(j < 4 ? pack_bf16x2(-s.x, -s.y) : pack_bf16x2(s.x, s.y));
        }
      }
      __syncwarp();  // read by all lanes: the stage may be filled again
      copy_round();
      stage = stage + 1 == kDepth ? 0 : stage + 1;
      if constexpr (kKind < 2) {
        double part[4] = {0.0, 0.0, 0.0, 0.0};  // four chains
        uint64_t f[kGroups];
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          const float2 v = pair_to_f32<__nv_bfloat16>(x[j]);
          f[j] = f32x2_pack(v.x, v.y);
          const double d0 = v.x, d1 = v.y;
          part[j & 3] = fma(d1, d1, fma(d0, d0, part[j & 3]));
        }
        double ss = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        const float rinv = __frsqrt_rn(static_cast<float>(ss * (1.0 / kD) + static_cast<double>(a.eps)));
        const uint64_t rr = f32x2_pack(rinv, rinv);
#pragma unroll
        for (int j = 0; j < kGroups; ++j)  // the norm's bf16 result
          f[j] = bf16x2_to_f32x2(f32x2_to_bf16x2(f32x2_mul(f32x2_mul(f[j], rr), wt[j])));
        // out[i] = y[i] cos[i] - y[i+64] sin[i];  out[i+64] = y[i+64] cos[i+64] + y[i] sin[i+64]
        // (products of bf16 are exact in fp32: one rounding each)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = f32x2_to_bf16x2(f32x2_fma(f[j], cs[j], f32x2_mul(f[j + 4], sn[j])));
          x[j + 4] = f32x2_to_bf16x2(f32x2_fma(f[j + 4], cs[j + 4], f32x2_mul(f[j], sn[j + 4])));
        }
      }
      if constexpr (kKind == 0) {
        uint8_t* dst = q_dst + i * 1024;
        if (live) {
#pragma unroll
          for (int j = 0; j < kGroups; ++j) *reinterpret_cast<uint32_t*>(dst + 32 * j) = x[j];
        }
      } else {
        uint32_t w0, w1, scale;
        quantise_row<__nv_bfloat16>(x, kKind == 2 ? a.v_inv : a.k_inv, g, w0, w1, scale);
        store_row(unit + i * unit_step, token, kKind == 2, live && slot_ok, g, w0, w1, scale);
      }
    };
    int r = lo;
    for (; r < min(hi, rq); ++r) round(std::integral_constant<int, 0>{}, r, r == lo);
    for (; r < min(hi, rq + rk); ++r) round(std::integral_constant<int, 1>{}, r - rq, r == lo);
    for (; r < hi; ++r) round(std::integral_constant<int, 2>{}, r - rq - rk, false);
  }
}

int sm_count() {
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Calls launch(first token, tokens, items, grid) for the tokens, as many at a time as the kernels' index takes, with
// at most `per_sm` blocks an SM. Eight are resident: the append takes two waves, whose second one evens out what
// does not divide (8192 tokens 11.4 us against 12.3 in one, 16384 21.2 against 22.3), the read, which waits for
// memory, one (10.0 and 18.0 against 10.3 and 18.3).
constexpr int kAppendBlocks = 16, kReadBlocks = 8;
template <typename Launch>
int in_launches(int64_t num_tokens, int kvh, int per_sm, Launch&& launch) {
  const int64_t per_group = 2 * static_cast<int64_t>(kvh), most_tokens = kMostItems / per_group * 4;
  const int64_t most_blocks = int64_t(sm_count()) * per_sm;
  for (int64_t first = 0; first < num_tokens; first += most_tokens) {
    const int64_t tokens = num_tokens - first < most_tokens ? num_tokens - first : most_tokens;
    const int64_t items = (tokens + 3) / 4 * per_group, want = (items + kWarps - 1) / kWarps;
    const int rc = launch(first, static_cast<int>(tokens), static_cast<int>(items),
                          dim3(static_cast<unsigned>(want < most_blocks ? want : most_blocks)));
    if (rc != NVK_OK) return rc;
  }
  return NVK_OK;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace
}  // namespace fp4
}  // namespace nvk

extern "C" int nvk_fp4_append(const void* key, const void* value, int64_t key_token_stride,
                              int64_t value_token_stride, void* kv_cache, const int64_t* slot_mapping,
                              int64_t num_tokens, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                              int dtype, float k_scale, float v_scale, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp4;
  const char* who = "fp4_append";
  if (num_tokens < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)num_tokens);
  int rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, k_scale, v_scale, who);
  if (rc != NVK_OK) return rc;
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_FP16)
    return fail(NVK_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 rows only)", who, dtype);
  if (num_tokens == 0) return NVK_OK;
  if (!key || !value || !slot_mapping) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  const int64_t row = static_cast<int64_t>(num_kv_heads) * kD;
  if (!aligned8(slot_mapping)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: slots must be 8-byte aligned", who);
  if (!aligned4(key) || !aligned4(value) || key_token_stride % 2 || value_token_stride % 2 ||
      (num_tokens > 1 && (key_token_stride < row || value_token_stride < row)))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: rows must be 4-byte aligned and token strides (%lld, %lld) cover a row",
                who, (long long)key_token_stride, (long long)value_token_stride);
  AppendArgs a;
  a.key = static_cast<const uint8_t*>(key);
  a.value = static_cast<const uint8_t*>(value);
  a.key_stride = key_token_stride * 2;
  a.value_stride = value_token_stride * 2;
  a.pool = static_cast<uint8_t*>(kv_cache);
  a.slots = slot_mapping;
  a.num_slots = static_cast<int64_t>(num_blocks) * block_size;
  a.kvh = num_kv_heads;
  a.upb_log2 = units_log2(block_size);
  a.per_token = divisor(2 * num_kv_heads);
  a.k_inv = 1.f / k_scale;
  a.v_inv = 1.f / v_scale;
  a.err = error_word;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return in_launches(num_tokens, num_kv_heads, kAppendBlocks, [&](int64_t first, int tokens, int items, dim3 grid) {
    AppendArgs b = a;
    b.num_tokens = tokens;
    b.items = items;
    b.key += first * a.key_stride;
    b.value += first * a.value_stride;
    b.slots += first;
    return check_cuda(dtype == NVK_DTYPE_BF16 ? launch_pdl(append_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, b)
                                              : launch_pdl(append_kernel<__half>, grid, dim3(kThreads), 0, st, b),
                      "fp4_append launch");
  });
}

extern "C" int nvk_fp4_read(void* key, void* value, const void* kv_cache, const int64_t* slot_mapping,
                            int64_t num_tokens, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                            int dtype, float k_scale, float v_scale, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp4;
  const char* who = "fp4_read";
  if (num_tokens < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)num_tokens);
  int rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, k_scale, v_scale, who);
  if (rc != NVK_OK) return rc;
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_FP16)
    return fail(NVK_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 rows only)", who, dtype);
  if (num_tokens == 0) return NVK_OK;
  if (!key || !value || !slot_mapping) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(key) || !aligned16(value) || !aligned8(slot_mapping))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: the rows must be 16-byte aligned, the slots 8-byte aligned", who);
  ReadArgs a;
  a.key = static_cast<uint8_t*>(key);
  a.value = static_cast<uint8_t*>(value);
  a.pool = static_cast<uint8_t*>(const_cast<void*>(kv_cache));
  a.slots = slot_mapping;
  a.num_slots = static_cast<int64_t>(num_blocks) * block_size;
  a.kvh = num_kv_heads;
  a.upb_log2 = units_log2(block_size);
  a.per_token = divisor(2 * num_kv_heads);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.err = error_word;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return in_launches(num_tokens, num_kv_heads, kReadBlocks, [&](int64_t first, int tokens, int items, dim3 grid) {
    ReadArgs b = a;
    b.num_tokens = tokens;
    b.items = items;
    b.key += first * num_kv_heads * (kD * 2);
    b.value += first * num_kv_heads * (kD * 2);
    b.slots += first;
    return check_cuda(dtype == NVK_DTYPE_BF16 ? launch_pdl(read_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, b)
                                              : launch_pdl(read_kernel<__half>, grid, dim3(kThreads), 0, st, b),
                      "fp4_read launch");
  });
}

extern "C" int nvk_fp4_qk_norm_rope_append(const void* query, const void* key, const void* value,
                                           int64_t query_stride, int64_t key_stride, int64_t value_stride,
                                           const void* q_weight, const void* k_weight, float eps,
                                           const float* cos_table, const float* sin_table, int max_position,
                                           const int64_t* positions, void* query_out, void* kv_cache,
                                           const int64_t* slot_mapping, int64_t num_tokens, int num_blocks,
                                           int block_size, int num_heads, int num_kv_heads, int head_dim,
                                           float k_scale, float v_scale, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp4;
  const char* who = "fp4_qk_norm_rope_append";
  if (num_tokens < 0 || num_heads <= 0 || max_position <= 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (tokens=%lld heads=%d max_position=%d)", who,
                (long long)num_tokens, num_heads, max_position);
  int rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, k_scale, v_scale, who);
  if (rc != NVK_OK) return rc;
  if (num_tokens == 0) return NVK_OK;
  if (num_tokens > (int64_t(1) << 30) || num_heads > (1 << 20))  // the item index: 32 bits
    return fail(NVK_ERR_UNSUPPORTED, "%s: %lld tokens or %d heads are above the kernel's range", who,
                (long long)num_tokens, num_heads);
  if (!query || !key || !value || !q_weight || !k_weight || !cos_table || !sin_table || !positions || !query_out ||
      !slot_mapping)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned4(query) || !aligned4(key) || !aligned4(value) || !aligned4(q_weight) || !aligned4(k_weight) ||
      !aligned4(query_out) || !aligned4(cos_table) || !aligned4(sin_table) || !aligned8(positions) ||
      !aligned8(slot_mapping) || query_stride % 2 || key_stride % 2 || value_stride % 2 ||
      (num_tokens > 1 && (query_stride < int64_t(num_heads) * kD || key_stride < int64_t(num_kv_heads) * kD ||
                          value_stride < int64_t(num_kv_heads) * kD)))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: rows and tables must be 4-byte aligned, positions and slots 8-byte aligned, and strides cover a row",
                who);
  NormArgs a;
  a.q = static_cast<const uint8_t*>(query);
  a.k = static_cast<const uint8_t*>(key);
  a.v = static_cast<const uint8_t*>(value);
  a.q_stride = query_stride * 2;
  a.k_stride = key_stride * 2;
  a.v_stride = value_stride * 2;
  a.q_weight = static_cast<const uint8_t*>(q_weight);
  a.k_weight = static_cast<const uint8_t*>(k_weight);
  a.cos_table = cos_table;
  a.sin_table = sin_table;
  a.max_pos = max_position;
  a.positions = positions;
  a.slots = slot_mapping;
  a.q_out = static_cast<uint8_t*>(query_out);
  a.pool = static_cast<uint8_t*>(kv_cache);
  a.num_slots = static_cast<int64_t>(num_blocks) * block_size;
  a.num_heads = num_heads;
  a.kvh = num_kv_heads;
  a.upb_log2 = units_log2(block_size);
  a.eps = eps;
  a.k_inv = 1.f / k_scale;
  a.v_inv = 1.f / v_scale;
  a.err = error_word;
  const int sms = sm_count();
  const int rounds = (num_heads + 3) / 4 + 2 * ((num_kv_heads + 3) / 4);
  // A token's rounds in `chunks` items of `chunk`: the split for which the warps of one resident wave end first, an
  // item's start (position, slot, the cos and sin rows) weighing a little more than a round. With 8 rounds a token:
  // 2048 tokens whole 10.5 us, in eighths 15.5; 2400 whole 15.8, in halves 14.1; 32768 whole 116.5, in halves 125.7.
  // A finer split has to win a thirty-second, which is as far as this estimate goes. Followed by the prefill attention
  // of a step (sequences of 256 over 768 cached tokens), coarser and finer, with the share that the estimate says:
  // 16 + 2 * 8 heads, 1500 tokens 35.3 and 34.0 (9 %), 5000 110.9 and 109.2 (6 %), 8192 116.3 and 115.6 (1 %; alone
  // 35.5 and 34.3, followed by a read of the rows 43.5 and 44.7); 32 + 2 * 8, 2400 tokens 83.8 and 81.9 (4 %), 10000
  // 236.6 and 238.1 (2 %; alone 54 and 61); 5 + 2 * 1, 2400 tokens 32.8 and 30.4 (8 %); 40 + 2 * 8, 8192 tokens 338.5
  // and 338.9 (6 %).
  const int64_t warps = int64_t(sms) * 2 * kWarps;
  int64_t best = 0;
  for (int n = 1; n <= rounds; n = n < 8 ? n + 1 : n < rounds && 2 * n > rounds ? rounds : 2 * n) {
    const int chunk = (rounds + n - 1) / n, chunks = (rounds + chunk - 1) / chunk;
    const int64_t cost = (num_tokens * chunks + warps - 1) / warps * (6 * chunk + 7);
    if (chunks > 1 && (cost >= best - best / 32 || num_tokens * chunks > kMostItems)) continue;
    best = cost, a.chunk = chunk, a.chunks = chunks;
  }
  a.items = static_cast<int>(num_tokens) * a.chunks;
  a.per_token = divisor(a.chunks);
  // 16-byte copies where every row and table allows them
  const bool wide = aligned16(query) && aligned16(key) && aligned16(value) && aligned16(cos_table) &&
                    aligned16(sin_table) && query_stride % 8 == 0 && key_stride % 8 == 0 && value_stride % 8 == 0;
  const void* kernel = wide ? reinterpret_cast<const void*>(&norm_rope_kernel<true>)
                            : reinterpret_cast<const void*>(&norm_rope_kernel<false>);
  if ((rc = ensure_dynamic_smem(kernel, sizeof(NormSmem))) != NVK_OK) return rc;
  const int want = (a.items + kWarps - 1) / kWarps, most = sms * 2;  // one resident wave
  const dim3 grid(want < most ? want : most);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return check_cuda(wide ? launch_pdl(norm_rope_kernel<true>, grid, dim3(kThreads), sizeof(NormSmem), st, a)
                         : launch_pdl(norm_rope_kernel<false>, grid, dim3(kThreads), sizeof(NormSmem), st, a),
                    "fp4_qk_norm_rope_append launch");
}
