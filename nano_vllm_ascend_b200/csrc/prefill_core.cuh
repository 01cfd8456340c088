// Causal prefill attention on the sm_100a tensor cores (tcgen05 + TMEM): the
// kernel body of paged_prefill.cu (bf16 K and V, copied by TMA) and of
// fp4_prefill.cu and fp8_prefill.cu (the 4- and 8-bit pools, whose tiles a
// warpgroup of their own decodes into the same shared-memory layout).
//
// Replaces torch_npu.npu_fused_infer_attention_score as called from
// src/nanovllm_ascend/layers/npu_prefill_attention.py:82-112 (TND layout,
// sparse_mode=3): paged mode reads the whole KV of a sequence (cached prefix
// + rows appended this step) through its block table with absolute kv
// lengths; dense mode reads contiguous K/V rows delimited by cumulative
// lengths. Masking is bottom-right aligned: query i of a sequence with Lq
// queries and Lk keys sees key j iff j <= Lk - Lq + i.
//
// Work item = 128 query rows of one sequence x two query heads of one GQA
// group ("streams" 0 and 1; one stream when the group size is odd). Both
// streams read the same 128-key K and V tiles (one pool block each), so each
// K/V byte staged in shared memory feeds two heads. The grid is persistent
// (one CTA per SM); CTA c takes items c, c + C, c + 2C, ... in an order that
// puts the heaviest query tiles first.
// Tensor memory (512 columns): S/P of stream s at s * 128, its O accumulator
// at 256 + s * 128.
//   warp 8 (producer): walks the item list and publishes each item's
//     descriptor through a 4-slot shared-memory ring (the other roles never
//     read the item metadata from global memory); per item the TMA loads of
//     the streams' Q tiles (once the previous item's last S has read their
//     buffers), then per key tile the K and V tiles (two 64-dim halves each,
//     128-byte swizzle = the canonical UMMA operand layout) into 2-stage
//     rings; block ids 32 at a time (one parallel load per warp).
//   warp 9 (MMA; the whole warp runs the loop, an elected lane issues):
//     per tile j and stream s, once the first 64 keys of P_s(j) are written,
//     O_s += P V over them, then over the other 64 (P read from TMEM where
//     the softmax wrote it over S_s, V MN-major from smem), and right behind
//     it S_s(j+1) = Q_s K(j+1)^T into the same columns. tcgen05.mma executes
//     in issue order, so S_s(j+1) overwrites P_s(j) only after the P V has
//     read it, and the tensor pipe has the other stream's work queued while
//     one stream's softmax runs. An item's first S tiles are issued behind
//     the previous item's last P V.
//   warps 0-3 / 4-7 (softmax of stream 0 / 1): thread r owns query row r =
//     TMEM lane r. Per tile the 128 scores of its row in one round of
//     tcgen05.ld, the mask, base-2 online softmax, P written as bf16 pairs
//     over the first 64 columns of S_s (tcgen05.st) in two halves, each
//     signalled once stored; lazy rescaling of O_s (only when the running
//     max grew by more than 2^8; S_s(j) having landed means P V_s(j-1),
//     issued before it, is complete). Per item, once its last P V_s has
//     completed, the normalised O_s rows go out through a staging buffer, 32
//     dims at a time: each warp stores the 64-byte pieces of the 32 rows that
//     its own lanes staged, eight per instruction (coalesced), and O_s is
//     released to the next item.
// Ten warps put three on one SM sub-partition, whose register file holds
// 3 x 32 x 168 registers: the kernel is held to 168 registers a thread.
//   4-bit pool, warps 12-15 (decoders; warps 10 and 11 idle): thread r owns
//     token row r of each K and V tile. It loads the row's packed words
//     straight into registers one tile ahead (in flight while the other of K
//     and V is decoded), turns them into fp16, which holds the values exactly,
//     and stores them where the TMA copy of a tile would have put them. All
//     operands are fp16 then: the softmax warps turn the next item's Q rows
//     into fp16, each scaled by a power of two into its range, between an
//     item's last P and its output, and P is fp16, three bits more exact than
//     bf16. Items are published one earlier, so that the next item's first
//     tiles are decoded behind this one's last. 16 warps have 128 registers a
//     thread at launch: the softmax warpgroups take 176, the other two give
//     them up.
//   8-bit pool: the same, but that a decoding warp has 32 token rows, two
//     units, and stores the codes as they are, as fp16; the softmax warps take
//     the units' exponents (see decode_chunks).
// What bounds it: the chain softmax -> P V + S -> softmax of a stream, of which
// two overlap (tensor pipe 42 % of active cycles, exp unit 43 %, issue 46 % with
// 4-bit K and V), and instruction fetch: 70 KB of code (4-bit), of which warps
// wait for what they run once an item. That is why the rare parts are short
// loops and one elected thread issues a whole product. Code that the roles ran
// in line before (masks over all registers, an election for every step, Q in
// the decoders): 89.8 us against 82.5 for 32 x 256 queries over 1024 keys, 16
// heads on 8 (60.2 GFLOP; with bf16 K and V 75.1 against 73.6). Exponents and
// sums two values an instruction: 80 us (with eight registers more for the
// softmax; 85 with spills of one), bf16 71.5, the same bits. Scores of any
// magnitude and NaN of V that a query does not see: 81.3 -> 82.1 -> 82.45 us.
// Measured and not taken for the 4-bit kernel, same work: scores read twice in
// a loop instead of held in registers 91.4 us; each thread storing its output
// row directly 98.2; Q by the two idle warps 86.2 or by the decoders 83.2 to
// 85.4; one loop over the tiles of all items 95.5; the upper half of the next S
// issued before the end of P 89.4 (products of 64 columns take as long as of
// 128); against 80: Q's largest exponents by the idle warps 82; a quarter of
// the exponentials as a polynomial, two values an instruction, 83 (left out
// altogether 79.6: the exponential unit is not what it waits for).
// Every mbarrier wait is bounded; on a timeout the CTA records the error,
// drains its in-flight copies and MMAs, frees TMEM and exits.
#pragma once

#include <climits>
#include <cstddef>

#include "fp4_kv.cuh"
#include "fp8_kv.cuh"
#include "host_common.h"
#include "nvk_common.cuh"
#include "tcgen05.cuh"

namespace nvk {
namespace prefill {

// What K and V are held in: bf16 rows, the 4-bit pool, the 8-bit pool. The latter two are decoded by warps of the kernel.
enum Held { kHeldBf16, kHeldFp4, kHeldFp8 };

constexpr int kD = 128;
constexpr int kRows = 128;                // query rows per item (UMMA M)
constexpr int kKeys = 128;                // keys per K/V tile: one 128-token pool block
constexpr int kHalfBytes = 128 * 128;     // one 64-dim half of a 128-row tile
constexpr int kTileBytes = 2 * kHalfBytes;
constexpr int kStages = 2;                // K and V ring depth
constexpr int kStreams = 2;               // query heads per item
constexpr int kStreamThreads = 128;       // softmax threads per stream
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kThreads = 10 * 32;
constexpr int kDecodeWarp0 = 12;          // quantised pools: warps 12-15
constexpr int kThreadsDecoding = 16 * 32;
// Registers a thread after the split of the decoding kernels' 512 x 128 (softmax, softmax, producer and MMA, decoders)
constexpr int kRegsSoftmax = 176, kRegsIssue = 64, kRegsDecode = 96;
// (8-bit: 184, 56 and 88 take 96.9 us for 97.4, within what repeats of one differ by, so that both kernels share one
// split; 184, 48 and 96 108.8, 168, 64 and 112 106.7: what is spilled)
static_assert(2 * kRegsSoftmax + kRegsIssue + kRegsDecode <= 4 * 128, "setmaxnreg shares exceed the launch's registers");
constexpr uint32_t kTmemCols = 512;       // S_0 | S_1 | O_0 | O_1, 128 columns each
constexpr uint32_t kColO = 256;
constexpr float kRescaleThreshold = 8.0f;
// 8-bit kernel: bounds of the factor from products to scores. Products are sums of 128 of rows below 2^16 and codes of
// up to 448 * 2^40, so below 2^72: at the least factor, which is normal times 2^-40, all scores are within 2^-14 of 0
// (weights round by 2^-11), and at the largest their differences stay finite.
constexpr float kLeastFactor = 0x1p-86f, kMostFactor = 0x1p53f;
constexpr float kFarScore = 1024.f;       // decoding kernels: scores whose rounding in fp32, 2^-14, would show in a weight
constexpr int kItemRing = 4;              // item descriptors published ahead by the producer

struct PrefillArgs {
  __nv_bfloat16* out;
  const int32_t* block_tables;
  const int32_t* cu_q;
  const int32_t* kv_lens;  // paged: absolute kv length per sequence
  const int32_t* cu_kv;    // dense: cumulative kv rows
  int* err;
  int bt_stride;
  int num_blocks;
  int num_heads;
  int qpk;
  int paired;  // two heads per item (GQA group size even)
  int paged;
  int batch;
  int qtiles;  // query tiles of the longest sequence
  float scale_log2;
  // a quantised pool
  const uint8_t* pool;
  int kvh, upb_log2, max_blocks, total_q;
  float out_scale;
};

// One work item: query tile qt of heads h0 .. h0 + streams - 1 of sequence b
// (n_kv < 0: no further item).
struct Item {
  int qt, h0, kvh, b, q0, lq, lk, kv_row0, n_kv;
  int k0;  // divided items: this CTA's first key, n_kv its tiles
};

struct PrefillSmem {
  alignas(1024) uint8_t q[kStreams][kTileBytes];
  alignas(1024) uint8_t k[kStages][kTileBytes];
  alignas(1024) uint8_t v[kStages][kTileBytes];
  alignas(1024) uint8_t stage[kStreams][kHalfBytes];  // epilogue: 64 dims of 128 output rows per stream
  Item items[kItemRing];
  alignas(16) uint8_t exps[4][2][kKeys / fp8::kUnitTokens];  // 8-bit pool, tile g at g % 4: K's and V's units, + 127
  alignas(16) int nan_from[kItemRing][fp4::kGroups];       // quantised pools: the first token that has a NaN in V's
                                                           // group (4 bits), or in V (8 bits: the first entry)
  uint64_t item_full[kItemRing];                 // items[i % ring] written (one phase per use)
  uint64_t q_full[kStreams], q_empty[kStreams];  // one phase per item
  uint64_t q_ready[kStreams];                    // 4-bit pool: Q_s is fp16 (one phase per item)
  uint64_t full_k[kStages], k_empty[kStages];
  uint64_t full_v[kStages], v_empty[kStages];
  uint64_t s_full[kStreams];   // S_s(j) in TMEM (and, in issue order, P V_s(j-1) done)
  uint64_t p_lo[kStreams];     // P_s(j) of keys 0-63 written by the stream's 128 softmax threads
  uint64_t p_hi[kStreams];     // P_s(j) of keys 64-127 written
  uint64_t o_ready[kStreams];  // an item's last P V_s complete (one phase per item)
  uint64_t o_free[kStreams];   // an item's O_s read out (one phase per item)
  uint64_t fin;
  uint32_t tmem_base;
  volatile int abort;
  Item whole;                  // divided items: the cluster's item
  int parts;                   // and how many CTAs hold a part of it
};

static_assert(sizeof(PrefillSmem) + 1024 <= 232448, "prefill shared memory exceeds one SM's 227 KB");

// The producer walks the item list; `next_item` skips items without rows and
// hands the ones whose rows see no key to `zero_rows`.
__device__ __forceinline__ int item_streams(const PrefillArgs& a) { return a.paired ? kStreams : 1; }

template <bool kDecoding>
__device__ __forceinline__ bool load_item(const PrefillArgs& a, int w, Item& it) {
  const int ns = item_streams(a);
  const int groups = a.num_heads / ns;  // head groups per sequence
  const int per_tile = groups * a.batch;
  const int t = w / per_tile;
  it.qt = a.qtiles - 1 - t;  // heaviest (last) query tiles first
  const int rem = w - t * per_tile;
  it.h0 = (rem % groups) * ns;
  it.kvh = it.h0 / a.qpk;  // both heads of a pair share it: h0 even, group size even
  it.b = rem / groups;
  it.q0 = a.cu_q[it.b];
  it.lq = a.cu_q[it.b + 1] - it.q0;
  // (asked at run time: without the question the bf16 kernel, which never gets in, takes 0.4 us of 74 longer)
  if (a.pool && it.lq > 0 && (it.q0 < 0 || it.lq > a.total_q - it.q0)) {  // rows that the query does not have
    if (a.err) atomicOr(a.err, kErrContextTooLong);
    return false;
  }
  if (it.qt * kRows >= it.lq) return false;
  it.lk = a.paged ? a.kv_lens[it.b] : (a.cu_kv[it.b + 1] - a.cu_kv[it.b]);
  if constexpr (kDecoding) {  // a length is held to [0, what the table reaches]: it bounds the item's work and the sums below
    const int64_t room = static_cast<int64_t>(a.max_blocks) << (a.upb_log2 + 4);
    if (it.lk > room) {
      if (a.err) atomicOr(a.err, kErrContextTooLong);
      it.lk = static_cast<int>(room);
    }
    it.lk = max(it.lk, 0);
  }
  it.kv_row0 = a.paged ? 0 : a.cu_kv[it.b];
  const int i_last = min(it.qt * kRows + kRows - 1, it.lq - 1);
  const int lim_last = min(it.lk - it.lq + i_last, it.lk - 1);
  it.n_kv = lim_last < 0 ? 0 : lim_last / kKeys + 1;
  return true;
}

template <bool kDecoding, typename ZeroRows>
__device__ __forceinline__ bool next_item(const PrefillArgs& a, int& w, int step, int total, Item& it,
                                          ZeroRows&& zero_rows) {
  for (; w < total; w += step) {
    if (!load_item<kDecoding>(a, w, it)) continue;
    if (it.n_kv == 0) {
      zero_rows(it);
      continue;
    }
    return true;
  }
  return false;
}

// The first 16 of 32 registers into 16 consecutive 32-bit TMEM columns of
// this thread's lane (warp-collective).
__device__ __forceinline__ void tmem_st16_first(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void flag_error(const PrefillArgs& a, PrefillSmem& sm, int code) {
  if (a.err) atomicOr(a.err, code);
  sm.abort = 1;
}

// The decoding kernels hold P as 2^7 p: p is at most 2^8 (see kRescaleThreshold),
// so fp16 takes it, with 11 bits down to p = 2^-21. (8-bit kernel: p 2^e in p's
// place. The largest one is held as 2^7 or more, so that a weight is off by
// 2^-11 of itself or by 2^-32 of the largest one, half of fp16's least step.)
template <bool kDecoding>
constexpr float kPShift = kDecoding ? 7.f : 0.f;

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr uint32_t umma_idesc_ab_bf16 = (1u << 7) | (1u << 10);

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// One token row of the 4-bit pool in registers: K (or V) codes and scales.
struct KRow {
  uint4 w[4];
  uint2 s;
};
struct VRow {
  uint2 w[8];
  uint4 s[2];  // the scales of the four tokens of its quad
};

__device__ __forceinline__ void load_row(KRow& k, const uint8_t* unit, int i) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
    k.w[t] = unit ? *reinterpret_cast<const uint4*>(unit + 64 * i + 16 * t) : make_uint4(0, 0, 0, 0);
  k.s = unit ? *reinterpret_cast<const uint2*>(unit + fp4::kOffKScale + 8 * i) : make_uint2(0, 0);
}
__device__ __forceinline__ void load_row(VRow& v, const uint8_t* unit, int i) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    v.w[g] = unit ? *reinterpret_cast<const uint2*>(unit + fp4::kOffV + 256 * (i >> 2) + 32 * g + 8 * (i & 3))
                  : make_uint2(0, 0);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    v.s[h] = unit ? *reinterpret_cast<const uint4*>(unit + fp4::kOffVScale + 32 * (i >> 2) + 16 * h)
                  : make_uint4(0, 0, 0, 0);
}

// Scale bytes of groups 2 k and 2 k + 1 (low two bytes of w), each as a pair of fp16; a NaN as 0 with kNoNan.
template <bool kNoNan = false>
__device__ __forceinline__ void scale_pairs(uint32_t w, uint32_t& s0, uint32_t& s1) {
  uint32_t lo, hi;
  fp4::e4m3_to_half2(w, lo, hi);
  if (kNoNan) asm("max.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0u));
  s0 = __byte_perm(lo, lo, 0x1010);
  s1 = __byte_perm(lo, lo, 0x3232);
}

// Eight codes (dims ascending from the low nibble) of one group into chunk c
// (dims 8 c .. 8 c + 7) of token row r of a tile in the 128-byte-swizzled layout.
__device__ __forceinline__ void put_chunk(uint32_t tile, int r, int c, uint32_t codes, uint32_t s) {
  uint32_t o[4];
  fp4::e2m1_to_half2(codes, o[0], o[1], o[2], o[3]);
  st_shared_v4(tile + (c >> 3) * kHalfBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4), fp4::hmul2(o[0], s),
               fp4::hmul2(o[1], s), fp4::hmul2(o[2], s), fp4::hmul2(o[3], s));
}

// Row r of a Q tile from bf16 to fp16 in place (see fp4_kv.cuh); returns what
// its scores have to be multiplied by. Short loops: fetching this code, once an
// item, costs as much as running it.
__device__ __forceinline__ float q_row_to_half(uint32_t tile, int r) {
  auto chunk = [&](int c) { return tile + (c >> 3) * kHalfBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
  uint32_t big = 0;
#pragma unroll 1
  for (int c0 = 0; c0 < 16; c0 += 4)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 v = ld_shared_v4(chunk(c0 + c));
      big = fp4::bf16x2_abs_max(fp4::bf16x2_abs_max(big, fp4::bf16x2_abs_max(v.x, v.y)),
                                fp4::bf16x2_abs_max(v.z, v.w));
    }
  const fp4::HalfRow row = fp4::half_row(big);
  auto half = [&](uint32_t w) { return fp4::bf16x2_to_half2(w, row.base); };
#pragma unroll 1
  for (int c0 = 0; c0 < 16; c0 += 2) {
    const uint32_t at0 = chunk(c0), at1 = chunk(c0 + 1);
    const uint4 u = ld_shared_v4(at0), v = ld_shared_v4(at1);
    st_shared_v4(at0, half(u.x), half(u.y), half(u.z), half(u.w));
    st_shared_v4(at1, half(v.x), half(v.y), half(v.z), half(v.w));
  }
  return row.up;
}

__device__ __forceinline__ void decode_row(const KRow& k, uint32_t tile, int r) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(k.w);  // word 4 t + p: groups 2 p and 2 p + 1
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t s[2];
    scale_pairs((p < 2 ? k.s.x : k.s.y) >> (16 * (p & 1)), s[0], s[1]);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        put_chunk(tile, r, 2 * (2 * p + e) + h, __byte_perm(w[8 * h + p], w[8 * h + 4 + p], e ? 0x7632 : 0x5410), s[e]);
  }
}
// The row's own scale bytes, of groups 0 to 3 and 4 to 7.
__device__ __forceinline__ uint2 scale_bytes(const VRow& v, int r) {
  const uint32_t pick = (r & 3) | ((4 + (r & 3)) << 4);  // v.s: word j holds group j of the quad's four tokens
  auto four = [&](const uint4& w) {
    return __byte_perm(__byte_perm(w.x, w.y, pick), __byte_perm(w.z, w.w, pick), 0x5410);
  };
  return make_uint2(four(v.s[0]), four(v.s[1]));
}
// A group of V whose scale is NaN is decoded as zeros: a weight of 0 times NaN
// would reach the queries that do not see the row. Its token is noted for the
// output, which turns to NaN where a query sees it.
__device__ __forceinline__ void note_nan(uint2 bytes, int token, int* nan_from) {
  if (((bytes.x + 0x01010101u) | (bytes.y + 0x01010101u)) & 0x80808080u) {  // from 0x7f alone
#pragma unroll 1
    for (int j = 0; j < fp4::kGroups; ++j) {
      if ((bytes.x & 0x7fu) == 0x7fu) atomicMin(nan_from + j, token);
      bytes.x = __funnelshift_r(bytes.x, bytes.y, 8);
      bytes.y >>= 8;
    }
  }
}
__device__ __forceinline__ void decode_row(const VRow& v, uint2 bytes, uint32_t tile, int r) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {  // groups 4 q .. 4 q + 3
    uint32_t s[4];
    scale_pairs<true>(q ? bytes.y : bytes.x, s[0], s[1]);
    scale_pairs<true>((q ? bytes.y : bytes.x) >> 16, s[2], s[3]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // dims 8 h .. 8 h + 7 of each group: a 4 x 4 transpose of bytes
      uint32_t x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = q ? v.w[4 * h + k].y : v.w[4 * h + k].x;
      const uint32_t a0 = __byte_perm(x[0], x[1], 0x5140), a1 = __byte_perm(x[0], x[1], 0x7362);
      const uint32_t b0 = __byte_perm(x[2], x[3], 0x5140), b1 = __byte_perm(x[2], x[3], 0x7362);
      put_chunk(tile, r, 2 * (4 * q + 0) + h, __byte_perm(a0, b0, 0x5410), s[0]);
      put_chunk(tile, r, 2 * (4 * q + 1) + h, __byte_perm(a0, b0, 0x7632), s[1]);
      put_chunk(tile, r, 2 * (4 * q + 2) + h, __byte_perm(a1, b1, 0x5410), s[2]);
      put_chunk(tile, r, 2 * (4 * q + 3) + h, __byte_perm(a1, b1, 0x7632), s[3]);
    }
  }
}

// The 8-bit pool: a decoding warp has the tile's tokens 32 w .. 32 w + 31, two
// units, in eight loads of 512 contiguous bytes: a lane takes a chunk of 16
// codes of four tokens a unit, such that eight lanes write two rows of four
// chunks each to the tile, without bank conflicts. The codes become fp16 as they
// are (one conversion for two), and the units' exponents go to the softmax
// warps, which take K's into the factor of the unit's 16 scores and V's into
// the exponents of its weights.
// A lane's token (of the four in 512 bytes) and chunk.
__device__ __forceinline__ int chunk_row(int lane) { return 2 * (lane >> 4) + (lane >> 2 & 1); }
__device__ __forceinline__ int chunk_of(int lane) { return 4 * (lane >> 3 & 1) + (lane & 3); }

struct Chunks {
  uint4 w[8];
};
// Load i of part 0 (K) or 1 (V) of two units: the tokens from `seen` on as zeros.
__device__ __forceinline__ uint4 load_chunk(const uint8_t* const (&unit)[2], int i, int part, int seen, int lane) {
  const uint8_t* from = unit[i >> 2];
  const int row = chunk_row(lane);
  return from && 4 * i + row < seen
             ? *reinterpret_cast<const uint4*>(from + part * fp8::kOffV + fp8::chunk_at(4 * (i & 3) + row, chunk_of(lane)))
             : make_uint4(0, 0, 0, 0);
}

// Chunks to the tile, from its token row r0 on, each followed by the load that
// takes its registers: `next(i)`. A row with a NaN holds nothing else: V's
// becomes zeros and its token is noted (see note_nan).
template <bool kIsV, typename Next>
__device__ __forceinline__ void decode_chunks(Chunks& x, uint32_t tile, int r0, int token, int* nan_from, int lane,
                                              Next&& next) {
  const int k = chunk_row(lane), l = chunk_of(lane);  // dims 16 l .. 16 l + 15
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint4 w = x.w[i];
    x.w[i] = next(i);
    if (kIsV && (w.x & 0x7fu) == 0x7fu) {
      w = make_uint4(0, 0, 0, 0);
      atomicMin(nan_from, token + 4 * i + k);
    }
    const int r = r0 + 4 * i + k;
    const uint32_t at = tile + (l >> 2) * kHalfBytes + r * 128 + (((2 * (l & 3)) ^ (r & 7)) << 4);
    auto eight = [&](uint32_t to, uint32_t a, uint32_t b) {
      uint32_t h[4];
      fp4::e4m3_to_half2(a, h[0], h[1]);
      fp4::e4m3_to_half2(b, h[2], h[3]);
      st_shared_v4(to, h[0], h[1], h[2], h[3]);
    };
    eight(at, w.x, w.y);
    eight(at ^ 16, w.z, w.w);
  }
}

// Divided items (8-bit pool): where there are few items, a cluster of CTAs takes
// one, each a run of its key tiles. Each leaves its O and softmax statistics in
// its shared memory, over the K and V tiles; then every CTA puts a share of the
// rows together, from all of them over distributed shared memory, the largest
// reference first as within a tile. A tile takes 2.0 us, the clusters' start,
// barriers and join 3 to 7: an item is divided where that saves kSavedTiles or
// more. (45 items on clusters of three: 10 tiles each 20.9 us, undivided 26.1; 8
// tiles 19.6 and 22.0; 6 tiles 18.2 and 18.0. Nine items on clusters of eight: 6
// tiles 11.9 and 17.6, 20 tiles 15.8 and 45.9. 128 queries over 8192 keys, 16
// heads on 8: 31.9 and 146; one query over 4097 19.4 and 78; 16 over 32784 96
// and 612.)
constexpr int kSavedTiles = 4, kMostParts = 8;
struct Part {
  float m, exp, l, sc;
};
__device__ __forceinline__ uint32_t part_chunk(int row, int c) {  // four dims of a row of O: offset in sm.k
  return row * (kD * 4) + ((c ^ (row & 7)) << 4);
}

// The output rows of this CTA, a share of the item's, by warps 0 to 7: a lane
// takes a part's statistics (of eight at most), then four dims of all parts. Not
// in line: its registers would be spilled in the softmax's loop (20 tiles of one
// CTA 54.2 us instead of 46.1).
[[maybe_unused]] static __device__ __noinline__ void join_parts(const PrefillArgs& a, PrefillSmem& sm, int rank, int ranks) {
  const Item& it = sm.whole;
  const int rows = min(kRows, it.lq - it.qt * kRows), share = (kRows + ranks - 1) / ranks, parts = sm.parts;
  const uint32_t o_at = smem_u32(sm.k), part_at = smem_u32(sm.v);
  const int lane = threadIdx.x & 31, p = lane & 7;
  const int end = min(rows, (rank + 1) * share);
#pragma unroll 1
  for (int row = rank * share + (threadIdx.x >> 5); row < end; row += 8) {
    const float4 x =
        p < parts ? ld_cluster_f4(part_at + row * sizeof(Part), p) : make_float4(0.f, -INFINITY, 0.f, 0.f);  // Part
    float4 y[kMostParts];
#pragma unroll
    for (int k = 0; k < kMostParts; ++k)
      y[k] = k < parts ? ld_cluster_f4(o_at + part_chunk(row, lane), k) : make_float4(0.f, 0.f, 0.f, 0.f);
    const bool any = x.y != -INFINITY;  // the row sees a key of the part
    float to = any ? x.x : -INFINITY;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, off));
    const float ref = any ? fmaf(x.x - to, x.w, x.y) : -INFINITY;
    float most = ref;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    const float by = any ? fast_exp2(ref - most) : 0.f;
    float l = x.z * by;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kMostParts; ++k) {
      const float w = __shfl_sync(0xffffffffu, by, k);
      o.x = fmaf(y[k].x, w, o.x), o.y = fmaf(y[k].y, w, o.y), o.z = fmaf(y[k].z, w, o.z), o.w = fmaf(y[k].w, w, o.w);
    }
    const float inv = l == 0.f ? 0.f : a.out_scale / l;
    __nv_bfloat16* out = a.out + (static_cast<int64_t>(it.q0 + it.qt * kRows + row) * a.num_heads + it.h0) * kD + 4 * lane;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
}

// kmap and vmap are read by the bf16 kernel only. kClusters: launched in clusters,
// each of which has at most one item, of one stream.
template <Held kHeld, bool kClusters = false>
__device__ __forceinline__ void prefill_body(const CUtensorMap& qmap, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                             const PrefillArgs& a) {
  constexpr bool kFp4 = kHeld == kHeldFp4;
  constexpr bool kDecoding = kHeld != kHeldBf16;  // fp16 operands
  constexpr bool kExps = kHeld == kHeldFp8;       // a tile's units have exponents
  pdl_launch_dependents();
  pdl_wait();
  const int ns = kClusters ? 1 : item_streams(a);
  const int total = a.qtiles * (a.num_heads / ns) * a.batch;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  extern __shared__ uint8_t smem_raw[];
  PrefillSmem& sm =
      *reinterpret_cast<PrefillSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full_k[s], kDecoding ? 128 : 1);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.full_v[s], kDecoding ? 128 : 1);
      mbar_init(&sm.v_empty[s], 1);
    }
    for (int s = 0; s < kStreams; ++s) {
      mbar_init(&sm.q_full[s], 1);
      mbar_init(&sm.q_ready[s], kStreamThreads);
      mbar_init(&sm.q_empty[s], 1);
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.p_lo[s], kStreamThreads);
      mbar_init(&sm.p_hi[s], kStreamThreads);
      mbar_init(&sm.o_ready[s], 1);
      mbar_init(&sm.o_free[s], kStreamThreads);
    }
    for (int i = 0; i < kItemRing; ++i) mbar_init(&sm.item_full[i], 1);
    mbar_init(&sm.fin, 1);
    sm.abort = 0;
    if constexpr (kClusters) sm.parts = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&sm.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  // The decoding kernels' register split: each role's branch starts with its
  // share (all four warps of a warpgroup name the same one).
  constexpr bool kSplit = kDecoding;

  if (warp == kProducerWarp) {
    // -------------------------------------------------------- producer ----
    if constexpr (kSplit) regs_dec<kRegsIssue>();
    if (lane == 0) {
      tma_prefetch_desc(&qmap);
      if constexpr (!kDecoding) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
      }
    }
    // Rows of an item that sees no key: zeros (two rows per warp instruction).
    auto zero_rows = [&](const Item& z) {
      const int rows = min(kRows, z.lq - z.qt * kRows);
      for (int s = 0; s < ns; ++s)
        for (int rr = lane >> 4; rr < rows; rr += 2) {
          __nv_bfloat16* row = a.out + (static_cast<int64_t>(z.q0 + z.qt * kRows + rr) * a.num_heads + z.h0 + s) * kD;
          *reinterpret_cast<uint4*>(row + (lane & 15) * 8) = make_uint4(0, 0, 0, 0);
        }
    };
    const int rank = kClusters ? cluster_rank() : 0, ranks = kClusters ? cluster_size() : 1;
    const int step = kClusters ? gridDim.x / ranks : gridDim.x;
    int w = kClusters ? blockIdx.x / ranks : blockIdx.x, qi = 0, g = 0, k_issued = 0, v_issued = 0;
    int q_extra = 0;  // streams that have a load of item qi, where that is not all of them
    bool ok = true;
    while (true) {
      Item it;
      bool have = next_item<kDecoding>(a, w, step, total, it, zero_rows);
      if constexpr (kClusters) {
        if (have) {
          int per = (it.n_kv + ranks - 1) / ranks;
          if (it.n_kv - per < kSavedTiles) per = it.n_kv;
          if (lane == 0) {
            sm.whole = it;
            sm.parts = (it.n_kv + per - 1) / per;
          }
          it.k0 = rank * per * kKeys;
          it.n_kv = min(per, it.n_kv - rank * per);
          have = it.n_kv > 0;
        }
      }
      if (lane == 0) {
        // The Q buffers, and with them the ring slot (read by every role
        // before the previous item's last S), are free once the previous
        // item's last S of each stream has completed. A decoding kernel fills
        // the slot before that wait: its last user, four items back, was done
        // when the last S of the item before the previous one had completed,
        // for which this loop has waited already.
        if (!kDecoding)
          for (int s = 0; s < ns && ok && qi > 0; ++s)
            if (!mbar_wait(&sm.q_empty[s], (qi - 1) & 1)) ok = false;
        Item& slot = sm.items[qi % kItemRing];
        slot = it;
        if (!have || !ok) slot.n_kv = -1;
        if constexpr (kDecoding) {
          int4* from = reinterpret_cast<int4*>(sm.nan_from[qi % kItemRing]);
          from[0] = from[1] = make_int4(INT_MAX, INT_MAX, INT_MAX, INT_MAX);
        }
        mbar_arrive(&sm.item_full[qi % kItemRing]);
        if (have && ok) {
          for (int s = 0; s < ns; ++s) {
            if (kDecoding && qi > 0 && !mbar_wait(&sm.q_empty[s], (qi - 1) & 1)) {
              ok = false;
              q_extra = s;
              break;
            }
            mbar_arrive_expect_tx(&sm.q_full[s], kTileBytes);
            tma_load_3d(sm.q[s], &qmap, &sm.q_full[s], 0, it.h0 + s, it.q0 + it.qt * kRows);
            tma_load_3d(sm.q[s] + kHalfBytes, &qmap, &sm.q_full[s], 64, it.h0 + s, it.q0 + it.qt * kRows);
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!have || !ok) break;
      if constexpr (!kDecoding) {
        const int32_t* bt = a.block_tables + static_cast<int64_t>(it.b) * a.bt_stride;
        int ids = 0;
        for (int j = 0; ok && j < it.n_kv; ++j, ++g) {
          if (__shfl_sync(0xffffffffu, sm.abort, 0)) { ok = false; break; }
          if ((j & 31) == 0 && a.paged) {  // block ids of tiles j .. j+31, one per lane
            const int jj = j + lane;
            int blk = 0;
            if (jj < it.n_kv) {
              blk = bt[jj];
              if (blk < 0 || blk >= a.num_blocks) {
                if (a.err) atomicOr(a.err, kErrBadBlockId);
                blk = a.num_blocks;  // fully outside the tensor map: zero fill
              }
            }
            ids = blk;
          }
          const int blk = __shfl_sync(0xffffffffu, ids, j & 31);
          const int row = a.paged ? blk * kKeys : it.kv_row0 + j * kKeys;
          const int st = g % kStages;
          if (lane == 0) {
            if (g >= kStages && !mbar_wait(&sm.k_empty[st], ((g / kStages) - 1) & 1)) {
              ok = false;
            } else {
              mbar_arrive_expect_tx(&sm.full_k[st], kTileBytes);
              tma_load_3d(sm.k[st], &kmap, &sm.full_k[st], 0, it.kvh, row);
              tma_load_3d(sm.k[st] + kHalfBytes, &kmap, &sm.full_k[st], 64, it.kvh, row);
              ++k_issued;
              if (g >= kStages && !mbar_wait(&sm.v_empty[st], ((g / kStages) - 1) & 1)) {
                ok = false;
              } else {
                mbar_arrive_expect_tx(&sm.full_v[st], kTileBytes);
                tma_load_3d(sm.v[st], &vmap, &sm.full_v[st], 0, it.kvh, row);
                tma_load_3d(sm.v[st] + kHalfBytes, &vmap, &sm.full_v[st], 64, it.kvh, row);
                ++v_issued;
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
      } else if (sm.abort) {
        ok = false;
      }
      ++qi;
      w += step;
      if (!ok) break;
    }
    if (lane == 0) {
      if (!ok) flag_error(a, sm, kErrWaitTimeout);
      // Drain every copy this CTA issued before it may exit (a Q buffer is
      // reloaded only after its previous load was consumed, so only the last
      // load of each stream can be in flight).
      for (int s = 0; s < ns; ++s)
        if (const int loads = qi + (s < q_extra ? 1 : 0); loads > 0) (void)mbar_wait(&sm.q_full[s], (loads - 1) & 1);
      for (int j = max(0, k_issued - kStages); j < k_issued; ++j)
        (void)mbar_wait(&sm.full_k[j % kStages], (j / kStages) & 1);
      for (int j = max(0, v_issued - kStages); j < v_issued; ++j)
        (void)mbar_wait(&sm.full_v[j % kStages], (j / kStages) & 1);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------- MMA ----
    if constexpr (kSplit) regs_dec<kRegsIssue>();
    // the operands' type fields: 1 for bf16, 0 for fp16
    constexpr uint32_t types = kDecoding ? umma_idesc_ab_bf16 : 0u;
    constexpr uint32_t idesc_qk = umma_idesc_bf16(kRows, kKeys, false) & ~types;
    constexpr uint32_t idesc_pv = umma_idesc_bf16(kRows, kD, true) & ~types;
    bool ok = true;
    auto wait_all = [](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
    auto commit = [](uint64_t* bar) {
      if (elect_one_sync()) umma_commit(bar);
      __syncwarp();
    };
    // One elected thread issues a whole product (electing for every step makes
    // the code several times as long). Steps move the descriptors' address
    // field, in units of 16 bytes.
    auto issue_s = [&](int s, int st) {  // S_s = Q_s K(stage st)^T
      if (elect_one_sync()) {
        const uint64_t qa = smem_desc_sw128(smem_u32(sm.q[s]), 16, 1024);
        const uint64_t kb = smem_desc_sw128(smem_u32(sm.k[st]), 16, 1024);
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4;
          umma_f16_ss(tmem + s * kKeys, qa + off, kb + off, idesc_qk, kk > 0);
        }
        umma_commit(&sm.s_full[s]);
      }
      __syncwarp();
    };
    // O_s (+)= P_s V(stage st) over the keys of 16-key steps kk0 .. kk0 + 3
    auto issue_pv = [&](int s, int st, int kk0, bool first) {
      if (elect_one_sync()) {
        const uint64_t vb = smem_desc_sw128(smem_u32(sm.v[st]), kHalfBytes, 1024);
#pragma unroll
        for (int kk = kk0; kk < kk0 + 4; ++kk)
          umma_f16_ts(tmem + kColO + s * kD, tmem + s * kKeys + kk * 8, vb + kk * (16 * 128 >> 4), idesc_pv,
                      (!first || kk > 0) ? 1u : 0u);
      }
      __syncwarp();
    };
    int qi = 0, g = 0;
    while (ok) {
      if (!wait_all(&sm.item_full[qi % kItemRing], (qi / kItemRing) & 1)) { ok = false; break; }
      const Item it = sm.items[qi % kItemRing];
      if (it.n_kv < 0) break;
      // First S tiles of the item: behind the previous item's last P V in
      // issue order, so they overwrite its P only after it was read.
      {
        const int st = g % kStages;
        if (!wait_all(&sm.full_k[st], (g / kStages) & 1)) { ok = false; break; }
        for (int s = 0; s < ns && ok; ++s) {
          if (!wait_all(kDecoding ? &sm.q_ready[s] : &sm.q_full[s], qi & 1)) { ok = false; break; }
          tc_fence_after();
          issue_s(s, st);
          if (it.n_kv == 1) commit(&sm.q_empty[s]);
        }
        if (!ok) break;
        commit(&sm.k_empty[st]);
      }
      for (int j = 0; j < it.n_kv && ok; ++j, ++g) {
        const int st = g % kStages, st1 = (g + 1) % kStages;
        const bool more = j + 1 < it.n_kv;
        if (!wait_all(&sm.full_v[st], (g / kStages) & 1) ||
            (more && !wait_all(&sm.full_k[st1], ((g + 1) / kStages) & 1))) {
          ok = false;
          break;
        }
        for (int s = 0; s < ns; ++s) {
          // the P V of the first 64 keys goes out while the softmax still
          // computes the exponentials of the other 64
          if (!wait_all(&sm.p_lo[s], g & 1) || (j == 0 && qi > 0 && !wait_all(&sm.o_free[s], (qi - 1) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_pv(s, st, 0, j == 0);
          if (!wait_all(&sm.p_hi[s], g & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_pv(s, st, 4, false);
          if (more) {
            issue_s(s, st1);
            if (j + 2 == it.n_kv) commit(&sm.q_empty[s]);  // the item's last S_s
          } else {
            commit(&sm.o_ready[s]);
          }
        }
        if (!ok) break;
        commit(&sm.v_empty[st]);
        if (more) commit(&sm.k_empty[st1]);
      }
      ++qi;
    }
    if (!ok && lane == 0) flag_error(a, sm, kErrWaitTimeout);
    // All MMAs of this CTA complete before TMEM is released.
    commit(&sm.fin);
    (void)mbar_wait(&sm.fin, 0);
  } else if (kDecoding && warp >= kDecodeWarp0) {
    // -------------------------------------------------------- decoders ----
    if constexpr (kSplit) regs_dec<kRegsDecode>();
    const int r = tid - kDecodeWarp0 * 32;  // token row of the tile
    const int i = r & (fp4::kUnitTokens - 1);
    int qi = 0, g = 0;
    bool ok = true;
    while (ok) {
      if (!__all_sync(0xffffffffu, mbar_wait(&sm.item_full[qi % kItemRing], (qi / kItemRing) & 1))) {
        ok = false;
        break;
      }
      const Item it = sm.items[qi % kItemRing];
      if (it.n_kv < 0) break;
      const int32_t* bt = a.block_tables + static_cast<int64_t>(it.b) * a.bt_stride;
      // The unit of token `tok`; nullptr (rows of zeros) past the sequence's
      // end and where the table leads nowhere.
      auto unit_of = [&](int tok) -> const uint8_t* {
        if (tok >= it.lk) return nullptr;
        const int u = tok >> 4;
        const int blk = bt[u >> a.upb_log2];
        if (blk < 0 || blk >= a.num_blocks) {
          if (a.err) atomicOr(a.err, kErrBadBlockId);
          return nullptr;
        }
        return a.pool + (((static_cast<int64_t>(blk) * a.kvh + it.kvh) << a.upb_log2) + (u & ((1 << a.upb_log2) - 1))) *
                            (kFp4 ? fp4::kUnitBytes : fp8::kUnitBytes);
      };
      // Tile j's K to `full_k` and V to `full_v`, once their stages are free, with the next tile's loads behind each.
      auto tile_of = [&](int j, auto&& decode_k, auto&& load_k, auto&& decode_v, auto&& load_v) {
        const int st = g % kStages;
        const uint32_t parity = ((g / kStages) - 1) & 1;
        if (sm.abort || (g >= kStages && !mbar_wait(&sm.k_empty[st], parity))) ok = false;
        if (!__all_sync(0xffffffffu, ok)) return ok = false;
        decode_k(smem_u32(sm.k[st]));
        fence_proxy_async_smem();
        mbar_arrive(&sm.full_k[st]);
        load_k();
        if (g >= kStages && !mbar_wait(&sm.v_empty[st], parity)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) return ok = false;
        decode_v(smem_u32(sm.v[st]));
        fence_proxy_async_smem();
        mbar_arrive(&sm.full_v[st]);
        load_v();
        return true;
      };
      int* nan_from = sm.nan_from[qi % kItemRing];
      if constexpr (kFp4) {
        KRow k;
        VRow v;
        const uint8_t* unit = unit_of(r);
        load_row(k, unit, i);
        load_row(v, unit, i);
        for (int j = 0; j < it.n_kv; ++j, ++g) {
          unit = j + 1 < it.n_kv ? unit_of((j + 1) * kKeys + r) : nullptr;
          if (!tile_of(
                  j, [&](uint32_t tile) { decode_row(k, tile, r); }, [&] { load_row(k, unit, i); },
                  [&](uint32_t tile) {
                    const uint2 bytes = scale_bytes(v, r);
                    note_nan(bytes, j * kKeys + r, nan_from);
                    decode_row(v, bytes, tile, r);
                  },
                  [&] { load_row(v, unit, i); }))
            break;
        }
      } else {
        // One set of registers: K's chunks make room for V's of the same tile, those for K's of the next one.
        const int r0 = r & ~31;  // the warp's first token row
        const int tok0 = kClusters ? it.k0 + r0 : r0;
        Chunks x;
        const uint8_t* unit[2] = {unit_of(tok0), unit_of(tok0 + 16)};
        int2 exps;  // lanes 0 and 1: of their unit
        auto load_exps = [&] {
          exps = make_int2(0, 0);
          const uint8_t* mine = lane == 0 ? unit[0] : unit[1];
          if (lane < 2 && mine) exps = *reinterpret_cast<const int2*>(mine + fp8::kOffExp);
        };
        load_exps();
#pragma unroll
        for (int n = 0; n < 8; ++n) x.w[n] = load_chunk(unit, n, 0, it.lk - tok0, lane);
        for (int j = 0; j < it.n_kv; ++j, ++g) {
          if (!tile_of(
                  j,
                  [&](uint32_t tile) {
                    // (The slot's last tile, four back, is done: the wait for this stage of K, whose last tile is two
                    // back, means that both streams' S of that tile, and with it P of the one before, were complete.)
                    if (lane < 2) {
                      sm.exps[g % 4][0][r0 / 16 + lane] = static_cast<uint8_t>(127 + fp8::held_exp(exps.x));
                      sm.exps[g % 4][1][r0 / 16 + lane] = static_cast<uint8_t>(127 + fp8::held_exp(exps.y));
                    }
                    const int seen = it.lk - j * kKeys - tok0;
                    decode_chunks<false>(x, tile, r0, 0, nullptr, lane,
                                         [&](int n) { return load_chunk(unit, n, 1, seen, lane); });
                  },
                  [&] {
                    const int next = j + 1 < it.n_kv ? (j + 1) * kKeys + tok0 : INT_MAX - 16;
                    unit[0] = unit_of(next);
                    unit[1] = unit_of(next + 16);
                    load_exps();
                  },
                  [&](uint32_t tile) {
                    const int seen = it.lk - (j + 1) * kKeys - tok0;
                    decode_chunks<true>(x, tile, r0, j * kKeys + tok0, nan_from, lane,
                                        [&](int n) { return load_chunk(unit, n, 0, seen, lane); });
                  },
                  [] {}))
            break;
        }
      }
      ++qi;
    }
    if (!ok) flag_error(a, sm, kErrWaitTimeout);
  } else if ((warp >> 2) < ns) {
    // --------------------------------------------------------- softmax ----
    if constexpr (kSplit) regs_inc<kRegsSoftmax>();
    const int s = warp >> 2;
    const int r = tid & (kStreamThreads - 1);  // query row within the tile = TMEM lane
    const uint32_t t_lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_s = tmem + s * kKeys + t_lane;
    const uint32_t tmem_o = tmem + kColO + s * kD + t_lane;
    float sc = a.scale_log2;
    uint8_t* stage = sm.stage[s];
    int qi = 0, g = 0;
    bool ok = true;
    Item it;
    // Item n's descriptor and, in the 4-bit kernel, this thread's row of its
    // Q, which becomes fp16 here, between an item's last P and its O: these
    // warps are eight, and have nothing to do while the last P V runs.
    auto begin_item = [&](int n) {
      if (!__all_sync(0xffffffffu, mbar_wait(&sm.item_full[n % kItemRing], (n / kItemRing) & 1))) return false;
      it = sm.items[n % kItemRing];
      if (kDecoding && it.n_kv > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.q_full[s], n & 1))) return false;
        sc = fp4::score_factor(q_row_to_half(smem_u32(sm.q[s]), r), a.scale_log2);
        if constexpr (kExps) sc = sc < kLeastFactor ? kLeastFactor : sc > kMostFactor ? kMostFactor : sc;  // NaN stays
        fence_proxy_async_smem();
        mbar_arrive(&sm.q_ready[s]);
      }
      return true;
    };
    if (kDecoding) ok = begin_item(0);
    while (ok) {
      if (!kDecoding && !begin_item(qi)) {
        ok = false;
        break;
      }
      if (it.n_kv < 0) break;
      const int i = it.qt * kRows + r;
      const int lim = ((i < it.lq) ? (it.lk - it.lq + i) : (it.lk - 1)) - (kClusters ? it.k0 : 0);
      // 8-bit kernel: weights are relative to p 2^e, e the unit's exponent of V: to the exponent `exp` beside m, and
      // the sum l takes 2^-e back (see fp8_decode.cu).
      float exp = -INFINITY;
      float m = kExps ? 0.f : -INFINITY, l = 0.f;  // m: the reference score in log2 units; in a decoding kernel its product q . k
      for (int j = 0; j < it.n_kv; ++j, ++g) {
        // warp-uniform outcome: the tcgen05.ld/st below need a converged warp
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.s_full[s], g & 1))) { ok = false; break; }
        tc_fence_after();
        const int kbase = j * kKeys;
        uint32_t sr[4][32];
        // A decoding kernel masks in tensor memory, in a loop: masking all of the row's registers at once is code that
        // runs once an item, and fetching it took longer (the instruction caches are full of the decoders' code).
        if (kDecoding && __any_sync(0xffffffffu, kbase + kKeys - 1 > lim)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int seen = lim - kbase - c * 32;  // the chunk's columns up to this one are seen
            tmem_ld32(tmem_s + c * 32, sr[0]);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e > seen) sr[0][e] = __float_as_uint(-INFINITY);
            tmem_st32(tmem_s + c * 32, sr[0]);
          }
          tmem_st_wait();
        }
        auto load_scores = [&] {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(tmem_s + c * 32, sr[c]);
          tmem_ld_wait();
        };
        load_scores();
        if (!kDecoding && kbase + kKeys - 1 > lim) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (kbase + c * 32 + e > lim) sr[c][e] = __float_as_uint(-INFINITY);
        }
        // 8-bit kernel: the exponents of the tile's units stay in four registers, a byte each.
        uint4 te = make_uint4(0, 0, 0, 0);
        if constexpr (kExps) te = ld_shared_v4(smem_u32(sm.exps[g % 4]));
        auto k_pow2 = [&](int u) {  // 2^e of K
          return __uint_as_float(__byte_perm(u < 4 ? te.x : te.y, 0, (u & 3) << 12 | 0x444) >> 1);
        };
        auto v_exp = [&](int u) {  // e of V: 2^23 + byte, less 2^23 + 127
          return __uint_as_float(__byte_perm(u < 4 ? te.z : te.w, 0x4b000000, 0x7540 + (u & 3))) - 8388735.f;
        };
        auto v_pow2_inv = [&](int u) {  // 2^-e of V
          return __uint_as_float(0x7f000000u - (__byte_perm(u < 4 ? te.z : te.w, 0, (u & 3) << 12 | 0x444) >> 1));
        };
        // The max is taken over raw scores (scale > 0), the scale folded into
        // the exponent's FMA below; max is exact, so its order is free.
        constexpr int kRuns = kExps ? kKeys / fp8::kUnitTokens : 4;  // units, or chunks
        float mx[kRuns];
#pragma unroll
        for (int u = 0; u < kRuns; ++u) {
          mx[u] = -INFINITY;
#pragma unroll
          for (int e = u * (kKeys / kRuns); e < (u + 1) * (kKeys / kRuns); e += 2)
            mx[u] = fmax3(mx[u], __uint_as_float(sr[e / 32][e % 32]), __uint_as_float(sr[e / 32][e % 32 + 1]));
        }
        bool resc;
        float alpha = 1.f, mu;
        if constexpr (kExps) {
          float mt = -INFINITY, most = -INFINITY;
#pragma unroll
          for (int u = 0; u < kRuns; ++u) {
            mx[u] *= k_pow2(u);
            mt = fmaxf(mt, mx[u]);
            most = fmaxf(most, fmaf(mx[u] - m, sc, v_exp(u) - exp));
          }
          resc = most > kRescaleThreshold;
          if (resc) {
            const float to = exp == -INFINITY ? mt : fmaxf(m, mt), old = fmaf(m - to, sc, exp);
            most = old;
#pragma unroll
            for (int u = 0; u < kRuns; ++u) most = fmaxf(most, fmaf(mx[u] - to, sc, v_exp(u)));
            alpha = fast_exp2(old - most);
            l *= alpha;
            m = to;
            exp = most;
          }
          mu = -m * sc;
        } else {
          const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * (kDecoding ? 1.f : sc);
          const float m_new = fmaxf(m, mt);
          resc = kDecoding ? (m_new - m) * sc > kRescaleThreshold : m_new > m + kRescaleThreshold;
          alpha = resc ? fast_exp2(kDecoding ? (m - m_new) * sc : m - m_new) : 1.f;
          if (resc) {
            l *= alpha;
            m = m_new;
          }
          mu = (m == -INFINITY) ? 0.f : kDecoding ? fmaf(-m, sc, kPShift<kDecoding>) : kPShift<kDecoding> - m;
        }
        // The decoding kernels far from 0, where the rounding of mu would reach the weights (and from 2^22 on lead P
        // out of fp16): the reference is subtracted from the products instead, which is exact where it matters.
        bool far = false;
        if (kDecoding && __any_sync(0xffffffffu, fabsf(mu) > kFarScore)) {
          far = true;
          const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            tmem_ld32(tmem_s + c * 32, sr[0]);
            tmem_ld_wait();
            float f[2] = {1.f, 1.f};
            if constexpr (kExps) {
              const uint32_t two = (c < 2 ? te.x : te.y) >> (16 * (c & 1));
              f[0] = __uint_as_float((two & 0xffu) << 23), f[1] = __uint_as_float((two & 0xff00u) << 15);
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
              sr[0][e] = __float_as_uint(kExps ? fmaf(__uint_as_float(sr[0][e]), f[e / 16], -ref)
                                               : __uint_as_float(sr[0][e]) - ref);
            tmem_st32(tmem_s + c * 32, sr[0]);
          }
          tmem_st_wait();
          load_scores();
          mu = kExps ? 0.f : kPShift<kDecoding>;
        }
        // (the exponent's part of the reference behind the products', which may be large)
        if constexpr (kExps) mu = exp == -INFINITY ? 0.f : mu + (kPShift<kDecoding> - exp);
        uint64_t sum[2] = {f32x2_pack(0.f, 0.f), f32x2_pack(0.f, 0.f)};  // independent add chains
        uint64_t sc2 = f32x2_pack(sc, sc), mu2 = f32x2_pack(mu, mu);
        // P over the first 64 columns of S_s (column k holds keys 2k and 2k+1
        // as a bf16 pair): word e of chunk c overwrites score e, already read.
        // Keys 0-63 are signalled first, so that their P V starts while the
        // exponentials of keys 64-127 are computed.
        auto exps = [&](int c) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (kExps && e % 8 == 0) {  // a unit begins
              const int u = 2 * c + e / 8;
              const float by = far ? sc : sc * k_pow2(u), add = mu + v_exp(u);
              sc2 = f32x2_pack(by, by), mu2 = f32x2_pack(add, add);
              sum[0] = sum[1] = f32x2_pack(0.f, 0.f);
            }
            float p0, p1;
            f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(sr[c][2 * e]), __uint_as_float(sr[c][2 * e + 1])), sc2, mu2),
                         p0, p1);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            sum[e & 1] = f32x2_add(sum[e & 1], f32x2_pack(p0, p1));
            sr[c][e] = kDecoding ? pack_half2(p0, p1) : pack_bf16x2(p0, p1);
            if (kExps && e % 8 == 7) {
              float s0, s1;
              f32x2_unpack(f32x2_add(sum[0], sum[1]), s0, s1);
              l = fmaf(s0 + s1, v_pow2_inv(2 * c + e / 8), l);
            }
          }
          tmem_st16_first(tmem_s + c * 16, sr[c]);
        };
        exps(0);
        exps(1);
        // O_s rescales (rarely) before any P V of this tile: S_s(j) landed,
        // so P V_s(j-1) is complete.
        if (j > 0 && __any_sync(0xffffffffu, resc)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(tmem_o + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tmem_o + c * 32, o);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sm.p_lo[s]);
        exps(2);
        exps(3);
        if constexpr (!kExps) {
          float s0, s1, s2, s3;
          f32x2_unpack(sum[0], s0, s1);
          f32x2_unpack(sum[1], s2, s3);
          l += (s0 + s1) + (s2 + s3);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sm.p_hi[s]);
      }
      if (!ok) break;
      // (8-bit kernel: the descriptor is read again, since its fields would be spilled in the loop above: 98.0 -> 97.2 us)
      if constexpr (kExps) it = sm.items[qi % kItemRing];
      const int rows = min(kRows, it.lq - it.qt * kRows);
      __nv_bfloat16* out = a.out + (static_cast<int64_t>(it.q0 + it.qt * kRows) * a.num_heads + it.h0 + s) * kD;
      if (kDecoding && !begin_item(qi + 1)) {
        ok = false;
        break;
      }
      // The item's last P V_s complete: normalise the O_s rows and store them
      // through stage[s], 32 dims at a time (its two halves in turn): thread r
      // writes its row's 64 bytes there (16-byte chunk c of row r at chunk
      // c ^ (r / 2 % 4): conflict free), then its warp stores the 32 pieces
      // that its lanes wrote, eight per instruction, so the global writes are
      // coalesced and no warp waits for another.
      if (!__all_sync(0xffffffffu, mbar_wait(&sm.o_ready[s], qi & 1))) { ok = false; break; }
      tc_fence_after();
      const float inv = kDecoding ? (l == 0.f ? 0.f : a.out_scale / l) : (l > 0.f ? 1.f / l : 0.f);
      // (`it` is the next item by now; this one's slot is filled again only behind its output)
      const Item& done = sm.items[qi % kItemRing];
      const int seen = kDecoding ? done.lk - done.lq + done.qt * kRows + r : 0;  // this row's last key
      if constexpr (kClusters) {
        if (sm.parts > 1) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(tmem_o + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              st_shared_v4(smem_u32(sm.k) + part_chunk(r, 8 * c + e), o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          if (seen >= sm.nan_from[qi % kItemRing][0]) l = __uint_as_float(0x7fffffffu);
          st_shared_v4(smem_u32(sm.v) + r * sizeof(Part), __float_as_uint(m), __float_as_uint(exp), __float_as_uint(l),
                       __float_as_uint(sc));  // (no item follows, so sc is still this one's)
          ++qi;
          continue;
        }
      }
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem_o + c * 32, o);
        tmem_ld_wait();
        if (c == 3) {  // O_s is read out: the next item's first P V_s may overwrite it
          tc_fence_before();
          mbar_arrive(&sm.o_free[s]);
        }
        const uint32_t half = smem_u32(stage + (c & 1) * (kRows * 64));
        float by[2] = {inv, inv};  // groups 2 c and 2 c + 1: NaN where the row sees one that V holds
        if constexpr (kDecoding)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (seen >= sm.nan_from[qi % kItemRing][kFp4 ? 2 * c + e : 0]) by[e] = __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const float f = by[q4 >> 1];
          const uint32_t x = pack_bf16x2(__uint_as_float(o[q4 * 8 + 0]) * f, __uint_as_float(o[q4 * 8 + 1]) * f);
          const uint32_t y = pack_bf16x2(__uint_as_float(o[q4 * 8 + 2]) * f, __uint_as_float(o[q4 * 8 + 3]) * f);
          const uint32_t z = pack_bf16x2(__uint_as_float(o[q4 * 8 + 4]) * f, __uint_as_float(o[q4 * 8 + 5]) * f);
          const uint32_t u = pack_bf16x2(__uint_as_float(o[q4 * 8 + 6]) * f, __uint_as_float(o[q4 * 8 + 7]) * f);
          st_shared_v4(half + r * 64 + ((q4 ^ ((r >> 1) & 3)) << 4), x, y, z, u);
        }
        __syncwarp();  // this warp's pieces are in this half, and the ones before them out of the other
        uint4 v[4];
        const int row0 = (warp & 3) * 32 + (lane >> 2), c16 = lane & 3;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[k] = ld_shared_v4(half + (row0 + 8 * k) * 64 + ((c16 ^ ((row0 >> 1) & 3)) << 4));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (row0 + 8 * k < rows)
            *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row0 + 8 * k) * a.num_heads * kD + c * 32 + c16 * 8) =
                v[k];
      }
      if (!ok) break;
      ++qi;
    }
    if (!ok) flag_error(a, sm, kErrWaitTimeout);
  } else if (kSplit && warp >= kProducerWarp && warp < kDecodeWarp0) {
    regs_dec<kRegsIssue>();  // the idle warps of the producer's warpgroup
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if constexpr (kClusters) {  // (every wait above ends, so all threads of the cluster come here)
    cluster_sync();
    if (warp < kProducerWarp && sm.parts > 1) join_parts(a, sm, cluster_rank(), cluster_size());
    __syncwarp();
    cluster_sync();  // the others have read this CTA's part
  }
  if (warp == kMmaWarp) {
    __syncwarp();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace prefill
}  // namespace nvk
