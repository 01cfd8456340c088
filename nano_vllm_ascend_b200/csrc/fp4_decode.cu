// Paged decode attention over the 4-bit KV pool, one query token a sequence:
//   out[b, h] = softmax(scale * q[b, h] . K_b^T) . V_b
// with K and V the values that the codes of fp4_kv.cuh stand for.
//
// HBM-bound: 144 bytes per (token, KV head) are read once. Tensor-core
// operands are made in registers, on the legacy m16n8k16 path: an A fragment
// can be filled straight from the packed codes (tcgen05 would need a second
// trip of four times the bytes through shared memory), and eight query heads
// are all the columns that there are.
//   S^T[16 tokens x 8 heads] = K[16 x 128] . Q^T, eight steps of one group each
//   O^T[16 dims x 8 heads] (8 tiles) += V^T[16 dims x 16 tokens] . P^T
// K and V enter as e2m1 -> fp16 (one conversion for two values): exact. K's
// scales multiply the fp32 sums of their groups, V's the weights: P s is
// rounded to fp16 twice (P, then the product: 2^-10 of a weight). 2^4 p is
// normal down to p = 2^-18, and the scales are held times a power of two that
// brings the largest one so far near 448, so that however small V is, the
// product loses nothing beside that. Q is scaled by a power of two into fp16's
// range, which holds its 8 bits exactly. Scores, maxima, sums and O are fp32;
// the last division is a product with an approximate reciprocal (2^-21, below
// bf16's half step of 2^-8; the exact one is 2 KB of code, and code that runs
// once costs its fetch).
//
// The schedule, the rings and the joins are in decode_core.cuh; a tile is two
// units (32 tokens, one copy of 4608 bytes), two in flight a warp: 74 to 147 KB
// an SM, where about 55 KB hide HBM's latency at full rate.
//
// What bounds it: with much to read, instruction issue (about 300 a unit and
// warp, 67 % of the slots; the ALU pipe at 59 % with 64 conversions of 2 values
// a unit, which run at half rate) and the power limit behind it (256 contexts
// of about 4096 tokens, 8 KV heads, 1.2 GB: 215 us = 5.6 TB/s alone, 240 to 253
// us in a long run at 1710 MHz); with little, latencies: launch, schedule and
// first bytes about 4 us, the pieces' meeting 1 to 2, a split pair's ticket and
// join 2 (one context of 100 tokens 4.9 us, 32 of 256 to 2304 16.9). The last
// comes from cuts inside pairs, which most are: 38 of 42 with 4 contexts up to
// 513 tokens, 141 of 147 with those 32.
#include <type_traits>

#include "decode_core.cuh"

namespace nvk {
namespace fp4 {
namespace {

using namespace decode;
using decode::kD;
using decode::kUnitTokens;

constexpr float kRescale = 3.f;  // log2 by which a score may pass the reference before that moves and O is rescaled
constexpr float kPShift = 4.f;   // P is held as 2^4 p: with p up to 2^3 and scales up to 480, P s fits fp16 (p goes
                                 // by differences of products, so that this holds for scores of any magnitude)
constexpr uint32_t kVScaleBytes = kGroups * kUnitTokens * 2;  // of one unit

struct State {
  uint32_t q;              // shared address of this lane's B fragments of Q^T (see load_q)
  float sc[2];             // factor from products to scores in log2 units, of heads 2 t and 2 t + 1
  float ref[2];            // p = 2^((product - ref) * sc + kPShift): their running largest product
  float thr[2];            // the product above which it moves: by kRescale in log2 units (-inf at first)
  float l[2];              // this lane's part of the sum of p
  float o[kGroups][4];     // O^T: dims 16 j + 2 g (heads 2 t, 2 t + 1), then 16 j + 2 g + 1 (the same)
  uint32_t room;           // V's scales, and so O, are held times 2^e (e of 0 to 15), such that the largest scale so
                           // far stays below 512; 8 e in every byte
};

// Q's rows of one pair as fragments: head g = lane / 4, dims 16 j + 4 t + {0, 1}
// and {2, 3}, t = lane % 4. They stay in shared memory (a lane reads only what
// it wrote): the 16 registers would cost spills.
__device__ __forceinline__ void load_q(const DecodeArgs& a, int b, int h, int g, int t, State& st) {
  uint2 raw[kGroups];
  const bool live = g < a.group;
  const __nv_bfloat16* row = a.q + (static_cast<int64_t>(b) * a.heads + h * a.group + (live ? g : 0)) * kD + 4 * t;
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
    raw[j] = live ? *reinterpret_cast<const uint2*>(row + 16 * j) : make_uint2(0, 0);
  uint32_t big = 0;
#pragma unroll
  for (int j = 0; j < kGroups; ++j) big = bf16x2_abs_max(big, bf16x2_abs_max(raw[j].x, raw[j].y));
  big = bf16x2_abs_max(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = bf16x2_abs_max(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const HalfRow half = half_row(big);
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
    st_shared_v2(st.q + 512 * (j >> 1) + 8 * (j & 1), bf16x2_to_half2(raw[j].x, half.base),
                 bf16x2_to_half2(raw[j].y, half.base));
  st.sc[0] = score_factor(__shfl_sync(0xffffffffu, half.up, 8 * t), a.scale_log2);
  st.sc[1] = score_factor(__shfl_sync(0xffffffffu, half.up, 8 * t + 4), a.scale_log2);
  st.ref[0] = st.ref[1] = 0.f;
  st.thr[0] = st.thr[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
  st.room = 15 * 0x08080808u;
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) st.o[j][c] = 0.f;
}

// A unit's V scales, word `lane`: group lane % 8 of the quad lane / 8. Tokens
// from `valid` on get scales of 0, so that nothing that their bytes hold (a NaN)
// meets their weights of 0.
template <bool kMask>
__device__ __forceinline__ uint32_t vscale_word(uint32_t unit, int valid, int lane) {
  uint32_t w = ld_shared(unit + kOffVScale + 4 * lane);
  if (kMask) {
    const int n = min(max(valid - 4 * (lane >> 3), 0), 4);
    w &= n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1;
  }
  return w;
}
// A scale byte's exponent field, its bits 3 to 6, has to be at most 15 - e.
__device__ __forceinline__ bool above(uint32_t w, uint32_t room) { return (w + room) & 0x80808080u; }
// Lowers the power of two to what the tile's scales allow, and O with it.
__device__ __forceinline__ void make_room(State& st, uint32_t w0, uint32_t w1) {
  uint32_t m = __vmaxu4(w0 & 0x78787878u, w1 & 0x78787878u);
  m = __vmaxu4(m, m >> 16);
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffu, (m >> 8) & 0xffu));
  const uint32_t old = st.room & 0xffu, now = min(old, 15u * 8 - m);
  st.room = now * 0x01010101u;
  if (!__any_sync(0xffffffffu, st.thr[0] != -INFINITY || st.thr[1] != -INFINITY)) return;  // O is 0 yet (or NaN)
  const float f = __uint_as_float((127u << 23) - ((old - now) << 20));
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) st.o[j][c] *= f;
}
// The words to fp16, once for the whole warp, times the power of two (exact).
__device__ __forceinline__ void convert_vscales(const State& st, uint32_t w, uint32_t to, int lane) {
  const int quad = lane >> 3, j = lane & 7;
  const uint32_t up = 0x3c003c00u + ((st.room & 0x00ff00ffu) << 7);
  uint32_t lo, hi;
  e4m3_to_half2(w, lo, hi);
  st_shared_v2(to + 64 * (j >> 1) + 16 * quad + 8 * (j & 1), hmul2(lo, up), hmul2(hi, up));
}

// Scores of one unit (without the factor sc): x[0], x[1] of token ta's heads
// 2 t and 2 t + 1, x[2], x[3] of token ta + 2's. Rows g and g + 8 of the S
// tile are these tokens, so that the transposed P has tokens 4 t .. 4 t + 3 in
// lane t, whose V words hold them.
template <bool kMask>
__device__ __forceinline__ void scores(const State& st, uint32_t unit, int valid, int g, int t, float (&x)[4]) {
  const int ta = 4 * (g >> 1) + (g & 1);
  const uint4 ka = ld_shared_v4(unit + 64 * ta + 16 * t), kb = ld_shared_v4(unit + 64 * (ta + 2) + 16 * t);
  const uint2 ksa = ld_shared_v2(unit + kOffKScale + 8 * ta), ksb = ld_shared_v2(unit + kOffKScale + 8 * (ta + 2));
  const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
  uint32_t sa[4], sb[4];
  e4m3_to_half2(ksa.x, sa[0], sa[1]);
  e4m3_to_half2(ksa.y, sa[2], sa[3]);
  e4m3_to_half2(ksb.x, sb[0], sb[1]);
  e4m3_to_half2(ksb.y, sb[2], sb[3]);
#pragma unroll
  for (int c = 0; c < 4; ++c) x[c] = 0.f;
  float y[4] = {0.f, 0.f, 0.f, 0.f};  // odd groups: two shorter chains of sums
#pragma unroll
  for (int w = 0; w < 4; ++w) {  // a word holds groups 2 w and 2 w + 1
    uint32_t p[4], q[4];
    e2m1_to_half2(wa[w], p[0], p[1], p[2], p[3]);
    e2m1_to_half2(wb[w], q[0], q[1], q[2], q[3]);
    float d[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
    const uint4 f = ld_shared_v4(st.q + 512 * w);
    mma_16816(d, p[0], q[0], p[1], q[1], f.x, f.y);
    mma_16816(e, p[2], q[2], p[3], q[3], f.z, f.w);
    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&sa[w]));
    const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&sb[w]));
    x[0] = fmaf(d[0], fa.x, x[0]), x[1] = fmaf(d[1], fa.x, x[1]);
    x[2] = fmaf(d[2], fb.x, x[2]), x[3] = fmaf(d[3], fb.x, x[3]);
    y[0] = fmaf(e[0], fa.y, y[0]), y[1] = fmaf(e[1], fa.y, y[1]);
    y[2] = fmaf(e[2], fb.y, y[2]), y[3] = fmaf(e[3], fb.y, y[3]);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) x[c] += y[c];
  if (kMask) {
    if (ta >= valid) x[0] = x[1] = -INFINITY;
    if (ta + 2 >= valid) x[2] = x[3] = -INFINITY;
  }
}

// O += V^T P^T of one unit; b0 and b1 are the fragments of P^T.
__device__ __forceinline__ void weigh(State& st, uint32_t unit, uint32_t vscale, int g, int t, uint32_t b0,
                                      uint32_t b1) {
  const uint4 va = ld_shared_v4(unit + kOffV + 256 * t + 32 * g);
  const uint4 vb = ld_shared_v4(unit + kOffV + 256 * t + 32 * g + 16);
#pragma unroll
  for (int w = 0; w < 2; ++w) {  // groups 4 w .. 4 w + 3; tokens 4 t .. 4 t + 3
    const uint32_t c0 = w ? va.y : va.x, c1 = w ? va.w : va.z;
    const uint32_t c2 = w ? vb.y : vb.x, c3 = w ? vb.w : vb.z;
    constexpr uint32_t kLow = 0x0f0f0f0fu;
    uint32_t lo01[4], hi01[4], lo23[4], hi23[4];
    auto spread = [](uint32_t v, uint32_t (&r)[4]) { e2m1_to_half2(v, r[0], r[1], r[2], r[3]); };
    spread((c0 & kLow) | ((c1 << 4) & ~kLow), lo01);
    spread(((c0 >> 4) & kLow) | (c1 & ~kLow), hi01);
    spread((c2 & kLow) | ((c3 << 4) & ~kLow), lo23);
    spread(((c2 >> 4) & kLow) | (c3 & ~kLow), hi23);
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const uint4 s = ld_shared_v4(vscale + 64 * (2 * w + (k >> 1)) + 16 * t);
      mma_16816(st.o[4 * w + k], lo01[k], hi01[k], lo23[k], hi23[k], hmul2(b0, s.x), hmul2(b1, s.y));
      mma_16816(st.o[4 * w + k + 1], lo01[k + 1], hi01[k + 1], lo23[k + 1], hi23[k + 1], hmul2(b0, s.z),
                hmul2(b1, s.w));
    }
  }
}

// One tile: its first `valid` tokens are the sequence's (kMask: fewer than all).
template <bool kMask>
__device__ __forceinline__ void attend(State& st, uint32_t tile, uint32_t vscale, int valid, int g, int t, int lane) {
  __syncwarp();  // the tile before this one is done with vscale
  const uint32_t w0 = vscale_word<kMask>(tile, valid, lane);
  const uint32_t w1 = vscale_word<kMask>(tile + kUnitBytes, valid - kUnitTokens, lane);
  float x[2][4];
  scores<kMask>(st, tile, valid, g, t, x[0]);
  if (__any_sync(0xffffffffu, above(w0, st.room) || above(w1, st.room))) make_room(st, w0, w1);
  convert_vscales(st, w0, vscale, lane);
  convert_vscales(st, w1, vscale + kVScaleBytes, lane);
  scores<kMask>(st, tile + kUnitBytes, valid - kUnitTokens, g, t, x[1]);
  const float hi0 = fmaxf(fmax3(x[0][0], x[0][2], x[1][0]), x[1][2]);
  const float hi1 = fmaxf(fmax3(x[0][1], x[0][3], x[1][1]), x[1][3]);
  if (__any_sync(0xffffffffu, hi0 > st.thr[0] || hi1 > st.thr[1])) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float m = e ? hi1 : hi0;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      const bool first = st.thr[e] == -INFINITY;
      m = first ? m : fmaxf(m, st.ref[e]);
      const float f = first ? 0.f : fast_exp2((st.ref[e] - m) * st.sc[e]);
      st.ref[e] = m == -INFINITY ? 0.f : m;
      st.thr[e] = __fadd_rd(m, __fdividef(kRescale, st.sc[e]));  // down: p stays within its bound
      st.l[e] *= f;
#pragma unroll
      for (int j = 0; j < kGroups; ++j) st.o[j][e] *= f, st.o[j][2 + e] *= f;
    }
  }
  uint32_t b[2][2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    auto weight = [&](int c) { return fast_exp2(fmaf(x[u][c] - st.ref[c & 1], st.sc[c & 1], kPShift)); };
    const float p0 = weight(0), p1 = weight(1), p2 = weight(2), p3 = weight(3);
    st.l[0] += p0 + p2;
    st.l[1] += p1 + p3;
    b[u][0] = movmatrix(half2_of(p0, p1));
    b[u][1] = movmatrix(half2_of(p2, p3));
  }
  __syncwarp();  // vscale is written
  weigh(st, tile, vscale, g, t, b[0][0], b[0][1]);
  weigh(st, tile + kUnitBytes, vscale + kVScaleBytes, g, t, b[1][0], b[1][1]);
}

// The format's part of decode_core.cuh's kernel.
template <int kWarpsOfF>
struct Format {
  static constexpr int kWarps = kWarpsOfF, kTileUnits = 2, kStages = 2;  // tiles in flight a warp
  static constexpr int kUnitBytes = fp4::kUnitBytes, kTileTokens = 2 * kUnitTokens, kTileBytes = 2 * kUnitBytes;
  // Tiles below which a CTA is not used. Fewer spread short work over more SMs but
  // give its joins more pieces (one sequence of 100 / 1000 tokens, 8 KV heads:
  // 4.9 / 6.8 us with 8; when it was chosen 4.8 / 7.1, and 6.0 / 8.3 with 16).
  static constexpr int kMinTiles = 8;
  static constexpr bool kExps = false;  // a piece's reference is its largest product alone
  using State = fp4::State;
  struct Scratch {
    uint2 vscale[2][kGroups / 2][4][2];  // [unit][j / 2][quad][j % 2]: V's scales of the quad's four tokens, fp16
  };

  static __device__ __forceinline__ void load_q(const DecodeArgs& a, int b, int h, int g, int t, State& st) {
    fp4::load_q(a, b, h, g, t, st);
  }
  template <bool kMask>
  static __device__ __forceinline__ void attend(State& st, uint32_t tile, uint32_t scratch, int valid, int g, int t,
                                                int lane) {
    fp4::attend<kMask>(st, tile, scratch, valid, g, t, lane);
  }
  // What brings O from how the state holds it to a piece's terms.
  static __device__ __forceinline__ float down(const State& st) {
    return __uint_as_float((127u << 23) - ((st.room & 0xffu) << 20));
  }
  static __device__ __forceinline__ float4 piece(const State& st, int e) {
    return make_float4(st.thr[e] == -INFINITY ? -INFINITY : st.ref[e], st.l[e], st.sc[e], 0.f);
  }
  // The first of the two neighbouring dims of which o[j] has a lane's part.
  static __device__ __forceinline__ int dim(int j, int g) { return 16 * j + 2 * g; }
};

// 16 warps where shared memory has room for the pieces of the group's heads
// beside their rings, else 12 (16 against 12 at two heads, 256 contexts of
// about 4096 tokens: 230 against 244 us).
constexpr int kFewHeads = 4;
static_assert(smem_bytes<Format<16>>(kFewHeads) <= 232448 && smem_bytes<Format<12>>(kMaxGroup) <= 232448,
              "decode shared memory exceeds the 227 KB per-CTA limit");

}  // namespace
}  // namespace fp4
}  // namespace nvk

extern "C" int nvk_fp4_paged_decode_workspace_size(int num_heads, int num_kv_heads, int head_dim, int num_ctas,
                                                   size_t* bytes) {
  using namespace nvk;
  const char* who = "fp4_paged_decode_workspace_size";
  if (!bytes) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (head_dim != fp4::kD) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", who, head_dim);
  int rc = decode::check_heads(num_heads, num_kv_heads, num_ctas, who), ctas = 0;
  if (rc != NVK_OK || (rc = decode::resolve_ctas(num_ctas, who, &ctas)) != NVK_OK) return rc;
  *bytes = decode::workspace_bytes(num_heads / num_kv_heads, ctas);
  return NVK_OK;
}

extern "C" int nvk_fp4_paged_decode(void* out, const void* query, const void* kv_cache, int num_blocks,
                                    int block_size, const int32_t* block_tables, int block_table_stride,
                                    int max_blocks_per_seq, const int32_t* context_lens, int batch, int num_heads,
                                    int num_kv_heads, int head_dim, float scale, float k_scale, float v_scale,
                                    int num_ctas, void* workspace, size_t workspace_bytes, nvk_stream_t stream) {
  return nvk_fp4_paged_decode_reporting(out, query, kv_cache, num_blocks, block_size, block_tables,
                                        block_table_stride, max_blocks_per_seq, context_lens, batch, num_heads,
                                        num_kv_heads, head_dim, scale, k_scale, v_scale, num_ctas, workspace,
                                        workspace_bytes, nullptr, stream);
}

extern "C" int nvk_fp4_paged_decode_reporting(void* out, const void* query, const void* kv_cache, int num_blocks,
                                              int block_size, const int32_t* block_tables, int block_table_stride,
                                              int max_blocks_per_seq, const int32_t* context_lens, int batch,
                                              int num_heads, int num_kv_heads, int head_dim, float scale,
                                              float k_scale, float v_scale, int num_ctas, void* workspace,
                                              size_t workspace_bytes, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp4;
  const char* who = "fp4_paged_decode";
  if (batch < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: batch %d", who, batch);
  int rc = check_heads(num_heads, num_kv_heads, num_ctas, who), ctas = 0;
  if (rc != NVK_OK) return rc;
  if ((rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, k_scale, v_scale, who)) != NVK_OK)
    return rc;
  DecodeArgs a;
  rc = prepare(a, ctas, out, query, kv_cache, num_blocks, units_log2(block_size), block_size, block_tables,
               block_table_stride, max_blocks_per_seq, context_lens, batch, num_heads, num_kv_heads, scale, num_ctas,
               workspace, workspace_bytes, error_word, who);
  if (rc != NVK_OK || batch == 0) return rc;
  a.scale_log2 = scale * 1.4426950408889634f * k_scale;
  a.v_scale = v_scale;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const char* what = "fp4_paged_decode launch";
  return a.group <= kFewHeads ? launch<Format<16>>(a, batch, ctas, kFewHeads, what, st)
                              : launch<Format<12>>(a, batch, ctas, kMaxGroup, what, st);
}
