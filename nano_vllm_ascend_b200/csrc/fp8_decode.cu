// Paged decode attention over the 8-bit KV pool, one query token a sequence:
//   out[b, h] = softmax(scale * q[b, h] . K_b^T) . V_b
// with K and V the values that the codes and exponents of fp8_kv.cuh stand for.
// The schedule, the rings and the joins are in decode_core.cuh.
//
// HBM-bound: 258 bytes per (token, KV head) are read once. Tensor-core operands
// are made in registers, as for the 4-bit pool (fp4_decode.cu says why):
//   S^T[16 tokens x 8 heads] = K[16 x 128] . Q^T, eight steps of 16 dims
//   O^T[16 dims x 8 heads] (8 tiles) += V^T[16 dims x 16 tokens] . P^T
// K and V enter as e4m3 -> fp16 (one conversion for two values): exact. A lane's
// words are whole 16-byte chunks: of K the 32 dims 32 t .. 32 t + 31 of tokens g
// and g + 8 (t = lane % 4, g = lane / 4), of V the dims 16 g .. 16 g + 15 of
// tokens 2 t, 2 t + 1, 2 t + 8 and 2 t + 9, whose bytes are paired by token; the
// order of the chunks in a row makes both free of bank conflicts. Q's fragments
// take the same order of dims.
//
// Exponents. K's multiplies the products: exact. V's is added to the exponent
// of the weights, so that what enters the tensor cores is p 2^e, and the sum of
// the weights takes p 2^e times 2^-e back (both in fp32, exact but for the
// smallest weights). Weights are relative to a reference that follows the
// largest p 2^e, not the largest p: p 2^e is held as fp16 where the largest one
// is held as 2^12 or more, normal down to 2^-26 of that and with a floor of
// 2^-37 of it, so that whatever the units' exponents are, what a token gives is
// right beside what the others give. Exponents are within 40 of 0, so that a
// weight times 2^-e stays in fp32's range.
// Measured: 256 contexts of 2048 to 6144 tokens (16 heads on 8, 2.16 GB) in 323
// to 341 us, 0.97 to 1.02 of the measured copy rate; two of 40960 tokens (32 on
// 8, 169 MB) in 33.3, 0.77: start, ends and the join of pieces; 77 ragged ones of
// up to 1499 tokens (10 on 2) in 14.0 where their 33 MB take 5: a CTA's share is
// four units a warp. A kernel of one warp a unit and dot products by lanes took
// 4900, 29200 and 1003 us.
#include <type_traits>

#include "decode_core.cuh"
#include "fp8_kv.cuh"

namespace nvk {
namespace fp8 {
namespace {

using namespace decode;
using decode::kD;
using decode::kUnitTokens;

constexpr float kRescale = 3.f;  // log2 by which a weight may pass the reference before that moves and O is rescaled
constexpr float kPShift = 12.f;  // weights are held times 2^12, so up to 2^15 in fp16

struct State {
  uint32_t q;     // shared address of this lane's B fragments of Q^T (see load_q)
  float sc[2];    // factor from products to scores in log2 units, of heads 2 t and 2 t + 1
  float ref[2];   // w = 2^((product - ref) * sc + e - exp + kPShift), e the unit's exponent of V: the largest product,
  float exp[2];   // and the largest exponent of a weight relative to it (-inf at first)
  float l[2];     // this lane's part of the sum of w 2^-e
  float o[8][4];  // O^T: dim 16 g + 2 j (heads 2 t, 2 t + 1), then 16 g + 2 j + 1 (the same)
};

// The factor from products to scores, as for the 4-bit pool, but below 2^53:
// with a row's largest entry below 2^16 and codes up to 448 * 2^40 the products
// are below 2^72, and their differences times the factor have to stay finite.
__device__ __forceinline__ float factor(float up, float scale_log2) {
  const float f = fp4::score_factor(up, scale_log2);
  return f > 9007199254740992.f ? 9007199254740992.f : f;  // NaN stays
}

// Q's rows of one pair as fragments: head g, dims 32 t + 4 j + {0, 1} and {2, 3} for step j.
__device__ __forceinline__ void load_q(const DecodeArgs& a, int b, int h, int g, int t, State& st) {
  uint4 raw[4];
  const bool live = g < a.group;
  const __nv_bfloat16* row = a.q + (static_cast<int64_t>(b) * a.heads + h * a.group + (live ? g : 0)) * kD + 32 * t;
#pragma unroll
  for (int w = 0; w < 4; ++w) raw[w] = live ? *reinterpret_cast<const uint4*>(row + 8 * w) : make_uint4(0, 0, 0, 0);
  uint32_t big = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    big = fp4::bf16x2_abs_max(big, fp4::bf16x2_abs_max(fp4::bf16x2_abs_max(raw[w].x, raw[w].y),
                                                       fp4::bf16x2_abs_max(raw[w].z, raw[w].w)));
  big = fp4::bf16x2_abs_max(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = fp4::bf16x2_abs_max(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const fp4::HalfRow half = fp4::half_row(big);
  auto to_half = [&](uint32_t w) { return fp4::bf16x2_to_half2(w, half.base); };
#pragma unroll
  for (int w = 0; w < 4; ++w)  // steps 2 w and 2 w + 1
    st_shared_v4(st.q + 512 * w, to_half(raw[w].x), to_half(raw[w].y), to_half(raw[w].z), to_half(raw[w].w));
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    st.sc[e] = factor(__shfl_sync(0xffffffffu, half.up, 8 * t + 4 * e), a.scale_log2);
    st.ref[e] = 0.f;
    st.exp[e] = -INFINITY;
    st.l[e] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) st.o[j][c] = 0.f;
}

// Products of one unit: x[0], x[1] of token g's heads 2 t and 2 t + 1, x[2], x[3] of token g + 8's.
template <bool kMask>
__device__ __forceinline__ void products(const State& st, uint32_t unit, int exp, int valid, int g, int t,
                                         float (&x)[4]) {
  const uint32_t row = unit + 128 * g, at = (32 * t) ^ (16 * g);  // chunk 2 t's place; g + 8 has the same
  const uint4 a0 = ld_shared_v4(row + at), a1 = ld_shared_v4(row + (at ^ 16));
  const uint4 b0 = ld_shared_v4(row + 1024 + at), b1 = ld_shared_v4(row + 1024 + (at ^ 16));
  const uint32_t wa[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
  const uint32_t wb[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
  float d[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};  // two shorter chains
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint4 f = ld_shared_v4(st.q + 512 * w);
    uint32_t la, ha, lb, hb;
    e4m3_to_half2(wa[2 * w], la, ha);
    e4m3_to_half2(wb[2 * w], lb, hb);
    mma_16816(d, la, lb, ha, hb, f.x, f.y);
    e4m3_to_half2(wa[2 * w + 1], la, ha);
    e4m3_to_half2(wb[2 * w + 1], lb, hb);
    mma_16816(e, la, lb, ha, hb, f.z, f.w);
  }
  const float by = pow2(exp);
#pragma unroll
  for (int c = 0; c < 4; ++c) x[c] = (d[c] + e[c]) * by;
  if (kMask) {
    if (g >= valid) x[0] = x[1] = -INFINITY;
    if (g + 8 >= valid) x[2] = x[3] = -INFINITY;
  }
}

// O += V^T P^T of one unit; b0 and b1 are the fragments of P^T. Tokens from
// `valid` on read as zeros, so that nothing that they hold (a NaN) meets their
// weights of 0.
template <bool kMask>
__device__ __forceinline__ void weigh(State& st, uint32_t unit, int valid, int g, int t, uint32_t b0, uint32_t b1) {
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 2 * t + (i & 1) + 4 * (i & 2);  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
    v[i] = ld_shared_v4(unit + kOffV + 128 * r + 16 * (g ^ (r & 7)));
    if (kMask && r >= valid) v[i] = make_uint4(0, 0, 0, 0);
  }
  const uint32_t* w[4] = {&v[0].x, &v[1].x, &v[2].x, &v[3].x};
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // dims 16 g + 4 i .. + 3: tiles 2 i and 2 i + 1
    uint32_t p[4], q[4];
    e4m3_to_half2(__byte_perm(w[0][i], w[1][i], 0x5140), p[0], p[1]);
    e4m3_to_half2(__byte_perm(w[0][i], w[1][i], 0x7362), p[2], p[3]);
    e4m3_to_half2(__byte_perm(w[2][i], w[3][i], 0x5140), q[0], q[1]);
    e4m3_to_half2(__byte_perm(w[2][i], w[3][i], 0x7362), q[2], q[3]);
    mma_16816(st.o[2 * i], p[0], p[1], q[0], q[1], b0, b1);
    mma_16816(st.o[2 * i + 1], p[2], p[3], q[2], q[3], b0, b1);
  }
}

// One tile: its first `valid` tokens are the sequence's (kMask: fewer than all).
template <bool kMask, int kUnits>
__device__ __forceinline__ void attend(State& st, uint32_t tile, int valid, int g, int t) {
  float x[kUnits][4], ve[kUnits];  // products, then the weights' exponents
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint2 exps = ld_shared_v2(tile + u * kUnitBytes + kOffExp);
    products<kMask>(st, tile + u * kUnitBytes, held_exp(exps.x), valid - u * kUnitTokens, g, t, x[u]);
    ve[u] = static_cast<float>(held_exp(exps.y));
  }
  float d[kUnits][4], most[2] = {-INFINITY, -INFINITY};
  auto exponents = [&] {
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        d[u][c] = fmaf(x[u][c] - st.ref[c & 1], st.sc[c & 1], ve[u] - st.exp[c & 1]);
        most[c & 1] = fmaxf(most[c & 1], d[u][c]);
      }
  };
  exponents();
  if (__any_sync(0xffffffffu, most[0] > kRescale || most[1] > kRescale)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      auto all = [](float m) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        return m;
      };
      float m = -INFINITY, n = -INFINITY;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) m = fmaxf(m, fmaxf(x[u][e], x[u][2 + e]));
      m = all(m);
      const bool first = st.exp[e] == -INFINITY;
      m = first ? m : fmaxf(m, st.ref[e]);
      m = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        n = fmaxf(n, fmaf(fmaxf(x[u][e], x[u][2 + e]) - m, st.sc[e], ve[u]));
      n = all(n);
      const float old = first ? -INFINITY : fmaf(st.ref[e] - m, st.sc[e], st.exp[e]);
      n = fmaxf(n, old);
      const float f = first ? 0.f : fast_exp2(old - n);
      st.ref[e] = m;
      st.exp[e] = n;
      st.l[e] *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) st.o[j][e] *= f, st.o[j][2 + e] *= f;
    }
    exponents();
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    auto weight = [&](int c) { return fast_exp2(d[u][c] + kPShift); };
    const float p0 = weight(0), p1 = weight(1), p2 = weight(2), p3 = weight(3);
    const float by = fast_exp2(-ve[u]);  // exact
    st.l[0] = fmaf(p0 + p2, by, st.l[0]);
    st.l[1] = fmaf(p1 + p3, by, st.l[1]);
    const uint32_t b0 = movmatrix(half2_of(p0, p1)), b1 = movmatrix(half2_of(p2, p3));
    weigh<kMask>(st, tile + u * kUnitBytes, valid - u * kUnitTokens, g, t, b0, b1);
  }
}

// The format's part of decode_core.cuh's kernel.
template <int kWarpsOfF, int kUnitsOfF, int kStagesOfF>
struct Format {
  static constexpr int kWarps = kWarpsOfF, kTileUnits = kUnitsOfF, kStages = kStagesOfF;
  static constexpr int kUnitBytes = fp8::kUnitBytes, kTileTokens = kTileUnits * kUnitTokens;
  static constexpr int kTileBytes = kTileUnits * kUnitBytes;
  // a CTA's least work: 8 units, four contexts of up to 513 tokens then take 6.6 us (16: 7.4; 32: 9.0; 6: 6.9; 4: 7.4)
  static constexpr int kMinTiles = 8 / kTileUnits;
  static constexpr bool kExps = true;  // a piece's reference is its largest product and an exponent
  using State = fp8::State;
  struct Scratch {};

  static __device__ __forceinline__ void load_q(const DecodeArgs& a, int b, int h, int g, int t, State& st) {
    fp8::load_q(a, b, h, g, t, st);
  }
  template <bool kMask>
  static __device__ __forceinline__ void attend(State& st, uint32_t tile, uint32_t, int valid, int g, int t, int) {
    fp8::attend<kMask, kTileUnits>(st, tile, valid, g, t);
  }
  static __device__ __forceinline__ float down(const State&) { return 1.f; }
  static __device__ __forceinline__ float4 piece(const State& st, int e) {
    return make_float4(st.exp[e] == -INFINITY ? -INFINITY : st.ref[e], st.l[e], st.sc[e], st.exp[e]);
  }
  static __device__ __forceinline__ int dim(int j, int g) { return 16 * g + 2 * j; }
};

// 14 warps, a unit a tile, two tiles in flight a warp: 28 units (116 KB) an SM, and 128 registers a thread. 64 contexts of 4096 tokens of 8 KV heads with two, five and eight heads a group: 85.5,
// 86.5 and 89.5 us; 16 warps (up to six heads fit) 89.2, 91.0 and none; 12 of three tiles 93.7 and 96.8 (five, eight); 10
// of tiles of two units 87.2, 90.9 and 93.4. 77 ragged contexts, five heads: 14.0, 14.3, 15.2 and 14.5.
using Only = Format<14, 1, 2>;
static_assert(smem_bytes<Only>(kMaxGroup) <= 232448, "decode shared memory exceeds the 227 KB per-CTA limit");

}  // namespace
}  // namespace fp8
}  // namespace nvk

extern "C" int nvk_fp8_paged_decode_workspace_size(int num_heads, int num_kv_heads, int head_dim, int num_ctas,
                                                   size_t* bytes) {
  using namespace nvk;
  const char* who = "fp8_paged_decode_workspace_size";
  if (!bytes) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (head_dim != fp8::kD) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", who, head_dim);
  int rc = decode::check_heads(num_heads, num_kv_heads, num_ctas, who), ctas = 0;
  if (rc != NVK_OK || (rc = decode::resolve_ctas(num_ctas, who, &ctas)) != NVK_OK) return rc;
  *bytes = decode::workspace_bytes(num_heads / num_kv_heads, ctas);
  return NVK_OK;
}

extern "C" int nvk_fp8_paged_decode(void* out, const void* query, const void* kv_cache, int num_blocks,
                                    int block_size, const int32_t* block_tables, int block_table_stride,
                                    int max_blocks_per_seq, const int32_t* context_lens, int batch, int num_heads,
                                    int num_kv_heads, int head_dim, float scale, int num_ctas, void* workspace,
                                    size_t workspace_bytes, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp8;
  const char* who = "fp8_paged_decode";
  if (batch < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: batch %d", who, batch);
  int rc = check_heads(num_heads, num_kv_heads, num_ctas, who), ctas = 0;
  if (rc != NVK_OK) return rc;
  if ((rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, who)) != NVK_OK) return rc;
  DecodeArgs a;
  rc = prepare(a, ctas, out, query, kv_cache, num_blocks, units_log2(block_size), block_size, block_tables,
               block_table_stride, max_blocks_per_seq, context_lens, batch, num_heads, num_kv_heads, scale, num_ctas,
               workspace, workspace_bytes, error_word, who);
  if (rc != NVK_OK || batch == 0) return rc;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.v_scale = 1.f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const char* what = "fp8_paged_decode launch";
  return launch<Only>(a, batch, ctas, kMaxGroup, what, st);
}
