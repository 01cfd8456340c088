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
// Data: every warp streams its tiles (two units, 32 tokens) through a ring of
// its own in shared memory, one bulk copy of 4608 contiguous bytes a tile (two
// copies where a block is one unit), two in flight: 74 to 147 KB an SM, where
// about 55 KB hide HBM's latency at full rate. No warp waits for another one's
// data.
//
// Schedule: the tiles of all (sequence, KV head) pairs, sequence
// major, are cut into equal contiguous ranges, one per CTA, each cut into
// equal ranges of its warps, wherever the cuts fall. A warp keeps its own
// running maximum (as a product of q and k: weights go by differences of
// products, so that they are right however large the scores are), sum and O;
// pairs that lie in one warp are written by it, the others' pieces meet in
// shared memory at the end, and pairs split over CTAs in the workspace, where
// the CTA that arrives last (a ticket) joins them. Nothing waits for another
// CTA.
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
#include "fp4_kv.cuh"

namespace nvk {
namespace fp4 {
namespace {

constexpr int kTileTokens = 2 * kUnitTokens;  // a warp's step
constexpr int kTileBytes = 2 * kUnitBytes;
constexpr int kStages = 2;       // tiles in flight a warp
constexpr int kMaxCtas = 1024;
// Tiles below which a CTA is not used. Fewer spread short work over more SMs but
// give its joins more pieces (one sequence of 100 / 1000 tokens, 8 KV heads:
// 4.9 / 6.8 us with 8; when it was chosen 4.8 / 7.1, and 6.0 / 8.3 with 16).
constexpr int kMinTiles = 8;
// CTAs that the longest pair may be cut over: the join reads the pieces of a
// pair one after another (one sequence of 40000 tokens, one KV head, 8 query
// heads: 18.3 us with 32, 21.2 with 48, 42 with 148; 2 heads: 12.9, 12.9, 15.1;
// beside four of 10 tokens, 8 heads, 19.7 against 47.2 over all 148).
// The longest one's tiles count, not the number of pairs: short and empty
// sequences beside it take no share of its pieces.
constexpr int kMostPieces = 32;
constexpr int kMaxGroup = 8;     // query heads per KV head: the columns of a fragment
constexpr float kRescale = 3.f;  // log2 by which a score may pass the reference before that moves and O is rescaled
constexpr float kPShift = 4.f;   // P is held as 2^4 p: with p up to 2^3 and scales up to 480, P s fits fp16 (p goes
                                 // by differences of products, so that this holds for scores of any magnitude)
constexpr size_t kTicketOffset = 256;
constexpr size_t kMlOffset = kTicketOffset + kMaxCtas * sizeof(int);
static_assert(kMlOffset == NVK_FP4_DECODE_ZEROED_BYTES, "what has to be zero is the error word and the tickets");

struct DecodeArgs {
  __nv_bfloat16* out;
  const __nv_bfloat16* q;
  const uint8_t* pool;
  const int32_t* tables;
  const int32_t* ctx;
  int* err;
  int* tickets;  // [CTAs], at zero between calls
  float4* ws_ml; // [CTAs][2][group] of a split pair's piece: see Smem's piece_ml
  float* ws_o;   // [CTAs][2][group][128]
  int batch, heads, kvh, group;
  int bt_stride, max_blocks, num_blocks, upb_log2;
  float scale_log2;  // scale * log2(e) * k_scale
  float v_scale;
};

// A pair that a CTA shares with others: end 0 began before the CTA's first tile,
// end 1 begins in the CTA and goes on behind its last.
struct End {
  int pair;    // -1: none
  int c0, c1;  // the CTAs that have a piece of it
  int last;    // this CTA's piece came last: it joins them
};

template <int kWarps>
struct Smem {
  alignas(128) uint8_t ring[kWarps][kStages][kTileBytes];  // a warp's last piece comes here when it has read them
  uint4 q[kWarps][kGroups / 2][32];  // fragments of Q, fp16
  uint2 vscale[kWarps][2][kGroups / 2][4][2];  // [unit][j / 2][quad][j % 2]: V's scales of the quad's four tokens, fp16
  uint64_t full[kWarps][kStages];
  int pre[2 * kWarps * 32 + 1];  // tiles before each sequence (of one KV head)
  int scan[kWarps], most[kWarps];
  int piece_pair[32];
  End end[2];
};
constexpr uint32_t kVScaleBytes = kGroups * kUnitTokens * 2;  // of one unit

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

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

__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st_shared_v2(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

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

__device__ __forceinline__ int ticket(int* p) {
  int v;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Orders this thread's shared-memory writes before later copies into them.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A unit of zeros in place of one that the table does not lead to (by the
// whole warp), ordered before the next copy into its place.
__device__ __forceinline__ void zero_unit(uint32_t unit, int lane) {
  for (int i = lane; i < kUnitBytes / 16; i += 32) st_shared_v4(unit + 16 * i, 0, 0, 0, 0);
  fence_proxy_async();
  __syncwarp();
}

__device__ __forceinline__ int seq_tiles(const DecodeArgs& a, int b, bool report) {
  int n = a.ctx[b];
  const int64_t most = static_cast<int64_t>(a.max_blocks) << (a.upb_log2 + 4);
  if (n > most) {
    if (report) atomicOr(a.err, kErrContextTooLong);
    n = static_cast<int>(most);
  }
  return n <= 0 ? 0 : (n - 1) / kTileTokens + 1;
}

template <int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 1) decode_kernel(const DecodeArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Sm = Smem<kWarps>;
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  // Pieces of pairs that are not one warp's: [2 * kWarps][group] (largest
  // product, or -inf; sum; sc, the pair's; unused), and [group][128] each: a
  // warp's first one in its own place, its last one in the warp's ring.
  float4* piece_ml = reinterpret_cast<float4*>(smem_raw + sizeof(Sm));
  float* piece_first = reinterpret_cast<float*>(piece_ml + 2 * kWarps * a.group);
  auto piece_o = [&](int p) {
    return (p & 1) ? reinterpret_cast<float*>(sm.ring[p >> 1]) : piece_first + (p >> 1) * a.group * kD;
  };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[warp][s], 1);
    fence_mbar_init();
  }
  pdl_launch_dependents();
  // The lengths and the tables are step metadata, which no kernel writes that
  // lets its dependents start early (see the entry point): they are read, and
  // the schedule made of them, while the kernel before this one drains.

  // ---- the prefix of tiles: two sequences a thread ----
  {
    const int b = 2 * tid;
    const int u0 = b < a.batch ? seq_tiles(a, b, blockIdx.x == 0) : 0;
    const int u1 = b + 1 < a.batch ? seq_tiles(a, b + 1, blockIdx.x == 0) : 0;
    int sum = u0 + u1;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += v;
    }
    const int most = __reduce_max_sync(0xffffffffu, max(u0, u1));
    if (lane == 31) sm.scan[warp] = sum, sm.most[warp] = most;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += sm.scan[w];
    const int at = before + sum - u0 - u1;
    if (b <= a.batch) sm.pre[b] = at;
    if (b + 1 <= a.batch) sm.pre[b + 1] = at + u0;
    if (b + 2 == a.batch) sm.pre[b + 2] = at + u0 + u1;
    if (tid < 32) sm.piece_pair[tid] = -1;
    __syncthreads();
  }
  auto zero_empty = [&] {  // the rows of sequences without context
    for (int b = blockIdx.x * kWarps + warp; b < a.batch; b += gridDim.x * kWarps) {
      if (sm.pre[b + 1] != sm.pre[b]) continue;
      uint32_t* row = reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(b) * a.heads * kD);
      for (int i = lane; i < a.heads * (kD / 2); i += 32) row[i] = 0;
    }
  };
  const int total = sm.pre[a.batch] * a.kvh;  // the entry point keeps it below 2^31
  int longest = 0;  // tiles of a pair
  for (int w = 0; w < (a.batch + 63) / 64; ++w) longest = max(longest, sm.most[w]);
  int ctas = min(static_cast<int>(gridDim.x), (total + kMinTiles - 1) / kMinTiles);
  if (static_cast<int64_t>(longest) * ctas > static_cast<int64_t>(total) * kMostPieces)
    ctas = static_cast<int>(static_cast<int64_t>(total) * kMostPieces / longest);
  const int c = blockIdx.x;
  if (c >= ctas) {
    pdl_wait();
    zero_empty();
    return;
  }
  // Even shares, the first ones a tile larger where it does not come out even.
  const int share = total / ctas, larger = total - share * ctas;
  const int clo = share * c + min(c, larger), chi = clo + share + (c < larger ? 1 : 0);
  const int wshare = (chi - clo) / kWarps, wlarger = (chi - clo) % kWarps;
  const int lo = clo + wshare * warp + min(warp, wlarger), hi = lo + wshare + (warp < wlarger ? 1 : 0);

  auto find_seq = [&](int x) {  // the sequence that tile x belongs to
    int b0 = 0, b1 = a.batch;   // pre[b0] * kvh <= x < pre[b1] * kvh
    while (b1 - b0 > 1) {
      const int mid = (b0 + b1) >> 1;
      if (sm.pre[mid] * a.kvh <= x) b0 = mid;
      else b1 = mid;
    }
    return b0;
  };
  if (warp == kWarps - 1 && lane < 2) {  // the pairs at this CTA's ends
    auto cta_of = [&](int x) {
      const int cut = larger * (share + 1);
      return x < cut ? x / (share + 1) : larger + (x - cut) / share;
    };
    const int x = lane == 0 ? clo : chi - 1;
    const int b = find_seq(x);
    const int tiles = sm.pre[b + 1] - sm.pre[b];
    const int h = (x - sm.pre[b] * a.kvh) / tiles;
    const int plo = sm.pre[b] * a.kvh + h * tiles, phi = plo + tiles;
    const bool split = lane == 0 ? plo < clo : plo >= clo && phi > chi;
    sm.end[lane] = End{split ? b * a.kvh + h : -1, cta_of(plo), cta_of(phi - 1), 0};
  }

  // Writes this warp's result of a pair as a piece (index 2 * warp + slot), or as the output.
  State st;
  st.q = smem_u32(&sm.q[warp][0][lane]);
  auto finish = [&](int b, int h, bool whole, int slot) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], off);
      st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], off);
    }
    const float down = __uint_as_float((127u << 23) - ((st.room & 0xffu) << 20));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = 2 * t + e;
      if (head >= a.group) continue;
      if (whole) {
        const float inv = st.l[e] == 0.f ? 0.f : __fdividef(a.v_scale, st.l[e]) * down;
        __nv_bfloat16* row = a.out + (static_cast<int64_t>(b) * a.heads + h * a.group + head) * kD + 2 * g;
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
          *reinterpret_cast<uint32_t*>(row + 16 * j) = pack_bf16x2(st.o[j][e] * inv, st.o[j][2 + e] * inv);
      } else {
        const int at = (2 * warp + slot) * a.group + head;
        if (g == 0) piece_ml[at] = make_float4(st.thr[e] == -INFINITY ? -INFINITY : st.ref[e], st.l[e], st.sc[e], 0.f);
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
          *reinterpret_cast<float2*>(piece_o(2 * warp + slot) + head * kD + 16 * j + 2 * g) =
              make_float2(st.o[j][e] * down, st.o[j][2 + e] * down);
      }
    }
    if (!whole && lane == 0) sm.piece_pair[2 * warp + slot] = b * a.kvh + h;
  };

  // ---- this warp's tiles ----
  const int n = hi - lo;
  constexpr int kFirst = 1 << 8, kLast = 1 << 9, kBad = 1 << 10, kBad2 = 1 << 11;
  // What lane i knows of the batch of 32 tiles that starts at lo + base: where
  // the units of tile base + i lie, whose it is, and its tokens with the flags
  // above.
  const uint8_t *next_at = nullptr, *next_at2 = nullptr;
  int next_pair = 0, next_info = 0;
  auto look_up = [&](int base) {
    if (base + lane >= n) return;
    const int x = lo + base + lane;
    const int b = find_seq(x);
    const int tiles = sm.pre[b + 1] - sm.pre[b];
    const int in_seq = x - sm.pre[b] * a.kvh;
    const int h = in_seq / tiles;
    const int tile = in_seq - h * tiles;
    const int64_t room = (static_cast<int64_t>(a.max_blocks) << (a.upb_log2 + 4));
    const int64_t left = min(static_cast<int64_t>(a.ctx[b]), room) - static_cast<int64_t>(tile) * kTileTokens;
    const int tokens = static_cast<int>(min(left, static_cast<int64_t>(kTileTokens)));
    next_pair = b * a.kvh + h;
    next_info = tokens | (tile == 0 ? kFirst : 0) | (tile == tiles - 1 ? kLast : 0);
    auto place = [&](int unit, int flag) {
      const int blk = a.tables[static_cast<int64_t>(b) * a.bt_stride + (unit >> a.upb_log2)];
      if (blk < 0 || blk >= a.num_blocks) next_info |= flag;
      return a.pool + ((((static_cast<int64_t>(blk) * a.kvh + h) << a.upb_log2) + (unit & ((1 << a.upb_log2) - 1))) *
                       kUnitBytes);
    };
    next_at = place(2 * tile, kBad);
    // blocks of one unit: the tile's second unit has a block of its own
    if (a.upb_log2 == 0 && tokens > kUnitTokens) next_at2 = place(2 * tile + 1, kBad2);
    else if (next_info & kBad) next_info |= kBad2;
  };
  auto fetch = [&](int i) {  // tile i into its stage, by the lane that knows it
    if (lane != (i & 31)) return;
    uint64_t* bar = &sm.full[warp][i % kStages];
    uint8_t* to = sm.ring[warp][i % kStages];
    const bool two = (next_info & 0xff) > kUnitTokens;
    if (a.upb_log2 > 0 && !(next_info & kBad)) {  // one copy
      mbar_arrive_expect_tx(bar, two ? kTileBytes : kUnitBytes);
      bulk_load(to, next_at, two ? kTileBytes : kUnitBytes, bar);
      return;
    }
    const bool one_ok = !(next_info & kBad), two_ok = two && !(next_info & kBad2);
    if (!one_ok || (two && !two_ok)) atomicOr(a.err, kErrBadBlockId);
    if (!one_ok && !two_ok) {
      mbar_arrive(bar);
      return;
    }
    mbar_arrive_expect_tx(bar, (one_ok ? kUnitBytes : 0) + (two_ok ? kUnitBytes : 0));
    if (one_ok) bulk_load(to, next_at, kUnitBytes, bar);
    if (two_ok) bulk_load(to + kUnitBytes, next_at2, kUnitBytes, bar);
  };
  look_up(0);
  pdl_wait();
  zero_empty();
  int issued = 0;
  for (; issued < min(n, kStages); ++issued) fetch(issued);
  int pair_now = next_pair, info_now = next_info;  // the batch that is being read
  bool ok = true, whole = false, open = false;
  int b = 0, h = 0, slot = 0;
  const uint32_t ring = smem_u32(sm.ring[warp]), vscale = smem_u32(sm.vscale[warp]);
  for (int i = 0; i < n; ++i) {
    if ((i & 31) == 0 && i > 0) pair_now = next_pair, info_now = next_info;
    const int info = __shfl_sync(0xffffffffu, info_now, i & 31);
    if (!open) {
      const int pair = __shfl_sync(0xffffffffu, pair_now, i & 31);
      b = pair / a.kvh;
      h = pair - b * a.kvh;
      load_q(a, b, h, g, t, st);
      whole = info & kFirst;
      slot = i == 0 ? 0 : 1;
      open = true;
    }
    const uint32_t tile = ring + (i % kStages) * kTileBytes;
    uint64_t* bar = &sm.full[warp][i % kStages];
    const uint32_t parity = (i / kStages) & 1;
    if (ok && !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)) && !__all_sync(0xffffffffu, mbar_wait(bar, parity))) {
      ok = false;
      if (lane == 0) atomicOr(a.err, kErrWaitTimeout);
    }
    const int tokens = info & 0xff;
    if (tokens == kTileTokens && !(info & (kBad | kBad2)) && ok) {
      attend<false>(st, tile, vscale, tokens, g, t, lane);
    } else {
      if (!ok || (info & kBad)) zero_unit(tile, lane);  // reads as zeros
      if (!ok || (info & kBad2)) zero_unit(tile + kUnitBytes, lane);
      attend<true>(st, tile, vscale, tokens, g, t, lane);
    }
    __syncwarp();  // every lane is done with the tile
    if (ok && issued < n) {
      if ((issued & 31) == 0) look_up(issued);
      fetch(issued);
      ++issued;
    }
    if ((info & kLast) || i == n - 1) {
      if (!ok)  // the ring takes the piece only after every copy into it has landed or been given up
        for (int k = max(i, issued - kStages); k < issued; ++k)
          (void)mbar_wait(&sm.full[warp][k % kStages], (k / kStages) & 1);
      finish(b, h, whole && (info & kLast), slot);
      open = false;
    }
  }
  __syncthreads();

  // ---- the pieces of one pair meet ----
  // Piece 2 w of warp w is what it had of a pair that began before it (or all
  // it had), piece 2 w + 1 of one that goes on behind it. A run of pieces of
  // one pair is its first one and then pieces 2 w of the warps after that.
  auto write_out = [&](int pair, int head, float l, const float4& o) {
    const float inv = l == 0.f ? 0.f : __fdividef(a.v_scale, l);
    const int pb = pair / a.kvh, ph = pair - pb * a.kvh;
    *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(pb) * a.heads + ph * a.group + head) * kD + 4 * lane) =
        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  };
  // a piece whose products were all -inf or NaN has the latter's NaN in its sum
  auto weight = [](float ref, float l, float m, float sc) {
    return ref == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2((ref - m) * sc);
  };
  auto warp_max = [](float m) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    return m;
  };
  auto warp_sum = [](float l) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    return l;
  };
  const int mine = sm.piece_pair[lane];  // lane p of every warp looks at piece p
  const uint32_t valid = __ballot_sync(0xffffffffu, mine >= 0);
  const uint32_t below = valid & ((1u << lane) - 1);
  const int prev = __shfl_sync(0xffffffffu, mine, below ? 31 - __clz(below) : 0);
  uint32_t starts = __ballot_sync(0xffffffffu, mine >= 0 && (below == 0 || prev != mine));
  for (int k = warp, at = 0; starts; at += a.group, starts &= starts - 1) {
    for (; k < at + a.group; k += kWarps) {  // task k: head k - at of this run
      const int head = k - at, first = __ffs(starts) - 1;
      const int pair = __shfl_sync(0xffffffffu, mine, first);
      const int count = __popc(__ballot_sync(0xffffffffu, mine == pair));
      const float4 ml = mine == pair ? piece_ml[lane * a.group + head] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      const float m = warp_max(ml.x);
      const float w = weight(ml.x, ml.y, m, ml.z), l = warp_sum(ml.y * w);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < count; ++i) {
        const int p = i == 0 ? first : 2 * ((first >> 1) + i);
        const float wp = __shfl_sync(0xffffffffu, w, p);
        const float4 v = *reinterpret_cast<const float4*>(piece_o(p) + head * kD + 4 * lane);
        o.x += wp * v.x, o.y += wp * v.y, o.z += wp * v.z, o.w += wp * v.w;
      }
      const int end = pair == sm.end[0].pair ? 0 : pair == sm.end[1].pair ? 1 : -1;
      if (end < 0) {
        write_out(pair, head, l, o);
      } else {
        const int64_t to = (static_cast<int64_t>(c) * 2 + end) * a.group + head;
        if (lane == first) a.ws_ml[to] = make_float4(m, l, ml.z, 0.f);
        *reinterpret_cast<float4*>(a.ws_o + to * kD + 4 * lane) = o;
      }
    }
  }
  // ---- pairs split over CTAs: the CTA whose piece comes last joins them ----
  __syncthreads();
  if (tid < 2 && sm.end[tid].pair >= 0) {
    const End e = sm.end[tid];
    // the CTA's pieces, which the barrier put before this, are out before the ticket; whoever takes
    // the last one sees all of them
    if (ticket(a.tickets + e.c0) == e.c1 - e.c0) {
      a.tickets[e.c0] = 0;  // every piece is in: nobody else touches it in this call
      sm.end[tid].last = 1;
    }
  }
  __syncthreads();
  // A task is a share of the pieces of one end and head: part, part + parts, ...,
  // kAhead loads in flight. Several parts meet in shared memory (the rings are done).
  constexpr int kAhead = 4;
  const int most = max(1, kWarps / (2 * a.group));
  auto parts_of = [&](const End& e) { return min(most, (e.c1 - e.c0 + kAhead) / kAhead); };
  float4* sum_o = reinterpret_cast<float4*>(sm.ring);
  float* sum_l = reinterpret_cast<float*>(sm.q);
  for (int k = warp; k < 2 * a.group * most; k += kWarps) {
    const int part = k / (2 * a.group), end = k & 1, head = (k >> 1) - part * a.group;
    const End e = sm.end[end];
    if (e.pair < 0 || !e.last || part >= parts_of(e)) continue;
    // the pair's piece in CTA i: its end 1 where it begins, its end 0 after that
    const int count = e.c1 - e.c0 + 1, parts = parts_of(e);
    auto at = [&](int i) { return (static_cast<int64_t>(e.c0 + i) * 2 + (i == 0 ? 1 : 0)) * a.group + head; };
    const float sc = __ldcg(&a.ws_ml[at(0)].z);
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = lane; i < count; i += 32) m = fmaxf(m, __ldcg(&a.ws_ml[at(i)].x));
    for (int i0 = part; i0 < count; i0 += kAhead * parts) {
      float4 v[kAhead];
      float2 ml[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + j * parts;
        ml[j] = i < count ? __ldcg(reinterpret_cast<const float2*>(a.ws_ml + at(i))) : make_float2(-INFINITY, 0.f);
        v[j] = i < count ? __ldcg(reinterpret_cast<const float4*>(a.ws_o + at(i) * kD + 4 * lane))
                         : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (i0 == part) m = warp_max(m);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float w = weight(ml[j].x, ml[j].y, m, sc);
        l += w * ml[j].y;
        o.x += w * v[j].x, o.y += w * v[j].y, o.z += w * v[j].z, o.w += w * v[j].w;
      }
    }
    if (parts == 1) {
      write_out(e.pair, head, l, o);
    } else {
      sum_o[k * 32 + lane] = o;
      if (lane == 0) sum_l[k] = l;
    }
  }
  __syncthreads();
  for (int k = warp; k < 2 * a.group; k += kWarps) {
    const End e = sm.end[k & 1];
    if (e.pair < 0 || !e.last || parts_of(e) == 1) continue;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int part = 0; part < parts_of(e); ++part) {
      const int i = k + part * 2 * a.group;
      const float4 v = sum_o[i * 32 + lane];
      l += sum_l[i];
      o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    }
    write_out(e.pair, k >> 1, l, o);
  }
}

template <int kWarps>
constexpr size_t smem_bytes(int group) {
  return sizeof(Smem<kWarps>) + static_cast<size_t>(kWarps) * group * (2 * sizeof(float4) + kD * sizeof(float));
}
// 16 warps where shared memory has room for the pieces of the group's heads
// beside their rings, else 12 (16 against 12 at two heads, 256 contexts of
// about 4096 tokens: 230 against 244 us).
constexpr int kFewHeads = 4;
static_assert(sizeof(Smem<16>) % 16 == 0 && sizeof(Smem<12>) % 16 == 0, "the pieces behind it are 16-byte aligned");
static_assert(smem_bytes<16>(kFewHeads) <= 232448 && smem_bytes<12>(kMaxGroup) <= 232448,
              "decode shared memory exceeds the 227 KB per-CTA limit");
static_assert(kStages * kTileBytes >= kMaxGroup * kD * 4, "a warp's ring takes its last piece");

// The sequences in launches of as many as the kernel's prefix holds.
template <int kWarps>
int launch(DecodeArgs a, int batch, int ctas, cudaStream_t stream) {
  const void* kernel = reinterpret_cast<const void*>(&decode_kernel<kWarps>);
  int rc = ensure_dynamic_smem(kernel, smem_bytes<kWarps>(kWarps == 16 ? kFewHeads : kMaxGroup));
  constexpr int kMaxSeqs = 2 * kWarps * 32;
  for (int left = batch; rc == NVK_OK && left > 0; left -= kMaxSeqs) {
    a.batch = left < kMaxSeqs ? left : kMaxSeqs;
    rc = check_cuda(launch_pdl(decode_kernel<kWarps>, dim3(ctas), dim3(kWarps * 32), smem_bytes<kWarps>(a.group),
                               stream, a),
                    "fp4_paged_decode launch");
    a.out += static_cast<int64_t>(kMaxSeqs) * a.heads * kD;
    a.q += static_cast<int64_t>(kMaxSeqs) * a.heads * kD;
    a.tables += static_cast<int64_t>(kMaxSeqs) * a.bt_stride;
    a.ctx += kMaxSeqs;
  }
  return rc;
}

size_t workspace_bytes(int group, int ctas) {
  return kMlOffset + static_cast<size_t>(ctas) * 2 * group * (sizeof(float4) + kD * sizeof(float));
}

int resolve_ctas(int num_ctas, int* out) {
  int ctas = num_ctas;
  if (ctas == 0) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&ctas, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return check_cuda(e, "fp4_paged_decode: SM count");
  }
  *out = ctas < kMaxCtas ? ctas : kMaxCtas;
  return NVK_OK;
}

int check_heads(int num_heads, int num_kv_heads, int num_ctas, const char* who) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_ctas < 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (heads=%d kv_heads=%d ctas=%d)", who, num_heads, num_kv_heads,
                num_ctas);
  if (num_heads % num_kv_heads != 0 || num_heads / num_kv_heads > kMaxGroup)
    return fail(NVK_ERR_UNSUPPORTED, "%s: %d query heads over %d KV heads (a GQA group of 1 to %d)", who, num_heads,
                num_kv_heads, kMaxGroup);
  return NVK_OK;
}

}  // namespace
}  // namespace fp4
}  // namespace nvk

extern "C" int nvk_fp4_paged_decode_workspace_size(int num_heads, int num_kv_heads, int head_dim, int num_ctas,
                                                   size_t* bytes) {
  using namespace nvk;
  using namespace nvk::fp4;
  const char* who = "fp4_paged_decode_workspace_size";
  if (!bytes) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (head_dim != kD) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", who, head_dim);
  int rc = check_heads(num_heads, num_kv_heads, num_ctas, who), ctas = 0;
  if (rc != NVK_OK || (rc = resolve_ctas(num_ctas, &ctas)) != NVK_OK) return rc;
  *bytes = workspace_bytes(num_heads / num_kv_heads, ctas);
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
                                              size_t workspace_bytes_given, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp4;
  const char* who = "fp4_paged_decode";
  if (batch < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: batch %d", who, batch);
  int rc = check_heads(num_heads, num_kv_heads, num_ctas, who);
  if (rc != NVK_OK) return rc;
  if ((rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, k_scale, v_scale, who)) != NVK_OK)
    return rc;
  if (!(scale > 0.f)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: scale %g is not positive", who, double(scale));
  if (max_blocks_per_seq <= 0 || block_table_stride < max_blocks_per_seq)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: block table stride %d below its %d columns", who, block_table_stride,
                max_blocks_per_seq);
  if (batch == 0) return NVK_OK;
  if (!out || !query || !block_tables || !context_lens || !workspace)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(out) || !aligned16(query) || !aligned16(workspace))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: q, out and workspace must be 16-byte aligned", who);
  const int upb_log2 = units_log2(block_size);
  const int64_t seqs = batch < 1024 ? batch : 1024;
  if (((seqs * max_blocks_per_seq * num_kv_heads) << upb_log2) > 0x7fffffffll ||
      (static_cast<int64_t>(max_blocks_per_seq) << upb_log2) > 0x7fffffffll / kUnitTokens)
    return fail(NVK_ERR_UNSUPPORTED, "%s: %d blocks of %d tokens a sequence and %d KV heads are above the kernel's range",
                who, max_blocks_per_seq, block_size, num_kv_heads);
  int ctas = 0;
  if ((rc = resolve_ctas(num_ctas, &ctas)) != NVK_OK) return rc;
  const int group = num_heads / num_kv_heads;
  if (workspace_bytes_given < workspace_bytes(group, ctas))
    return fail(NVK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes_given,
                workspace_bytes(group, ctas));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  DecodeArgs a;
  a.pool = static_cast<const uint8_t*>(kv_cache);
  a.err = error_word ? error_word : reinterpret_cast<int*>(ws);
  a.tickets = reinterpret_cast<int*>(ws + kTicketOffset);
  a.ws_ml = reinterpret_cast<float4*>(ws + kMlOffset);
  a.ws_o = reinterpret_cast<float*>(ws + kMlOffset + static_cast<size_t>(ctas) * 2 * group * sizeof(float4));
  a.heads = num_heads;
  a.kvh = num_kv_heads;
  a.group = group;
  a.bt_stride = block_table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks;
  a.upb_log2 = upb_log2;
  a.scale_log2 = scale * 1.4426950408889634f * k_scale;
  a.v_scale = v_scale;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.q = static_cast<const __nv_bfloat16*>(query);
  a.tables = block_tables;
  a.ctx = context_lens;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return group <= kFewHeads ? launch<16>(a, batch, ctas, st) : launch<12>(a, batch, ctas, st);
}
