// Paged decode attention over a quantised KV pool, one query token a sequence:
// the schedule, the rings and the joins that fp4_decode.cu (the 4-bit pool) and
// fp8_decode.cu (the 8-bit pool) share. What hangs on the pool's format is a
// struct F of theirs: the size of its units, Q's fragments, and a tile's scores,
// weights and products with V.
//
// Data: every warp streams its tiles (F::kTileUnits units of 16 tokens) through
// a ring of its own in shared memory, one bulk copy of contiguous bytes a tile
// (a copy for each unit where a block is one unit), F::kStages in flight. No
// warp waits for another one's data.
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
#pragma once

#include <type_traits>

#include "fp4_kv.cuh"

namespace nvk {
namespace decode {

constexpr int kD = 128;
constexpr int kUnitTokens = 16;
constexpr int kMaxCtas = 1024;
// CTAs that the longest pair may be cut over: the join reads the pieces of a
// pair one after another (one sequence of 40000 tokens, one KV head, 8 query
// heads: 18.3 us with 32, 21.2 with 48, 42 with 148; 2 heads: 12.9, 12.9, 15.1;
// beside four of 10 tokens, 8 heads, 19.7 against 47.2 over all 148).
// The longest one's tiles count, not the number of pairs: short and empty
// sequences beside it take no share of its pieces.
constexpr int kMostPieces = 32;
constexpr int kMaxGroup = 8;     // query heads per KV head: the columns of a fragment
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
  float scale_log2;  // scale * log2(e) (* k_scale)
  float v_scale;
};

// A pair that a CTA shares with others: end 0 began before the CTA's first tile,
// end 1 begins in the CTA and goes on behind its last.
struct End {
  int pair;    // -1: none
  int c0, c1;  // the CTAs that have a piece of it
  int last;    // this CTA's piece came last: it joins them
};

template <typename F>
struct Smem {
  alignas(128) uint8_t ring[F::kWarps][F::kStages][F::kTileBytes];  // a warp's last piece comes here when it has read them
  uint4 q[F::kWarps][4][32];  // fragments of Q, fp16
  typename F::Scratch scratch[F::kWarps];
  uint64_t full[F::kWarps][F::kStages];
  int pre[2 * F::kWarps * 32 + 1];  // tiles before each sequence (of one KV head)
  int scan[F::kWarps], most[F::kWarps];
  int piece_pair[32];
  End end[2];
};

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

__device__ __forceinline__ int ticket(int* p) {
  int v;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Orders this thread's shared-memory writes before later copies into them.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A unit of zeros in place of one that the table does not lead to (by the
// whole warp), ordered before the next copy into its place.
template <typename F>
__device__ __forceinline__ void zero_unit(uint32_t unit, int lane) {
  for (int i = lane; i < F::kUnitBytes / 16; i += 32) st_shared_v4(unit + 16 * i, 0, 0, 0, 0);
  fence_proxy_async();
  __syncwarp();
}

template <typename F>
__device__ __forceinline__ int seq_tiles(const DecodeArgs& a, int b, bool report) {
  int n = a.ctx[b];
  const int64_t most = static_cast<int64_t>(a.max_blocks) << (a.upb_log2 + 4);
  if (n > most) {
    if (report) atomicOr(a.err, kErrContextTooLong);
    n = static_cast<int>(most);
  }
  return n <= 0 ? 0 : (n - 1) / F::kTileTokens + 1;
}

template <typename F>
__global__ void __launch_bounds__(F::kWarps * 32, 1) decode_kernel(const DecodeArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr int kWarps = F::kWarps, kStages = F::kStages, kTileTokens = F::kTileTokens, kTileBytes = F::kTileBytes;
  constexpr int kUnitBytes = F::kUnitBytes;
  constexpr bool kTwo = F::kTileUnits == 2;
  static_assert(F::kTileUnits == 1 || kTwo, "a tile is one unit or two");
  using Sm = Smem<F>;
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  // Pieces of pairs that are not one warp's: [2 * kWarps][group] (largest
  // product, or -inf; sum; sc, the pair's; the reference's exponent, see
  // F::kExps), and [group][128] each: a
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
    const int u0 = b < a.batch ? seq_tiles<F>(a, b, blockIdx.x == 0) : 0;
    const int u1 = b + 1 < a.batch ? seq_tiles<F>(a, b + 1, blockIdx.x == 0) : 0;
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
  int ctas = min(static_cast<int>(gridDim.x), (total + F::kMinTiles - 1) / F::kMinTiles);
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
  typename F::State st;
  st.q = smem_u32(&sm.q[warp][0][lane]);
  auto finish = [&](int b, int h, bool whole, int slot) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], off);
      st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], off);
    }
    const float down = F::down(st);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = 2 * t + e;
      if (head >= a.group) continue;
      if (whole) {
        const float inv = st.l[e] == 0.f ? 0.f : __fdividef(a.v_scale, st.l[e]) * down;
        __nv_bfloat16* row = a.out + (static_cast<int64_t>(b) * a.heads + h * a.group + head) * kD + F::dim(0, g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint32_t*>(row + F::dim(j, 0)) = pack_bf16x2(st.o[j][e] * inv, st.o[j][2 + e] * inv);
      } else {
        const int at = (2 * warp + slot) * a.group + head;
        if (g == 0) piece_ml[at] = F::piece(st, e);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float2*>(piece_o(2 * warp + slot) + head * kD + F::dim(j, g)) =
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
    next_at = place(F::kTileUnits * tile, kBad);
    if constexpr (!kTwo) return;
    // blocks of one unit: the tile's second unit has a block of its own
    if (a.upb_log2 == 0 && tokens > kUnitTokens) next_at2 = place(2 * tile + 1, kBad2);
    else if (next_info & kBad) next_info |= kBad2;
  };
  auto fetch = [&](int i) {  // tile i into its stage, by the lane that knows it
    if (lane != (i & 31)) return;
    uint64_t* bar = &sm.full[warp][i % kStages];
    uint8_t* to = sm.ring[warp][i % kStages];
    const bool two = kTwo && (next_info & 0xff) > kUnitTokens;
    if ((!kTwo || a.upb_log2 > 0) && !(next_info & kBad)) {  // one copy
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
  const uint32_t ring = smem_u32(sm.ring[warp]), scratch = smem_u32(&sm.scratch[warp]);
  for (int i = 0; i < n; ++i) {
    if ((i & 31) == 0 && i > 0) pair_now = next_pair, info_now = next_info;
    const int info = __shfl_sync(0xffffffffu, info_now, i & 31);
    if (!open) {
      const int pair = __shfl_sync(0xffffffffu, pair_now, i & 31);
      b = pair / a.kvh;
      h = pair - b * a.kvh;
      F::load_q(a, b, h, g, t, st);
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
      F::template attend<false>(st, tile, scratch, tokens, g, t, lane);
    } else {
      if (!ok || (info & kBad)) zero_unit<F>(tile, lane);  // reads as zeros
      if (kTwo && (!ok || (info & kBad2))) zero_unit<F>(tile + kUnitBytes, lane);
      F::template attend<true>(st, tile, scratch, tokens, g, t, lane);
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
  // (what a piece holds of it is relative to its reference: see F::kExps for the exponents)
  auto weight = [](float ref, float l, float m, float sc, float exp, float most) {
    return ref == -INFINITY ? (l == 0.f ? 0.f : 1.f)
                            : fast_exp2(F::kExps ? fmaf(ref - m, sc, exp - most) : (ref - m) * sc);
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
      const float most = F::kExps ? warp_max(ml.x == -INFINITY ? -INFINITY : fmaf(ml.x - m, ml.z, ml.w)) : 0.f;
      const float w = weight(ml.x, ml.y, m, ml.z, ml.w, most), l = warp_sum(ml.y * w);
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
        if (lane == first) a.ws_ml[to] = make_float4(m, l, ml.z, F::kExps ? most : 0.f);
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
    float m = -INFINITY, most = 0.f, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = lane; i < count; i += 32) m = fmaxf(m, __ldcg(&a.ws_ml[at(i)].x));
    if constexpr (F::kExps) {
      m = warp_max(m);
      most = -INFINITY;
      for (int i = lane; i < count; i += 32) {
        const float4 v = __ldcg(a.ws_ml + at(i));
        if (v.x != -INFINITY) most = fmaxf(most, fmaf(v.x - m, sc, v.w));
      }
      most = warp_max(most);
    }
    for (int i0 = part; i0 < count; i0 += kAhead * parts) {
      float4 v[kAhead];
      using Ml = std::conditional_t<F::kExps, float4, float2>;
      Ml ml[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + j * parts;
        if (i < count) ml[j] = __ldcg(reinterpret_cast<const Ml*>(a.ws_ml + at(i)));
        else ml[j].x = -INFINITY, ml[j].y = 0.f;
        v[j] = i < count ? __ldcg(reinterpret_cast<const float4*>(a.ws_o + at(i) * kD + 4 * lane))
                         : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (!F::kExps && i0 == part) m = warp_max(m);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        float exp = 0.f;
        if constexpr (F::kExps) exp = ml[j].w;
        const float w = weight(ml[j].x, ml[j].y, m, sc, exp, most);
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

// With the pieces of `group` heads of every warp.
template <typename F>
constexpr size_t smem_bytes(int group) {
  return sizeof(Smem<F>) + static_cast<size_t>(F::kWarps) * group * (2 * sizeof(float4) + kD * sizeof(float));
}

// The sequences in launches of as many as the kernel's prefix holds; `most` heads a group are the most that F takes.
template <typename F>
int launch(DecodeArgs a, int batch, int ctas, int most, const char* what, cudaStream_t stream) {
  static_assert(sizeof(Smem<F>) % 16 == 0, "the pieces behind it are 16-byte aligned");
  static_assert(F::kStages * F::kTileBytes >= kMaxGroup * kD * 4, "a warp's ring takes its last piece");
  const void* kernel = reinterpret_cast<const void*>(&decode_kernel<F>);
  int rc = ensure_dynamic_smem(kernel, smem_bytes<F>(most));
  constexpr int kMaxSeqs = 2 * F::kWarps * 32;
  for (int left = batch; rc == NVK_OK && left > 0; left -= kMaxSeqs) {
    a.batch = left < kMaxSeqs ? left : kMaxSeqs;
    rc = check_cuda(launch_pdl(decode_kernel<F>, dim3(ctas), dim3(F::kWarps * 32), smem_bytes<F>(a.group), stream, a),
                    what);
    a.out += static_cast<int64_t>(kMaxSeqs) * a.heads * kD;
    a.q += static_cast<int64_t>(kMaxSeqs) * a.heads * kD;
    a.tables += static_cast<int64_t>(kMaxSeqs) * a.bt_stride;
    a.ctx += kMaxSeqs;
  }
  return rc;
}

inline size_t workspace_bytes(int group, int ctas) {
  return kMlOffset + static_cast<size_t>(ctas) * 2 * group * (sizeof(float4) + kD * sizeof(float));
}

inline int resolve_ctas(int num_ctas, const char* who, int* out) {
  int ctas = num_ctas;
  if (ctas == 0) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&ctas, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return check_cuda(e, who);
  }
  *out = ctas < kMaxCtas ? ctas : kMaxCtas;
  return NVK_OK;
}

inline int check_heads(int num_heads, int num_kv_heads, int num_ctas, const char* who) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_ctas < 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (heads=%d kv_heads=%d ctas=%d)", who, num_heads, num_kv_heads,
                num_ctas);
  if (num_heads % num_kv_heads != 0 || num_heads / num_kv_heads > kMaxGroup)
    return fail(NVK_ERR_UNSUPPORTED, "%s: %d query heads over %d KV heads (a GQA group of 1 to %d)", who, num_heads,
                num_kv_heads, kMaxGroup);
  return NVK_OK;
}

// What both entry points do behind the pool's own checks: the other checks, and the arguments that do not hang on the
// format (scale_log2, v_scale and the launch are the caller's).
inline int prepare(DecodeArgs& a, int& ctas, void* out, const void* query, const void* kv_cache, int num_blocks,
                   int upb_log2, int block_size, const int32_t* block_tables, int block_table_stride,
                   int max_blocks_per_seq, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                   float scale, int num_ctas, void* workspace, size_t workspace_bytes_given, int* error_word,
                   const char* who) {
  if (!(scale > 0.f)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: scale %g is not positive", who, double(scale));
  if (max_blocks_per_seq <= 0 || block_table_stride < max_blocks_per_seq)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: block table stride %d below its %d columns", who, block_table_stride,
                max_blocks_per_seq);
  if (batch == 0) return NVK_OK;
  if (!out || !query || !block_tables || !context_lens || !workspace)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(out) || !aligned16(query) || !aligned16(workspace))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: q, out and workspace must be 16-byte aligned", who);
  const int64_t seqs = batch < 1024 ? batch : 1024;
  if (((seqs * max_blocks_per_seq * num_kv_heads) << upb_log2) > 0x7fffffffll ||
      (static_cast<int64_t>(max_blocks_per_seq) << upb_log2) > 0x7fffffffll / kUnitTokens)
    return fail(NVK_ERR_UNSUPPORTED, "%s: %d blocks of %d tokens a sequence and %d KV heads are above the kernel's range",
                who, max_blocks_per_seq, block_size, num_kv_heads);
  const int rc = resolve_ctas(num_ctas, who, &ctas);
  if (rc != NVK_OK) return rc;
  const int group = num_heads / num_kv_heads;
  if (workspace_bytes_given < workspace_bytes(group, ctas))
    return fail(NVK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes_given,
                workspace_bytes(group, ctas));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
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
  a.out = static_cast<__nv_bfloat16*>(out);
  a.q = static_cast<const __nv_bfloat16*>(query);
  a.tables = block_tables;
  a.ctx = context_lens;
  return NVK_OK;
}

}  // namespace decode
}  // namespace nvk
