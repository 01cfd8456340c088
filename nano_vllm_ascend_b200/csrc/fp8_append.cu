// Quantising append into the 8-bit KV pool, and the read of its rows. The
// pool's format is in fp8_kv.cuh.
//
// Append. A unit's exponent is that of the unit's largest value, so the rows
// that a call writes into one unit have to meet: its owner, the call's token
// at the lowest offset, gathers the unit's up to 16 rows of one head's K or V
// in one warp (16 bytes of a row a lane, two rows a load instruction), which
// finds the largest magnitude, sets the exponent, writes the codes, and brings
// the rows that were there to a larger exponent or, where the unit's first
// token is written, makes them zeros.
// Which tokens share a unit:
//  - up to kScanTokens: every block looks through the call's slots for those
//    of its one token's unit;
//  - above: index_kernel writes each token's number to index[slot], and the
//    blocks look the units' 16 entries of their 16 tokens up. The index needs no
//    clearing: entry i of slot s counts only if slots[i] is s, whatever else the
//    memory held.
// (8 heads, bf16, rows of a prompt and rows of as many sequences: the scan takes
// 6.1 and 7.5 us at 512 tokens, the index 4.9 and 8.3; 3.9 and 4.8 against 4.8
// and 7.7 at 256; 9.1 and 13.4 against 6.1 and 13.0 at 1024. Up to 512 a caller
// needs no workspace.)
// A prompt's rows fill their units, so that one token of 16 owns work; a decode
// step's all do. A block's units are therefore shared by up to kMostShares
// blocks, as far as that keeps four on an SM busy: 1024 rows of as many
// sequences 43.7 -> 13.0 us, of a prompt 6.1 either way; 32 rows 4.4 -> 3.3.
// (Four tokens a block instead of 16 in the indexed form: 15.4 us for a prompt's
// 8192 rows instead of 10.5.) The blocks of a chunk find their shares by a list
// that each makes for itself, so it is in the tokens' order.
// Bound by latency when short (3.3 us for a decode step's 32 rows, of which 2
// are a launch in a graph) and by the loads of rows when long: 8192 rows of 8
// heads in bf16, 50.5 MB, take 10.1 us, 7.7 at the copy rate.
// Slots must differ; of two rows for one slot, one is written whole.
#include <algorithm>

#include "fp8_kv.cuh"

namespace nvk {
namespace fp8 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMostChunk = 16;     // tokens of a block
constexpr int kScanTokens = 512;
constexpr int kMostShares = 16;

struct AppendArgs {
  const uint8_t* key;
  const uint8_t* value;
  int64_t key_stride, value_stride;  // bytes between tokens
  uint8_t* pool;
  const int64_t* slots;
  const int32_t* index;    // null: look through the slots
  int64_t num_slots;
  int tokens, chunk, kvh, upb_log2;
  int* err;
};

__global__ void __launch_bounds__(kThreads) index_kernel(const int64_t* slots, int32_t* index, int tokens,
                                                         int64_t num_slots) {
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= tokens) return;
  const int64_t s = slots[i];
  if (s >= 0 && s < num_slots) index[s] = i;
}

template <typename T>
constexpr uint32_t kInf = 0x7f80u;
template <>
constexpr uint32_t kInf<__half> = 0x7c00u;

template <typename T>
__device__ __forceinline__ float bits_to_float(uint32_t b) {
  return pair_to_f32<T>(b).x;
}

// Eight neighbouring elements of a row.
template <bool kWide>
__device__ __forceinline__ uint4 load8(const uint8_t* p) {
  if constexpr (kWide) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  auto two = [&](int i) { return h[i] | (static_cast<uint32_t>(h[i + 1]) << 16); };
  return make_uint4(two(0), two(2), two(4), two(6));
}

template <typename T>
__device__ __forceinline__ uint2 codes_of(const uint4& x, float inv) {
  auto two = [&](uint32_t w) {
    const float2 f = pair_to_f32<T>(w);
    return floats_to_e4m3x2(f.x * inv, f.y * inv);
  };
  return make_uint2(two(x.x) | (two(x.y) << 16), two(x.z) | (two(x.w) << 16));
}
// Codes to the exponent that is larger by -log2(by).
__device__ __forceinline__ uint32_t moved(uint32_t w, float by) {
  uint32_t lo, hi;
  e4m3_to_half2(w, lo, hi);
  const float2 a = pair_to_f32<__half>(lo), b = pair_to_f32<__half>(hi);
  return floats_to_e4m3x2(a.x * by, a.y * by) | (floats_to_e4m3x2(b.x * by, b.y * by) << 16);
}

template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads, 4) append_kernel(const AppendArgs a) {
  __shared__ int member[kMostChunk][kUnitTokens];  // the token that writes each offset of the unit, or -1
  __shared__ int64_t unit_of[kMostChunk];          // -1: no unit of the pool
  __shared__ int owners[kMostChunk];               // the block's tokens that own their unit, in order
  __shared__ int num_owners;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int first = blockIdx.x * a.chunk, count = min(a.chunk, a.tokens - first);
  if (tid < count) {
    const int64_t s = a.slots[first + tid];
    const bool ok = s >= 0 && s < a.num_slots;
    unit_of[tid] = ok ? s >> 4 : -1;
    if (!ok && a.err) atomicOr(a.err, kErrBadSlot);
  }
  for (int i = tid; i < count * kUnitTokens; i += kThreads) (&member[0][0])[i] = -1;
  __syncthreads();
  if (a.index) {
    for (int i = tid; i < count * kUnitTokens; i += kThreads) {
      const int64_t u = unit_of[i >> 4];
      if (u < 0) continue;
      const int64_t s = u * kUnitTokens + (i & 15);
      const int j = a.index[s];
      if (j >= 0 && j < a.tokens && a.slots[j] == s) (&member[0][0])[i] = j;
    }
  } else {
    for (int j = tid; j < a.tokens; j += kThreads) {
      const int64_t s = a.slots[j];
      if (s < 0) continue;
      for (int c = 0; c < count; ++c)
        if (s >> 4 == unit_of[c]) atomicMax(&member[c][s & 15], j);
    }
  }
  __syncthreads();
  if (warp == 0) {
    // Every block of the chunk (gridDim.y of them) makes this list for itself and takes a share of it by place, so the
    // order has to be the same in all of them.
    static_assert(kMostChunk <= 32, "a block's tokens are lanes of one warp");
    int low = -1;
    if (lane < count)
      for (int o = kUnitTokens - 1; o >= 0; --o)
        if (member[lane][o] >= 0) low = member[lane][o];
    const bool owns = lane < count && low == first + lane;
    const uint32_t all = __ballot_sync(0xffffffffu, owns);
    if (owns) owners[__popc(all & ((1u << lane) - 1))] = lane;
    if (lane == 0) num_owners = __popc(all);
  }
  __syncthreads();
  const int per_unit = 2 * a.kvh, items = num_owners * per_unit;
  const int half = lane >> 4, part = lane & 15;  // this lane's dims: 8 part .. 8 part + 7 of every other row
  for (int w = blockIdx.y * kWarps + warp; w < items; w += gridDim.y * kWarps) {
    const int c = owners[w / per_unit], rest = w % per_unit, kv = rest >= a.kvh, head = rest - kv * a.kvh;
    uint8_t* unit = unit_at(a.pool, unit_of[c], head, a.kvh, a.upb_log2);
    int* exp_at = reinterpret_cast<int*>(unit + kOffExp) + kv;
    const int e_old = held_exp(*exp_at);
    const uint8_t* rows = (kv ? a.value : a.key) + static_cast<int64_t>(head) * kD * 2 + 16 * part;
    const int64_t stride = kv ? a.value_stride : a.key_stride;
    uint4 x[8];
    uint32_t here = 0;  // bit p: row 2 p + half is written
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int j = member[c][2 * p + half];
      x[p] = j >= 0 ? load8<kWide>(rows + j * stride) : make_uint4(0, 0, 0, 0);
      here |= (j >= 0) << p;
    }
    uint32_t big = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      constexpr uint32_t kMag = 0x7fff7fffu;
      big = __vmaxu2(big, __vmaxu2(__vmaxu2(x[p].x & kMag, x[p].y & kMag), __vmaxu2(x[p].z & kMag, x[p].w & kMag)));
    }
    big = __reduce_max_sync(0xffffffffu, max(big & 0xffffu, big >> 16));
    uint32_t nan_rows = 0;  // bit p
    if (big >= kInf<T>) {   // infinities and NaN do not count, and a row with a NaN is one throughout
      big = 0;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const uint32_t words[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
        bool nan = false;
        for (int i = 0; i < 8; ++i) {
          const uint32_t m = words[i >> 1] >> (16 * (i & 1)) & 0x7fffu;
          if (m > kInf<T>) nan = true;
          if (m < kInf<T>) big = max(big, m);
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, nan);
        if (votes >> (16 * half) & 0xffffu) nan_rows |= 1u << p;
      }
      big = __reduce_max_sync(0xffffffffu, big);
    }
    const int e_new = exponent_for(bits_to_float<T>(big));
    const bool anew = member[c][0] >= 0;
    const int e = anew ? e_new : max(e_old, e_new);
    const float inv = pow2(-e);
    uint8_t* codes = unit + kv * kOffV + 8 * (part & 1);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int r = 2 * p + half;
      uint2* at = reinterpret_cast<uint2*>(codes + chunk_at(r, part >> 1));
      if (here >> p & 1) {
        *at = nan_rows >> p & 1 ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : codes_of<T>(x[p], inv);
      } else if (anew) {
        *at = make_uint2(0, 0);
      } else if (e > e_old) {
        const uint2 old = *at;
        const float by = pow2(e_old - e);
        *at = make_uint2(moved(old.x, by), moved(old.y, by));
      }
    }
    if (lane == 0) *exp_at = e;
  }
}

struct ReadArgs {
  uint8_t* key;
  uint8_t* value;
  uint8_t* pool;
  const int64_t* slots;
  int64_t num_slots, tokens, items;
  int kvh, upb_log2;
  int* err;
};

// A warp takes K or V of one head of 16 of the call's tokens, which mostly are
// one unit's: 2 KB that lie together, two rows a load (16 lanes of eight codes),
// all in flight, and whole rows out. Neighbouring warps take the other heads, so
// that both sides' lines and pages are used while they are open. (Row by row in
// the order of the output, 128 bytes from a place of their own each, 28672 to
// 35712 tokens of 8 heads ran at 3.9 to 4.4 TB/s however many were in flight.)
// Sixteen tokens that are a unit in order share an address and an exponent.
// HBM-bound: 32768 rows of 8 heads, 202 MB, in 34.4 us (5.9 TB/s, 0.90 of the
// measured copy rate); with an exponent and an address a row 38.7. Five blocks
// an SM: 44.9 us with the append of 8192 rows, four 45.9, six 46.7, eight 54.4.
template <typename T>
__global__ void __launch_bounds__(kThreads, 5) read_kernel(const ReadArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, half = lane >> 4, part = lane & 15;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); item < a.items;
       item += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int per_group = 2 * a.kvh;
    int64_t group;
    if (a.items <= 0x7fffffff) group = static_cast<uint32_t>(item) / static_cast<uint32_t>(per_group);
    else group = item / per_group;
    const int rest = static_cast<int>(item - group * per_group), kv = rest >= a.kvh, head = rest - kv * a.kvh;
    const int64_t first = group * kUnitTokens;
    const int count = static_cast<int>(min(static_cast<int64_t>(kUnitTokens), a.tokens - first));
    int64_t mine = -1;
    if (part < count) {
      mine = a.slots[first + part];
      if (mine < 0 || mine >= a.num_slots) {
        if (rest == 0 && half == 0 && a.err) atomicOr(a.err, kErrBadSlot);
        mine = -1;
      }
    }
    uint2 w[8];
    float by[8];
    const int64_t begin = __shfl_sync(0xffffffffu, mine, 0);
    if (__all_sync(0xffffffffu, begin >= 0 && mine == begin + part && (begin & 15) == 0)) {  // a unit, in order
      const uint8_t* unit = unit_at(a.pool, begin >> 4, head, a.kvh, a.upb_log2);
      const float one = pow2(held_exp(reinterpret_cast<const int*>(unit + kOffExp)[kv]));
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        w[n] = *reinterpret_cast<const uint2*>(unit + kv * kOffV + chunk_at(2 * n + half, part >> 1) + 8 * (part & 1));
        by[n] = one;
      }
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int64_t slot = __shfl_sync(0xffffffffu, mine, 2 * n + half);
        w[n] = make_uint2(0, 0);
        by[n] = 1.f;
        if (slot >= 0) {
          const uint8_t* unit = unit_at(a.pool, slot >> 4, head, a.kvh, a.upb_log2);
          by[n] = pow2(held_exp(reinterpret_cast<const int*>(unit + kOffExp)[kv]));
          w[n] = *reinterpret_cast<const uint2*>(unit + kv * kOffV + chunk_at(slot & 15, part >> 1) + 8 * (part & 1));
        }
      }
    }
    uint8_t* out = (kv ? a.value : a.key) + ((first * a.kvh + head) * kD + 8 * part) * 2;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int r = 2 * n + half;
      if (r >= count) continue;
      auto two = [&](uint32_t h) {
        const float2 f = pair_to_f32<__half>(h);
        return f32_to_pair<T>(f.x * by[n], f.y * by[n]);
      };
      uint32_t h[4];
      e4m3_to_half2(w[n].x, h[0], h[1]);
      e4m3_to_half2(w[n].y, h[2], h[3]);
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r) * a.kvh * (kD * 2)) =
          make_uint4(two(h[0]), two(h[1]), two(h[2]), two(h[3]));
    }
  }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace fp8
}  // namespace nvk

extern "C" int nvk_fp8_append_workspace_size(int64_t num_tokens, int64_t num_slots, size_t* bytes) {
  using namespace nvk;
  if (!bytes || num_tokens < 0 || num_slots < 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "fp8_append_workspace_size: null pointer or negative size");
  *bytes = num_tokens > fp8::kScanTokens ? static_cast<size_t>(num_slots) * sizeof(int32_t) : 0;
  return NVK_OK;
}

extern "C" int nvk_fp8_append(const void* key, const void* value, int64_t key_token_stride,
                              int64_t value_token_stride, void* kv_cache, const int64_t* slot_mapping,
                              int64_t num_tokens, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                              int dtype, void* workspace, size_t workspace_bytes, int* error_word,
                              nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp8;
  const char* who = "fp8_append";
  if (num_tokens < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)num_tokens);
  int rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, who);
  if (rc != NVK_OK) return rc;
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_FP16)
    return fail(NVK_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 rows only)", who, dtype);
  if (num_tokens == 0) return NVK_OK;
  if (num_tokens > (int64_t(1) << 30))
    return fail(NVK_ERR_UNSUPPORTED, "%s: %lld tokens are above the kernel's range", who, (long long)num_tokens);
  if (!key || !value || !slot_mapping) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  const int64_t row = static_cast<int64_t>(num_kv_heads) * kD;
  if (!aligned(slot_mapping, 8) || !aligned(key, 2) || !aligned(value, 2))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: slots must be 8-byte aligned, rows 2-byte aligned", who);
  if (num_tokens > 1 && (key_token_stride < row || value_token_stride < row))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: token strides (%lld, %lld) must cover a row", who,
                (long long)key_token_stride, (long long)value_token_stride);
  AppendArgs a;
  a.key = static_cast<const uint8_t*>(key);
  a.value = static_cast<const uint8_t*>(value);
  a.key_stride = key_token_stride * 2;
  a.value_stride = value_token_stride * 2;
  a.pool = static_cast<uint8_t*>(kv_cache);
  a.slots = slot_mapping;
  a.num_slots = static_cast<int64_t>(num_blocks) * block_size;
  a.tokens = static_cast<int>(num_tokens);
  a.kvh = num_kv_heads;
  a.upb_log2 = units_log2(block_size);
  a.err = error_word;
  a.index = nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (num_tokens > kScanTokens) {
    if (workspace_bytes < static_cast<size_t>(a.num_slots) * sizeof(int32_t) || !workspace)
      return fail(NVK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes,
                  static_cast<size_t>(a.num_slots) * sizeof(int32_t));
    if (!aligned(workspace, 4)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: workspace must be 4-byte aligned", who);
    a.index = static_cast<int32_t*>(workspace);
    rc = check_cuda(launch_pdl(index_kernel, dim3((a.tokens + kThreads - 1) / kThreads), dim3(kThreads), 0, st,
                               slot_mapping, static_cast<int32_t*>(workspace), a.tokens, a.num_slots),
                    "fp8_append index launch");
    if (rc != NVK_OK) return rc;
    a.chunk = kMostChunk;
  } else {
    a.chunk = 1;
  }
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int blocks = (a.tokens + a.chunk - 1) / a.chunk, rounds = (2 * a.kvh * a.chunk + kWarps - 1) / kWarps;
  const dim3 grid(blocks, std::clamp(4 * sms / blocks, 1, std::min(rounds, kMostShares)));
  const bool wide = aligned16(key) && aligned16(value) && key_token_stride % 8 == 0 && value_token_stride % 8 == 0;
  auto launch = [&](auto kernel) { return check_cuda(launch_pdl(kernel, grid, dim3(kThreads), 0, st, a), "fp8_append launch"); };
  if (dtype == NVK_DTYPE_BF16)
    return wide ? launch(append_kernel<__nv_bfloat16, true>) : launch(append_kernel<__nv_bfloat16, false>);
  return wide ? launch(append_kernel<__half, true>) : launch(append_kernel<__half, false>);
}

extern "C" int nvk_fp8_read(void* key, void* value, const void* kv_cache, const int64_t* slot_mapping,
                            int64_t num_tokens, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                            int dtype, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::fp8;
  const char* who = "fp8_read";
  if (num_tokens < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: %lld tokens", who, (long long)num_tokens);
  int rc = check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, who);
  if (rc != NVK_OK) return rc;
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_FP16)
    return fail(NVK_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 rows only)", who, dtype);
  if (num_tokens == 0) return NVK_OK;
  if (!key || !value || !slot_mapping) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(key) || !aligned16(value) || !aligned(slot_mapping, 8))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: the rows must be 16-byte aligned, the slots 8-byte aligned", who);
  ReadArgs a;
  a.key = static_cast<uint8_t*>(key);
  a.value = static_cast<uint8_t*>(value);
  a.pool = static_cast<uint8_t*>(const_cast<void*>(kv_cache));
  a.slots = slot_mapping;
  a.num_slots = static_cast<int64_t>(num_blocks) * block_size;
  a.tokens = num_tokens;
  a.items = (num_tokens + kUnitTokens - 1) / kUnitTokens * 2 * num_kv_heads;
  a.kvh = num_kv_heads;
  a.upb_log2 = units_log2(block_size);
  a.err = error_word;
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t want = (a.items + kWarps - 1) / kWarps, most = int64_t(sms) * 32;
  const dim3 grid(static_cast<unsigned>(want < most ? want : most));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return check_cuda(dtype == NVK_DTYPE_BF16 ? launch_pdl(read_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, a)
                                            : launch_pdl(read_kernel<__half>, grid, dim3(kThreads), 0, st, a),
                    "fp8_read launch");
}
