// Rotary positions of q's and k's heads, with their RMS norm where weights are
// given. Over the first R dims of a head of D, in pairs (a, b) = (y_i, y_i+R/2)
// ("half") or (y_2i, y_2i+1) ("interleaved"):
//   y = x, or x * rsqrt(mean(x^2) + eps) * w
//   out = ((a cos - b sin) f, (b cos + a sin) f),  angle = position * inv_freq_i
// and out = y from dim R on. Everything between the loads and the one rounding
// at the end is fp32; the angle is made in 64 bits, in half turns and less whole
// turns: off by at most 2^-26 of a turn (fp32's rounding of what is left) and
// 2^-52 of itself (the roundings of the position and of its product with the
// frequency, which is as far off itself), so by less than 2^-24 of a turn below
// 2^30 radians and by 2^-12 of a radian at 2^40. A table would have to be read,
// and ends somewhere.
//
// HBM-bound: every row is read and written once.
// row_kernel (whole vectors of V elements): a lane takes V pairs of a row, so
// that a pair never leaves its lane: dims V p .. of the head's first half of R
// and the same of its second ("half"), or 2 V neighbouring dims. A row is
// D / 2V lanes, a warp takes the rows of one token (or a share of them, where
// there are few tokens) that many at a time, the next ones' loads ahead of this
// one's arithmetic, and makes the token's cosines and sines once: a pair or two
// a lane, exchanged in shared memory. V is 8 where rows allow 16-byte loads,
// else 2. any_kernel takes what is left: odd halves, rows at odd addresses,
// heads above 256 dims.
// Measured: 8191 tokens of 40 heads of 128, half of each turned, 168 MB, 29.6 us
// (5.7 TB/s, 0.87 of the measured copy rate); by any_kernel's way, a row a warp
// and elements one by one, 173. Blocks of four warps, 64 registers: of eight 34.7
// (their last wave leaves SMs idle), of two 30.0; two rows ahead 29.8; ten
// blocks an SM (48 registers, spills) 38. A decode step's 32 tokens: 2.5 us,
// of which 2 are a launch in a graph.
#include "host_common.h"
#include "nvk_common.cuh"

#include <cuda_fp16.h>

#include <type_traits>

namespace nvk {
namespace rotary {
namespace {

constexpr int kThreads = 256;
constexpr int kMostDim = 512;

struct Args {
  const uint8_t* in[2];   // q, k
  uint8_t* out[2];
  const uint8_t* weight[2];
  int64_t in_stride[2], out_stride[2];  // elements between tokens
  const double* inv_freq;
  const int64_t* positions;
  int64_t tokens;
  int heads[2];
  int dim, rotated, interleaved;
  float factor, eps;
};

// cos and sin of position * inv_freq, times the factor. The product by 1 / pi
// keeps its rounding error (and 1 / pi its next bits), so that a far angle, as
// rounded to a double, loses nothing on its way into [-1, 1] half turns.
__device__ __forceinline__ float2 turn(int64_t position, double inv_freq, float factor) {
  constexpr double kInvPi = 0x1.45f306dc9c883p-2, kInvPiRest = -0x1.6b01ec5417056p-56;
  const double angle = static_cast<double>(position) * inv_freq, turns = angle * kInvPi;
  const double rest = fma(angle, kInvPiRest, fma(angle, kInvPi, -turns));
  const float x = static_cast<float>(fma(-2.0, rint(0.5 * turns), turns) + rest);
  float s, c;
  sincospif(x, &s, &c);
  return make_float2(c * factor, s * factor);
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }

// A block takes a token, a warp a row at a time, a pair (or two dims) a lane.
template <typename T>
__global__ void __launch_bounds__(kThreads) any_kernel(const Args a) {
  __shared__ float2 cs[kMostDim / 2];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = a.rotated / 2, pairs = a.dim / 2;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    __syncthreads();
    for (int i = threadIdx.x; i < half; i += kThreads) cs[i] = turn(a.positions[t], a.inv_freq[i], a.factor);
    __syncthreads();
    for (int r = warp; r < a.heads[0] + a.heads[1]; r += kThreads / 32) {
      const int which = r >= a.heads[0], h = r - which * a.heads[0];
      const T* x = reinterpret_cast<const T*>(a.in[which]) + t * a.in_stride[which] + static_cast<int64_t>(h) * a.dim;
      T* y = reinterpret_cast<T*>(a.out[which]) + t * a.out_stride[which] + static_cast<int64_t>(h) * a.dim;
      const T* w = reinterpret_cast<const T*>(a.weight[which]);
      // pair i: the dims of rotated pair i, or the next two of the rest
      auto dims = [&](int i, int& d0, int& d1) {
        if (i >= half || a.interleaved) d0 = 2 * i, d1 = d0 + 1;
        else d0 = i, d1 = i + half;
      };
      float u[kMostDim / 64], v[kMostDim / 64], sum = 0.f;
#pragma unroll
      for (int k = 0; k < kMostDim / 64; ++k) {
        const int i = 32 * k + lane;
        if (i >= pairs) continue;
        int d0, d1;
        dims(i, d0, d1);
        u[k] = to_float(x[d0]), v[k] = to_float(x[d1]);
        sum += u[k] * u[k] + v[k] * v[k];
      }
      float rinv = 1.f;
      if (w) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        rinv = rsqrtf(sum / a.dim + a.eps);
      }
#pragma unroll
      for (int k = 0; k < kMostDim / 64; ++k) {
        const int i = 32 * k + lane;
        if (i >= pairs) continue;
        int d0, d1;
        dims(i, d0, d1);
        float p = u[k], q = v[k];
        if (w) p = p * rinv * to_float(w[d0]), q = q * rinv * to_float(w[d1]);
        if (i < half) {
          const float2 c = cs[i];
          const float p0 = p;
          p = p * c.x - q * c.y;
          q = q * c.x + p0 * c.y;
        }
        y[d0] = from_float<T>(p), y[d1] = from_float<T>(q);
      }
    }
  }
}

// V elements of type T as fp32, and back.
template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(bf16lo_to_f32(w), bf16hi_to_f32(w));
}
template <typename T>
__device__ __forceinline__ uint32_t two_rounded(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}
template <int V>
struct Words {
  uint32_t w[V / 2];
};
template <int V>
__device__ __forceinline__ Words<V> load_words(const void* p) {
  Words<V> r;
  if constexpr (V == 8) {
    const uint4 v = *static_cast<const uint4*>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else {
    r.w[0] = *static_cast<const uint32_t*>(p);
  }
  return r;
}
template <int V>
__device__ __forceinline__ void store_words(void* p, const Words<V>& r) {
  if constexpr (V == 8) *static_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else *static_cast<uint32_t*>(p) = r.w[0];
}

constexpr int kRowWarps = 4;
constexpr int kRowBlocks = 8;  // an SM: 64 registers a thread, 32 warps
constexpr int kRowMostDim = 256;

// `share` rows of a token a warp; `group` lanes a row (a power of two).
template <typename T, int V, bool kNorm, bool kInterleaved>
__global__ void __launch_bounds__(32 * kRowWarps, kRowBlocks) row_kernel(const Args a, int share, int shares, int group) {
  __shared__ float2 turns[kRowWarps][kRowMostDim / 2];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float2* cs = turns[warp];
  const int half = a.rotated / 2, per_row = a.dim / (2 * V), at_once = 32 / group;
  const int p = lane & (group - 1), sub = lane / group;
  const bool live = p < per_row, rotates = V * p < half;
  // the lane's dims: V from d0 and V from d1
  const int d0 = rotates && !kInterleaved ? V * p : 2 * V * p, d1 = d0 + (rotates && !kInterleaved ? half : V);
  const int rows = a.heads[0] + a.heads[1];
  const int64_t items = a.tokens * shares;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kRowWarps + warp; item < items;
       item += static_cast<int64_t>(gridDim.x) * kRowWarps) {
    const int64_t t = item / shares;
    const int first = static_cast<int>(item - t * shares) * share, end = min(first + share, rows);
    auto place = [&](bool out, int r) -> uint8_t* {  // row r of the token, q's heads and then k's
      const bool k = r >= a.heads[0];
      const uint8_t* base = out ? (k ? a.out[1] : a.out[0]) : (k ? a.in[1] : a.in[0]);
      const int64_t stride = out ? (k ? a.out_stride[1] : a.out_stride[0]) : (k ? a.in_stride[1] : a.in_stride[0]);
      return const_cast<uint8_t*>(base) + 2 * (t * stride + static_cast<int64_t>(k ? r - a.heads[0] : r) * a.dim);
    };
    Words<V> x0{}, x1{};
    auto load = [&](int r) {
      if (!live || r >= end) return;
      const uint8_t* row = place(false, r);
      x0 = load_words<V>(row + 2 * d0);
      x1 = load_words<V>(row + 2 * d1);
    };
    load(first + sub);
    const int64_t position = a.positions[t];
    __syncwarp();  // the token before this one is done with cs
    for (int i = lane; i < half; i += 32) cs[i] = turn(position, a.inv_freq[i], a.factor);
    __syncwarp();
    float2 c[V];
    if (rotates) {
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = cs[V * p + i];
    }
    for (int r0 = first; r0 < end; r0 += at_once) {
      const int r = r0 + sub;
      float y[2 * V];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 u = two_floats<T>(x0.w[i]), v = two_floats<T>(x1.w[i]);
        y[2 * i] = u.x, y[2 * i + 1] = u.y, y[V + 2 * i] = v.x, y[V + 2 * i + 1] = v.y;
      }
      load(r + at_once);
      if constexpr (kNorm) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) sum += live ? y[i] * y[i] : 0.f;
        for (int off = group / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const float rinv = rsqrtf(sum / a.dim + a.eps);
        const uint8_t* w = r >= a.heads[0] ? a.weight[1] : a.weight[0];
        if (live && r < end) {
          const Words<V> w0 = load_words<V>(w + 2 * d0), w1 = load_words<V>(w + 2 * d1);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const float2 u = two_floats<T>(w0.w[i]), v = two_floats<T>(w1.w[i]);
            y[2 * i] *= rinv * u.x, y[2 * i + 1] *= rinv * u.y, y[V + 2 * i] *= rinv * v.x, y[V + 2 * i + 1] *= rinv * v.y;
          }
        }
      }
      if (rotates) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float& u = y[kInterleaved ? 2 * i : i];
          float& v = y[kInterleaved ? 2 * i + 1 : V + i];
          const float u0 = u;
          u = u * c[i].x - v * c[i].y;
          v = v * c[i].x + u0 * c[i].y;
        }
      }
      if (live && r < end) {
        Words<V> o0, o1;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          o0.w[i] = two_rounded<T>(y[2 * i], y[2 * i + 1]);
          o1.w[i] = two_rounded<T>(y[V + 2 * i], y[V + 2 * i + 1]);
        }
        uint8_t* row = place(true, r);
        store_words<V>(row + 2 * d0, o0);
        store_words<V>(row + 2 * d1, o1);
      }
    }
  }
}

template <typename T, int V>
int launch_rows(const Args& a, bool norm, int sms, cudaStream_t st) {
  const int per_row = a.dim / (2 * V);
  int group = 1;
  while (group < per_row) group *= 2;
  const int rows = a.heads[0] + a.heads[1], at_once = 32 / group;
  // A warp takes a whole token, which makes the cosines and sines least often, unless that leaves SMs without 16 warps.
  const int64_t want = int64_t(sms) * 16;
  int share = rows;
  if (a.tokens < want) {
    const int64_t shares = (want + a.tokens - 1) / a.tokens;
    share = static_cast<int>((rows + shares - 1) / shares);
    share = (share + at_once - 1) / at_once * at_once;
    if (share > rows) share = rows;
  }
  const int shares = (rows + share - 1) / share;
  const int64_t blocks = (a.tokens * shares + kRowWarps - 1) / kRowWarps, most = int64_t(sms) * 64;
  const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most));
  auto go = [&](auto kernel) {
    return check_cuda(launch_pdl(kernel, grid, dim3(32 * kRowWarps), 0, st, a, share, shares, group), "rotary launch");
  };
  if (norm) return a.interleaved ? go(row_kernel<T, V, true, true>) : go(row_kernel<T, V, true, false>);
  return a.interleaved ? go(row_kernel<T, V, false, true>) : go(row_kernel<T, V, false, false>);
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace rotary
}  // namespace nvk

extern "C" int nvk_rotary(void* query_out, void* key_out, const void* query, const void* key,
                          int64_t query_out_stride, int64_t key_out_stride, int64_t query_stride, int64_t key_stride,
                          const void* q_weight, const void* k_weight, float eps, const double* inv_freq,
                          const int64_t* positions, float attention_scale, int64_t num_tokens, int num_heads,
                          int num_kv_heads, int head_dim, int rotary_dim, int interleaved, int dtype,
                          nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::rotary;
  const char* who = "rotary";
  if (num_tokens < 0 || num_heads < 0 || num_kv_heads < 0 || num_heads > 65535 || num_kv_heads > 65535)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (tokens=%lld heads=%d kv_heads=%d)", who,
                (long long)num_tokens, num_heads, num_kv_heads);
  if (head_dim < 2 || head_dim > kMostDim || head_dim % 2)
    return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (even, 2 to %d)", who, head_dim, kMostDim);
  if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: rotary_dim %d is not even and in [2, head_dim]", who, rotary_dim);
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_FP16)
    return fail(NVK_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or fp16 rows only)", who, dtype);
  if (num_tokens == 0 || num_heads + num_kv_heads == 0) return NVK_OK;
  if (!inv_freq || !positions || (num_heads && (!query || !query_out)) || (num_kv_heads && (!key || !key_out)))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (num_heads == 0) q_weight = nullptr;  // not used, whatever it is
  if (num_kv_heads == 0) k_weight = nullptr;
  if (!q_weight != !k_weight && num_heads && num_kv_heads)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: norm weights for only one of q and k", who);
  if (!aligned(inv_freq, 8) || !aligned(positions, 8) || !aligned(query, 2) || !aligned(key, 2) ||
      !aligned(query_out, 2) || !aligned(key_out, 2) || !aligned(q_weight, 2) || !aligned(k_weight, 2))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: a tensor is not aligned to its elements", who);
  const int64_t q_row = static_cast<int64_t>(num_heads) * head_dim, k_row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (num_tokens > 1 && (query_stride < q_row || query_out_stride < q_row || key_stride < k_row || key_out_stride < k_row))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: token strides must cover a row", who);
  Args a{{static_cast<const uint8_t*>(query), static_cast<const uint8_t*>(key)},
         {static_cast<uint8_t*>(query_out), static_cast<uint8_t*>(key_out)},
         {static_cast<const uint8_t*>(q_weight), static_cast<const uint8_t*>(k_weight)},
         {query_stride, key_stride},
         {query_out_stride, key_out_stride},
         inv_freq, positions, num_tokens, {num_heads, num_kv_heads}, head_dim, rotary_dim, interleaved ? 1 : 0,
         attention_scale, eps};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // Whole vectors of `v` elements: rows at their multiples, and no vector across the end of the rotated dims (or the
  // middle of them, where the halves are apart).
  auto vectors = [&](int v) {
    auto rows_at = [&](const void* p, int64_t stride, int heads) {
      return heads == 0 || (aligned(p, 2 * v) && (stride % v == 0 || num_tokens == 1));
    };
    return head_dim <= kRowMostDim && head_dim <= 64 * v && head_dim % (2 * v) == 0 && rotary_dim % (2 * v) == 0 &&
           rows_at(query, query_stride, num_heads) && rows_at(query_out, query_out_stride, num_heads) &&
           rows_at(key, key_stride, num_kv_heads) && rows_at(key_out, key_out_stride, num_kv_heads) &&
           aligned(q_weight, 2 * v) && aligned(k_weight, 2 * v);
  };
  const bool norm = q_weight || k_weight, bf16 = dtype == NVK_DTYPE_BF16;
  if (vectors(8)) return bf16 ? launch_rows<__nv_bfloat16, 8>(a, norm, sms, st) : launch_rows<__half, 8>(a, norm, sms, st);
  if (vectors(2)) return bf16 ? launch_rows<__nv_bfloat16, 2>(a, norm, sms, st) : launch_rows<__half, 2>(a, norm, sms, st);
  const dim3 grid(static_cast<unsigned>(num_tokens < int64_t(sms) * 8 ? num_tokens : int64_t(sms) * 8));
  return check_cuda(dtype == NVK_DTYPE_BF16 ? launch_pdl(any_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, a)
                                            : launch_pdl(any_kernel<__half>, grid, dim3(kThreads), 0, st, a),
                    "rotary launch");
}
