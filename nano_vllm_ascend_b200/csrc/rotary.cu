// Rotary positions of q's and k's heads, with their RMS norm where weights are
// given. Over the first R dims of a head of D, in pairs (a, b) = (y_i, y_i+R/2)
// ("half") or (y_2i, y_2i+1) ("interleaved"):
//   y = x, or x * rsqrt(mean(x^2) + eps) * w
//   out = ((a cos - b sin) f, (b cos + a sin) f),  angle = position * inv_freq_i
// and out = y from dim R on. Everything between the loads and the one rounding
// at the end is fp32; the angle is made in 64 bits, in half turns and less whole
// turns, so that its error is 2^-24 of a turn at any position: a table would
// have to be read, and ends somewhere.
//
// HBM-bound: every row is read and written once.
#include "host_common.h"
#include "nvk_common.cuh"

#include <cuda_fp16.h>

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
// keeps its rounding error (and 1 / pi its next bits), so that a far angle loses
// nothing on its way into [-1, 1] half turns.
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
  const dim3 grid(static_cast<unsigned>(num_tokens < 148 * 8 ? num_tokens : 148 * 8));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return check_cuda(dtype == NVK_DTYPE_BF16 ? launch_pdl(any_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, a)
                                            : launch_pdl(any_kernel<__half>, grid, dim3(kThreads), 0, st, a),
                    "rotary launch");
}
