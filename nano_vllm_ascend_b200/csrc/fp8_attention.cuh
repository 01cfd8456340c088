// Attention over the 8-bit KV pool, the plain way: a warp takes one head of one
// query row and goes through its keys one by one, four dims a lane.
#pragma once

#include "fp8_kv.cuh"

namespace nvk {
namespace fp8 {

struct AttentionArgs {
  __nv_bfloat16* out;
  const __nv_bfloat16* q;
  const uint8_t* pool;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* cu_q;  // null: one query row a sequence
  int* err;
  int64_t total_q;
  int batch, heads, kvh, bt_stride, max_blocks, num_blocks, upb_log2;
  float scale_log2;
};

static __global__ void __launch_bounds__(256) attention_kernel(const AttentionArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t items = a.total_q * a.heads;
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); w < items;
       w += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t row = w / a.heads;
    const int head = static_cast<int>(w - row * a.heads), h = head / (a.heads / a.kvh);
    int b = static_cast<int>(row), lq = 1, i = 0;
    if (a.cu_q) {
      b = -1;
      for (int s = 0; s < a.batch; ++s)
        if (row >= a.cu_q[s] && row < a.cu_q[s + 1]) b = s;
      if (b < 0) continue;
      lq = a.cu_q[b + 1] - a.cu_q[b];
      i = static_cast<int>(row) - a.cu_q[b];
    }
    int64_t lk = a.lens[b];
    const int64_t room = static_cast<int64_t>(a.max_blocks) << (a.upb_log2 + 4);
    if (lk > room) {
      lk = room;
      if (a.err) atomicOr(a.err, kErrContextTooLong);
    }
    const int64_t seen = min(lk - lq + i + 1, lk);
    const uint2 qw = *reinterpret_cast<const uint2*>(a.q + w * kD + 4 * lane);
    const float2 q0 = pair_to_f32<__nv_bfloat16>(qw.x), q1 = pair_to_f32<__nv_bfloat16>(qw.y);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t t = 0; t < seen; ++t) {
      const int u = static_cast<int>(t >> 4), r = static_cast<int>(t & 15);
      const int blk = a.tables[static_cast<int64_t>(b) * a.bt_stride + (u >> a.upb_log2)];
      float2 k0{}, k1{}, v0{}, v1{};
      if (blk >= 0 && blk < a.num_blocks) {
        const uint8_t* unit = a.pool + (((static_cast<int64_t>(blk) * a.kvh + h) << a.upb_log2) +
                                        (u & ((1 << a.upb_log2) - 1))) * kUnitBytes;
        const int at = chunk_at(r, lane >> 2) + 4 * (lane & 3);
        const int* exps = reinterpret_cast<const int*>(unit + kOffExp);
        auto four = [&](uint32_t word, int e, float2& lo, float2& hi) {
          uint32_t x, y;
          e4m3_to_half2(word, x, y);
          const float by = pow2(held_exp(e));
          lo = pair_to_f32<__half>(x), hi = pair_to_f32<__half>(y);
          lo.x *= by, lo.y *= by, hi.x *= by, hi.y *= by;
        };
        four(*reinterpret_cast<const uint32_t*>(unit + at), exps[0], k0, k1);
        four(*reinterpret_cast<const uint32_t*>(unit + kOffV + at), exps[1], v0, v1);
      } else if (a.err) {
        atomicOr(a.err, kErrBadBlockId);
      }
      float s = q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (s > m) {
        const float f = m == -INFINITY ? 0.f : fast_exp2((m - s) * a.scale_log2);
        l *= f;
        for (int e = 0; e < 4; ++e) o[e] *= f;
        m = s;
      }
      const float p = fast_exp2((s - m) * a.scale_log2);
      l += p;
      o[0] += p * v0.x, o[1] += p * v0.y, o[2] += p * v1.x, o[3] += p * v1.y;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(a.out + w * kD + 4 * lane) =
        make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  }
}

inline int launch_attention(const AttentionArgs& a, cudaStream_t st, const char* what) {
  const int64_t want = (a.total_q * a.heads + 7) / 8;
  return check_cuda(launch_pdl(attention_kernel, dim3(static_cast<unsigned>(want < 148 * 8 ? want : 148 * 8)),
                               dim3(256), 0, st, a),
                    what);
}

}  // namespace fp8
}  // namespace nvk
