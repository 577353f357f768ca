// Decode attention over the 8-bit paged KV cache: one new token per sequence.
//
//   out[b, h] = sum_j softmax_j(scale * q[b, h] . K^[j]) V^[j],  j < context_lens[b]
// with K^ = e4m3 * 2^(byte - 127) per (token, kv head) row, V^ the same; the
// g = Hq / Hk query heads of a group share a kv head. A row of length 0 gives
// zeros.
//
// One CTA per (row, kv head): four warps take the tokens in turn, a lane holds
// four dims of each of the group's heads, with a running maximum and sum per
// warp, merged at the end.
#pragma once
#include "fp8_cache.cuh"

namespace nkv {

constexpr int kDecode8Warps = 4;

struct Decode8Params {
  const __nv_bfloat16* q;
  int64_t q_stride_token, q_stride_head;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const uint8_t* k_exp;
  const uint8_t* v_exp;
  int64_t num_blocks;
  const int32_t* block_tables;
  const int32_t* context_lens;
  int max_blocks;
  int block_size;
  int batch;
  int num_kv_heads;
  int g;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_stride_token;
};

__device__ __forceinline__ float4 e4m3x4_to_float4(uint32_t w, float s) {
  const uint32_t a = e4m3x2_to_f16x2(w), b = e4m3x2_hi_to_f16x2(w);
  const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return make_float4(fa.x * s, fa.y * s, fb.x * s, fb.y * s);
}

template <int G>
__global__ void __launch_bounds__(kDecode8Warps * 32) paged_decode_fp8_kernel(const Decode8Params p) {
  __shared__ float so[kDecode8Warps][G][128], sm[kDecode8Warps][G], sl[kDecode8Warps][G];
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.num_kv_heads, h = blockIdx.x % p.num_kv_heads;
  int len = p.context_lens[b];
  if (len > p.max_blocks * p.block_size) {
    if (threadIdx.x == 0) raise_error(NKV_DEVERR_DECODE_BLOCK);
    len = p.max_blocks * p.block_size;
  }
  float4 q[G], o[G];
  float m[G], l[G];
#pragma unroll
  for (int r = 0; r < G; ++r) {
    q[r] = o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[r] = -INFINITY;
    l[r] = 0.f;
    if (r < p.g) {
      const uint2 u = *reinterpret_cast<const uint2*>(p.q + b * p.q_stride_token +
                                                      (h * p.g + r) * p.q_stride_head + 4 * lane);
      q[r] = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                         __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
    }
  }
  for (int t = warp; t < len; t += kDecode8Warps) {
    const int bi = t / p.block_size, off = t - bi * p.block_size;
    const int32_t blk = p.block_tables[static_cast<int64_t>(b) * p.max_blocks + bi];
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0) raise_error(NKV_DEVERR_DECODE_BLOCK);
      continue;
    }
    const int64_t row = ((static_cast<int64_t>(blk) * p.block_size + off) * p.num_kv_heads + h) * 128 + 4 * lane;
    const int64_t e = (static_cast<int64_t>(blk) * p.num_kv_heads + h) * p.block_size + off;
    const float4 k = e4m3x4_to_float4(*reinterpret_cast<const uint32_t*>(p.k_cache + row),
                                      exp_byte_to_float(p.k_exp[e]));
    const float4 v = e4m3x4_to_float4(*reinterpret_cast<const uint32_t*>(p.v_cache + row),
                                      exp_byte_to_float(p.v_exp[e]));
#pragma unroll
    for (int r = 0; r < G; ++r) {
      float s = q[r].x * k.x + q[r].y * k.y + q[r].z * k.z + q[r].w * k.w;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= p.scale_log2;
      const float m_new = fmaxf(m[r], s);
      const float a = exp2f(m[r] - m_new), w = exp2f(s - m_new);
      m[r] = m_new;
      l[r] = l[r] * a + w;
      o[r] = make_float4(o[r].x * a + w * v.x, o[r].y * a + w * v.y, o[r].z * a + w * v.z,
                         o[r].w * a + w * v.w);
    }
  }
#pragma unroll
  for (int r = 0; r < G; ++r) {
    *reinterpret_cast<float4*>(&so[warp][r][4 * lane]) = o[r];
    if (lane == 0) {
      sm[warp][r] = m[r];
      sl[warp][r] = l[r];
    }
  }
  __syncthreads();
  for (int r = warp; r < p.g; r += kDecode8Warps) {
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < kDecode8Warps; ++w) M = fmaxf(M, sm[w][r]);
    for (int w = 0; w < kDecode8Warps; ++w) {
      const float f = sm[w][r] == -INFINITY ? 0.f : exp2f(sm[w][r] - M);
      const float4 x = *reinterpret_cast<const float4*>(&so[w][r][4 * lane]);
      L += sl[w][r] * f;
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    uint2 u;
    u.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    u.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(p.out + b * p.out_stride_token + (h * p.g + r) * 128 + 4 * lane) = u;
  }
}

}  // namespace nkv
