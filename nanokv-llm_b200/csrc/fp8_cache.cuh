// Rows of the 8-bit KV cache: quantised store and read-back.
//
// A row x[128] of one (token, kv head) is held as 128 e4m3 values and one
// exponent byte: with a = max of the finite |x_i|,
//   k = the smallest integer with a <= 448 * 2^k, kept in [-117, 119]
//       (a == 0: -117),   byte = k + 127,
//   q_i = e4m3(clamp(x_i * 2^-k, -448, 448)), round to nearest even.
// A power-of-two scale costs e4m3 no precision (only range at the subnormal
// end), makes the scaling exact on both sides -- x * 2^-k and q * 2^k are bf16
// numbers -- and needs one byte. The bounds on k keep every q * 2^k a finite
// bf16 number, normal or 0 .. 2^-126-sized. An infinity is held as the largest
// number of its row, a NaN as NaN.
//
// Layouts: values [num_blocks, block_size, Hk, 128] like the bf16 cache,
// exponent bytes [num_blocks, Hk, block_size], so that the bytes of one
// (block, kv head) lie together: a decode tile of 128 tokens takes 128 bytes.
//
// Both kernels only move data: 8 lanes take one row, lane m its elements
// [8 m, 8 m + 8) and [64 + 8 m, 64 + 8 m + 8), so that every access of a row
// covers whole sectors and the row maximum is three shuffles.
#pragma once
#include <cuda_fp8.h>

#include "nkv_common.cuh"
#include "qk_norm_rope.cuh"

namespace nkv {

constexpr int kRows8Warps = 8;      // warps per CTA
constexpr int kRows8PerLane = 2;    // rows a group of 8 lanes takes at a time
constexpr int kLoad8Tokens = 512;   // most tokens of one CTA of the read-back
constexpr int kRow8MinExp = -117;
constexpr int kRow8MaxExp = 119;

// 2^(byte - 127) for byte in [1, 254]; byte 0 gives 0, byte 255 infinity.
__device__ __forceinline__ float exp_byte_to_float(uint32_t byte) {
  return __uint_as_float(byte << 23);
}

// k of a row from its maximum's bf16 bits (finite): a = 1.f * 2^e needs
// k = e - 8 while 1.f <= 1.75 (448 = 1.75 * 2^8), else e - 7. Zero and subnormal
// maxima have a zero exponent field and land below the lower bound.
__device__ __forceinline__ int row8_exponent(uint32_t bits) {
  const int k = static_cast<int>(bits >> 7) - 127 - 8 + ((bits & 0x7fu) > 0x60u ? 1 : 0);
  return min(max(k, kRow8MinExp), kRow8MaxExp);
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// bf16 bits of the largest finite magnitude among the 16 elements that each of
// a row's 8 lanes holds (magnitudes of bf16 numbers order as their bits do).
__device__ __forceinline__ uint32_t row8_top(const uint4 (&raw)[2], unsigned mask) {
  const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
  auto reduce = [&](uint32_t v) {
    v = max_u16x2(v, __shfl_xor_sync(mask, v, 1));
    v = max_u16x2(v, __shfl_xor_sync(mask, v, 2));
    v = max_u16x2(v, __shfl_xor_sync(mask, v, 4));
    return max(v & 0xffffu, v >> 16);
  };
  uint32_t v = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) v = max_u16x2(v, w[j] & 0x7fff7fffu);
  uint32_t top = reduce(v);
  if (top >= 0x7f80u) {  // infinities and NaN do not set the scale
    v = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t a = w[j] & 0x7fff7fffu;
      v = max_u16x2(v, ((a & 0xffffu) < 0x7f80u ? a & 0xffffu : 0u) | (a < 0x7f800000u ? a & 0xffff0000u : 0u));
    }
    top = reduce(v);
  }
  return top;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// The two e4m3 values of the low 16 bits of v, exact in f16.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo;\n\tmov.b32 {lo, _}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 hi;\n\tmov.b32 {_, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(v));
  return r;
}

struct Rows8Params {
  uint8_t* cache[2];   // K, V values
  uint8_t* exps[2];    // K, V exponent bytes
  int64_t num_blocks;
  int num_kv_heads;
  int block_size;
  // store: the step's bf16 rows and their slots
  const __nv_bfloat16* src[2];
  int64_t src_stride[2];
  const int32_t* slot_mapping;
  // load: the packed bf16 rows and where each sequence's pages are
  __nv_bfloat16* dst[2];
  int64_t dst_stride[2];
  const int32_t* block_tables;
  const int32_t* cu_seqlens;
  int max_blocks;
  int batch;
  int num_tokens;
  int cta_tokens;      // tokens of one CTA
};

// What a group of 8 lanes does in a CTA: a token's rows are its K heads, then
// its V heads; the CTA's 32 groups take `width` rows of `tokens` tokens at a
// time, a group always the same row of its tokens, so that only the token
// changes from one access to the next.
struct Rows8Group {
  int which, h, first, tokens;  // K (0) or V (1), kv head, first token, tokens of a pass
};
__device__ __forceinline__ bool rows8_group(int row0, int num_kv_heads, Rows8Group& g) {
  constexpr int kGroups = kRows8Warps * 4;
  const int width = min(2 * num_kv_heads - row0, kGroups);
  const int group = threadIdx.x >> 3;
  g.tokens = kGroups / width;
  g.first = group / width;
  const int row = row0 + group - g.first * width;
  g.which = row >= num_kv_heads ? 1 : 0;
  g.h = row - g.which * num_kv_heads;
  return g.first < g.tokens;
}

// Both kernels: a pass takes kRows8PerLane tokens a group, their loads first,
// then the arithmetic and the stores.
__global__ void __launch_bounds__(kRows8Warps * 32) store_kvcache_fp8_kernel(const Rows8Params p) {
  allow_dependent_launch();
  grid_dependency_wait();
  const int m = threadIdx.x & 7;
  const unsigned mask = 0xffu << (threadIdx.x & 24);  // this row's 8 lanes, all on the same path
  const int t0 = blockIdx.x * p.cta_tokens;
  const int tokens = min(p.cta_tokens, p.num_tokens - t0);
  const int64_t num_slots = p.num_blocks * p.block_size;
  for (int row0 = 0; row0 < 2 * p.num_kv_heads; row0 += kRows8Warps * 4) {
    Rows8Group g;
    if (!rows8_group(row0, p.num_kv_heads, g)) continue;
    const int64_t src_stride = p.src_stride[g.which];
    const __nv_bfloat16* src = p.src[g.which] + t0 * src_stride + g.h * 128 + 8 * m;
    uint8_t* values = p.cache[g.which] + g.h * 128 + 8 * m;
    uint8_t* exps = p.exps[g.which] + static_cast<int64_t>(g.h) * p.block_size;
    for (int t = g.first; t < tokens; t += g.tokens * kRows8PerLane) {
      int32_t slot[kRows8PerLane];
      uint4 raw[kRows8PerLane][2];
#pragma unroll
      for (int i = 0; i < kRows8PerLane; ++i) {
        const int tt = t + i * g.tokens;
        slot[i] = -1;
        if (tt >= tokens) continue;
        slot[i] = ldg_nc_s32(p.slot_mapping + t0 + tt);
        // read whatever the slot is: no wait before the loads
        const uint4* at = reinterpret_cast<const uint4*>(src + tt * src_stride);
        raw[i][0] = ldg_nc_v4(at);
        raw[i][1] = ldg_nc_v4(at + 8);
      }
#pragma unroll
      for (int i = 0; i < kRows8PerLane; ++i) {
        if (slot[i] == -1) continue;
        if (slot[i] < 0 || slot[i] >= num_slots) {
          if (m == 0) raise_error(NKV_DEVERR_STORE_SLOT);
          continue;
        }
        float x[2][8];
        bf8_to_f8(raw[i][0], x[0]);
        bf8_to_f8(raw[i][1], x[1]);
        const int k = row8_exponent(row8_top(raw[i], mask));
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
        uint2 q[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float(&v)[8] = x[half];
          q[half] = make_uint2(e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                               e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
        }
        uint2* dst = reinterpret_cast<uint2*>(values + static_cast<int64_t>(slot[i]) * p.num_kv_heads * 128);
        dst[0] = q[0];
        dst[8] = q[1];
        if (m == 0) {
          const int blk = slot[i] / p.block_size;
          exps[static_cast<int64_t>(blk) * p.num_kv_heads * p.block_size + (slot[i] - blk * p.block_size)] =
              static_cast<uint8_t>(k + 127);
        }
      }
    }
  }
}

// A CTA finds its tokens' pages first (a search, then a table entry: four or
// five loads in turn, once for the CTA), then streams their rows.
__global__ void __launch_bounds__(kRows8Warps * 32) load_kvcache_fp8_kernel(const Rows8Params p) {
  __shared__ int2 places[kLoad8Tokens];  // block, offset in it; block -1: left as it is, -2: reads as zeros
  allow_dependent_launch();
  grid_dependency_wait();
  const int t0 = blockIdx.x * p.cta_tokens;
  const int tokens = min(p.cta_tokens, p.num_tokens - t0);
  for (int i = threadIdx.x; i < tokens; i += kRows8Warps * 32) {
    const int t = t0 + i;
    // the sequence of packed row t: the last b with cu_seqlens[b] <= t
    int lo = 0, hi = p.batch;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(p.cu_seqlens + mid) <= t) lo = mid;
      else hi = mid - 1;
    }
    // before the first sequence or behind the last one: left as it is
    const int pos = lo < p.batch ? t - __ldg(p.cu_seqlens + lo) : -1;
    int2 place = make_int2(-1, 0);
    if (pos >= 0) {
      const int bi = pos / p.block_size;
      if (bi >= p.max_blocks) {
        raise_error(NKV_DEVERR_PREFILL_RANGE);
      } else {
        place = make_int2(__ldg(p.block_tables + static_cast<int64_t>(lo) * p.max_blocks + bi),
                          pos - bi * p.block_size);
        if (place.x < 0 || place.x >= p.num_blocks) {
          raise_error(NKV_DEVERR_DECODE_BLOCK);
          place.x = -2;
        }
      }
    }
    places[i] = place;
  }
  __syncthreads();
  const int m = threadIdx.x & 7;
  for (int row0 = 0; row0 < 2 * p.num_kv_heads; row0 += kRows8Warps * 4) {
    Rows8Group g;
    if (!rows8_group(row0, p.num_kv_heads, g)) continue;
    const int64_t dst_stride = p.dst_stride[g.which];
    __nv_bfloat16* out = p.dst[g.which] + t0 * dst_stride + g.h * 128 + 8 * m;
    const int64_t block_rows = static_cast<int64_t>(p.num_kv_heads) * p.block_size;
    const uint8_t* values = p.cache[g.which] + g.h * 128 + 8 * m;
    const uint8_t* exps = p.exps[g.which] + static_cast<int64_t>(g.h) * p.block_size;
    for (int t = g.first; t < tokens; t += g.tokens * kRows8PerLane) {
      int blk[kRows8PerLane];
      uint2 raw[kRows8PerLane][2];
      uint32_t byte[kRows8PerLane];
#pragma unroll
      for (int i = 0; i < kRows8PerLane; ++i) {
        const int tt = t + i * g.tokens;
        const int2 place = tt < tokens ? places[tt] : make_int2(-1, 0);
        blk[i] = place.x;
        raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
        byte[i] = 0u;
        if (place.x >= 0) {
          const int64_t base = place.x * block_rows;
          const uint2* src =
              reinterpret_cast<const uint2*>(values + (base + place.y * p.num_kv_heads) * 128);
          raw[i][0] = __ldg(src);
          raw[i][1] = __ldg(src + 8);
          byte[i] = __ldg(exps + base + place.y);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows8PerLane; ++i) {
        if (blk[i] == -1) continue;
        const float s = exp_byte_to_float(byte[i]);
        uint4* dst = reinterpret_cast<uint4*>(out + (t + i * g.tokens) * dst_stride);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t w[2] = {raw[i][half].x, raw[i][half].y};
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t a = e4m3x2_to_f16x2(w[j]), b = e4m3x2_hi_to_f16x2(w[j]);
            const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
            const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
            o[2 * j] = pack_bf16x2(fa.x * s, fa.y * s);
            o[2 * j + 1] = pack_bf16x2(fb.x * s, fb.y * s);
          }
          dst[8 * half] = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
  }
}

}  // namespace nkv
