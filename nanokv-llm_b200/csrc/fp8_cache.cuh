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
constexpr int kRows8PerLane = 4;    // rows each group of 8 lanes takes
constexpr int kRows8PerWarp = 4 * kRows8PerLane;
constexpr int kLoad8Tokens = 512;   // most tokens of one CTA of the read-back
constexpr int kRow8MinExp = -117;
constexpr int kRow8MaxExp = 119;

// 2^(byte - 127) for byte in [1, 254]; byte 0 gives 0, byte 255 infinity.
__device__ __forceinline__ float exp_byte_to_float(uint32_t byte) {
  return __uint_as_float(byte << 23);
}

// k of the row maximum a (finite, >= 0): a = 1.f * 2^e needs k = e - 8 while
// 1.f <= 1.75 (448 = 1.75 * 2^8), else e - 7. bf16 subnormals have a zero
// exponent field and land below the lower bound either way.
__device__ __forceinline__ int row8_exponent(float a) {
  const uint32_t bits = __float_as_uint(a);
  const int e = static_cast<int>(bits >> 23) - 127;
  const int k = e - 8 + ((bits & 0x007fffffu) > 0x00600000u ? 1 : 0);
  return min(max(k, kRow8MinExp), kRow8MaxExp);
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
  uint32_t num_rows;   // tokens x 2 x Hk
  int cta_tokens;      // read-back: tokens of one CTA
};

// Row `r` of the call: token, K (0) or V (1), kv head. The rows of a token are
// its K heads, then its V heads.
struct Row8 {
  int t, which, h;
};
__device__ __forceinline__ Row8 row8_of(uint32_t r, int num_kv_heads) {
  const uint32_t per_token = 2u * num_kv_heads;
  const uint32_t t = r / per_token;
  const int rest = static_cast<int>(r - t * per_token);
  const int which = rest >= num_kv_heads ? 1 : 0;
  return Row8{static_cast<int>(t), which, rest - which * num_kv_heads};
}

// Rows in three steps -- where they are, all loads, the arithmetic and the
// stores -- so that a lane has eight 16-byte loads in flight.
__global__ void __launch_bounds__(kRows8Warps * 32) store_kvcache_fp8_kernel(const Rows8Params p) {
  allow_dependent_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int m = lane & 7;
  const int sub = lane >> 3;  // row within the warp's four
  const uint32_t base = (blockIdx.x * kRows8Warps + (threadIdx.x >> 5)) * kRows8PerWarp;
  const int64_t num_slots = p.num_blocks * p.block_size;
  int32_t slot[kRows8PerLane];
  Row8 row[kRows8PerLane];
  uint4 raw[kRows8PerLane][2];
#pragma unroll
  for (int i = 0; i < kRows8PerLane; ++i) {
    const uint32_t r = base + 4 * i + sub;
    row[i] = row8_of(min(r, p.num_rows - 1), p.num_kv_heads);
    slot[i] = r < p.num_rows ? ldg_nc_s32(p.slot_mapping + row[i].t) : -1;
  }
#pragma unroll
  for (int i = 0; i < kRows8PerLane; ++i) {
    // rows that are not written are read all the same: no branch before the loads
    const uint4* src = reinterpret_cast<const uint4*>(
        p.src[row[i].which] + row[i].t * p.src_stride[row[i].which] + row[i].h * 128 + 8 * m);
    raw[i][0] = ldg_nc_v4(src);
    raw[i][1] = ldg_nc_v4(src + 8);
  }
#pragma unroll
  for (int i = 0; i < kRows8PerLane; ++i) {
    if (slot[i] == -1) continue;
    if (slot[i] < 0 || slot[i] >= num_slots) {
      if (m == 0) raise_error(NKV_DEVERR_STORE_SLOT);
      continue;
    }
    float x[16];
    {
      float half[8];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf8_to_f8(raw[i][s], half);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[8 * s + j] = half[j];
      }
    }
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float v = fabsf(x[j]);
      if (v < INFINITY) a = fmaxf(a, v);  // infinities and NaN do not set the scale
    }
    const unsigned mask = 0xffu << (8 * sub);  // this row's 8 lanes, all on the same path
    a = fmaxf(a, __shfl_xor_sync(mask, a, 1));
    a = fmaxf(a, __shfl_xor_sync(mask, a, 2));
    a = fmaxf(a, __shfl_xor_sync(mask, a, 4));
    const int k = row8_exponent(a);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[j] = e4m3x4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
    uint2* dst = reinterpret_cast<uint2*>(
        p.cache[row[i].which] + (static_cast<int64_t>(slot[i]) * p.num_kv_heads + row[i].h) * 128 + 8 * m);
    dst[0] = make_uint2(q[0], q[1]);
    dst[8] = make_uint2(q[2], q[3]);
    if (m == 0) {
      const int blk = slot[i] / p.block_size;
      p.exps[row[i].which][(static_cast<int64_t>(blk) * p.num_kv_heads + row[i].h) * p.block_size +
                           (slot[i] - blk * p.block_size)] = static_cast<uint8_t>(k + 127);
    }
  }
}

// A CTA finds its tokens' slots first (a search, then a table entry: four or
// five loads in turn, once for the CTA), then streams their rows.
__global__ void __launch_bounds__(kRows8Warps * 32) load_kvcache_fp8_kernel(const Rows8Params p) {
  __shared__ int32_t slots[kLoad8Tokens];  // -1: left as it is, -2: no page, reads as zeros
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
    int slot = -1;
    if (pos >= 0) {
      const int bi = pos / p.block_size;
      if (bi >= p.max_blocks) {
        raise_error(NKV_DEVERR_PREFILL_RANGE);
      } else {
        const int32_t blk = __ldg(p.block_tables + static_cast<int64_t>(lo) * p.max_blocks + bi);
        if (blk >= 0 && blk < p.num_blocks) {
          slot = blk * p.block_size + pos - bi * p.block_size;
        } else {
          raise_error(NKV_DEVERR_DECODE_BLOCK);
          slot = -2;
        }
      }
    }
    slots[i] = slot;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int m = lane & 7;
  const int sub = lane >> 3;
  const uint32_t rows = static_cast<uint32_t>(tokens) * 2u * p.num_kv_heads;
  for (uint32_t r0 = (threadIdx.x >> 5) * kRows8PerWarp; r0 < rows; r0 += kRows8Warps * kRows8PerWarp) {
    Row8 row[kRows8PerLane];
    int slot[kRows8PerLane];
    uint2 raw[kRows8PerLane][2];
    uint32_t byte[kRows8PerLane];
#pragma unroll
    for (int i = 0; i < kRows8PerLane; ++i) {
      const uint32_t r = r0 + 4 * i + sub;
      row[i] = row8_of(min(r, rows - 1), p.num_kv_heads);
      slot[i] = r < rows ? slots[row[i].t] : -1;
      raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
      byte[i] = 0u;
      if (slot[i] >= 0) {
        const uint2* src = reinterpret_cast<const uint2*>(
            p.cache[row[i].which] + (static_cast<int64_t>(slot[i]) * p.num_kv_heads + row[i].h) * 128 + 8 * m);
        const int blk = slot[i] / p.block_size;
        raw[i][0] = __ldg(src);
        raw[i][1] = __ldg(src + 8);
        byte[i] = __ldg(p.exps[row[i].which] +
                        (static_cast<int64_t>(blk) * p.num_kv_heads + row[i].h) * p.block_size +
                        (slot[i] - blk * p.block_size));
      }
    }
#pragma unroll
    for (int i = 0; i < kRows8PerLane; ++i) {
      if (slot[i] == -1) continue;
      const float s = exp_byte_to_float(byte[i]);
      uint4* dst = reinterpret_cast<uint4*>(p.dst[row[i].which] +
                                            (t0 + row[i].t) * p.dst_stride[row[i].which] + row[i].h * 128 + 8 * m);
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

}  // namespace nkv
