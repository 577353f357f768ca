// Decode attention over the 8-bit paged KV cache: one new token per sequence.
//
//   out[b, h] = sum_j softmax_j(scale * q[b, h] . K^[j]) V^[j],  j < context_lens[b]
// with K^ = e4m3 * 2^(byte - 127) per (token, kv head) row, V^ the same; the
// g = Hq / Hk query heads of a group share a kv head. A row of length 0 gives
// zeros.
//
// What bounds it: HBM. A cached token of a kv head is 258 bytes and 4 g * 128
// FLOP, 2 g FLOP a byte.
//
// Split and join. The work of a call is the 128-token tiles of every (row, kv
// head) pair (64 tokens of two heads where kv heads pair up) in the order (head,
// row, tile); CTA c of n takes T / n of the T tiles, the first T mod n CTAs one
// more. (Heads outermost: CTAs n / Hk apart then read the same tokens of
// different heads at the same time, neighbours in memory.) The ranges are equal
// whatever the lengths, and which tiles they hold depends on the lengths alone:
// results are the same every time. A CTA finishes the pairs that lie inside its
// range; of a pair that it shares with others it leaves the raw (m, l, O) in the
// workspace (at most two: at its range's start and end), which a second kernel,
// launched behind the first with programmatic dependence, joins in the CTAs'
// order. No counters, so the workspace needs no content and outlives nothing.
//
// Calls of at most one (row, kv head) per SM whose time is latency are launched
// as thread-block clusters of 1 to 8 CTAs instead, a cluster per (row, kv head):
// no scan of the lengths and no second launch, the CTAs' parts are joined through
// distributed shared memory by the same kernel.
//
// One CTA per SM: two producer warps walk the range and keep a ring of tiles
// full (TMA for K and V, 128-byte rows, 128B swizzle; bulk copies for the
// exponent bytes and the group's q rows), two groups of four consumer
// warps take the tiles in turn, 32 tokens a warp, with a running softmax per
// warp; at the end of a pair a merger warp joins their states while they go on.
//
// Arithmetic. e4m3 is exact in f16, so K and V go to the tensor cores as f16
// (mma.sync m16n8k16, 32-bit sums; groups of 1 to 16 heads are too narrow for
// 64-row tcgen05 tiles). mma.sync takes e4m3 operands too, with sums as exact,
// but rearranges them on every use (a warp's dependent products 52 cycles
// apart, f16 24): with q and the weights split in two e4m3 terms instead of K
// and V converted, 128 rows of 8 kv heads took 226 us for 192. Products are
// transposed, S^T = K Q^T and O^T = V^T P^T: tokens and dims fill the 16 rows,
// the heads the 8 columns; groups of 9 to 16 heads give the two consumer groups
// eight each, and every tile to both.
//   * q is scaled by the power of two that brings its row's maximum into
//     [1, 2) and rounded to f16: 11 bits for a bf16's 8, so only elements
//     below 2^-14 of the maximum lose any (at most 2^-25 of the maximum).
//   * K's exponents and that power of two multiply the 32-bit scores.
//   * V's exponents go into the weights: w_j = 2^(s_j + k_j - M + 15) with M the
//     running maximum of s_j + k_j (s in log2 units), so w <= 2^15 (f16 reaches
//     65,504) and has f16's full 11 bits down to 2^-29 of the largest, however
//     far the rows' scales are apart; below it is off by at most 2^-40 of the
//     largest. The softmax's own maximum m and sum l are kept beside it in 32
//     bits; at the end O is multiplied by 2^-15 and by 2^(M - m).
// Rows of 8-bit values come out of ldmatrix as 16-bit pairs: for K two dims of
// a token (the k order of the product is permuted to match, in q's fragments
// too), for V, transposed, two dims of two tokens; one byte permute makes them
// two tokens of each dim, and the dims of a fragment's upper and lower 8 rows
// are the odd and the even ones.
#pragma once
#include <cuda_fp16.h>

#include "fp8_cache.cuh"
#include "tcgen05.cuh"

namespace nkv {

constexpr int kDecode8Tile = 128;  // rows of 128 values of a tile: tokens x kv heads
constexpr int kDecode8Warps = 8;  // consumers: two groups of four, which take the tiles in turn
constexpr int kDecode8Merger = kDecode8Warps + 2;  // after two producers, K's and V's
template <bool kCluster>
constexpr int kDecode8Threads = (kDecode8Merger + (kCluster ? 0 : 1)) * 32;
constexpr int kDecode8TileBytes = kDecode8Tile * 128;
constexpr int kDecode8MaxCtas = 160;
constexpr int kDecode8ORow = 132;   // floats of one row of a partial: O[128], m, l, 2 of padding
constexpr int kDecode8JoinWarps = 16;  // at most; no fewer than the q heads of a tile
constexpr int kDecode8MaxCluster = 8;
constexpr int kDecode8WeightExp = 15;  // the largest weight is 2^this

template <int G, int NH>
struct Decode8Shape {
  static_assert(G == 1 || G == 2 || G == 4 || G == 8 || G == 16, "padded group width");
  static_assert(NH == 1 || (NH == 2 && G <= 8), "kv heads of a tile");
  static constexpr int kTokens = kDecode8Tile / NH;  // tokens of a tile
  static constexpr int kWarpHeads = G <= 8 ? G : 8;  // q heads of a consumer warp
  static constexpr int kStages = NH * G <= 4 ? 6 : 5;
  static constexpr int kQBytes = (NH * G < 4 ? 4 : NH * G) * 256;
  // [K][V][q rows][K exponents][V exponents], 1024-byte aligned
  static constexpr int kStageBytes = 2 * kDecode8TileBytes + kQBytes + 1024;
  // the warps' (O, m, l) of a pair, as many pairs as fit beside the ring
  static constexpr int kStateFloats = kDecode8Warps * kWarpHeads * kDecode8ORow;
  static constexpr int kSlots = G <= 4 && !(G == 4 && NH == 1) ? 2 : 1;
  static constexpr int kBarOffset = kStages * kStageBytes + kSlots * kStateFloats * 4;
  static constexpr int kSmemBytes = kBarOffset + (2 * kStages + 2 * kSlots) * 8 + kStages * 16 + kSlots * 16 + 32 + 1024;
};

// What CTA c leaves for the join: the pair that begins in its range and goes
// on in the next CTAs', and how many CTAs share it (0: none).
struct Decode8Split {
  int32_t pair, pieces;
};

struct Decode8Params {
  const __nv_bfloat16* q;
  int64_t q_stride_token, q_stride_head;
  const uint8_t* k_exp;
  const uint8_t* v_exp;
  int64_t num_blocks;
  const int32_t* block_tables;
  const int32_t* context_lens;
  int max_blocks;
  int block_size;
  int box_rows;   // tokens of one TMA box: min(block_size, tokens of a tile)
  int box_heads;  // kv heads of one: a tile's where its tokens lie in one page, else 1
  int batch;
  int num_kv_heads;
  int g;
  int rows;       // q heads of a tile's kv heads
  int join_rows;  // of them, how many a CTA of the join takes
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_stride_token;
  int cluster;           // CTAs of a cluster, one cluster per (row, kv head) that joins by itself
  Decode8Split* splits;  // [CTAs]
  float* parts;          // [CTAs][2][rows][kDecode8ORow]: range's first pair, last pair
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(  // registers only: left to the compiler to schedule
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// Length of row b, kept inside its block table.
__device__ __forceinline__ int decode8_length(const Decode8Params& p, int b) {
  int len = max(__ldg(p.context_lens + b), 0);
  if (len > p.max_blocks * p.block_size) {
    raise_error(NKV_DEVERR_DECODE_BLOCK);
    len = p.max_blocks * p.block_size;
  }
  return len;
}

template <int NH>
__device__ __forceinline__ int decode8_tiles(int len) {
  return (len + kDecode8Tile / NH - 1) / (kDecode8Tile / NH);
}

__device__ __forceinline__ void decode8_store(__nv_bfloat16* dst, float4 v, float f) {
  uint2 u;
  u.x = pack_bf16x2(v.x * f, v.y * f);
  u.y = pack_bf16x2(v.z * f, v.w * f);
  *reinterpret_cast<uint2*>(dst) = u;
}

// kCluster: launched as clusters of p.cluster CTAs, one per (row, kv head). (A
// kernel of its own: the join's code in the split form cost it 3 %.)
template <int G, int NH, bool kCluster>
__global__ void __launch_bounds__(kDecode8Threads<kCluster>, 1)
paged_decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const Decode8Params p) {
  using S = Decode8Shape<G, NH>;
  constexpr int kTokens = S::kTokens;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  constexpr int kSlots = S::kSlots;
  float* state = reinterpret_cast<float*>(smem + kStages * S::kStageBytes);  // [slots]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::kBarOffset);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* state_full = empty_bar + kStages;  // per slot: written by all consumer warps
  uint64_t* state_empty = state_full + kSlots;  // and read again
  // per stage: row (-1: no more tiles), head, flags | valid tokens << 8; per slot the same
  int4* meta = reinterpret_cast<int4*>(smem + (S::kBarOffset + (2 * kStages + 2 * kSlots) * 8 + 15) / 16 * 16);
  int4* slot_meta = meta + kStages;
  volatile int* abort_flag = reinterpret_cast<int*>(slot_meta + kSlots);
  __shared__ int warp_tiles[kDecode8Merger + 1];
  __shared__ int4 first_tile;  // the range's first row, tile of it, the row's length and tiles
  enum { kFirst = 1, kLast = 2, kPartial = 4, kPartialSlot1 = 8, kFinal = 16 };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 2);
      mbar_init(smem_u32(&empty_bar[s]), kDecode8Warps);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(smem_u32(&state_full[s]), kDecode8Warps);
      mbar_init(smem_u32(&state_empty[s]), kCluster ? kDecode8Warps : 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == kDecode8Warps * 32) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  // Lengths and tables into L2 before the wait (a hint: what the kernel ahead
  // may still write is written there too); a cache's stream has evicted them
  // since the last call, and the first tile waits for two such loads in turn.
  {
    const int64_t lines = (p.batch * 4 + 127) / 128;
    const int64_t all = lines + (static_cast<int64_t>(p.batch) * p.max_blocks * 4 + 127) / 128;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x; i < min(all, 4 * step); i += step)
      prefetch_l2(i < lines ? reinterpret_cast<const char*>(p.context_lens) + i * 128
                            : reinterpret_cast<const char*>(p.block_tables) + (i - lines) * 128);
  }
  __syncthreads();
  grid_dependency_wait();
  allow_dependent_launch();

  const int csize = p.cluster;
  if (kCluster && static_cast<int>(cluster_nctarank()) != csize) {
    if (threadIdx.x == 0) raise_error(NKV_DEVERR_LAUNCH_SHAPE);
    return;
  }
  const int groups = p.num_kv_heads / NH;  // of kv heads, one a tile
  const int g = p.g;
  const float NEG_INF = -INFINITY;
  // Sum of the consumer warps' states of one of a tile's q heads, this lane's
  // four dims: M, L, acc. With two kv heads a tile, every other pair of warps;
  // with more than eight heads, every other group of four.
  auto merge_row = [&](const float* st, int row, float& M, float& L, float4& acc) {
    constexpr int kHeads = S::kWarpHeads;
    constexpr int kStates = G > 8 ? 4 : kDecode8Warps / NH;
    const int part = G > 8 ? row >> 3 : NH == 1 ? 0 : row / g;  // eight heads; or a kv head's
    const int first = G > 8 ? part * 4 : part * 2;              // its first warp
    const float* src = st + (first * kHeads + row - part * (G > 8 ? 8 : g)) * kDecode8ORow;
    auto of = [](int w) { return NH == 1 ? w : (w >> 1) * 4 + (w & 1); };
    float2 ml[kStates];
    M = NEG_INF;
#pragma unroll
    for (int w = 0; w < kStates; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(src + of(w) * kHeads * kDecode8ORow + 128);
      M = fmaxf(M, ml[w].x);
    }
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kStates; ++w) {
      const float f = ml[w].x == NEG_INF ? 0.f : fast_exp2(ml[w].x - M);
      const float4 x = *reinterpret_cast<const float4*>(src + of(w) * kHeads * kDecode8ORow + 4 * lane);
      L += ml[w].y * f;
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
  };

  // ---- the call's tiles and this CTA's range of them (the split form). Every
  // thread sums the tiles of a few rows in turn; the one whose rows hold the
  // range's first tile finds the row.
  int total = 0, head_tiles = 0, ctas = 1, u = 0, left = 0, head_first = 0;
  if constexpr (!kCluster) {
    const int per = (p.batch + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
    const int row0 = min(static_cast<int>(threadIdx.x) * per, p.batch), row1 = min(row0 + per, p.batch);
    int mine = 0;
#pragma unroll 4
    for (int i = row0; i < row1; ++i) mine += decode8_tiles<NH>(decode8_length(p, i));
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) warp_tiles[warp] = incl;
    __syncthreads();
    int before = incl - mine;
#pragma unroll
    for (int w = 0; w <= kDecode8Merger; ++w) {
      const int x = warp_tiles[w];
      if (w < warp) before += x;
      head_tiles += x;
    }
    total = head_tiles * groups;
    ctas = max(min(static_cast<int>(gridDim.x), total), 1);
    const int c = static_cast<int>(blockIdx.x);
    const int share = total / ctas, more = total - share * ctas;  // the first `more` CTAs take one more
    if (c < ctas) {
      u = c * share + min(c, more);
      left = share + (c < more ? 1 : 0);
    }
    head_first = left > 0 ? u / head_tiles : 0;
    const int rest = u - head_first * head_tiles;
    if (mine > 0 && rest >= before && rest < before + mine) {
      int at = before;
      for (int i = row0;; ++i) {
        const int len = decode8_length(p, i), n = decode8_tiles<NH>(len);
        if (rest < at + n) {
          first_tile = make_int4(i, rest - at, len, n);
          break;
        }
        at += n;
      }
    }
    __syncthreads();
  }

  // A merged row of (b, h): the output or, if the pair is shared with other
  // CTAs, this one's part.
  auto put_row = [&](int slot, int b, int h, int flags, int row) {
    float M, L;
    float4 acc;
    merge_row(state + slot * S::kStateFloats, row, M, L, acc);
    if (!(flags & kPartial)) {
      decode8_store(p.out + b * p.out_stride_token + (h * p.rows + row) * 128 + 4 * lane, acc,
                    L > 0.f ? 1.f / L : 0.f);
    } else {
      float* dst = p.parts + ((blockIdx.x * 2 + (flags & kPartialSlot1 ? 1 : 0)) * p.rows + row) * kDecode8ORow;
      *reinterpret_cast<float4*>(dst + 4 * lane) = acc;
      if (lane == 0) *reinterpret_cast<float2*>(dst + 128) = make_float2(M, L);
    }
  };

  if (!kCluster && warp == kDecode8Merger) {
    // -------------------------------------------------------------- merger
    // Joins the states of a pair while the consumers go on with the next one;
    // the last pair of the range they join themselves.
    for (uint32_t n = 0;; ++n) {
      const int slot = static_cast<int>(n % kSlots);
      if (!mbar_wait_bounded(smem_u32(&state_full[slot]), (n / kSlots) & 1u)) {
        *abort_flag = 1;
        return;
      }
      const int4 sm = slot_meta[slot];
      const int b = sm.x, h = sm.y, flags = sm.z;
      if (b < 0 || (flags & kFinal)) return;
#pragma unroll 2
      for (int row = 0; row < p.rows; ++row) put_row(slot, b, h, flags, row);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&state_empty[slot]));
    }
  }

  if (warp >= kDecode8Warps) {
    // ----------------------------------------------------------- producers
    // Both walk the same tiles; one copies K, its exponents and q, the other V
    // and its exponents. A lane holds the position of one box (min(block_size,
    // 128) tokens) of the 32 ahead and issues that box's copies itself, so a
    // tile costs no division, shuffle or table load.
    const bool for_k = warp == kDecode8Warps;
    const CUtensorMap* tm = for_k ? &tm_k : &tm_v;
    const uint8_t* exps = for_k ? p.k_exp : p.v_exp;
    const uint32_t value_off = for_k ? 0u : static_cast<uint32_t>(kDecode8TileBytes);
    const uint32_t exp_off = 2 * kDecode8TileBytes + S::kQBytes + (for_k ? 0u : static_cast<uint32_t>(kDecode8Tile));
    const uint64_t policy = l2_policy_evict_first();
    const uint32_t q_bytes = for_k ? static_cast<uint32_t>(p.rows) * 256u : 0u;
    const int box_shift = 31 - __clz(p.box_rows);
    const int tile_boxes = kTokens >> box_shift;
    const int page_boxes = p.block_size >> box_shift;
    // of a page: a shift where it is a power of two (every usual size)
    const int page_shift = (page_boxes & (page_boxes - 1)) == 0 ? 31 - __clz(page_boxes) : -1;
    auto page_of = [&](int box) { return page_shift >= 0 ? box >> page_shift : box / page_boxes; };
    // ---- its first row, head and tile
    int b = 0, h = 0, t = 0, len = 0, ntiles = 0;
    if (kCluster) {
      const int pair = static_cast<int>(blockIdx.x) / csize, rank = static_cast<int>(blockIdx.x) % csize;
      b = pair / groups;
      h = pair - b * groups;
      len = decode8_length(p, b);
      ntiles = decode8_tiles<NH>(len);
      t = rank * ntiles / csize;
      left = (rank + 1) * ntiles / csize - t;
    } else if (left > 0) {
      const int4 at = first_tile;
      b = at.x;
      h = head_first;
      t = at.y;
      len = at.z;
      ntiles = at.w;
    }
    // the lengths of 32 rows from lens0, one per lane
    int lens0 = -32, my_len = 0;
    auto load_lengths = [&](int first) {
      lens0 = first;
      my_len = first + lane < p.batch ? decode8_length(p, first + lane) : 0;
    };
    // the first row with tokens at or after (head, row)
    auto seek = [&](int& head, int& row) {
      while (true) {
        if (row >= p.batch) {
          row = 0;
          ++head;
        }
        if (row < lens0 || row >= lens0 + 32) load_lengths(row);
        const unsigned some = __ballot_sync(0xffffffffu, my_len > 0) & (0xffffffffu << (row - lens0));
        if (some != 0u) {
          row = lens0 + __ffs(some) - 1;
          return;
        }
        row = lens0 + 32;
      }
    };
    // the table entry of this lane's box, first + lane, of a row
    auto load_entry = [&](int row, int first) {
      const int page = page_of(first + lane);
      return page < p.max_blocks
                 ? __ldg(p.block_tables + static_cast<int64_t>(row) * p.max_blocks + page)
                 : -1;
    };
    int box0 = 0, slot = 0;   // the window's first box; this lane's box's first slot
    const uint8_t* exp_src = exps;
    unsigned good = 0u;       // the window's boxes that have a page
    auto set_window = [&](int first, int blk) {
      box0 = first;
      const bool ok = blk >= 0 && blk < p.num_blocks;
      const int off = (first + lane - page_of(first + lane) * page_boxes) << box_shift;
      // no page: rows far outside the tensor, which TMA fills with zeros
      slot = ok ? blk * p.block_size + off : -2 * kDecode8Tile;
      exp_src = exps + (static_cast<int64_t>(blk) * p.num_kv_heads + h * NH) * p.block_size + off;
      good = __ballot_sync(0xffffffffu, ok);
    };
    if (left > 0) set_window(t * tile_boxes, load_entry(b, t * tile_boxes));
    int stage = 0;
    uint32_t phase = 0;
    int64_t issued = 0;
    bool ok = true;
    auto wait_empty = [&]() {
      const uint32_t bar = smem_u32(&empty_bar[stage]);
      for (uint32_t i = 0; i < kWaitPollLimit; ++i) {
        if (mbar_try_wait(bar, phase ^ 1u)) return true;
        if (*abort_flag != 0) return false;
      }
      raise_error(NKV_DEVERR_WAIT_TIMEOUT);
      return false;
    };
    Decode8Split split{0, 0};
    while (left > 0 && ok) {
      // ---- tiles [t, t + count) of (b, h)
      const int count = min(left, ntiles - t);
      const int seg_flags = (count == ntiles ? 0 : kPartial) | (t == 0 ? kPartialSlot1 : 0) |
                            (count == left ? kFinal : 0);
      if (!kCluster && t == 0 && count != ntiles) {
        // the CTA that takes the pair's last tile
        const int last = u + ntiles - 1, share = total / ctas, more = total - share * ctas;
        const int cta = last < more * (share + 1) ? last / (share + 1) : more + (last - more * (share + 1)) / share;
        split.pair = b * groups + h;
        split.pieces = cta - static_cast<int>(blockIdx.x) + 1;
      }
      int next_h = h, next_b = b + 1, next_len = 0, next_ent = -1;
      for (int j = 0; j < count; ++j) {
        int first = (t + j) * tile_boxes - box0;  // the tile's first box within the window
        if (first >= 32) {
          set_window(box0 + first, load_entry(b, box0 + first));
          first = 0;
        }
        const int valid = min(kTokens, len - (t + j) * kTokens);
        const int boxes = (valid + p.box_rows - 1) >> box_shift;
        const int at = lane - first;
        const unsigned with_exps = (good >> first) & (0xffu >> (8 - boxes));
        if (with_exps != 0xffu >> (8 - boxes)) {
          // A box without a page: its values are filled with zeros, its exponent
          // bytes (what the stage held last, maybe 255) here, so that its tokens
          // count as zero keys and values. Before the stage is published.
          ok = wait_empty();
          if (ok && at >= 0 && at < boxes && !((good >> lane) & 1u)) {
            for (int x = 0; x < NH * p.box_rows; x += 16)
              *reinterpret_cast<uint4*>(smem + stage * S::kStageBytes + exp_off + x / p.box_rows * kTokens +
                                        (at << box_shift) + x % p.box_rows) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_shared();
            raise_error(NKV_DEVERR_DECODE_BLOCK);
          }
          ok = __all_sync(0xffffffffu, ok) != 0;
        }
        if (ok && at >= 0 && at < boxes) {
          ok = wait_empty();
          if (ok) {
            const uint32_t sbase = smem_u32(smem + stage * S::kStageBytes);
            const uint32_t bar = smem_u32(&full_bar[stage]);
            if (at == 0) {
              if (for_k) {
                meta[stage] =
                    make_int4(b, h, seg_flags | (j == 0 ? kFirst : 0) | (j == count - 1 ? kLast : 0) | (valid << 8), 0);
              }
              mbar_arrive_expect_tx(bar, (((boxes * 128u + __popc(with_exps)) * NH) << box_shift) +
                                             (j == 0 ? q_bytes : 0u));
              if (for_k && j == 0) {
                const __nv_bfloat16* src =
                    p.q + b * p.q_stride_token + static_cast<int64_t>(h) * p.rows * p.q_stride_head;
                const uint32_t sq = sbase + 2 * kDecode8TileBytes;
                if (p.q_stride_head == 128) {
                  bulk_load_row(sq, src, q_bytes, bar);
                } else {
                  for (int r = 0; r < p.rows; ++r) bulk_load_row(sq + r * 256, src + r * p.q_stride_head, 256, bar);
                }
              }
            }
            for (int hh = 0; hh < NH; hh += p.box_heads)
              tma_load_3d(sbase + value_off + static_cast<uint32_t>((hh * kTokens + (at << box_shift)) * 128), tm,
                          bar, 0, slot, h * NH + hh, policy);
            if ((good >> lane) & 1u) {
#pragma unroll
              for (int hh = 0; hh < NH; ++hh)
                bulk_load_row(sbase + exp_off + hh * kTokens + (at << box_shift), exp_src + hh * p.block_size,
                              p.box_rows, bar);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (!ok) break;
        ++issued;
        if (j == 0 && left > count) {
          // the next row: its length is at hand, its table entries are requested now
          seek(next_h, next_b);
          next_len = __shfl_sync(0xffffffffu, my_len, next_b - lens0);
          next_ent = load_entry(next_b, 0);
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      u += count;
      left -= count;
      t = 0;
      h = next_h;
      b = next_b;
      len = next_len;
      ntiles = decode8_tiles<NH>(len);
      set_window(0, next_ent);
    }
    if (lane == 0) {
      if (for_k && !kCluster) p.splits[blockIdx.x] = split;
      if (ok && wait_empty()) {
        if (for_k) meta[stage].x = -1;
        mbar_arrive(smem_u32(&full_bar[stage]));
      } else {
        *abort_flag = 1;
        // after a wait that gave up: leave no copy in flight behind
        for (int64_t i = max(issued - kStages, static_cast<int64_t>(0)); i < issued; ++i)
          mbar_wait_bounded(smem_u32(&full_bar[i % kStages]), static_cast<uint32_t>(i / kStages) & 1u);
      }
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int gid = lane >> 2;
  const int tig = lane & 3;
  // rows without a token
  for (int b = blockIdx.x; !kCluster && b < p.batch; b += gridDim.x) {
    if (__ldg(p.context_lens + b) > 0 && p.max_blocks > 0) continue;
    uint4* dst = reinterpret_cast<uint4*>(p.out + b * p.out_stride_token);
    for (int i = threadIdx.x; i < groups * p.rows * 16; i += kDecode8Warps * 32) dst[i] = make_uint4(0u, 0u, 0u, 0u);
  }

  float o[8][4];  // O^T: dims 16 dm + 2 gid (+ 1 for [2], [3]), heads 2 tig (+ 1 for odd)
  float m_run[2], l_run[2], w_run[2];
  uint32_t qb[8][2];  // q's B fragments
  float qs[2];
  int stage = 0;
  uint32_t phase = 0;
  uint32_t merges = 0;
  uint32_t turn = G > 8 ? 0u : warp >> 2;  // even: the tile is this group's
  // the warp's 32 rows of a tile: tokens tok_base .. of its kvh-th kv head
  const int row_base = (warp & 3) * 32;
  const int kvh = NH == 1 ? 0 : (warp & 3) >> 1;
  const int tok_base = row_base - kvh * kTokens;
  const int head0 = G > 8 ? (warp >> 2) * 8 : 0;  // its first q head
  const int heads = min(g - head0, S::kWarpHeads);
  while (true) {
    if (!mbar_wait_bounded(smem_u32(&full_bar[stage]), phase)) {
      *abort_flag = 1;
      break;
    }
    const int4 tile = meta[stage];
    const int b = tile.x, h = tile.y, flags = tile.z;
    if (b < 0) break;
    const int valid = flags >> 8;
    const uint8_t* sp = smem + stage * S::kStageBytes;
    const uint8_t* sexp = sp + 2 * kDecode8TileBytes + S::kQBytes;

    if (flags & kFirst) {
#pragma unroll
      for (int dm = 0; dm < 8; ++dm) o[dm][0] = o[dm][1] = o[dm][2] = o[dm][3] = 0.f;
      m_run[0] = m_run[1] = w_run[0] = w_run[1] = NEG_INF;
      l_run[0] = l_run[1] = 0.f;
      // q's B fragments: head gid, dims 16 kk + 4 tig .. + 3
      uint2 raw[8];
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        raw[kk] = make_uint2(0u, 0u);
        if (gid < heads)
          raw[kk] = *reinterpret_cast<const uint2*>(sp + 2 * kDecode8TileBytes + (kvh * g + head0 + gid) * 256 +
                                                    kk * 32 + tig * 8);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(__uint_as_float(raw[kk].x << 16)),
                                     fabsf(__uint_as_float(raw[kk].x & 0xffff0000u))),
                               fmaxf(fabsf(__uint_as_float(raw[kk].y << 16)),
                                     fabsf(__uint_as_float(raw[kk].y & 0xffff0000u)))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
      const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        qb[kk][0] = pack_f16x2(__uint_as_float(raw[kk].x << 16) * down,
                               __uint_as_float(raw[kk].x & 0xffff0000u) * down);
        qb[kk][1] = pack_f16x2(__uint_as_float(raw[kk].y << 16) * down,
                               __uint_as_float(raw[kk].y & 0xffff0000u) * down);
      }
      const float up = __uint_as_float(e << 23) * p.scale_log2;
      qs[0] = __shfl_sync(0xffffffffu, up, 8 * tig);
      qs[1] = __shfl_sync(0xffffffffu, up, 8 * tig + 4);
    }

    const bool mine = G > 8 || (turn++ & 1u) == 0u;
    if (mine && tok_base < valid) {
      const uint32_t sK = smem_u32(sp);
      const uint32_t sV = sK + kDecode8TileBytes;
      const int mi = lane >> 3;
      const int lrow = row_base + (mi & 1) * 8 + (lane & 7);
      // ---- S^T = K Q^T: two 16-token tiles, 8 steps of 16 dims. All loads first
      // (each waits for none of the others), even and odd steps in sums of their
      // own.
      uint32_t raw[2][4][4];  // [token tile][pair of 16-byte chunks]: tokens 0-7 / 8-15 of the first, of the second
#pragma unroll
      for (int kp = 0; kp < 4; ++kp)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
          ldsm_x4(sK + swz128(lrow + 16 * mt, 2 * kp + (mi >> 1)), raw[mt][kp][0], raw[mt][kp][1],
                  raw[mt][kp][2], raw[mt][kp][3]);
      float s[2][4], s_odd[2][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[mt][c] = s_odd[mt][c] = 0.f;
#pragma unroll
      for (int kp = 0; kp < 4; ++kp) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t(&r)[4] = raw[mt][kp];
          mma_f16_16816(s[mt], e4m3x2_to_f16x2(r[0]), e4m3x2_to_f16x2(r[1]), e4m3x2_hi_to_f16x2(r[0]),
                        e4m3x2_hi_to_f16x2(r[1]), qb[2 * kp][0], qb[2 * kp][1]);
          mma_f16_16816(s_odd[mt], e4m3x2_to_f16x2(r[2]), e4m3x2_to_f16x2(r[3]), e4m3x2_hi_to_f16x2(r[2]),
                        e4m3x2_hi_to_f16x2(r[3]), qb[2 * kp + 1][0], qb[2 * kp + 1][1]);
        }
      }
      // ---- the rest of the tile into registers, then the stage goes back to the
      // producer: what a warp holds of the ring is not in flight from memory
      const bool partial = tok_base + 32 > valid;
      float vk[2][2];
      float ks[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int at = row_base + 16 * mt + 8 * r + gid;
          ks[mt][r] = exp_byte_to_float(sexp[at]);
          vk[mt][r] = static_cast<float>(static_cast<int>(sexp[kDecode8Tile + at]) - 127);
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int dp = 0; dp < 4; ++dp)
          ldsm_x4_trans(sV + swz128(lrow + 16 * mt, 2 * dp + (mi >> 1)), raw[mt][dp][0], raw[mt][dp][1],
                        raw[mt][dp][2], raw[mt][dp][3]);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty_bar[stage]));
      // ---- scores in log2 units, running maxima
      float mx[2] = {NEG_INF, NEG_INF}, wx[2] = {NEG_INF, NEG_INF};
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = (s[mt][c] + s_odd[mt][c]) * (ks[mt][c >> 1] * qs[c & 1]);
          if (partial && tok_base + 16 * mt + 8 * (c >> 1) + gid >= valid) v = NEG_INF;
          s[mt][c] = v;
          mx[c & 1] = fmaxf(mx[c & 1], v);
          wx[c & 1] = fmaxf(wx[c & 1], v + vk[mt][c >> 1]);
        }
      }
      float m_use[2], w_low[2], w_scale[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
          wx[e] = fmaxf(wx[e], __shfl_xor_sync(0xffffffffu, wx[e], x));
        }
        const float m_new = fmaxf(m_run[e], mx[e]);
        const float w_new = fmaxf(w_run[e], wx[e]);
        m_use[e] = m_new == NEG_INF ? 0.f : m_new;
        const float w_use = w_new == NEG_INF ? 0.f : w_new;
        w_low[e] = w_use - kDecode8WeightExp;
        l_run[e] *= fast_exp2(m_run[e] - m_use[e]);
        w_scale[e] = fast_exp2(w_run[e] - w_use);
        m_run[e] = m_new;
        w_run[e] = w_new;
      }
      uint32_t wb[2][2];  // the weights as B fragments (two tokens of a head)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        float w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          l_run[c & 1] += fast_exp2(s[mt][c] - m_use[c & 1]);
          w[c] = fast_exp2(s[mt][c] + vk[mt][c >> 1] - w_low[c & 1]);
        }
        wb[mt][0] = movmatrix_trans(pack_f16x2(w[0], w[1]));
        wb[mt][1] = movmatrix_trans(pack_f16x2(w[2], w[3]));
      }
      // the maxima seldom move after the first tiles
      if (__any_sync(0xffffffffu, w_scale[0] != 1.f || w_scale[1] != 1.f)) {
#pragma unroll
        for (int dm = 0; dm < 8; ++dm) {
          o[dm][0] *= w_scale[0];
          o[dm][1] *= w_scale[1];
          o[dm][2] *= w_scale[0];
          o[dm][3] *= w_scale[1];
        }
      }
      if (partial) {  // V of tokens past the end counts as 0
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const int tk = tok_base + 16 * mt + 2 * tig;
          const uint32_t keep_lo = (tk < valid ? 0x0000ffffu : 0u) | (tk + 1 < valid ? 0xffff0000u : 0u);
          const uint32_t keep_hi = (tk + 8 < valid ? 0x0000ffffu : 0u) | (tk + 9 < valid ? 0xffff0000u : 0u);
#pragma unroll
          for (int dp = 0; dp < 4; ++dp) {
            raw[mt][dp][0] &= keep_lo;
            raw[mt][dp][1] &= keep_hi;
            raw[mt][dp][2] &= keep_lo;
            raw[mt][dp][3] &= keep_hi;
          }
        }
      }
      // ---- O^T += V^T P^T: two steps of 16 tokens, 8 tiles of 16 dims
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int dm = 0; dm < 8; ++dm) {
          // bytes: token 2 tig dims 2 gid, 2 gid + 1, token 2 tig + 1 the same
          const uint32_t lo = __byte_perm(raw[mt][dm >> 1][2 * (dm & 1)], 0u, 0x3120);
          const uint32_t hi = __byte_perm(raw[mt][dm >> 1][2 * (dm & 1) + 1], 0u, 0x3120);
          mma_f16_16816(o[dm], e4m3x2_to_f16x2(lo), e4m3x2_hi_to_f16x2(lo), e4m3x2_to_f16x2(hi),
                        e4m3x2_hi_to_f16x2(hi), wb[mt][0], wb[mt][1]);
        }
      }
    } else {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty_bar[stage]));
    }
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1u;
    }
    if (!(flags & kLast)) continue;

    // ---- the pair's tiles in this CTA are done: the warp's state to shared memory
    const int slot = static_cast<int>(merges % kSlots);
    if (!mbar_wait_bounded(smem_u32(&state_empty[slot]), ((merges / kSlots) & 1u) ^ 1u)) {
      *abort_flag = 1;
      break;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[e];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      const int head = 2 * tig + e;
      if (head < heads) {
        const float m = m_run[e];
        const float f = m == NEG_INF ? 0.f : fast_exp2(w_run[e] - m);
        constexpr float kDown = 1.f / (1 << kDecode8WeightExp);
        float* dst = state + slot * S::kStateFloats + (warp * S::kWarpHeads + head) * kDecode8ORow;
#pragma unroll
        for (int dm = 0; dm < 8; ++dm)
          *reinterpret_cast<float2*>(dst + 16 * dm + 2 * gid) = make_float2(o[dm][e] * kDown * f, o[dm][2 + e] * kDown * f);
        if (gid == 0) *reinterpret_cast<float2*>(dst + 128) = make_float2(m, l);
      }
    }
    if (!kCluster && threadIdx.x == 0) {
      slot_meta[slot] = tile;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&state_full[slot]));
    if (kCluster || (flags & kFinal)) {
      if (!mbar_wait_bounded(smem_u32(&state_full[slot]), (merges / kSlots) & 1u)) {
        *abort_flag = 1;
        break;
      }
      for (int row = warp; row < p.rows; row += kDecode8Warps) {
        if constexpr (kCluster) {
          float M, L;
          float4 acc;
          merge_row(state + slot * S::kStateFloats, row, M, L, acc);
          // every tile of this CTA is consumed: the ring's memory is free
          float* dst = reinterpret_cast<float*>(smem) + row * kDecode8ORow;
          *reinterpret_cast<float4*>(dst + 4 * lane) = acc;
          if (lane == 0) *reinterpret_cast<float2*>(dst + 128) = make_float2(M, L);
        } else {
          put_row(slot, b, h, flags, row);
        }
      }
      if (!kCluster) return;
    }
    ++merges;
  }
  if constexpr (!kCluster) {
    // no tile fell to this CTA: the end marker for the merger
    const int slot = static_cast<int>(merges % kSlots);
    if (!mbar_wait_bounded(smem_u32(&state_empty[slot]), ((merges / kSlots) & 1u) ^ 1u)) *abort_flag = 1;
    if (threadIdx.x == 0) slot_meta[slot].x = -1;
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&state_full[slot]));
    return;
  }

  // ---- cluster launch: the CTAs' rows are joined through distributed shared
  // memory, in rank order, each CTA taking some of the group's heads (eight a
  // round: a single CTA with 9 to 16 heads takes two)
  const int rank = static_cast<int>(blockIdx.x) % csize;
  const int pair = static_cast<int>(blockIdx.x) / csize;
  if (merges == 0) {  // no tile fell to this CTA
    for (int row = warp; row < p.rows; row += kDecode8Warps) {
      float* dst = reinterpret_cast<float*>(smem) + row * kDecode8ORow;
      *reinterpret_cast<float4*>(dst + 4 * lane) = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane == 0) *reinterpret_cast<float2*>(dst + 128) = make_float2(NEG_INF, 0.f);
    }
  }
  __syncwarp();
  cluster_sync_all();
  for (int row = warp * csize + rank; row < p.rows; row += kDecode8Warps * csize) {
    float4 x[kDecode8MaxCluster];
    float2 ml[kDecode8MaxCluster];
    float M = NEG_INF;
#pragma unroll
    for (int c = 0; c < kDecode8MaxCluster; ++c) {
      ml[c] = make_float2(NEG_INF, 0.f);
      x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < csize) {
        const uint32_t src = mapa_shared(smem_u32(smem) + row * kDecode8ORow * 4, c);
        x[c] = ld_cluster_f32x4(src + 16 * lane);
        ml[c] = ld_cluster_f32x2(src + 512);
        M = fmaxf(M, ml[c].x);
      }
    }
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kDecode8MaxCluster; ++c) {
      const float f = ml[c].x == NEG_INF ? 0.f : fast_exp2(ml[c].x - M);
      L += ml[c].y * f;
      acc.x += x[c].x * f;
      acc.y += x[c].y * f;
      acc.z += x[c].z * f;
      acc.w += x[c].w * f;
    }
    decode8_store(p.out + (pair / groups) * p.out_stride_token + ((pair % groups) * p.rows + row) * 128 + 4 * lane, acc,
                  L > 0.f ? 1.f / L : 0.f);
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while another reads its rows
}

// Joins the pieces of the pair that begins in CTA blockIdx.x's range and goes
// on in later ones, join_rows of its q heads from join_rows * blockIdx.y on:
// `parts` warps for each head, each summing every parts-th piece, then one of
// them their sums, always in the same order.
__global__ void __launch_bounds__(kDecode8JoinWarps * 32) decode_fp8_join_kernel(const Decode8Params p) {
  __shared__ float sums[kDecode8JoinWarps][kDecode8ORow];
  grid_dependency_wait();
  allow_dependent_launch();
  const Decode8Split split = p.splits[blockIdx.x];
  if (split.pieces == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int parts = blockDim.x >> 5;
  while (parts * p.join_rows > static_cast<int>(blockDim.x >> 5)) parts >>= 1;
  const int in_cta = warp / parts, part = warp - in_cta * parts;
  const int row = blockIdx.y * p.join_rows + in_cta;
  const bool live = in_cta < p.join_rows && row < p.rows;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    // piece 0 is the range's last pair of this CTA, piece i the first of CTA + i
    auto piece = [&](int i) {
      return p.parts + ((static_cast<int>(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + row) * kDecode8ORow;
    };
    // eight pieces' loads at a time, then one rescaling of the sums so far
    for (int i = part; i < split.pieces; i += 8 * parts) {
      float2 ml[8];
      float4 x[8];
      float top = M;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i + k * parts < split.pieces) {
          const float* src = piece(i + k * parts);
          ml[k] = *reinterpret_cast<const float2*>(src + 128);
          x[k] = *reinterpret_cast<const float4*>(src + 4 * lane);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
      const float keep = M == -INFINITY ? 0.f : fast_exp2(M - top);
      M = top;
      L *= keep;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - top);
        L += ml[k].y * f;
        acc.x += x[k].x * f;
        acc.y += x[k].y * f;
        acc.z += x[k].z * f;
        acc.w += x[k].w * f;
      }
    }
  }
  *reinterpret_cast<float4*>(&sums[warp][4 * lane]) = acc;
  if (lane == 0) *reinterpret_cast<float2*>(&sums[warp][128]) = make_float2(M, L);
  __syncthreads();
  if (!live || part != 0) return;
  for (int w = 1; w < parts; ++w) M = fmaxf(M, sums[warp + w][128]);
  L = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < parts; ++w) {
    const float* src = sums[warp + w];
    const float f = src[128] == -INFINITY ? 0.f : fast_exp2(src[128] - M);
    const float4 x = *reinterpret_cast<const float4*>(src + 4 * lane);
    L += src[129] * f;
    acc.x += x.x * f;
    acc.y += x.y * f;
    acc.z += x.z * f;
    acc.w += x.w * f;
  }
  const int groups = p.num_kv_heads * p.g / p.rows;
  const int b = split.pair / groups, h = split.pair - b * groups;
  decode8_store(p.out + b * p.out_stride_token + (h * p.rows + row) * 128 + 4 * lane, acc,
                L > 0.f ? 1.f / L : 0.f);
}

}  // namespace nkv
