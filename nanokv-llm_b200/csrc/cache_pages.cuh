// Pages of a paged KV cache: copying, forking, freeing and compacting.
//
// State, all on the device: block_tables [rows, max_blocks] (-1 = no page),
// context_lens [rows], ref_counts [num_pages] (how many table entries name a
// page; <= 0 = free). A page is block_size tokens of every cache tensor. A
// cache tensor is described by a region: `lead` copies (layers, K / V) of
// num_pages contiguous pages; a page consists of segments of
// block_size * token_bytes bytes (one for the K / V values, one per kv head
// for exponent bytes), so the first n tokens of a page are the first
// n * token_bytes bytes of every segment.
//
// An operation is a plan -- which page goes where and how many of its tokens,
// made by one CTA from the tables and counts -- and a copy of the plan's pages
// over all regions. Everything is decided on the device: nothing is read back,
// and the calls can be captured in a CUDA graph. Free pages are taken lowest
// first, so results do not depend on the order of atomics.
#pragma once
#include "nkv_common.cuh"

namespace nkv {

constexpr int kPagePlanThreads = 1024;
constexpr int kPageCopyThreads = 256;
constexpr int kPageCopyBytes = 32768;  // bytes of one copy item

struct PageRegion {
  uint8_t* base;
  int64_t lead_stride;  // bytes
  int64_t page_bytes;
  int64_t seg_bytes;
  int64_t token_bytes;
  int64_t first_item;     // items of the regions before this one, per page
  int items_per_page;     // items of one page of one lead index
};

// One page of a plan: tokens [0, ntok) of page src go to page dst; dst < 0:
// nothing to do.
struct PageMove {
  int32_t src, dst, ntok, pad;
};

template <int N>
struct PageRegions {
  PageRegion r[N];
  int num;
  int64_t items_per_move;  // over all regions and lead indices
};

// ---------------------------------------------------------------- copy
template <int N>
__global__ void __launch_bounds__(kPageCopyThreads)
page_copy_kernel(const __grid_constant__ PageRegions<N> rg, const PageMove* moves,
                 const int32_t* num_moves_dev, int num_moves, int block_size) {
  allow_dependent_launch();
  grid_dependency_wait();
  const int n = num_moves_dev != nullptr ? min(*num_moves_dev, num_moves) : num_moves;
  const int64_t total = n * rg.items_per_move;
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int64_t mv = item / rg.items_per_move;
    const int64_t rest = item - mv * rg.items_per_move;
    const PageMove move = moves[mv];
    if (move.dst < 0 || move.ntok <= 0) continue;
    int lo = 0, hi = rg.num - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (rg.r[mid].first_item <= rest) lo = mid;
      else hi = mid - 1;
    }
    const PageRegion& r = rg.r[lo];
    const int64_t in_region = rest - r.first_item;
    const int64_t lead = in_region / r.items_per_page;
    const int64_t from = (in_region - lead * r.items_per_page) * kPageCopyBytes;
    const int bytes = static_cast<int>(min(static_cast<int64_t>(kPageCopyBytes), r.page_bytes - from));
    const int64_t live = move.ntok * r.token_bytes;  // bytes of each segment that are copied
    const uint8_t* src = r.base + lead * r.lead_stride + move.src * r.page_bytes + from;
    uint8_t* dst = r.base + lead * r.lead_stride + move.dst * r.page_bytes + from;
    const bool whole = live >= r.seg_bytes;
    for (int v = threadIdx.x; v < bytes / 16; v += kPageCopyThreads) {
      const int64_t off = from + 16 * v;
      int64_t keep = 16;
      if (!whole) keep = live - off % r.seg_bytes;
      if (keep >= 16) {
        reinterpret_cast<uint4*>(dst)[v] = reinterpret_cast<const uint4*>(src)[v];
      } else {
        for (int64_t i = 0; i < keep; ++i) dst[16 * v + i] = src[16 * v + i];
      }
    }
  }
}

// ---------------------------------------------------------------- plan helpers
// Exclusive prefix sum of one value per thread over the CTA; `sum` gets the total.
__device__ __forceinline__ int block_exclusive_sum(int v, int* warp_sums, int& sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous round's sums are read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < kPagePlanThreads / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  sum = total;
  return before + x - v;
}

// Drops one reference to page p (already known to be in range).
__device__ __forceinline__ void page_release(int32_t* ref_counts, int32_t p) {
  if (atomicSub(ref_counts + p, 1) <= 0) {  // already free: undone and flagged
    atomicAdd(ref_counts + p, 1);
    raise_error(NKV_DEVERR_PAGES);
  }
}

// ---------------------------------------------------------------- copy plan
struct PageCopyPlanParams {
  const int32_t* src;
  const int32_t* dst;
  int n;
  int64_t num_pages;
  int block_size;
  PageMove* moves;
};

__device__ __forceinline__ bool bit_of(const uint32_t* map, int64_t i) {
  return (map[i >> 5] >> (i & 31)) & 1u;
}

// A pair is copied when both pages exist, no other pair writes its target and
// no pair reads it (any order of the copies then gives the same result).
__global__ void __launch_bounds__(kPagePlanThreads) page_copy_plan_kernel(const PageCopyPlanParams p) {
  extern __shared__ uint32_t maps[];  // read, written, written twice: a bit per page each
  const int64_t words = (p.num_pages + 31) / 32;
  uint32_t *read = maps, *written = maps + words, *twice = written + words;
  allow_dependent_launch();
  grid_dependency_wait();
  for (int64_t i = threadIdx.x; i < 3 * words; i += kPagePlanThreads) maps[i] = 0u;
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const int32_t s = p.src[i], d = p.dst[i];
    if (s < 0 || s >= p.num_pages || d < 0 || d >= p.num_pages) continue;
    atomicOr(read + (s >> 5), 1u << (s & 31));
    if (atomicOr(written + (d >> 5), 1u << (d & 31)) >> (d & 31) & 1u)
      atomicOr(twice + (d >> 5), 1u << (d & 31));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const int32_t s = p.src[i], d = p.dst[i];
    const bool skip = s == -1 && d == -1;  // padding
    bool ok = s >= 0 && s < p.num_pages && d >= 0 && d < p.num_pages;
    if (ok) ok = !bit_of(twice, d) && !bit_of(read, d);
    if (!ok && !skip) raise_error(NKV_DEVERR_PAGES);
    p.moves[i] = PageMove{s, ok ? d : -1, p.block_size, 0};
  }
}

// ---------------------------------------------------------------- fork plan
struct PageForkParams {
  int32_t* block_tables;
  int max_blocks;
  int num_rows;
  int32_t* context_lens;
  int32_t* ref_counts;
  int64_t num_pages;
  int block_size;
  const int32_t* src_rows;
  const int32_t* dst_rows;
  int n;
  int32_t* out_pages;  // [n]: the page that holds the fork's last tokens, -1: none needed, -2: not forked
  PageMove* moves;     // [n]
  int32_t* free_list;  // [n] scratch
};

__global__ void __launch_bounds__(kPagePlanThreads) page_fork_plan_kernel(const PageForkParams p) {
  extern __shared__ uint32_t maps[];  // rows read, written, written twice
  __shared__ int warp_sums[kPagePlanThreads / 32];
  const int words = (p.num_rows + 31) / 32;
  uint32_t *read = maps, *written = maps + words, *twice = written + words;
  allow_dependent_launch();
  grid_dependency_wait();
  for (int i = threadIdx.x; i < 3 * words; i += kPagePlanThreads) maps[i] = 0u;
  __syncthreads();
  // ---- which forks can be made: rows in range, the target named once and no source
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const int32_t s = p.src_rows[i], d = p.dst_rows[i];
    if (s < 0 || s >= p.num_rows || d < 0 || d >= p.num_rows) continue;
    atomicOr(read + (s >> 5), 1u << (s & 31));
    if (atomicOr(written + (d >> 5), 1u << (d & 31)) >> (d & 31) & 1u)
      atomicOr(twice + (d >> 5), 1u << (d & 31));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const int32_t s = p.src_rows[i], d = p.dst_rows[i];
    const bool skip = s == -1 && d == -1;  // padding
    bool ok = s >= 0 && s < p.num_rows && d >= 0 && d < p.num_rows;
    if (ok) ok = !bit_of(twice, d) && !bit_of(read, d);
    int len = 0;
    if (ok) {
      len = p.context_lens[s];
      ok = len >= 0 && len <= static_cast<int64_t>(p.max_blocks) * p.block_size;
    }
    if (!ok && !skip) raise_error(NKV_DEVERR_PAGES);
    // src: the source's length until the pages are known
    p.moves[i] = PageMove{len, ok ? 0 : -1, len % p.block_size, 0};
    p.out_pages[i] = ok ? -1 : -2;
  }
  __syncthreads();
  // ---- the targets' old pages are released
  const int64_t entries = static_cast<int64_t>(p.n) * p.max_blocks;
  for (int64_t e = threadIdx.x; e < entries; e += kPagePlanThreads) {
    const int i = static_cast<int>(e / p.max_blocks);
    if (p.moves[i].dst < 0) continue;
    int32_t* at = p.block_tables + static_cast<int64_t>(p.dst_rows[i]) * p.max_blocks + e % p.max_blocks;
    const int32_t old = *at;
    if (old >= 0) {
      if (old < p.num_pages) page_release(p.ref_counts, old);
      else raise_error(NKV_DEVERR_PAGES);
      *at = -1;
    }
  }
  __syncthreads();
  // ---- the lowest free pages, as many as forks want one
  int want = 0;
  for (int base = 0; base < p.n; base += kPagePlanThreads) {
    const int i = base + threadIdx.x;
    int sum;
    block_exclusive_sum(i < p.n && p.moves[i].dst >= 0 && p.moves[i].ntok > 0, warp_sums, sum);
    want += sum;
  }
  int found = 0;
  for (int64_t base = 0; base < p.num_pages && found < want; base += kPagePlanThreads) {
    const int64_t page = base + threadIdx.x;
    const bool free = page < p.num_pages && __ldcg(p.ref_counts + page) <= 0;
    int sum;
    const int rank = found + block_exclusive_sum(free, warp_sums, sum);
    if (free && rank < want) p.free_list[rank] = static_cast<int32_t>(page);
    found += sum;
  }
  found = min(found, want);
  __syncthreads();
  // ---- a page for every fork with a partial one, in the forks' order
  int given = 0;
  for (int base = 0; base < p.n; base += kPagePlanThreads) {
    const int i = base + threadIdx.x;
    const bool wants = i < p.n && p.moves[i].dst >= 0 && p.moves[i].ntok > 0;
    int sum;
    const int rank = given + block_exclusive_sum(wants, warp_sums, sum);
    given += sum;
    if (i >= p.n) continue;
    const PageMove m = p.moves[i];
    if (m.dst < 0) continue;
    const int32_t s = p.src_rows[i], d = p.dst_rows[i];
    if (wants) {
      const int32_t from = p.block_tables[static_cast<int64_t>(s) * p.max_blocks + m.src / p.block_size];
      if (rank >= found || from < 0 || from >= p.num_pages) {  // no page left, or none to copy
        raise_error(NKV_DEVERR_PAGES);
        p.moves[i] = PageMove{0, -1, 0, 0};
        p.out_pages[i] = -2;
        p.context_lens[d] = 0;
        continue;
      }
      const int32_t to = p.free_list[rank];
      p.ref_counts[to] = 1;
      p.block_tables[static_cast<int64_t>(d) * p.max_blocks + m.src / p.block_size] = to;
      p.out_pages[i] = to;
      p.moves[i] = PageMove{from, to, m.ntok, 1 + m.src / p.block_size};
    } else {
      p.moves[i] = PageMove{0, -1, 0, 1 + m.src / p.block_size};
    }
    p.context_lens[d] = m.src;
  }
  __syncthreads();
  // ---- full pages are shared (pad: 1 + how many, 0 = not forked)
  for (int64_t e = threadIdx.x; e < entries; e += kPagePlanThreads) {
    const int i = static_cast<int>(e / p.max_blocks);
    const int j = static_cast<int>(e % p.max_blocks);
    if (j >= p.moves[i].pad - 1) continue;
    const int32_t page = p.block_tables[static_cast<int64_t>(p.src_rows[i]) * p.max_blocks + j];
    if (page >= 0 && page < p.num_pages) atomicAdd(p.ref_counts + page, 1);
    else raise_error(NKV_DEVERR_PAGES);
    p.block_tables[static_cast<int64_t>(p.dst_rows[i]) * p.max_blocks + j] = page;
  }
}

// ---------------------------------------------------------------- free
struct PageFreeParams {
  int32_t* block_tables;
  int max_blocks;
  int num_rows;
  int32_t* context_lens;
  int32_t* ref_counts;
  int64_t num_pages;
  int block_size;
  const int32_t* rows;
  int n;
  int trim;
};

// One CTA per named row. The exchange makes a row that is named twice lose its
// pages once.
__global__ void __launch_bounds__(256) page_free_kernel(const PageFreeParams p) {
  allow_dependent_launch();
  grid_dependency_wait();
  const int32_t row = p.rows[blockIdx.x];
  if (row == -1) return;  // padding
  if (row < 0 || row >= p.num_rows) {
    if (threadIdx.x == 0) raise_error(NKV_DEVERR_PAGES);
    return;
  }
  int keep = 0;
  if (p.trim) {
    const int len = p.context_lens[row];
    keep = len > 0 ? (len - 1) / p.block_size + 1 : 0;
  }
  for (int j = keep + threadIdx.x; j < p.max_blocks; j += blockDim.x) {
    const int32_t page = atomicExch(p.block_tables + static_cast<int64_t>(row) * p.max_blocks + j, -1);
    if (page < 0) continue;
    if (page < p.num_pages) page_release(p.ref_counts, page);
    else raise_error(NKV_DEVERR_PAGES);
  }
  if (!p.trim && threadIdx.x == 0) p.context_lens[row] = 0;
}

// ---------------------------------------------------------------- compact plan
struct PageCompactParams {
  const int32_t* block_tables;
  int32_t* out_block_tables;  // may be block_tables
  int64_t entries;            // rows * max_blocks
  const int32_t* ref_counts;
  int32_t* out_ref_counts;    // may be ref_counts
  int64_t num_pages;
  int block_size;
  int32_t* out_num_live;
  PageMove* moves;
  int32_t* num_moves;
  int32_t* remap;             // [num_pages]: where a moved page went, -1 = stays, -2 = free
};

// With n live pages, the i-th live page at or past n goes to the i-th free
// page before n, both counted upwards.
__global__ void __launch_bounds__(kPagePlanThreads) page_compact_plan_kernel(const PageCompactParams p) {
  __shared__ int warp_sums[kPagePlanThreads / 32];
  allow_dependent_launch();
  grid_dependency_wait();
  int live = 0;
  for (int64_t base = 0; base < p.num_pages; base += kPagePlanThreads) {
    const int64_t page = base + threadIdx.x;
    int sum;
    block_exclusive_sum(page < p.num_pages && p.ref_counts[page] > 0, warp_sums, sum);
    live += sum;
  }
  int holes = 0, movers = 0;
  for (int64_t base = 0; base < p.num_pages; base += kPagePlanThreads) {
    const int64_t page = base + threadIdx.x;
    const bool in = page < p.num_pages;
    const bool used = in && p.ref_counts[page] > 0;
    const bool hole = in && !used && page < live, mover = used && page >= live;
    int hole_sum, mover_sum;
    const int hole_at = holes + block_exclusive_sum(hole, warp_sums, hole_sum);
    const int mover_at = movers + block_exclusive_sum(mover, warp_sums, mover_sum);
    if (hole) p.moves[hole_at].dst = static_cast<int32_t>(page);
    if (mover) p.moves[mover_at].src = static_cast<int32_t>(page);
    if (in) {
      p.remap[page] = used ? -1 : -2;
      if (p.out_ref_counts != p.ref_counts) p.out_ref_counts[page] = p.ref_counts[page];
    }
    holes += hole_sum;
    movers += mover_sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPagePlanThreads) {
    const int32_t from = p.moves[i].src, to = p.moves[i].dst;
    p.moves[i].ntok = p.block_size;
    p.remap[from] = to;
    p.out_ref_counts[to] = p.ref_counts[from];
    p.out_ref_counts[from] = 0;
  }
  if (threadIdx.x == 0) {
    *p.num_moves = movers;
    *p.out_num_live = live;
  }
}

__global__ void __launch_bounds__(256) page_remap_kernel(const PageCompactParams p) {
  allow_dependent_launch();
  grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= p.entries) return;
  int32_t page = p.block_tables[i];
  if (page >= 0) {
    if (page < p.num_pages) {
      const int32_t to = p.remap[page];
      if (to >= 0) page = to;
      else if (to == -2) raise_error(NKV_DEVERR_PAGES);  // a table names a free page
    } else {
      raise_error(NKV_DEVERR_PAGES);
    }
  }
  p.out_block_tables[i] = page;
}

}  // namespace nkv
