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
constexpr int kPageCopyBytes = 65536;  // bytes of one copy item

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
// nothing to copy. shared: full pages that a fork shares.
struct PageMove {
  int32_t src, dst, ntok, shared;
};

template <int N>
struct PageRegions {
  PageRegion r[N];
  int num;
  int64_t items_per_move;  // over all regions and lead indices
};

// ---------------------------------------------------------------- copy
// Tables and counts that follow a plan, updated by the kernel that copies its
// pages (they touch nothing that the copies touch).
struct PageTables {
  const int32_t* in;       // block tables
  int32_t* out;            // the same for a fork, may be for a compaction
  int64_t entries;         // compaction: rows * max_blocks; fork: forks * max_blocks; 0: none
  int max_blocks;
  int64_t num_pages;
  // fork: the rows' full pages are shared
  const int32_t* src_rows; // null: compaction
  const int32_t* dst_rows;
  int32_t* ref_counts;
  // compaction: where a page went
  const int32_t* remap;
};

__device__ __forceinline__ void page_share(const PageTables& t, const PageMove* moves, int64_t e) {
  const int i = static_cast<int>(e / t.max_blocks);
  const int j = static_cast<int>(e - static_cast<int64_t>(i) * t.max_blocks);
  if (j >= moves[i].shared) return;
  const int32_t page = t.in[static_cast<int64_t>(t.src_rows[i]) * t.max_blocks + j];
  if (page < 0 || page >= t.num_pages) {  // no page of the cache: the branch lacks it too
    raise_error(NKV_DEVERR_PAGES);
    return;
  }
  const int32_t held = atomicAdd(t.ref_counts + page, 1);
  if (held <= 0) {  // by nobody: flagged, the source's reference too
    raise_error(NKV_DEVERR_PAGES);
    atomicAdd(t.ref_counts + page, 1 - held);
  }
  t.out[static_cast<int64_t>(t.dst_rows[i]) * t.max_blocks + j] = page;
}

__device__ __forceinline__ void page_remap(const PageTables& t, int64_t e) {
  int32_t page = t.in[e];
  if (page >= 0) {
    const int32_t to = page < t.num_pages ? t.remap[page] : -2;
    if (to >= 0) page = to;
    else if (to == -2) raise_error(NKV_DEVERR_PAGES);  // a table names a free page, or none of the cache
  }
  t.out[e] = page;
}

// Bound by HBM: each move reads a page and writes one (a partial page that several
// branches get is read for each, partly from L2). A CTA takes items of 64 KB,
// every thread sixteen 16-byte loads and then their stores, so that a CTA has
// 64 KB in flight. (Bulk copies through shared memory measured the same or
// slower but for many forks: 21 pages of 28 layers 200 us each way, a pool of
// 512 pages 180 against 178; items of 32 KB: 101 instead of 92 us for 144 forks
// with partial pages, whose skipped items are twice as many.)
template <int N>
__global__ void __launch_bounds__(kPageCopyThreads)
page_copy_kernel(const __grid_constant__ PageRegions<N> rg, const PageMove* moves,
                 const int32_t* num_moves_dev, int num_moves, const PageTables tables) {
  constexpr int kVecs = kPageCopyBytes / 16 / kPageCopyThreads;
  allow_dependent_launch();
  grid_dependency_wait();
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kPageCopyThreads;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kPageCopyThreads + threadIdx.x; e < tables.entries;
       e += stride) {
    if (tables.src_rows != nullptr) page_share(tables, moves, e);
    else page_remap(tables, e);
  }
  if (rg.items_per_move == 0) return;
  const int n = num_moves_dev != nullptr ? min(*num_moves_dev, num_moves) : num_moves;
  // item (mv, rest) and the step of a whole grid, without a division per item
  int64_t mv = blockIdx.x / rg.items_per_move;
  int64_t rest = blockIdx.x - mv * rg.items_per_move;
  const int64_t step_mv = gridDim.x / rg.items_per_move;
  const int64_t step_rest = gridDim.x - step_mv * rg.items_per_move;
  for (; mv < n; mv += step_mv, rest += step_rest) {
    if (rest >= rg.items_per_move) {
      rest -= rg.items_per_move;
      if (++mv >= n) break;
    }
    const PageMove move = moves[mv];
    if (move.dst < 0 || move.ntok <= 0) continue;
    int lo = 0, hi = rg.num - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (rg.r[mid].first_item <= rest) lo = mid;
      else hi = mid - 1;
    }
    const PageRegion& r = rg.r[lo];
    const uint32_t in_region = static_cast<uint32_t>(rest - r.first_item);
    const uint32_t lead = in_region / static_cast<uint32_t>(r.items_per_page);
    const int64_t from = static_cast<int64_t>(in_region - lead * r.items_per_page) * kPageCopyBytes;
    const int64_t live = move.ntok * r.token_bytes;  // bytes of each segment that are copied
    const bool one_seg = r.seg_bytes == r.page_bytes;
    if (one_seg && from >= live) continue;
    int bytes = static_cast<int>(min(static_cast<int64_t>(kPageCopyBytes), r.page_bytes - from));
    const bool whole = live >= r.seg_bytes;
    const uint8_t* src = r.base + lead * r.lead_stride + move.src * r.page_bytes + from;
    uint8_t* dst = r.base + lead * r.lead_stride + move.dst * r.page_bytes + from;
    // Whole 16-byte units of the item that are copied; a segment's last, partial
    // unit (exponent bytes) goes byte by byte.
    if (one_seg && !whole) bytes = static_cast<int>(min(static_cast<int64_t>(bytes), live - from));
    const bool plain = (whole || one_seg) && bytes % 16 == 0;
    if (plain) {
      const int vecs = bytes / 16;
      uint4 v[kVecs];
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const int i = threadIdx.x + k * kPageCopyThreads;
        if (i < vecs) v[k] = __ldcs(reinterpret_cast<const uint4*>(src) + i);
      }
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const int i = threadIdx.x + k * kPageCopyThreads;
        if (i < vecs) __stcs(reinterpret_cast<uint4*>(dst) + i, v[k]);
      }
      continue;
    }
    const uint32_t seg = static_cast<uint32_t>(min(r.seg_bytes, static_cast<int64_t>(0x7fffffff)));
    for (int i = threadIdx.x; i < (bytes + 15) / 16; i += kPageCopyThreads) {
      const int64_t off = from + 16 * i;
      int64_t keep = live - (one_seg ? off : off % seg);
      if (keep >= 16) {
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
      } else {
        for (int64_t k = 0; k < keep; ++k) dst[16 * i + k] = src[16 * i + k];
      }
    }
  }
}

// ---------------------------------------------------------------- plan helpers
// Exclusive prefix sum of one value per warp over the CTA, the same for all
// lanes of a warp; `sum` gets the total.
__device__ __forceinline__ int warps_exclusive_sum(int v, int* warp_sums, int& sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // the previous round's sums are read
  if (lane == 0) warp_sums[warp] = v;
  __syncthreads();
  int x = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  sum = __shfl_sync(0xffffffffu, x, 31);
  return __shfl_sync(0xffffffffu, x, warp) - v;
}

// Which of a warp's next 512 pages are in use: bit `lane` of mask k is page
// base + 32 k + lane. Pages past the end count as neither (see `in`).
constexpr int kPageMasks = 16;
constexpr int kPagesPerRound = kPagePlanThreads * kPageMasks;
__device__ __forceinline__ void page_masks(const int32_t* ref_counts, int64_t base, int64_t num_pages,
                                           uint32_t (&used)[kPageMasks], uint32_t (&in)[kPageMasks]) {
  const int lane = threadIdx.x & 31;
  int32_t ref[kPageMasks];
#pragma unroll
  for (int k = 0; k < kPageMasks; ++k) {
    const int64_t page = base + 32 * k + lane;
    ref[k] = page < num_pages ? __ldcg(ref_counts + page) : 0;
  }
#pragma unroll
  for (int k = 0; k < kPageMasks; ++k) {
    used[k] = __ballot_sync(0xffffffffu, ref[k] > 0);
    in[k] = __ballot_sync(0xffffffffu, base + 32 * k + lane < num_pages);
  }
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
    p.moves[i] = PageMove{s, ok ? d : -1, 0x7fffffff, 0};  // every token
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
};

// A fork as the planning CTA holds it in shared memory; dst = -1: not made.
// src is the source row, then the page of its last, partial tokens. page is the
// new page, -1: none needed, -2: none to copy from, below: not found yet.
struct PageFork {
  int32_t src, dst, len, page;
};

// Decides which forks can be made, releases the targets' old pages and hands
// out a page to every fork with a partial one. (The full pages are shared by
// the kernel that copies.) One CTA: the phases depend on each other, and each
// is a round or two of loads.
__global__ void __launch_bounds__(kPagePlanThreads) page_fork_plan_kernel(const PageForkParams p) {
  extern __shared__ uint32_t maps[];  // rows read, written, written twice; then the forks
  __shared__ int warp_sums[kPagePlanThreads / 32];
  const int words = (p.num_rows + 31) / 32;
  uint32_t *read = maps, *written = maps + words, *twice = written + words;
  PageFork* forks = reinterpret_cast<PageFork*>(maps + (3 * words + 3) / 4 * 4);
  int32_t* tail = reinterpret_cast<int32_t*>(forks + p.n);  // a fork's partial page; by_rank later on
  for (int i = threadIdx.x; i < 3 * words; i += kPagePlanThreads) maps[i] = 0u;
  __syncthreads();
  allow_dependent_launch();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // ---- which forks can be made: rows in range, the target named once and no source
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const int32_t s = p.src_rows[i], d = p.dst_rows[i];
    forks[i] = PageFork{s, d, 0, -1};
    tail[i] = -1;
    if (s < 0 || s >= p.num_rows || d < 0 || d >= p.num_rows) continue;
    forks[i].len = p.context_lens[s];
    atomicOr(read + (s >> 5), 1u << (s & 31));
    if (atomicOr(written + (d >> 5), 1u << (d & 31)) >> (d & 31) & 1u)
      atomicOr(twice + (d >> 5), 1u << (d & 31));
  }
  __syncthreads();
  bool partial = false;
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const PageFork f = forks[i];
    const bool skip = f.src == -1 && f.dst == -1;  // padding
    bool ok = f.src >= 0 && f.src < p.num_rows && f.dst >= 0 && f.dst < p.num_rows;
    if (ok) ok = !bit_of(twice, f.dst) && !bit_of(read, f.dst);
    if (ok) ok = f.len >= 0 && f.len <= static_cast<int64_t>(p.max_blocks) * p.block_size;
    if (!ok && !skip) raise_error(NKV_DEVERR_PAGES);
    if (!ok) forks[i].dst = -1;
    else if (f.len % p.block_size != 0) partial = true;
  }
  const bool hands_out = __syncthreads_or(partial);  // pages, to forks with a partial one
  // ---- the targets' old pages are released: a warp per target, its entries in
  // rounds of 128 loads
  for (int i = warp; i < p.n; i += kPagePlanThreads / 32) {
    const int32_t d = forks[i].dst;
    if (d < 0) continue;
    int32_t* row = p.block_tables + static_cast<int64_t>(d) * p.max_blocks;
    for (int j0 = 0; j0 < p.max_blocks; j0 += 128) {
      int32_t old[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + 32 * k + lane;
        old[k] = j < p.max_blocks ? row[j] : -1;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (old[k] < 0) continue;
        if (old[k] < p.num_pages) page_release(p.ref_counts, old[k]);
        else raise_error(NKV_DEVERR_PAGES);
        row[j0 + 32 * k + lane] = -1;
      }
    }
  }
  __syncthreads();
  // ---- the sources' pages: one that nobody holds could be handed out below. A
  // full one is flagged and given the source's reference; of a partial one, or one
  // that is not there, no fork is made. (Where none is handed out the sharing finds
  // a full one.) Enough threads a fork for its table in one round, 32 at most.
  if (hands_out) {
    int shift = 0;
    while (shift < 5 && (1 << shift) < p.max_blocks) ++shift;
    for (int i = threadIdx.x >> shift; i < p.n; i += kPagePlanThreads >> shift) {
      const PageFork f = forks[i];
      if (f.dst < 0) continue;
      const int32_t* from = p.block_tables + static_cast<int64_t>(f.src) * p.max_blocks;
      const int full = f.len / p.block_size;
      const int used = full + (f.len > full * p.block_size ? 1 : 0);
      for (int j = threadIdx.x & ((1 << shift) - 1); j < used; j += 1 << shift) {
        const int32_t page = from[j];
        const bool there = page >= 0 && page < p.num_pages;
        const bool held = there && __ldcg(p.ref_counts + page) > 0;
        if (j == full) {
          if (held) tail[i] = page;
          else forks[i].page = -2;
        } else if (there && !held) {
          raise_error(NKV_DEVERR_PAGES);
          atomicMax(p.ref_counts + page, 1);
        }
      }
    }
    __syncthreads();
  }
  // ---- rank of every fork with a partial page among those, in order
  int want = 0;
  for (int base = 0; base < p.n; base += kPagePlanThreads) {
    const int i = base + threadIdx.x;
    int32_t page = i < p.n && forks[i].dst >= 0 ? forks[i].page : -2;
    const int32_t from = page != -2 ? tail[i] : -1;
    if (from >= 0) page = -3;
    const unsigned mask = __ballot_sync(0xffffffffu, page == -3);
    int sum;
    const int before = want + warps_exclusive_sum(__popc(mask), warp_sums, sum);
    if (page == -3) page -= before + __popc(mask & ((1u << lane) - 1u));
    if (i < p.n) {
      forks[i].src = from;
      forks[i].page = page;
    }
    want += sum;
  }
  __syncthreads();
  // ---- the lowest free pages: rank r's page to the fork of rank r. The forks
  // with a partial page, in order, start at `by_rank` (their indices).
  int32_t* by_rank = tail;
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads)
    if (forks[i].page <= -3) by_rank[-3 - forks[i].page] = i;
  int found = 0;
  for (int64_t base = 0; base < p.num_pages && found < want; base += kPagesPerRound) {
    uint32_t used[kPageMasks], in[kPageMasks];
    const int64_t first = base + warp * 32 * kPageMasks;
    page_masks(p.ref_counts, first, p.num_pages, used, in);
    int mine = 0;
#pragma unroll
    for (int k = 0; k < kPageMasks; ++k) mine += __popc(in[k] & ~used[k]);
    int sum;
    int rank = found + warps_exclusive_sum(mine, warp_sums, sum);
#pragma unroll
    for (int k = 0; k < kPageMasks; ++k) {
      const uint32_t free = in[k] & ~used[k];
      const int r = rank + __popc(free & ((1u << lane) - 1u));
      if ((free >> lane & 1u) && r < want) forks[by_rank[r]].page = static_cast<int32_t>(first + 32 * k + lane);
      rank += __popc(free);
    }
    found += sum;
  }
  __syncthreads();
  // ---- the plan
  for (int i = threadIdx.x; i < p.n; i += kPagePlanThreads) {
    const PageFork f = forks[i];
    PageMove m{0, -1, 0, 0};
    int32_t out = -2;
    if (f.dst >= 0) {
      const int full = f.len / p.block_size;
      const bool made = f.page >= -1;
      if (!made) {  // no page left, or none to copy: the target stays empty
        raise_error(NKV_DEVERR_PAGES);
      } else {
        out = f.page;
        m.shared = full;
        if (f.page >= 0) {
          p.ref_counts[f.page] = 1;
          p.block_tables[static_cast<int64_t>(f.dst) * p.max_blocks + full] = f.page;
          m.src = f.src;
          m.dst = f.page;
          m.ntok = f.len - full * p.block_size;
        }
      }
      p.context_lens[f.dst] = made ? f.len : 0;
    }
    p.moves[i] = m;
    p.out_pages[i] = out;
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

// ---------------------------------------------------------------- shared rows
struct PageSharedParams {
  const int32_t* rows;
  int32_t* out_rows;  // may be rows
  int n;
  const int32_t* block_tables;
  int max_blocks;
  int num_rows;
  const int32_t* lens;  // null: the pages are a row's first
  const int32_t* ref_counts;
  int64_t num_pages;
  int block_size;
  int window_blocks;
  int pages;
};

// A warp per named row: which of them may be rewritten in place.
__global__ void __launch_bounds__(32) page_shared_kernel(const PageSharedParams p) {
  const int i = blockIdx.x, lane = threadIdx.x;
  int32_t row = p.rows[i];
  if (row != -1 && (row < 0 || row >= p.num_rows)) {
    if (lane == 0) raise_error(NKV_DEVERR_PAGES);
    row = -1;
  }
  if (row >= 0) {
    const int first = p.lens != nullptr ? p.lens[row] / p.block_size - p.window_blocks : 0;
    bool shared = false;
    for (int j = max(first, 0) + lane; j < min(first + p.pages, p.max_blocks); j += 32) {
      const int32_t page = p.block_tables[static_cast<int64_t>(row) * p.max_blocks + j];
      if (page >= 0 && page < p.num_pages && p.ref_counts[page] > 1) shared = true;
    }
    if (__any_sync(0xffffffffu, shared)) {
      if (lane == 0) raise_error(NKV_DEVERR_PAGES);
      row = -1;
    }
  }
  if (lane == 0) p.out_rows[i] = row;
}

// ---------------------------------------------------------------- compact plan
struct PageCompactParams {
  const int32_t* ref_counts;
  int32_t* out_ref_counts;    // may be ref_counts
  int64_t num_pages;
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t used[kPageMasks], in[kPageMasks];
  const int64_t warp_first = warp * 32 * kPageMasks;
  // pages in use, and those of them below `bound`
  auto count = [&](int64_t bound) {
    int mine = 0;
    for (int64_t base = 0; base < min(p.num_pages, bound); base += kPagesPerRound) {
      page_masks(p.ref_counts, base + warp_first, min(p.num_pages, bound), used, in);
#pragma unroll
      for (int k = 0; k < kPageMasks; ++k) mine += __popc(used[k]);
    }
    int sum;
    warps_exclusive_sum(mine, warp_sums, sum);
    return sum;
  };
  const int live = count(p.num_pages);
  const int settled = count(live);  // already among the first `live`
  int before_round = 0;             // pages in use in the rounds before
  for (int64_t base = 0; base < p.num_pages; base += kPagesPerRound) {
    const int64_t first = base + warp_first;
    page_masks(p.ref_counts, first, p.num_pages, used, in);
    int mine = 0;
#pragma unroll
    for (int k = 0; k < kPageMasks; ++k) mine += __popc(used[k]);
    int sum;
    int before = before_round + warps_exclusive_sum(mine, warp_sums, sum);
    before_round += sum;
#pragma unroll
    for (int k = 0; k < kPageMasks; ++k) {
      const int64_t page = first + 32 * k + lane;
      const int below = before + __popc(used[k] & ((1u << lane) - 1u));  // in use before this page
      const bool is_used = used[k] >> lane & 1u;
      if (page < p.num_pages) {
        p.remap[page] = is_used ? -1 : -2;
        if (p.out_ref_counts != p.ref_counts) p.out_ref_counts[page] = p.ref_counts[page];
        if (!is_used && page < live) p.moves[page - below].dst = static_cast<int32_t>(page);
        if (is_used && page >= live) p.moves[below - settled].src = static_cast<int32_t>(page);
      }
      before += __popc(used[k]);
    }
  }
  __syncthreads();
  const int movers = live - settled;
  for (int i = threadIdx.x; i < movers; i += kPagePlanThreads) {
    const int32_t from = p.moves[i].src, to = p.moves[i].dst;
    p.moves[i].ntok = 0x7fffffff;  // every token
    p.remap[from] = to;
    p.out_ref_counts[to] = p.ref_counts[from];
    p.out_ref_counts[from] = 0;
  }
  if (threadIdx.x == 0) {
    *p.num_moves = movers;
    *p.out_num_live = live;
  }
}

}  // namespace nkv
