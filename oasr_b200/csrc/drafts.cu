// Trees of drafted tokens: who sees whom, and the accepted tokens' rows moved together in the pages.
#include <cmath>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ob {
namespace drafts {
namespace {

constexpr int kMaxNodes = 1024;

// A block takes eight words (256 columns) of a tree's masks, a thread up to four nodes of it.  Node i knows the nodes between itself and its
// `up` (the parent at first); in a round it takes over what `up` knows and goes on to up's `up`, so a way of n steps takes log2(n) rounds
// (walked step by step, 256 trees of 255 nodes, 256 of width 24, take 45 us).  A node whose way ends elsewhere than in node 0 (a parent that is
// not an earlier node) is padding: no bits, depth -1.
constexpr int kTreeWords = 8, kTreeThreads = 256;

template <int kNodes>   // of a thread
__global__ void __launch_bounds__(kTreeThreads) draft_tree_kernel(uint32_t* mask, int32_t* depth, const int32_t* parents, const int T, const int words) {
  __shared__ uint4 bits[kNodes * kTreeThreads][2];
  __shared__ int2 way[kNodes * kTreeThreads];   // up, steps to it
  const int b = blockIdx.x, w0 = blockIdx.y * kTreeWords;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  uint32_t mine[kNodes][kTreeWords];
  int2 at[kNodes];
  bool open = false;
#pragma unroll
  for (int x = 0; x < kNodes; ++x) {
    const int i = x * kTreeThreads + threadIdx.x;
    at[x] = make_int2(0, 0);
    if (i > 0 && i < T) {
      const int p = parents[static_cast<int64_t>(b) * T + i];
      at[x] = make_int2(p >= 0 && p < i ? p : -1, 1);
    }
    open |= at[x].x > 0;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) mine[x][w] = i >> 5 == w0 + w ? 1u << (i & 31) : 0u;
  }
  while (__syncthreads_or(open)) {   // (also: nobody reads what is written next)
#pragma unroll
    for (int x = 0; x < kNodes; ++x) {
      const int i = x * kTreeThreads + threadIdx.x;
      bits[i][0] = make_uint4(mine[x][0], mine[x][1], mine[x][2], mine[x][3]);
      bits[i][1] = make_uint4(mine[x][4], mine[x][5], mine[x][6], mine[x][7]);
      way[i] = at[x];
    }
    __syncthreads();
    open = false;
#pragma unroll
    for (int x = 0; x < kNodes; ++x) {
      const int up = at[x].x;
      if (up <= 0) continue;
      const uint4 lo = bits[up][0], hi = bits[up][1];
      const int2 next = way[up];
      mine[x][0] |= lo.x, mine[x][1] |= lo.y, mine[x][2] |= lo.z, mine[x][3] |= lo.w;
      mine[x][4] |= hi.x, mine[x][5] |= hi.y, mine[x][6] |= hi.z, mine[x][7] |= hi.w;
      at[x] = make_int2(next.x, at[x].y + next.y);
      open |= next.x > 0;
    }
  }
#pragma unroll
  for (int x = 0; x < kNodes; ++x) {
    const int i = x * kTreeThreads + threadIdx.x;
    if (i >= T) continue;
    const bool inside = at[x].x == 0;
    const int64_t row = static_cast<int64_t>(b) * T + i;
    if (w0 == 0) {
      mine[x][0] |= 1u;
      depth[row] = inside ? at[x].y : -1;
    }
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w)
      if (w0 + w < words) mask[row * words + w0 + w] = inside ? mine[x][w] : 0u;
  }
}

// One pool: `layers` of them, each (blocks, outer, block_size) rows of row_bytes.
struct Pool {
  uint8_t* p;
  int64_t layer_bytes;
  uint32_t layers, outer, row_bytes, unit;   // unit: bytes that a thread moves of a row (1 to 16)
  uint32_t blocks;                           // that move its columns
};
constexpr int kMaxPools = 64;
struct Move {
  Pool pool[kMaxPools];
  const int32_t *block_table, *offset, *path, *counts;
  int64_t blocks_per_seq, block_size, num_blocks;
  int pools, T;
};

// A column is `unit` bytes of a row of one head of one layer.  A block moves 32 columns (the lanes) of one sequence, 64 rows at a time, eight to a
// warp: all are loaded, and when the whole block has them, stored.  The path ascends, so a row's place lies below all rows that are loaded later.
// (A thread with its column's rows all to itself, eight at a time, left 96 paths of 24 rows in 16 layers of 4-bit pages at 51 us.)
constexpr int kMoveThreads = 256, kMoveRows = 64, kOfThread = kMoveRows * 32 / kMoveThreads;

template <typename U>
__device__ __forceinline__ void move_rows(uint8_t* base, const int64_t* from, const int64_t* to, const int n, const int64_t stride) {
  U v[kOfThread];
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int x = 0; x < kOfThread; ++x) {
    const int i = x * (kMoveThreads / 32) + warp;
    if (base && i < n && from[i] >= 0) v[x] = *reinterpret_cast<const U*>(base + from[i] * stride);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kOfThread; ++x) {
    const int i = x * (kMoveThreads / 32) + warp;
    if (base && i < n && from[i] >= 0) *reinterpret_cast<U*>(base + to[i] * stride) = v[x];
  }
}

__global__ void __launch_bounds__(kMoveThreads) commit_drafts_kernel(const __grid_constant__ Move a) {
  __shared__ int64_t from[kMoveRows], to[kMoveRows];   // in rows of one head; -1: nothing to move
  __shared__ int end;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  const int32_t* path = a.path + static_cast<int64_t>(b) * a.T;
  const int64_t offset = a.offset[b];
  const int count = min(max(a.counts[b], 0), a.T);
  // a block's columns are of one pool
  uint32_t block = blockIdx.x;
  int k = 0;
  for (; k + 1 < a.pools && block >= a.pool[k].blocks; ++k) block -= a.pool[k].blocks;
  const Pool& pool = a.pool[k];
  const uint32_t of_row = pool.row_bytes / pool.unit, column = block * 32 + lane, rest = column / of_row;
  const uint32_t o = rest % pool.outer, layer = rest / pool.outer;
  uint8_t* const base = layer < pool.layers
                            ? pool.p + layer * pool.layer_bytes + (static_cast<int64_t>(o) * a.block_size * pool.row_bytes + (column - rest * of_row) * pool.unit)
                            : nullptr;
  // page (or -1) and slot of a position below 2^32
  auto place = [&](int64_t pos, int64_t& page, int& slot) {
    const uint32_t at = static_cast<uint32_t>(pos), blk = at / static_cast<uint32_t>(a.block_size);
    page = pos >= 0 && blk < a.blocks_per_seq ? table[blk] : -1;
    if (page >= a.num_blocks) page = -1;
    slot = static_cast<int>(at - blk * static_cast<uint32_t>(a.block_size));
  };
  for (int i0 = 0; i0 < count; i0 += kMoveRows) {
    if (threadIdx.x == 0) end = count;
    __syncthreads();   // (also: the rows before are stored)
    if (threadIdx.x < kMoveRows) {
      const int i = i0 + static_cast<int>(threadIdx.x), p = i < count ? path[i] : -1;
      if (i < count && p <= (i > 0 ? path[i - 1] : -1)) atomicMin(&end, i);   // an entry that does not ascend ends the path
      int64_t f = -1, t = -1;
      int sf = 0, st = 0;
      if (p >= 0 && p != i) place(offset + p, f, sf), place(offset + i, t, st);
      const int64_t page_rows = pool.outer * a.block_size;
      from[threadIdx.x] = f >= 0 && t >= 0 ? f * page_rows + sf : -1;
      to[threadIdx.x] = t * page_rows + st;
    }
    __syncthreads();
    const int n = min(end - i0, kMoveRows);
    switch (pool.unit) {
      case 16: move_rows<uint4>(base, from, to, n, pool.row_bytes); break;
      case 8: move_rows<uint2>(base, from, to, n, pool.row_bytes); break;
      case 4: move_rows<uint32_t>(base, from, to, n, pool.row_bytes); break;
      case 2: move_rows<uint16_t>(base, from, to, n, pool.row_bytes); break;
      default: move_rows<uint8_t>(base, from, to, n, pool.row_bytes); break;
    }
    if (n < kMoveRows) break;
  }
}

}  // namespace
}  // namespace drafts
}  // namespace ob

extern "C" int oasr_b200_draft_tree(uint32_t* mask, int32_t* depth, const int32_t* parents, int64_t B, int64_t T, int64_t words, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && T >= 0, OASR_ERR_INVALID, "draft_tree: bad shape");
  OB_REQUIRE(T <= drafts::kMaxNodes, OASR_ERR_UNSUPPORTED, "draft_tree: trees of up to %d nodes (got %lld)", drafts::kMaxNodes, (long long)T);
  OB_REQUIRE(B <= 0x7fffffff && words == (T + 31) / 32, OASR_ERR_INVALID, "draft_tree: batch too large, or not a word for each 32 nodes");
  if (B == 0 || T == 0) return OASR_OK;
  OB_REQUIRE(mask && depth && parents, OASR_ERR_INVALID, "draft_tree: null pointer argument");
  OB_REQUIRE(is_aligned(mask, 4) && is_aligned(depth, 4) && is_aligned(parents, 4), OASR_ERR_ALIGN, "draft_tree: operands must be aligned to their elements");
  const dim3 grid(static_cast<unsigned>(B), static_cast<unsigned>((words + drafts::kTreeWords - 1) / drafts::kTreeWords));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T <= drafts::kTreeThreads)
    launch_pdl(drafts::draft_tree_kernel<1>, grid, dim3(drafts::kTreeThreads), 0, st, mask, depth, parents, static_cast<int>(T), static_cast<int>(words));
  else
    launch_pdl(drafts::draft_tree_kernel<drafts::kMaxNodes / drafts::kTreeThreads>, grid, dim3(drafts::kTreeThreads), 0, st, mask, depth, parents,
               static_cast<int>(T), static_cast<int>(words));
  return check_launch("draft_tree launch");
}

extern "C" int oasr_b200_commit_drafts(const oasr_b200_draft_pool* pools, int64_t num_pools, const int32_t* block_table, const int32_t* offset,
                                       const int32_t* path, const int32_t* counts, int64_t B, int64_t T, int64_t blocks_per_seq, int64_t block_size,
                                       int64_t num_blocks, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && T >= 0 && num_pools >= 0 && blocks_per_seq >= 0 && block_size > 0 && num_blocks > 0, OASR_ERR_INVALID, "commit_drafts: bad shape");
  OB_REQUIRE(B <= 65535 && T <= 0x7fffff && num_blocks <= 0x7fffffff && block_size <= 0x7fffffff, OASR_ERR_INVALID, "commit_drafts: batch, tree or pool too large");
  if (B == 0 || T == 0 || num_pools == 0 || blocks_per_seq == 0) return OASR_OK;
  OB_REQUIRE(pools && block_table && offset && path && counts, OASR_ERR_INVALID, "commit_drafts: null pointer argument");
  OB_REQUIRE(is_aligned(block_table, 4) && is_aligned(offset, 4) && is_aligned(path, 4) && is_aligned(counts, 4), OASR_ERR_ALIGN,
             "commit_drafts: operands must be aligned to their elements");
  for (int64_t i = 0; i < num_pools; ++i)
    OB_REQUIRE(pools[i].data && pools[i].layers > 0 && pools[i].outer > 0 && pools[i].row_bytes > 0 && pools[i].layers <= 0x7fff &&
                   pools[i].outer <= 0xffff && pools[i].row_bytes <= 0xffffff && pools[i].layers * pools[i].outer * pools[i].row_bytes <= 0x1ffffff,
               OASR_ERR_INVALID, "commit_drafts: bad pool, or rows too large");
  for (int64_t done = 0; done < num_pools; done += drafts::kMaxPools) {
    drafts::Move a{};
    a.block_table = block_table, a.offset = offset, a.path = path, a.counts = counts;
    a.blocks_per_seq = blocks_per_seq, a.block_size = block_size, a.num_blocks = num_blocks, a.T = static_cast<int>(T);
    int64_t all = 0;
    for (; a.pools < drafts::kMaxPools && done + a.pools < num_pools; ++a.pools) {
      const oasr_b200_draft_pool& p = pools[done + a.pools];
      const uint64_t bits = reinterpret_cast<uintptr_t>(p.data) | static_cast<uint64_t>(p.row_bytes) | 16u;
      const int64_t unit = static_cast<int64_t>(bits & (~bits + 1));   // (a layer is a whole number of rows)
      const int64_t blocks = (p.layers * p.outer * (p.row_bytes / unit) + 31) / 32;
      a.pool[a.pools] = drafts::Pool{static_cast<uint8_t*>(p.data), num_blocks * p.outer * block_size * p.row_bytes, static_cast<uint32_t>(p.layers),
                                     static_cast<uint32_t>(p.outer), static_cast<uint32_t>(p.row_bytes), static_cast<uint32_t>(unit), static_cast<uint32_t>(blocks)};
      all += blocks;
    }
    launch_pdl(drafts::commit_drafts_kernel, dim3(static_cast<unsigned>(all), static_cast<unsigned>(B)), dim3(drafts::kMoveThreads), 0,
               static_cast<cudaStream_t>(stream), a);
    const int rc = check_launch("commit_drafts launch");
    if (rc != OASR_OK) return rc;
  }
  return OASR_OK;
}
