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
// (walked step by step, 256 trees of 255 nodes, 256 of width 24, take 45 us; so 7.2).  A node whose way ends elsewhere than in node 0 (a parent that is
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
  uint32_t wide_bits, of_block, blocks;      // a strip has up to 2^wide_bits units; strips of a block; blocks
};
constexpr int kMaxPools = 64;
struct Move {
  Pool pool[kMaxPools];
  const int32_t *block_table, *offset, *path, *counts;
  int64_t blocks_per_seq, block_size, num_blocks;
  int pools, T;
};

// A block moves some strips of one pool (up to 32 units of the rows of one head of one layer), for one sequence, 64 rows at a time: all rows are
// loaded, and when the whole block has them, stored.  The path ascends, so a row's place lies below all rows that are loaded later.
// A warp's lanes are 2^wide_bits units of each of 32 >> wide_bits rows: rows of 4-bit codes and scales are 64 and 8 bytes, and lie together by
// head.  A thread has eight rows (or two or four of each of four or two strips, where a row is one unit or two).
// (96 paths of 24 rows in 16 layers of 4-bit pages: 27 us; 51 with a thread to a column of all rows, 36 with heads on neighbouring lanes.)
constexpr int kMoveThreads = 256, kMoveRows = 64, kOfThread = 8;

__device__ __forceinline__ uint4 load_unit(const uint8_t* p, uint32_t unit) {
  uint4 v = make_uint4(0, 0, 0, 0);
  switch (unit) {
    case 16: v = *reinterpret_cast<const uint4*>(p); break;
    case 8: {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      v.x = w.x, v.y = w.y;
      break;
    }
    case 4: v.x = *reinterpret_cast<const uint32_t*>(p); break;
    case 2: v.x = *reinterpret_cast<const uint16_t*>(p); break;
    default: v.x = *p; break;
  }
  return v;
}
__device__ __forceinline__ void store_unit(uint8_t* p, const uint4& v, uint32_t unit) {
  switch (unit) {
    case 16: *reinterpret_cast<uint4*>(p) = v; break;
    case 8: *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y); break;
    case 4: *reinterpret_cast<uint32_t*>(p) = v.x; break;
    case 2: *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(v.x); break;
    default: *p = static_cast<uint8_t>(v.x); break;
  }
}

__global__ void __launch_bounds__(kMoveThreads) commit_drafts_kernel(const __grid_constant__ Move a) {
  __shared__ int64_t from[kMoveRows], to[kMoveRows];   // page * block_size and slot in the low half, the page in the high one; -1: nothing to move
  __shared__ int end;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int b = blockIdx.y;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  const int32_t* path = a.path + static_cast<int64_t>(b) * a.T;
  const int64_t offset = a.offset[b];
  const int count = min(max(a.counts[b], 0), a.T);
  // page (or -1) and slot of a position below 2^32
  auto place = [&](int64_t pos, int64_t& page, int& slot) {
    const uint32_t at = static_cast<uint32_t>(pos), blk = at / static_cast<uint32_t>(a.block_size);
    page = pos >= 0 && blk < a.blocks_per_seq ? table[blk] : -1;
    if (page >= a.num_blocks) page = -1;
    slot = static_cast<int>(at - blk * static_cast<uint32_t>(a.block_size));
  };
  uint32_t block = blockIdx.x;
  int k = 0;
  for (; k + 1 < a.pools && block >= a.pool[k].blocks; ++k) block -= a.pool[k].blocks;
  const Pool& pool = a.pool[k];
  const uint32_t of_row = pool.row_bytes / pool.unit, of_head = (of_row + 31) / 32;   // units of a row; strips of a head
  const uint32_t all_strips = pool.layers * pool.outer * of_head, bits = pool.wide_bits, more = bits > 2 ? bits - 2 : 0;   // 2^more warps share a strip
  const uint32_t strip0 = block * pool.of_block + (bits >= 2 ? warp >> more : warp * (4u >> bits));
  const uint32_t passes = bits >= 2 ? 8u : 2u << bits, row0 = lane >> bits, rows = 32u >> bits;
  const int64_t head_bytes = a.block_size * pool.row_bytes, page_bytes = pool.outer * head_bytes;
  auto strip_at = [&](uint32_t strip) -> uint8_t* {   // the lane's unit of its row 0; null: none
    const uint32_t head = strip / of_head, unit = (strip - head * of_head) * 32 + (lane & ((1u << bits) - 1)), layer = head / pool.outer;
    return strip < all_strips && unit < of_row ? pool.p + layer * pool.layer_bytes + (head - layer * pool.outer) * head_bytes + unit * pool.unit : nullptr;
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
      from[threadIdx.x] = f >= 0 && t >= 0 ? f << 32 | sf : -1;
      to[threadIdx.x] = t << 32 | st;
    }
    __syncthreads();
    const int n = min(end - i0, kMoveRows);
    uint4 v[kOfThread];
    uint32_t moved = 0;
    uint8_t* p = nullptr;   // row 0 of the strip
    auto row_of = [&](int x) { return (((x & (passes - 1)) << more) + (warp & ((1u << more) - 1))) * rows + row0; };
    auto at = [&](int64_t place) { return p + (place >> 32) * page_bytes + static_cast<uint32_t>(place) * static_cast<int64_t>(pool.row_bytes); };
#pragma unroll
    for (int x = 0; x < kOfThread; ++x) {
      if ((x & (passes - 1)) == 0) p = strip_at(strip0 + x / passes);
      const int i = row_of(x);
      if (p && i < n && from[i] >= 0) v[x] = load_unit(at(from[i]), pool.unit), moved |= 1u << x;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kOfThread; ++x) {
      if (passes < kOfThread && (x & (passes - 1)) == 0) p = strip_at(strip0 + x / passes);
      if (moved >> x & 1u) store_unit(at(to[row_of(x)]), v[x], pool.unit);
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
  // A row that lies in two pools would be moved twice.  (Pools mostly ascend or descend: then each lies beside all before it.)
  const auto begin = [](const oasr_b200_draft_pool& p) { return static_cast<unsigned __int128>(reinterpret_cast<uintptr_t>(p.data)); };
  const auto end = [&](const oasr_b200_draft_pool& p) {
    return begin(p) + static_cast<unsigned __int128>(p.layers * p.outer * p.row_bytes) * static_cast<uint64_t>(num_blocks * block_size);
  };
  unsigned __int128 lowest = begin(pools[0]), highest = end(pools[0]);
  for (int64_t i = 1; i < num_pools; ++i) {
    const unsigned __int128 b0 = begin(pools[i]), b1 = end(pools[i]);
    if (b0 < highest && lowest < b1)
      for (int64_t k = 0; k < i; ++k)
        OB_REQUIRE(b0 >= end(pools[k]) || begin(pools[k]) >= b1, OASR_ERR_INVALID, "commit_drafts: pools %lld and %lld share memory", (long long)k, (long long)i);
    lowest = b0 < lowest ? b0 : lowest, highest = b1 > highest ? b1 : highest;
  }
  for (int64_t done = 0; done < num_pools; done += drafts::kMaxPools) {
    drafts::Move a{};
    a.block_table = block_table, a.offset = offset, a.path = path, a.counts = counts;
    a.blocks_per_seq = blocks_per_seq, a.block_size = block_size, a.num_blocks = num_blocks, a.T = static_cast<int>(T);
    int64_t all = 0;
    for (; a.pools < drafts::kMaxPools && done + a.pools < num_pools; ++a.pools) {
      const oasr_b200_draft_pool& p = pools[done + a.pools];
      const uint64_t bits = reinterpret_cast<uintptr_t>(p.data) | static_cast<uint64_t>(p.row_bytes) | 16u;
      const int64_t unit = static_cast<int64_t>(bits & (~bits + 1));   // (a layer is a whole number of rows)
      const int64_t of_row = p.row_bytes / unit, strips = p.layers * p.outer * ((of_row + 31) / 32);
      uint32_t wide_bits = 0;
      while (wide_bits < 5 && (1 << wide_bits) < of_row) ++wide_bits;
      const int64_t of_block = 32 >> wide_bits, blocks = (strips + of_block - 1) / of_block;
      a.pool[a.pools] = drafts::Pool{static_cast<uint8_t*>(p.data), num_blocks * p.outer * block_size * p.row_bytes, static_cast<uint32_t>(p.layers),
                                     static_cast<uint32_t>(p.outer), static_cast<uint32_t>(p.row_bytes), static_cast<uint32_t>(unit), wide_bits,
                                     static_cast<uint32_t>(of_block), static_cast<uint32_t>(blocks)};
      all += blocks;
    }
    launch_pdl(drafts::commit_drafts_kernel, dim3(static_cast<unsigned>(all), static_cast<unsigned>(B)), dim3(drafts::kMoveThreads), 0,
               static_cast<cudaStream_t>(stream), a);
    const int rc = check_launch("commit_drafts launch");
    if (rc != OASR_OK) return rc;
  }
  return OASR_OK;
}
