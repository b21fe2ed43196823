// Trees of drafted tokens: who sees whom, and the accepted tokens' rows moved together in the pages.
#include <cmath>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ob {
namespace drafts {
namespace {

constexpr int kMaxNodes = 1024;

// A warp per node, its mask's words in the lanes: the way to node 0 is walked from parent to parent in shared memory.  A node
// whose way ends elsewhere (a parent that is not an earlier node) is padding: no bits, depth -1.
__global__ void __launch_bounds__(256) draft_tree_kernel(uint32_t* mask, int32_t* depth, const int32_t* parents, const int T, const int words) {
  __shared__ int32_t parent[kMaxNodes];
  const int lane = threadIdx.x & 31, b = blockIdx.x;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  for (int i = threadIdx.x; i < T; i += 256) parent[i] = parents[static_cast<int64_t>(b) * T + i];
  __syncthreads();
  for (int i = blockIdx.y * 8 + (threadIdx.x >> 5); i < T; i += gridDim.y * 8) {
    uint32_t bits = 0;
    int at = i, steps = 0;
    while (at > 0) {   // (parents lie before their children, so this ends)
      if (lane == at >> 5) bits |= 1u << (at & 31);
      const int p = parent[at];
      at = p < at ? p : -1;
      ++steps;
    }
    if (lane == 0 && at == 0) bits |= 1u;
    const bool inside = at == 0;
    const int64_t row = static_cast<int64_t>(b) * T + i;
    if (lane < words) mask[row * words + lane] = inside ? bits : 0u;
    if (lane == 0) depth[row] = inside ? steps : -1;
  }
}

// One pool: `layers` of them, each (blocks, outer, block_size) rows of row_bytes.
struct Pool {
  uint8_t* p;
  int64_t layer_bytes;
  int32_t layers, outer, row_bytes, unit;   // unit: bytes that a thread moves of a row (1 to 16)
};
constexpr int kMaxPools = 64;
struct Move {
  Pool pool[kMaxPools];
  const int32_t *block_table, *offset, *path, *counts;
  int64_t blocks_per_seq, block_size, num_blocks;
  int pools, T;
};

// A thread moves one column of one pool, `unit` bytes wide, of all rows of a sequence.  The path ascends, so row i's place was read before it
// is written: of eight rows at a time, all are loaded before the first is stored.
template <typename U>
__device__ __forceinline__ void move_column(uint8_t* base, const int64_t (&from)[8], const int64_t (&to)[8], const int n, const int64_t stride) {
  U v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n && from[i] >= 0 && to[i] >= 0) v[i] = *reinterpret_cast<const U*>(base + from[i] * stride);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n && from[i] >= 0 && to[i] >= 0) *reinterpret_cast<U*>(base + to[i] * stride) = v[i];
}

__global__ void __launch_bounds__(256) commit_drafts_kernel(const __grid_constant__ Move a) {
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int b = blockIdx.y;
  // the thread's column
  int64_t column = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  int k = 0;
  int64_t of_row = 0;
  for (; k < a.pools; ++k) {
    of_row = a.pool[k].row_bytes / a.pool[k].unit;
    const int64_t all = of_row * a.pool[k].outer * a.pool[k].layers;
    if (column < all) break;
    column -= all;
  }
  const bool active = k < a.pools;
  const Pool& pool = a.pool[active ? k : 0];
  const int64_t piece = column % of_row, rest = column / of_row;
  const int o = static_cast<int>(rest % pool.outer), layer = static_cast<int>(rest / pool.outer);
  // row (page, slot) lies at (page * outer + o) * block_size + slot rows of row_bytes
  uint8_t* const base = active ? pool.p + layer * pool.layer_bytes + static_cast<int64_t>(o) * a.block_size * pool.row_bytes + piece * pool.unit : nullptr;

  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  const int32_t* path = a.path + static_cast<int64_t>(b) * a.T;
  const int64_t offset = a.offset[b];
  const int count = min(max(a.counts[b], 0), a.T);
  auto row_of = [&](int64_t pos) -> int64_t {   // in rows of a pool's head `o`; -1: no such row
    if (pos < 0) return -1;
    const int64_t block = pos / a.block_size;
    if (block >= a.blocks_per_seq) return -1;
    const int32_t page = table[block];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.num_blocks)) return -1;
    return static_cast<int64_t>(page) * pool.outer * a.block_size + (pos - block * a.block_size);
  };
  int before = -1;
  for (int i0 = 0; i0 < count; i0 += 8) {
    int64_t from[8], to[8];
    int n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      from[i] = to[i] = -1;
      if (n == i && i0 + i < count) {
        const int p = path[i0 + i];
        if (p > before) {   // an entry that does not ascend ends the path
          n = i + 1;
          before = p;
          if (p != i0 + i) from[i] = row_of(offset + p), to[i] = row_of(offset + i0 + i);
        }
      }
    }
    if (active) {
      switch (pool.unit) {
        case 16: move_column<uint4>(base, from, to, n, pool.row_bytes); break;
        case 8: move_column<uint2>(base, from, to, n, pool.row_bytes); break;
        case 4: move_column<uint32_t>(base, from, to, n, pool.row_bytes); break;
        case 2: move_column<uint16_t>(base, from, to, n, pool.row_bytes); break;
        default: move_column<uint8_t>(base, from, to, n, pool.row_bytes); break;
      }
    }
    if (n < 8) break;
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
  // few sequences: a tree's nodes over several blocks
  const int64_t ways = (T + 7) / 8, spread = B >= sm_count() ? 1 : (2 * sm_count() + B - 1) / B;
  launch_pdl(drafts::draft_tree_kernel, dim3(static_cast<unsigned>(B), static_cast<unsigned>(ways < spread ? ways : spread)), dim3(256), 0,
             static_cast<cudaStream_t>(stream), mask, depth, parents, static_cast<int>(T), static_cast<int>(words));
  return check_launch("draft_tree launch");
}

extern "C" int oasr_b200_commit_drafts(const oasr_b200_draft_pool* pools, int64_t num_pools, const int32_t* block_table, const int32_t* offset,
                                       const int32_t* path, const int32_t* counts, int64_t B, int64_t T, int64_t blocks_per_seq, int64_t block_size,
                                       int64_t num_blocks, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && T >= 0 && num_pools >= 0 && blocks_per_seq >= 0 && block_size > 0 && num_blocks > 0, OASR_ERR_INVALID, "commit_drafts: bad shape");
  OB_REQUIRE(B <= 65535 && T <= 0x7fffff && num_blocks <= 0x7fffffff, OASR_ERR_INVALID, "commit_drafts: batch, tree or pool too large");
  if (B == 0 || T == 0 || num_pools == 0 || blocks_per_seq == 0) return OASR_OK;
  OB_REQUIRE(pools && block_table && offset && path && counts, OASR_ERR_INVALID, "commit_drafts: null pointer argument");
  OB_REQUIRE(is_aligned(block_table, 4) && is_aligned(offset, 4) && is_aligned(path, 4) && is_aligned(counts, 4), OASR_ERR_ALIGN,
             "commit_drafts: operands must be aligned to their elements");
  for (int64_t i = 0; i < num_pools; ++i)
    OB_REQUIRE(pools[i].data && pools[i].layers > 0 && pools[i].outer > 0 && pools[i].row_bytes > 0 && pools[i].layers <= 0x7fffffff &&
                   pools[i].outer <= 0x7fffffff && pools[i].row_bytes <= 0x7fffffff,
               OASR_ERR_INVALID, "commit_drafts: bad pool");
  for (int64_t done = 0; done < num_pools; done += drafts::kMaxPools) {
    drafts::Move a{};
    a.block_table = block_table, a.offset = offset, a.path = path, a.counts = counts;
    a.blocks_per_seq = blocks_per_seq, a.block_size = block_size, a.num_blocks = num_blocks, a.T = static_cast<int>(T);
    int64_t columns = 0;
    for (; a.pools < drafts::kMaxPools && done + a.pools < num_pools; ++a.pools) {
      const oasr_b200_draft_pool& p = pools[done + a.pools];
      const uint64_t bits = reinterpret_cast<uintptr_t>(p.data) | static_cast<uint64_t>(p.row_bytes) | 16u;
      const int unit = static_cast<int>(bits & (~bits + 1));   // (a layer is a whole number of rows)
      a.pool[a.pools] = drafts::Pool{static_cast<uint8_t*>(p.data), num_blocks * p.outer * block_size * p.row_bytes, static_cast<int32_t>(p.layers),
                                     static_cast<int32_t>(p.outer), static_cast<int32_t>(p.row_bytes), unit};
      columns += p.layers * p.outer * (p.row_bytes / unit);
    }
    OB_REQUIRE((columns + 255) / 256 <= 0x7fffffff, OASR_ERR_INVALID, "commit_drafts: too many rows for one call");
    launch_pdl(drafts::commit_drafts_kernel, dim3(static_cast<unsigned>((columns + 255) / 256), static_cast<unsigned>(B)), dim3(256), 0,
               static_cast<cudaStream_t>(stream), a);
    const int rc = check_launch("commit_drafts launch");
    if (rc != OASR_OK) return rc;
  }
  return OASR_OK;
}
