// What the kernels of attention over 16-bit pages with a tree of drafted tokens share.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace ob {
namespace fmha_tree {

struct Args {
  void* out;
  const void *q, *k, *v;
  const int32_t *block_table, *seqlens, *seqstarts, *q_lens;
  const uint32_t* mask;          // null: row t sees the drafted keys 0 .. t
  float* parts;                  // null, or the partial results of `splits` blocks a group
  int64_t qs_b, qs_h, qs_t, os_b, os_h, os_t;
  int64_t mask_b;                // words from one sequence's mask to the next one's; 0: one for all
  int64_t blocks_per_seq, block_size, num_blocks;
  int B, H, Hkv, Tq, mask_words, splits;
  int longest_first;             // sequences in the order of their lengths
  float scale_log2;
};

constexpr int kMostOfCluster = 8;   // blocks of the form for many rows that share a cache as a cluster; more leave partial results

constexpr float kEmpty = -3.4028235e38f;   // below every score; a row's maximum before its first key

// A weight is 2^((score - m) unit + kBelow), m a maximum of the row's scores that moves when one passes it by kLag (in powers of two).  The difference
// comes first: score unit - m unit as one multiply-add is off by many powers of two where scores are large.  (It takes 0.5 us of 18.1 for 37 trees of 21;
// choosing between the two by the row's maximum 1.7.)  In fp16 weights lie up to 2^15, are rounded by half a step down to 2^-21 of the maximum, and
// vanish below 2^-32 of it.  (Relative to the maximum itself, 2^-14 and 2^-25: many keys of little weight behind one of much were lost.)  bf16 has the
// exponents of fp32.
template <typename T>
constexpr float kBelow = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr float kLag = 8.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2(e) times the size of the scale (the queries have its sign); zero would make a number of -inf
__device__ __forceinline__ float unit_of(const Args& a) { return fmaxf(fabsf(a.scale_log2), 1.2e-38f); }

// A sequence as every block of it sees it.
struct Sequence {
  int start, end, prefix, live;   // keys [start, end); the first drafted key (may be below zero); rows that count

  __device__ __forceinline__ Sequence(const Args& a, int b) {
    const int len = max(a.seqlens[b], 0), capacity = static_cast<int>(a.blocks_per_seq * a.block_size);
    live = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
    start = a.seqstarts ? max(a.seqstarts[b], 0) : 0;
    end = min(len, capacity);
    prefix = len - live;
  }
};

// Whether row t sees drafted key u (u >= 0)
__device__ __forceinline__ bool sees(const Args& a, const uint32_t* words, int t, int u, int live) {
  if (u >= live) return false;
  if (words == nullptr) return u <= t;
  return u < a.mask_words * 32 && (words[u >> 5] >> (u & 31) & 1u);
}
__device__ __forceinline__ const uint32_t* mask_row(const Args& a, int b, int t) {
  return a.mask ? a.mask + b * a.mask_b + static_cast<int64_t>(t) * a.mask_words : nullptr;
}

// Partial results of one (split, group, row block of `rows` rows): maxima, sums and outputs; rows x (maximum, sum), then rows x D of output, or in the
// form for many rows the maxima, the sums, then D x rows of output.
template <int D>
__host__ __device__ constexpr int64_t part_floats(int rows) { return static_cast<int64_t>(rows) * (D + 2); }

// The form for many rows (fmha_tree_wide.cu): tensor memory, 128 or 256 rows a block.
int run_wide(const Args& a, int head_dim, int dtype, int block_rows, int64_t groups, int row_blocks, cudaStream_t s);

}  // namespace fmha_tree
}  // namespace ob
