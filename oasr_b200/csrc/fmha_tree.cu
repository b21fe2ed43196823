// Attention of a tree of drafted tokens over 16-bit pages:
//
//   out[t] = sum_j softmax_j(scale q_t . k_j) v_j      over the keys  j < P  and  j = P + u  with bit u of mask[t],  start <= j < the table's end,
//
// P = len - q_len: the drafted rows' own keys are the last ones of the cache.  A single token is a tree of one node, a chunk a chain
// (no mask: bits 0 .. t).  A row that sees nothing, and rows t >= q_len, are zeros.
//
// Keys are the M side of both products (mma.m16n8k16: S^T = K Q^T, O^T = V^T P^T), the rows of all query heads that share a key
// head the N side, so that a single token wastes 7 of 8 columns and not 15 of 16 rows.  P takes one transpose in registers
// (movmatrix) between the two.  Weights are rounded to the type before they meet the values, as in the package's other attention; their
// sum, the maximum and the output are fp32.  What weights are relative to (m) moves only when a score passes it by far (kLag).
// Every warp walks its own tiles of 16 keys (always of one page) with its own maximum, sum and output, behind its own ring of tiles in
// shared memory that asynchronous copies fill; the warps of a block meet in shared memory at the end, and the blocks that share a long
// cache through partial results that a second, small kernel joins.
// Bound by memory where caches are long (64 chains of 5 over 500 to 6000 keys, 32 heads over 8 of 128: 140 us, 0.94 of the measured copy rate), by the start and end of
// blocks where they are short (37 trees of 21 over up to 1001 keys, 8 heads of 64: 18.1 us, floor 6.6; one token over 300 keys 4.4 us).  21 rows run as 32.
#include <cmath>

#include "common.cuh"
#include "fmha_tree.cuh"
#include "sm100_ptx.cuh"
#include "smem_limit.cuh"

namespace ob {
namespace fmha_tree {

int g_path = 0;   // tunable "fmha_tree_path": 0 by size, 1 the few-row form, 2 the form for many rows

namespace {

template <typename T>
struct Op;
template <>
struct Op<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static constexpr uint32_t kExponent = 0x7c00u;
};
template <>
struct Op<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static constexpr uint32_t kExponent = 0x7f80u;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void ldmatrix(uint32_t p, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t p, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() {   // all but the last N groups of copies have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kKeys = 16;

// A tile of 16 keys in the ring, K then V; the 16-byte pieces of row r lie at piece ^ (r & 7).  With four stages only three blocks of four warps of 64 dims
// have a place on an SM, with three stages four: 64 sequences of 4000 keys, 8 heads, 4 rows 99.6 and 81.7 us, 16 rows 110 and 87 (200 sequences of 2000
// keys, 4 heads: 65 and 68, 68 and 76).
template <int D>
struct Ring {
  static constexpr int kRow = 2 * D, kHalf = kKeys * kRow, kBytes = 2 * kHalf, kStages = 3;
  static __device__ __forceinline__ int at(int row, int piece) { return row * kRow + ((piece ^ (row & 7)) << 4); }
};

template <int D, int NT, int kWarps>
struct Merge {   // the warps' maxima, sums and outputs
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  float o[kWarps][8 * NT][D + 4];
};

template <int D, int NT, int kWarps>
struct Smem {
  static constexpr int kRings = kWarps * Ring<D>::kStages * Ring<D>::kBytes;
  static constexpr int kQ = NT == 4 ? 8 * NT * 2 * D : 0;   // 32 rows of queries are too many for registers
  static constexpr int kMerge = sizeof(Merge<D, NT, kWarps>);
  static constexpr int kBytes = (kRings > kMerge ? kRings : kMerge) + kQ;
};

// The n-th longest sequence, where blocks outnumber their places: a long one that starts last would end alone.  `lens` has room for B + 1.  Every block
// ranks all sequences against all: of 256 that takes 15 to 20 us, more than it gives, and beyond 64 they stay in their own order.
constexpr int kMostInOrder = 64;
template <int kThreads>
__device__ __forceinline__ int nth_longest(const Args& a, int n, int32_t* lens) {
  for (int i = threadIdx.x; i < a.B; i += kThreads) {
    const Sequence s(a, i);
    lens[i] = s.live > 0 ? max(s.end - s.start, 0) : 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.B; i += kThreads) {
    const int mine = lens[i];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < a.B; ++j) {
      const int other = lens[j];
      before += other > mine || (other == mine && j < i);
    }
    if (before == n) lens[a.B] = i;
  }
  __syncthreads();
  const int b = lens[a.B];
  __syncthreads();   // the room is used for other things
  return b;
}

template <typename T, int D, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, D == 128 ? 8 / kWarps : kWarps == 8 ? 2 : NT == 4 ? 3 : 4) fmha_tree_kernel(const Args a, const int row_blocks) {
  using R = Ring<D>;
  using S = Smem<D, NT, kWarps>;
  constexpr int NR = 8 * NT, KD = D / 16;   // rows; steps of 16 dims
  extern __shared__ __align__(128) uint8_t smem[];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int split = static_cast<int>(blockIdx.x) % a.splits, group = static_cast<int>(blockIdx.x) / a.splits;
  int at = group;
  const int rb = at % row_blocks;
  at /= row_blocks;
  const int hk = at % a.Hkv;
  int b = at / a.Hkv;
  if constexpr (kWarps == 4) {   // (eight: all blocks have a place)
    if (a.longest_first) b = nth_longest<kWarps * 32>(a, b, reinterpret_cast<int32_t*>(smem));
  }
  const int share = a.H / a.Hkv, rows = share * a.Tq, row0 = rb * NR;
  const Sequence seq(a, b);

  // tiles of this block: a run of the sequence's, dealt to the warps one by one
  const int tile0 = seq.start / kKeys, tile1 = row0 < seq.live * share ? max((seq.end + kKeys - 1) / kKeys, tile0) : tile0;
  const int per = (tile1 - tile0 + a.splits - 1) / a.splits;
  const int last = min(tile0 + (split + 1) * per, tile1);
  int tile = tile0 + split * per + warp;

  const int units = static_cast<int>(a.block_size) / kKeys, table_len = static_cast<int>(a.blocks_per_seq);
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  const int64_t row_bytes = static_cast<int64_t>(a.Hkv) * R::kRow;
  const uint8_t* const kp = static_cast<const uint8_t*>(a.k) + hk * R::kRow;
  const uint8_t* const vp = static_cast<const uint8_t*>(a.v) + hk * R::kRow;
  int ahead_block = tile / units, ahead_unit = tile - ahead_block * units;
  const int step_blocks = kWarps / units, step_units = kWarps - step_blocks * units;
  struct Place {
    int page, unit;
  };
  auto look_ahead = [&]() {   // the place of the next tile of the walk
    const Place p{ahead_block < table_len ? table[ahead_block] : -1, ahead_unit};
    ahead_block += step_blocks;
    ahead_unit += step_units;
    if (ahead_unit >= units) ahead_unit -= units, ++ahead_block;
    return p;
  };
  const uint32_t ring = ptx::smem_u32(smem) + warp * (R::kStages * R::kBytes);
  constexpr int kPieces = D / 8, kRowsPass = 32 / kPieces, kPasses = kKeys / kRowsPass;   // 16-byte pieces of a row; rows a pass of the warp
  const int copy_row = lane / kPieces, copy_piece = lane % kPieces;
  uint32_t there = 0;   // bit i: the tile i steps on has a page
  auto fetch = [&](const Place& p, uint32_t stage) {
    const bool known = static_cast<uint32_t>(p.page) < static_cast<uint32_t>(a.num_blocks);
    there |= (known ? 1u : 0u) << (R::kStages - 1);
    const int64_t first = (known ? static_cast<int64_t>(p.page) : 0) * a.block_size + p.unit * kKeys;   // (a tile without a page reads page 0 and is masked)
    const int64_t off = (first + copy_row) * row_bytes + copy_piece * 16;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const uint32_t dst = stage + R::at(copy_row + i * kRowsPass, copy_piece);
      copy16(dst, kp + off + i * kRowsPass * row_bytes);
      copy16(dst + R::kHalf, vp + off + i * kRowsPass * row_bytes);
    }
  };
#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) {
    there >>= 1;
    const Place p = look_ahead();
    if (tile + i * kWarps < last) fetch(p, ring + i * R::kBytes);
    commit_copies();
  }
  Place next = look_ahead();

  // ---- queries as the second operand (column g), with the sign of the scale
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const float unit = unit_of(a);
  auto q_row = [&](int r) { return static_cast<const T*>(a.q) + b * a.qs_b + (hk * share + r % share) * a.qs_h + static_cast<int64_t>(r / share) * a.qs_t; };
  uint32_t qf[NT == 4 ? 1 : NT][NT == 4 ? 1 : KD][2];
  const uint32_t q_smem = ptx::smem_u32(smem) + (S::kBytes - S::kQ);
  if constexpr (NT < 4) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + n * 8 + g;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(q_row(r < rows ? r : 0)) + t;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        qf[n][k][0] = r < rows ? q[k * 8] ^ flip : 0u;
        qf[n][k][1] = r < rows ? q[k * 8 + 4] ^ flip : 0u;
      }
    }
  } else {
    for (int i = threadIdx.x; i < NR * kPieces; i += kWarps * 32) {
      const int r = i / kPieces, p = i % kPieces;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row0 + r < rows) v = reinterpret_cast<const uint4*>(q_row(row0 + r))[p];
      *reinterpret_cast<uint4*>(smem + (S::kBytes - S::kQ) + R::at(r, p)) = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
    }
    __syncthreads();
  }

  float o[NT][KD][4] = {}, m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = kEmpty, l[n][0] = l[n][1] = 0.f;

  // addresses within a tile, as ldmatrix takes them: K rows are the operand's rows, V rows its columns
  const int k_row = lane & 15, k_piece = lane >> 4, v_row = (lane & 7) + (lane >> 4) * 8, v_piece = lane >> 3 & 1;
  uint32_t stage = ring, free_stage = ring + (R::kStages - 1) * R::kBytes;
  for (; tile < last; tile += kWarps) {
    copies_but<R::kStages - 2>();
    __syncwarp();                       // the tile is there for all lanes, and the last one is read by all
    there >>= 1;
    if (tile + (R::kStages - 1) * kWarps < last) fetch(next, free_stage);
    commit_copies();
    next = look_ahead();
    const int j0 = tile * kKeys;
    const bool known = there & 1u, whole = known && j0 >= seq.start && j0 + kKeys <= min(seq.prefix, seq.end);   // nothing to mask

    // ---- scores: keys g and g + 8, columns 2 t (+ 1)
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      uint32_t kf[4];
      ldmatrix(stage + R::at(k_row, 2 * k + k_piece), kf);
      if constexpr (NT < 4) {
#pragma unroll
        for (int n = 0; n < NT; ++n) Op<T>::mma(s[n], kf, qf[n][k][0], qf[n][k][1]);
      } else {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {   // two column tiles' operands: rows 8 n .. 8 n + 15, both halves of the step
          uint32_t qs[4];
          ldmatrix(q_smem + R::at(8 * n + (lane & 7) + (lane >> 4) * 8, 2 * k + (lane >> 3 & 1)), qs);
          Op<T>::mma(s[n], kf, qs[0], qs[1]);
          Op<T>::mma(s[n + 1], kf, qs[2], qs[3]);
        }
      }
    }
    bool odd = false;
    if (!whole) {
      // the rows' bits of the tile's 16 keys; all words are asked for before the first is looked at
      const int u = j0 - seq.prefix, w = u >> 5, off = u & 31;
      auto first = [](int n) { return n >= 16 ? 0xffffu : n <= 0 ? 0u : (1u << n) - 1; };
      const uint32_t in = known ? first(seq.end - j0) & ~first(seq.start - j0) : 0u, before = first(-u), live = first(seq.live - u) & ~before;
      uint32_t lo[NT][2], hi[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int tq = min((row0 + n * 8 + 2 * t + c) / share, a.Tq - 1);
          const uint32_t* words = mask_row(a, b, tq);
          lo[n][c] = words ? (w >= 0 && w < a.mask_words ? words[w] : 0u) : first(tq + 1 - u);
          hi[n][c] = words && w + 1 >= 0 && w + 1 < a.mask_words ? words[w + 1] : 0u;
        }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t tree = a.mask ? __funnelshift_r(lo[n][c], hi[n][c], off) : lo[n][c], seen = ((tree & live) | before) & in;
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (!(seen >> (g + 8 * x) & 1u)) s[n][2 * x + c] = -INFINITY;
        }
      // Values that no row sees are zeros, as a weight of zero does not undo a NaN.
#pragma unroll 1
      for (int i = 0; i < kPasses; ++i) {
        const int row = copy_row + i * kRowsPass, j = j0 + row;
        uint4* p = reinterpret_cast<uint4*>(smem + (stage - ptx::smem_u32(smem)) + R::kHalf + R::at(row, copy_piece));
        if (!known || j < seq.start || j >= seq.end) {
          *p = make_uint4(0, 0, 0, 0);
        } else if (j >= seq.prefix) {
          const uint4 v = *p;
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int x = 0; x < 4; ++x)
            odd |= (w[x] & Op<T>::kExponent) == Op<T>::kExponent || (w[x] >> 16 & Op<T>::kExponent) == Op<T>::kExponent;
        }
      }
      odd = __any_sync(0xffffffffu, odd);
      __syncwarp();
    }

    // ---- weights
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) raise |= (fmaxf(s[n][c], s[n][2 + c]) - m[n][c]) * unit > kLag;
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = fmaxf(s[n][c], s[n][2 + c]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          v = fmaxf(v, m[n][c]);
          const float f = ex2((m[n][c] - v) * unit);
          m[n][c] = v;
          l[n][c] *= f;
#pragma unroll
          for (int i = 0; i < KD; ++i) o[n][i][c] *= f, o[n][i][2 + c] *= f;
        }
    }
    uint32_t pf[NT][2];   // after the transpose the lane has keys 2 t (+ 1) and 2 t + 8 (+ 1) of row g
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float e0 = ex2(fmaf(s[n][2 * x] - m[n][0], unit, kBelow<T>)), e1 = ex2(fmaf(s[n][2 * x + 1] - m[n][1], unit, kBelow<T>));
        l[n][0] += e0;
        l[n][1] += e1;
        pf[n][x] = transpose8x8(Op<T>::pack(e0, e1));
      }
    }
    if (odd) {   // values of drafted keys that are not finite reach the rows that see them by hand, and no other
      T* const vs = reinterpret_cast<T*>(smem + (stage - ptx::smem_u32(smem)) + R::kHalf);
      for (int x = 0; x < kKeys; ++x) {
        const int u = j0 + x - seq.prefix;
        if (u < 0 || j0 + x >= seq.end || j0 + x < seq.start) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int tq = min((row0 + n * 8 + 2 * t + c) / share, a.Tq - 1);
            if (!sees(a, mask_row(a, b, tq), tq, u, seq.live)) continue;
#pragma unroll
            for (int i = 0; i < KD; ++i)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const float v = Elem<T>::to_f(vs[R::at(x, 2 * i + y) / 2 + g]);
                if (!(fabsf(v) < INFINITY)) o[n][i][2 * y + c] += v;
              }
          }
      }
      __syncwarp();
      for (int i = 0; i < kPasses; ++i) {
        if (j0 + copy_row + i * kRowsPass < seq.prefix) continue;
        T* p = vs + R::at(copy_row + i * kRowsPass, copy_piece) / 2;
        for (int x = 0; x < 8; ++x)
          if (!(fabsf(Elem<T>::to_f(p[x])) < INFINITY)) p[x] = Elem<T>::from_f(0.f);
      }
      __syncwarp();
    }
    // ---- output: dims 16 i + g (+ 8), rows 2 t (+ 1)
#pragma unroll
    for (int i = 0; i < KD; ++i) {
      uint32_t vf[4];
      ldmatrix_trans(stage + R::kHalf + R::at(v_row, 2 * i + v_piece), vf);
#pragma unroll
      for (int n = 0; n < NT; ++n) Op<T>::mma(o[n][i], vf, pf[n][0], pf[n][1]);
    }
    free_stage = stage;
    stage = stage == ring + (R::kStages - 1) * R::kBytes ? ring : stage + R::kBytes;
  }
  copies_but<0>();

  // ---- the warps meet
  using M = Merge<D, NT, kWarps>;
  M& sh = *reinterpret_cast<M*>(smem);
  __syncthreads();   // the rings are done with
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float v = l[n][c];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      const int r = n * 8 + 2 * t + c;
      if (g == 0) sh.m[warp][r] = m[n][c], sh.l[warp][r] = v;
#pragma unroll
      for (int i = 0; i < KD; ++i) sh.o[warp][r][16 * i + g] = o[n][i][c], sh.o[warp][r][16 * i + 8 + g] = o[n][i][2 + c];
    }
  __syncthreads();
  float* const part = a.parts ? a.parts + (static_cast<int64_t>(split) * (gridDim.x / a.splits) + group) * part_floats<D>(NR) : nullptr;
  for (int i = threadIdx.x; i < NR * (D / 8); i += kWarps * 32) {
    const int n = i / (D / 8), d = i % (D / 8) * 8, r = row0 + n;
    if (r >= rows) break;
    float top = sh.m[0][n], sum = 0.f, acc[8] = {};
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh.m[w][n]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2((sh.m[w][n] - top) * unit);
      const float4 a0 = *reinterpret_cast<const float4*>(&sh.o[w][n][d]), a1 = *reinterpret_cast<const float4*>(&sh.o[w][n][d + 4]);
      sum = fmaf(f, sh.l[w][n], sum);
      acc[0] = fmaf(f, a0.x, acc[0]), acc[1] = fmaf(f, a0.y, acc[1]), acc[2] = fmaf(f, a0.z, acc[2]), acc[3] = fmaf(f, a0.w, acc[3]);
      acc[4] = fmaf(f, a1.x, acc[4]), acc[5] = fmaf(f, a1.y, acc[5]), acc[6] = fmaf(f, a1.z, acc[6]), acc[7] = fmaf(f, a1.w, acc[7]);
    }
    if (part) {
      if (d == 0) part[2 * n] = top, part[2 * n + 1] = sum;
      float4* dst = reinterpret_cast<float4*>(part + 2 * NR + n * D + d);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      continue;
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // NaN stays
    const int tq = r / share;
    Pack<T> out;
#pragma unroll
    for (int x = 0; x < 8; ++x) out.v[x] = Elem<T>::from_f(tq < seq.live ? acc[x] * inv : 0.f);
    st128(static_cast<T*>(a.out) + b * a.os_b + (hk * share + r - tq * share) * a.os_h + static_cast<int64_t>(tq) * a.os_t + d, out);
  }
}

// Joins the partial results of a group's blocks: `kWays` warps a row, each with its share of the parts (one warp alone took 20 us for 74 of them).
template <typename T, int D, int kWays>
__global__ void __launch_bounds__(256) fmha_tree_join_kernel(const Args a, const int row_blocks, const int NR, const int groups) {
  constexpr int kRows = 8 / kWays, kV = D / 32;
  __shared__ float tops[8], sums[8], outs[8][D];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, way = warp % kWays;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kRows + warp / kWays, group = item / NR;
  const int n = static_cast<int>(item - group * NR), rb = static_cast<int>(group % row_blocks), at = static_cast<int>(group / row_blocks);
  const int hk = at % a.Hkv, b = at / a.Hkv, share = a.H / a.Hkv, r = rb * NR + n;
  const bool there = group < groups && r < share * a.Tq;
  const int64_t part = part_floats<D>(NR), step = part * groups;
  const float* src = a.parts + group * part;
  const float unit = unit_of(a);
  float top = kEmpty, sum = 0.f, acc[kV] = {};
  if (there) {
    for (int s = way + lane * kWays; s < a.splits; s += 32 * kWays) top = fmaxf(top, src[s * step + 2 * n]);
    top = warp_max(top);
#pragma unroll 4
    for (int s = way; s < a.splits; s += kWays) {
      const float* p = src + s * step;
      const float2 ml = *reinterpret_cast<const float2*>(p + 2 * n);
      const float f = ex2((ml.x - top) * unit);
      float v[kV];
#pragma unroll
      for (int x = 0; x < kV; ++x) v[x] = p[2 * NR + n * D + lane * kV + x];
      sum = fmaf(f, ml.y, sum);
#pragma unroll
      for (int x = 0; x < kV; ++x) acc[x] = fmaf(f, v[x], acc[x]);
    }
  }
  if constexpr (kWays > 1) {
    if (lane == 0) tops[warp] = top, sums[warp] = sum;
#pragma unroll
    for (int x = 0; x < kV; ++x) outs[warp][lane * kV + x] = acc[x];
    __syncthreads();
    if (way) return;
#pragma unroll
    for (int w = 1; w < kWays; ++w) top = fmaxf(top, tops[warp + w]);
    const float own = ex2((tops[warp] - top) * unit);
    sum *= own;
#pragma unroll
    for (int x = 0; x < kV; ++x) acc[x] *= own;
#pragma unroll
    for (int w = 1; w < kWays; ++w) {
      const float f = ex2((tops[warp + w] - top) * unit);
      sum = fmaf(f, sums[warp + w], sum);
#pragma unroll
      for (int x = 0; x < kV; ++x) acc[x] = fmaf(f, outs[warp + w][lane * kV + x], acc[x]);
    }
  }
  if (!there) return;
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // NaN stays
  const int tq = r / share, live = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
  T* out = static_cast<T*>(a.out) + b * a.os_b + (hk * share + r - tq * share) * a.os_h + static_cast<int64_t>(tq) * a.os_t + lane * kV;
#pragma unroll
  for (int x = 0; x < kV; ++x) out[x] = Elem<T>::from_f(tq < live ? acc[x] * inv : 0.f);
}

struct Plan {
  int rows, row_blocks, splits;   // rows of a block; blocks of rows of a (sequence, key head); blocks that share a cache
  int64_t groups;
  bool wide, parts;   // the form for many rows; blocks that share a cache leave partial results
  bool longest_first;
  int warps;   // of a block of the few-row form
};

// How a call is cut.  An SM holds 16 warps of the few-row form at 64 dims (12 in blocks of four with 32 rows, for their registers) and 8 at 128: eight to a
// block as long as all blocks fit, else four
// (37 trees of 21 over up to 1001 keys, 8 heads of 64: 18.7 us with four).  Blocks that share a cache: until the SMs are full, as long as each warp has
// four tiles, and if that saves more than the second kernel costs, some 6 us, at 0.4 us a tile (the same trees in two parts: 24 us).  The
// block table's width stands for the lengths, which are on the GPU.
Plan plan(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t D, int64_t keys, int64_t pool_rows) {
  Plan p;
  const int64_t rows = H / Hkv * Tq;
  // Which form: measured in us, few rows against many, rows of 4 heads a key head.  128 dims, 64 groups of 6000 keys: 32 rows 42 / 45, 48 rows 60 / 45, 256
  // rows 206 / 63; 512 groups of 3000: 131 / 170, 217 / 172, 789 / 250.  64 dims, 64 of 6000: 29 / 34, 45 / 35, 146 / 57.  Few blocks over short caches are
  // the few-row form's whatever their rows: 128 dims, 8 groups of 1000: 48 rows 15 / 19, 256 rows 16 / 25 (where the rule is wrong it costs little: 64 dims,
  // 64 groups of 1000, 64 rows 17 / 15).
  const bool short_and_few = keys <= 2048 && (rows + 31) / 32 * B * Hkv <= sm_count();
  p.wide = pool_rows <= 0x7fffffff - 128 && (g_path ? g_path == 2 : rows > 32 && !short_and_few);
  if (p.wide) {
    p.rows = rows <= 128 ? 128 : 256;
    p.row_blocks = static_cast<int>((rows + p.rows - 1) / p.rows);
    p.groups = B * Hkv * p.row_blocks;
    // Blocks that share a cache: until each SM has one, as long as each has four steps.  Up to eight are a cluster (as many as its size allows in groups of
    // 18 SMs), which saves the partial results and the kernel that joins them: 64 groups of 256 rows of 128 dims over 6000 keys, two blocks each: 63 us, 77
    // through partial results (some of it from tiles asked for ahead of the queries).  More than eight only where that shortens the walk by more than two
    // steps: two groups of 112 rows of 128 dims over 100003 keys, 74 blocks each: 32 us.
    const int64_t most = keys / 512, steps = keys / 128;
    int64_t s = p.groups > 0 ? sm_count() / p.groups : 1;
    s = s < most ? s : most;
    if (s > kMostOfCluster && steps / kMostOfCluster - steps / s <= 2) s = kMostOfCluster;
    while (s > 1 && s <= kMostOfCluster && p.groups > sm_count() / 18 * (18 / s)) --s;
    p.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
    p.parts = p.splits > kMostOfCluster;
    p.longest_first = false;
    return p;
  }
  p.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  p.row_blocks = static_cast<int>((rows + p.rows - 1) / p.rows);
  p.groups = B * Hkv * p.row_blocks;
  const int64_t warps = sm_count() * (D == 64 ? 16 : 8);
  p.warps = p.groups * 8 <= warps ? 8 : 4;
  const int64_t slots = warps / p.warps, most = keys / (p.warps * kKeys * 4);
  int64_t s = p.groups > 0 ? slots / p.groups : 1;
  s = s < most ? s : most;
  if (keys * (s - 1) < 16 * p.warps * 16 * s) s = 1;
  p.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
  p.parts = p.splits > 1;
  // (64 sequences of 500 to 6000 keys, 8 heads of 128, 20 rows: 127 us, 159 in their own order; of 300 keys each: 26 and 25.  With 64 dims more blocks have a
  // place at once, and there is nothing to gain: 113 and 112.)
  p.longest_first = D == 128 && B > 1 && B <= kMostInOrder && p.groups > slots && keys >= 2048;
  return p;
}

template <typename T, int D, int NT, int kWarps>
int launch(const Args& a, const Plan& p, cudaStream_t s) {
  using S = Smem<D, NT, kWarps>;
  static SmemLimit limit;
  const cudaError_t e = limit.raise(fmha_tree_kernel<T, D, NT, kWarps>, S::kBytes);
  if (e != cudaSuccess) return set_error(OASR_ERR_CUDA, "fmha_tree: shared memory limit: %s", cudaGetErrorString(e));
  launch_pdl(fmha_tree_kernel<T, D, NT, kWarps>, dim3(static_cast<unsigned>(p.groups * p.splits)), dim3(kWarps * 32), S::kBytes, s, a, p.row_blocks);
  return check_launch("fmha_tree launch");
}
template <typename T, int D, int NT>
int launch(const Args& a, const Plan& p, cudaStream_t s) {
  return p.warps == 8 ? launch<T, D, NT, 8>(a, p, s) : launch<T, D, NT, 4>(a, p, s);
}

template <typename T, int D>
int run(const Args& a, const Plan& p, int dtype, cudaStream_t s) {
  if (p.wide) return run_wide(a, D, dtype, p.rows, p.groups, p.row_blocks, s);
  const int rc = p.rows == 8 ? launch<T, D, 1>(a, p, s) : p.rows == 16 ? launch<T, D, 2>(a, p, s) : launch<T, D, 4>(a, p, s);
  if (rc != OASR_OK || p.splits == 1) return rc;
  const int64_t rows = p.groups * p.rows;
  const auto join = [&](auto kern, int ways) {
    launch_pdl(kern, dim3(static_cast<unsigned>((rows * ways + 7) / 8)), dim3(256), 0, s, a, p.row_blocks, p.rows, static_cast<int>(p.groups));
  };
  if (p.splits <= 4) join(fmha_tree_join_kernel<T, D, 1>, 1);
  else join(fmha_tree_join_kernel<T, D, 8>, 8);
  return check_launch("fmha_tree join launch");
}

}  // namespace
}  // namespace fmha_tree
}  // namespace ob

extern "C" int64_t oasr_b200_fmha_tree_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t D, int64_t blocks_per_seq,
                                                       int64_t block_size, int64_t num_blocks) {
  using namespace ob::fmha_tree;
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || Tq <= 0 || (D != 64 && D != 128) || blocks_per_seq < 0 || block_size <= 0) return 0;
  const Plan p = plan(B, H, Hkv, Tq, D, blocks_per_seq * block_size, num_blocks * block_size);
  return p.parts ? p.splits * p.groups * (D == 64 ? part_floats<64>(p.rows) : part_floats<128>(p.rows)) * 4 : 0;
}

extern "C" int oasr_b200_fmha_tree(void* out, const int64_t* out_strides, const void* q, const int64_t* q_strides, const void* k_pool,
                                   const void* v_pool, const int32_t* block_table, const int32_t* seqlens, const int32_t* seqstarts,
                                   const int32_t* q_lens, const uint32_t* mask, int64_t mask_stride, int64_t mask_words, void* workspace,
                                   int64_t workspace_bytes, int64_t blocks_per_seq, int64_t block_size, int64_t num_blocks, int64_t B, int64_t H,
                                   int64_t Hkv, int64_t Tq, int64_t D, double scale, int dtype, void* stream) {
  using namespace ob;
  using namespace ob::fmha_tree;
  OB_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && Tq >= 0 && D > 0 && blocks_per_seq >= 0 && num_blocks > 0, OASR_ERR_INVALID, "fmha_tree: bad shape");
  OB_REQUIRE(H % Hkv == 0, OASR_ERR_INVALID, "fmha_tree: H (%lld) must be divisible by H_kv (%lld)", (long long)H, (long long)Hkv);
  OB_REQUIRE(D == 64 || D == 128, OASR_ERR_UNSUPPORTED, "fmha_tree: head_dim %lld is not supported (64 and 128 are)", (long long)D);
  OB_REQUIRE(block_size > 0 && block_size % 16 == 0, OASR_ERR_UNSUPPORTED, "fmha_tree: the block size must be a multiple of 16 (got %lld)",
             (long long)block_size);
  // (a position and the tiles that a walk looks ahead fit 32 bits)
  OB_REQUIRE(B <= 65535 && H <= 65535 && Tq <= 0x7fff && num_blocks <= 0x7fffffff && block_size <= 0x7fffff && blocks_per_seq <= 0x7fffff00 &&
                 blocks_per_seq * block_size <= 0x7fff0000,
             OASR_ERR_INVALID, "fmha_tree: batch, head count or length too large");
  // (a scale that is no number would pass for one of zero: scores and scale meet in fmaxf)
  OB_REQUIRE(std::isfinite(static_cast<float>(scale * 1.4426950408889634)), OASR_ERR_INVALID, "fmha_tree: softmax_scale must be a finite number");
  if (B == 0 || Tq == 0) return OASR_OK;
  OB_REQUIRE(out && out_strides && q && q_strides && k_pool && v_pool && (block_table || blocks_per_seq == 0) && seqlens, OASR_ERR_INVALID,
             "fmha_tree: null pointer argument");
  OB_REQUIRE(!mask || (mask_words * 32 >= Tq && mask_words <= 0x7fff && mask_stride >= 0), OASR_ERR_INVALID,
             "fmha_tree: a mask has a word for each 32 of %lld rows (got %lld)", (long long)Tq, (long long)mask_words);
  for (int i = 0; i < 3; ++i)
    OB_REQUIRE(out_strides[i] % 8 == 0 && q_strides[i] % 8 == 0, OASR_ERR_ALIGN, "fmha_tree: strides must be multiples of 8 elements");
  OB_REQUIRE(is_aligned(out, 16) && is_aligned(q, 16) && is_aligned(k_pool, 16) && is_aligned(v_pool, 16) && is_aligned(mask, 4) && is_aligned(workspace, 16),
             OASR_ERR_ALIGN, "fmha_tree: operands must be 16-byte aligned");
  const Plan p = plan(B, H, Hkv, Tq, D, blocks_per_seq * block_size, num_blocks * block_size);
  OB_REQUIRE(p.groups * p.splits <= 0x7fffffff && p.groups * p.rows <= 0x7fffffff, OASR_ERR_INVALID, "fmha_tree: too many rows for one call");
  const int64_t need = oasr_b200_fmha_tree_workspace_bytes(B, H, Hkv, Tq, D, blocks_per_seq, block_size, num_blocks);
  OB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), OASR_ERR_INVALID, "fmha_tree: %lld bytes of workspace needed, %lld given", (long long)need,
             (long long)workspace_bytes);
  const Args a{out, q, k_pool, v_pool, block_table, seqlens, seqstarts, q_lens, mask, need ? static_cast<float*>(workspace) : nullptr, q_strides[0], q_strides[1],
               q_strides[2], out_strides[0], out_strides[1], out_strides[2], mask_stride, blocks_per_seq, block_size, num_blocks, static_cast<int>(B),
               static_cast<int>(H), static_cast<int>(Hkv), static_cast<int>(Tq), static_cast<int>(mask_words), p.splits, p.longest_first,
               static_cast<float>(scale * 1.4426950408889634)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int { return D == 64 ? run<T_, 64>(a, p, dtype, st) : run<T_, 128>(a, p, dtype, st); });
}
