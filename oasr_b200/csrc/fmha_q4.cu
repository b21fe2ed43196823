// Attention over 4-bit pages (q4.cuh):
//
//   out[r] = sum_j softmax_j(scale q_r . k_j) v_j      over start <= j < len, and with `causal` j <= len - q_len + t
//
// Query row t of sequence b stands at position len[b] - q_len[b] + t, so one rule serves a single token, a chunk and a whole
// prompt whose keys are in the pages already.  A row that sees nothing, and rows t >= q_len[b], are zeros.
//
// Keys are the M side of both products (mma.m16n8k16: S^T = K Q^T over the group's dims, O^T = V^T P^T), query rows the N side,
// so a single token wastes 7 of 8 columns and not 15 of 16 rows, and a code needs no transpose: as MMA operands' row, column
// and contraction orders are free, each lane takes whole 32-bit words of codes of whichever keys and dims its fragment stands
// for.  Per 32 keys of a warp, with g = lane / 4 and t = lane % 4:
//   K   the lane holds words t G .. t G + G - 1 (an octet of each group) of keys g + 8 x.  The operand, fp16 for either
//       type, is the code n - 8 itself: a LOP3 puts two of them behind an exponent, a half2 subtraction or multiply-add takes the offset
//       off (left in the products, to be taken off in their sums, it costs the scores 2^-13 of sum |q| times the largest code).  Each
//       row of queries is brought to 2^10 by a power of two (bf16 reaches further than fp16; exact but for what is 2^-34 of the
//       row's largest); a group's sums are scaled in fp32 afterwards.  So a score is a sum of exact products in fp32.
//   V   the lane holds words g D / 64 (+ 1) of keys 8 x + 2 t and 8 x + 2 t + 1.  Here the operand is (n - 8) * scale, exact in the
//       type (q4.cuh).  In bf16 the second nibble has no room behind an exponent: left alone it is the number n 2^-129 (gradual
//       underflow joins the normal numbers at n = 8), which one FMA takes to (n - 8) / 4.
//   P   the scores' fragment is the transpose of what the second product reads: movmatrix.  Weights are rounded to the type (their
//       sum, the maximum and the output are fp32), as in the package's attention over 16-bit pages: each is off by half a step at
//       most, which with the result's own rounding makes an error of 1.2 to 1.35 times that of rounding the result alone.  Exact
//       weights would be a second operand and as many products again.
// The ALU (logic, shifts, permutes: half a warp instruction a clock) is the busiest unit; the FMA pipe, which does the rest of the
// conversion, is not.
// The running maximum moves only when a score passes it by 2^8: numerator and denominator hold the same factor whatever is
// subtracted, so that only their range counts (weights stay below 2^8, finite in either type).  Most tiles need one vote in the place
// of a reduction over the lanes.
// Every warp walks its own tiles with its own maximum, sum and output, and has its own ring of tiles in shared memory, filled by
// asynchronous copies (a tile is two runs of 16 keys of a page): no registers wait for memory, no warp for another.  One to eight
// warps of a block, or the blocks of a cluster, share a (sequence, key head, rows) and meet in shared memory at the end.
//
// B200: 64 sequences of 6000 keys, 32 heads of 128 over 8 key heads, one token each: 112-120 us (442 MB, 3.8 TB/s), bound by
// instructions (some 730 of a warp for 32 keys; ALU 0.55 busy, FMA 0.48, issue slots 0.68).  256 chunks of 16 rows over up to 1001 keys,
// 8 heads of 64: 49 us, a third of it a block's start (lengths, pages, first tile) and end.
#include <cmath>

#include "common.cuh"
#include "fmha_q4.cuh"
#include "q4.cuh"
#include "sm100_ptx.cuh"
#include "smem_limit.cuh"

namespace ob {
namespace fmha_q4 {

int g_path = 0;   // tunable "fmha_q4_path": 0 by size, 1 the few-row form, 2 the prompt form

namespace {

// D = A B + C in fp16 with fp32 accumulators
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void copy16(uint32_t dst, uint64_t src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void copies_but() {   // all but the last N groups of copies have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void lds(uint32_t p, uint32_t* r) {
  if constexpr (N == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(p));
  else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(p));
  else asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p));
}

constexpr int kMaxParts = 4;   // blocks of a cluster

// A tile of 32 keys in the ring: codes of K and V, then their scales.  In rows of 64 bytes the upper two 16-byte pieces of every
// second pair of rows change places with the lower two, which halves the V reads' bank conflicts (their rows are 2 t apart).
template <int D>
struct Tile {
  static constexpr int kRow = D / 2, kCodes = 32 * kRow, kScales = 32 * (D / 32) * 2;
  static constexpr int kK = 0, kV = kCodes, kKs = 2 * kCodes, kVs = 2 * kCodes + kScales, kBytes = 2 * kCodes + 2 * kScales;
  static constexpr int kStages = D == 64 ? 4 : 3;
  static __device__ __forceinline__ int at(int row, int byte) { return row * kRow + (D == 128 ? byte ^ ((row & 2) << 4) : byte); }
};

template <int D, int NT, int kWarps>
struct Merge {   // a warp's, and then the block's, maxima, sums and outputs
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  float o[kWarps][8 * NT][D + 4];
};

template <typename T, int D, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, (NT == 1 ? (D == 64 ? 20 : 16) : NT == 2 ? (D == 64 ? 16 : 12) : 8) / kWarps)
fmha_q4_kernel(const Args a, const int parts, const int ways, const int row_blocks, const int groups) {
  constexpr int G = D / 32, VW = G / 2;   // groups of a row; words of a V row that a lane holds
  constexpr int NR = 8 * NT;
  using Ring = Tile<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  Merge<D, NT, kWarps>& sh = *reinterpret_cast<Merge<D, NT, kWarps>*>(smem);   // after the walk, in the rings' place
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int part = blockIdx.x % parts;
  // `ways` warps of the block share a group (sequence, key head, rows)
  const int group = static_cast<int>(blockIdx.x / parts) * (kWarps / ways) + warp / ways, way = warp % ways;
  int at = min(group, groups - 1);
  const int rb = at % row_blocks;
  at /= row_blocks;
  const int hk = at % a.Hkv, b = at / a.Hkv;
  const int share = a.H / a.Hkv;
  const int rows = group < groups ? share * a.Tq : 0, row0 = rb * NR;
  const int len = max(a.seqlens[b], 0), q_len = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
  const int capacity = static_cast<int>(a.blocks_per_seq * a.block_size);
  const int start = a.seqstarts ? max(a.seqstarts[b], 0) : 0;

  // A tile's halves are 16 keys of one page each: half h of tile i is unit 2 i + h, in block (2 i + h) / units of the table.  The
  // walk keeps quotient and remainder, and looks a block up two tiles ahead.
  const int units = static_cast<int>(a.block_size) / 16, table_len = static_cast<int>(a.blocks_per_seq);
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  const int step = ways * parts, step_blocks = 2 * step / units, step_units = 2 * step - step_blocks * units;
  int tile = start / 32 + part * ways + way;
  struct Place {
    int page0, page1;   // as the table has them
    int unit;           // of the first half in its block; the second's is the next one, or the next block's first
  };
  int ahead_block = 2 * tile / units, ahead_unit = 2 * tile - ahead_block * units;
  auto look_ahead = [&]() {   // the place of the next tile of the walk
    Place p;
    p.unit = ahead_unit;
    const int block1 = ahead_block + (ahead_unit + 1 == units);
    p.page0 = ahead_block < table_len ? table[ahead_block] : -1;
    p.page1 = block1 < table_len ? table[block1] : -1;
    ahead_block += step_blocks;
    ahead_unit += step_units;
    if (ahead_unit >= units) ahead_unit -= units, ++ahead_block;
    return p;
  };
  Place first[Ring::kStages];   // the look-ups of the first tiles are on their way while the lengths are
#pragma unroll
  for (int i = 0; i < Ring::kStages; ++i) first[i] = look_ahead();

  // keys that a row may see: [start, limit)
  auto limit_of = [&](int r) {
    if (r >= rows) return 0;
    const int tq = r / share;
    if (tq >= q_len) return 0;
    int end = min(len, capacity);
    if (a.causal) end = static_cast<int>(min(static_cast<int64_t>(end), static_cast<int64_t>(len) - q_len + tq + 1));
    return max(end, 0);
  };
  int limit[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    limit[n][0] = limit_of(row0 + n * 8 + 2 * t);
    limit[n][1] = limit_of(row0 + n * 8 + 2 * t + 1);
  }
  // rows are in the order of their positions, so the last one that counts sees the most and the first one the least
  const int last_row = min(min(row0 + NR, rows), q_len * share) - 1;
  const int end = last_row >= row0 ? limit_of(last_row) : 0;
  const int all_end = last_row >= row0 ? limit_of(row0) : 0;   // padding rows see nothing, and nobody reads what they hold

  const int tile_end = (end + 31) / 32;
  auto known = [&](int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_blocks); };
  // copies of a tile: a half's codes are one run of 16 rows, its scales another
  const uint32_t ring = ptx::smem_u32(smem) + warp * (Ring::kStages * Ring::kBytes);
  constexpr int kPieces = Ring::kCodes / 2 / 16;      // of a half: 32 or 64
  const uint32_t to = Ring::at(lane * 16 / Ring::kRow, lane * 16 % Ring::kRow);
  constexpr int kScalePieces = Ring::kScales / 16;    // of a tile's K or V: 8 or 16 lanes
  const bool scale_lane = lane < 2 * kScalePieces, scale_half = lane % kScalePieces >= kScalePieces / 2;
  const uint64_t k_codes = reinterpret_cast<uint64_t>(a.k_codes) + lane * 16, v_codes = reinterpret_cast<uint64_t>(a.v_codes) + lane * 16;
  const uint64_t scales = reinterpret_cast<uint64_t>(lane >= kScalePieces ? a.v_scales : a.k_scales) + lane % (kScalePieces / 2) * 16;
  const uint32_t page_bytes = a.Hkv * static_cast<uint32_t>(a.block_size) * Ring::kRow, head_bytes = hk * static_cast<uint32_t>(a.block_size) * Ring::kRow;
  uint32_t there = 0;   // two bits a tile in the ring: its halves have pages
  auto fetch = [&](const Place& p, uint32_t stage) {
    // a half without a page reads page 0 and is masked
    const bool k0 = known(p.page0), k1 = known(p.page1);
    const int unit1 = p.unit + 1 == units ? 0 : p.unit + 1;
    const uint64_t o0 = static_cast<uint64_t>(k0 ? static_cast<uint32_t>(p.page0) : 0u) * page_bytes + (head_bytes + static_cast<uint32_t>(p.unit) * (16 * Ring::kRow));
    const uint64_t o1 = static_cast<uint64_t>(k1 ? static_cast<uint32_t>(p.page1) : 0u) * page_bytes + (head_bytes + static_cast<uint32_t>(unit1) * (16 * Ring::kRow));
#pragma unroll
    for (int i = 0; i < kPieces / 32; ++i) {          // 512 bytes further: 8 or 16 rows, the same place in the row
      copy16(stage + Ring::kK + to + i * 512, k_codes + o0 + i * 512);
      copy16(stage + Ring::kK + to + Ring::kCodes / 2 + i * 512, k_codes + o1 + i * 512);
      copy16(stage + Ring::kV + to + i * 512, v_codes + o0 + i * 512);
      copy16(stage + Ring::kV + to + Ring::kCodes / 2 + i * 512, v_codes + o1 + i * 512);
    }
    if (scale_lane) copy16(stage + Ring::kKs + lane * 16, scales + ((scale_half ? o1 : o0) >> 3));   // a row has an eighth of its codes' bytes
    there |= (k0 ? 1u : 0u) << (2 * Ring::kStages - 2) | (k1 ? 2u : 0u) << (2 * Ring::kStages - 2);
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

#pragma unroll
  for (int i = 0; i < Ring::kStages - 1; ++i) {
    there >>= 2;
    if (tile + i * step < tile_end) fetch(first[i], ring + i * Ring::kBytes);
    commit();
  }
  Place next = first[Ring::kStages - 1];
  // ---- queries as the second operand: column g, dims of octet t of each group
  uint32_t qf[NT][G][4];
  float unit[NT][2];   // takes a column's sums to scores in the log2 domain
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + n * 8 + g;
    const T* q = static_cast<const T*>(a.q) + b * a.qs_b + (hk * share + r % share) * a.qs_h + static_cast<int64_t>(r / share) * a.qs_t;
    Pack<T> x[G];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      if (r < rows) x[k] = ld128(q + k * 32 + t * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (r >= rows) x[k].v[i] = Elem<T>::from_f(0.f);
        top = q4::max_nan(top, fabsf(Elem<T>::to_f(x[k].v[i])));
      }
    }
    top = q4::max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = q4::max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = max(static_cast<int>(__float_as_uint(top) >> 23) & 255, 12);   // biased exponent of the row's largest
    const float lift = __uint_as_float(static_cast<uint32_t>(264 - e) << 23);     // 2^(137 - e)
    const float down = __uint_as_float(static_cast<uint32_t>(max(e - 10, 1)) << 23) * fabsf(a.scale_log2);
    unit[n][0] = fmaxf(__shfl_sync(0xffffffffu, down, 8 * t), 1.2e-38f);           // a scale of zero leaves masked scores at -inf
    unit[n][1] = fmaxf(__shfl_sync(0xffffffffu, down, 8 * t + 4), 1.2e-38f);
    const float signed_lift = a.scale_log2 < 0.f ? -lift : lift;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = Elem<T>::to_f(x[k].v[i]) * signed_lift;
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[n][k][i] = half2_bits(__floats2half2_rn(y[i], y[i + 4]));
    }
  }

  float o[NT][VW * 4][4] = {}, m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = kEmpty, l[n][0] = l[n][1] = 0.f;

  const uint32_t k_lane = g * Ring::kRow + Ring::at(g, t * (G * 4)) % Ring::kRow;
  const uint32_t v_lane = 2 * t * Ring::kRow + Ring::at(2 * t, g * (VW * 4)) % Ring::kRow;
  uint32_t stage = ring, free_stage = ring + (Ring::kStages - 1) * Ring::kBytes;
  for (; tile < tile_end; tile += step) {
    copies_but<Ring::kStages - 2>();
    __syncwarp();                                      // the tile is there for all lanes, and the last one is read by all
    there >>= 2;
    if (tile + (Ring::kStages - 1) * step < tile_end) fetch(next, free_stage);
    commit();
    next = look_ahead();
    const int j0 = tile * 32;
    const bool whole = j0 >= start && j0 + 32 <= all_end && (there & 3) == 3;   // nothing to mask

    // ---- scores: m-tile i has keys 16 i + g and 16 i + 8 + g, columns 2 t (+ 1)
    float s[NT][2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t kw[2][G], ks[2][G / 2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 16 * i + 8 * x;
        lds<G>(stage + k_lane + (Ring::kK + row * Ring::kRow), kw[x]);
        lds<G / 2>(stage + g * (G * 2) + (Ring::kKs + row * (G * 2)), ks[x]);
      }
#pragma unroll
      for (int k = 0; k < G; ++k) {
        float sc[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          sc[x] = k & 1 ? Op<T>::high_f(ks[x][k / 2]) : Op<T>::low_f(ks[x][k / 2]);
        }
        const uint32_t wa = kw[0][k], wb = kw[1][k], ha = wa >> 8, hb = wb >> 8;
        const uint32_t af[8] = {low_codes(wa), low_codes(wb), second_codes(wa), second_codes(wb), low_codes(ha), low_codes(hb), second_codes(ha), second_codes(hb)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float c[4] = {};
          mma_f16(c, af, qf[n][k][0], qf[n][k][1], c);
          mma_f16(c, af + 4, qf[n][k][2], qf[n][k][3], c);
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][i][x] = k == 0 ? sc[x >> 1] * c[x] : fmaf(sc[x >> 1], c[x], s[n][i][x]);
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = j0 + 16 * i + 8 * (x >> 1) + g;
            if (!(there >> i & 1) || j < start || j >= limit[n][x & 1]) s[n][i][x] = -INFINITY;
          }
    }

    // ---- weights
    float top[NT][2];
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = fmaxf(fmaxf(s[n][0][c], s[n][0][2 + c]), fmaxf(s[n][1][c], s[n][1][2 + c])) * unit[n][c];
        raise |= top[n][c] > m[n][c] + 8.f;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = top[n][c];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          v = fmaxf(v, m[n][c]);
          const float f = ex2(m[n][c] - v);
          m[n][c] = v;
          l[n][c] *= f;
#pragma unroll
          for (int i = 0; i < VW * 4; ++i) o[n][i][c] *= f, o[n][i][2 + c] *= f;
        }
    }
    uint32_t pf[NT][4];   // block x: keys 8 x + g; after the transpose the lane has keys 8 x + 2 t (+ 1) of row g
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float e0 = ex2(fmaf(s[n][x >> 1][(x & 1) * 2], unit[n][0], -m[n][0]));
        const float e1 = ex2(fmaf(s[n][x >> 1][(x & 1) * 2 + 1], unit[n][1], -m[n][1]));
        l[n][0] += e0;
        l[n][1] += e1;
        pf[n][x] = transpose8x8(Op<T>::pack(e0, e1));
      }
    }

    // ---- output: dims of the lane's words, keys 8 x + 2 t and 8 x + 2 t + 1 of block x
    uint32_t vw[4][2][VW], sp[VW][4];
    const uint32_t own = g & 1 ? 0x7632u : 0x5410u;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int row = 8 * x + 2 * t;
#pragma unroll
      for (int y = 0; y < 2; ++y) lds<VW>(stage + v_lane + (Ring::kV + (8 * x + y) * Ring::kRow), vw[x][y]);
      uint32_t s2[2];
      if constexpr (G == 2) {   // a key's two scales are a word; the lane's group is g % 2
        lds<2>(stage + Ring::kVs + row * 4, s2);
        sp[0][x] = __byte_perm(s2[0], s2[1], own);
      } else {                  // its words 2 g and 2 g + 1 are of groups 0, 1 (g even) or 2, 3
        lds<1>(stage + Ring::kVs + row * 8 + (g & 1) * 4, s2);
        lds<1>(stage + Ring::kVs + row * 8 + 8 + (g & 1) * 4, s2 + 1);
        sp[0][x] = lows(s2[0], s2[1]);
        sp[VW - 1][x] = highs(s2[0], s2[1]);
      }
    }
    if (!whole) {   // a key that some row of the block does not see must not reach it as 0 * NaN: those rows' outputs take it by hand
      bool odd = false;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int j = j0 + 8 * x + 2 * t + y;
          const bool seen = (there >> (x >> 1) & 1) && j >= start && j < end;
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const unsigned short h = static_cast<unsigned short>(sp[w][x] >> (16 * y));
            if (seen && fabsf(Elem<T>::to_f(*reinterpret_cast<const T*>(&h))) < INFINITY) continue;
            odd |= seen;
            sp[w][x] &= y ? 0x0000ffffu : 0xffff0000u;
          }
        }
      if (__any_sync(0xffffffffu, odd)) {
        for (int x = 0; x < 32; ++x) {
          const int j = j0 + x;
          if (!(there >> (x >> 4) & 1) || j < start || j >= end) continue;
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const T* sc = reinterpret_cast<const T*>(smem + (stage - ptx::smem_u32(smem)) + Ring::kVs) + x * G + (g * VW + w) % G;
            if (fabsf(Elem<T>::to_f(*sc)) < INFINITY) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                if (j < limit[n][c])
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[n][w * 4 + i][c] = o[n][w * 4 + i][2 + c] = __uint_as_float(0x7fffffffu);
          }
        }
      }
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      uint32_t st[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) st[x] = Op<T>::steep(sp[w][x]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // dims 2 i, 2 i + 1 of the octet: byte i of the words
        uint32_t d0[4], d1[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t src = __byte_perm(vw[x][0][w], vw[x][1][w], 0x4400 + 0x1111 * i);
          d0[x] = Op<T>::low(src, sp[w][x]);
          d1[x] = Op<T>::second(src, st[x]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          Op<T>::mma(o[n][w * 4 + i], d0[0], d1[0], d0[1], d1[1], pf[n][0], pf[n][1]);
          Op<T>::mma(o[n][w * 4 + i], d0[2], d1[2], d0[3], d1[3], pf[n][2], pf[n][3]);
        }
      }
    }
    free_stage = stage;
    stage = stage == ring + (Ring::kStages - 1) * Ring::kBytes ? ring : stage + Ring::kBytes;
  }

  // ---- the warps of a group meet, then the blocks of the cluster
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
      for (int w = 0; w < VW; ++w) {
        const int dim = q4::octet_of_word(g * VW + w, G) * 8;
        float* dst = &sh.o[warp][r][dim];
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[n][w * 4 + i][c], o[n][w * 4 + i][2 + c]);
      }
    }
  __syncthreads();
  if (parts > 1) {   // the block's own sum over its warps goes into the first warp's place
    for (int i = threadIdx.x; i < NR * (D / 4); i += kWarps * 32) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float top = sh.m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh.m[w][r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sh.m[w][r] - top);
        const float4 v = *reinterpret_cast<const float4*>(&sh.o[w][r][d]);
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
      }
      *reinterpret_cast<float4*>(&sh.o[0][r][d]) = acc;
    }
    __syncthreads();
    if (threadIdx.x < NR) {
      const int r = threadIdx.x;
      float top = sh.m[0][r], sum = 0.f;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh.m[w][r]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum = fmaf(sh.l[w][r], ex2(sh.m[w][r] - top), sum);
      sh.m[0][r] = top, sh.l[0][r] = sum;
    }
    ptx::cluster_sync();
  }
  // Rows of the warp's own group, dealt over its warps; with a cluster (the block is one group) over those of all blocks.
  const int first_warp = warp - way;
  for (int i = (part * ways + way) * 32 + lane; i < NR * (D / 8); i += parts * ways * 32) {
    const int n = i / (D / 8), d = i % (D / 8) * 8, r = row0 + n;
    if (r >= rows) continue;
    float top = kEmpty, sum = 0.f, acc[8] = {};
    if (parts == 1) {
      for (int w = first_warp; w < first_warp + ways; ++w) top = fmaxf(top, sh.m[w][n]);
      for (int w = first_warp; w < first_warp + ways; ++w) {
        const float f = ex2(sh.m[w][n] - top);
        const float4 a0 = *reinterpret_cast<const float4*>(&sh.o[w][n][d]), a1 = *reinterpret_cast<const float4*>(&sh.o[w][n][d + 4]);
        sum = fmaf(f, sh.l[w][n], sum);
        acc[0] = fmaf(f, a0.x, acc[0]), acc[1] = fmaf(f, a0.y, acc[1]), acc[2] = fmaf(f, a0.z, acc[2]), acc[3] = fmaf(f, a0.w, acc[3]);
        acc[4] = fmaf(f, a1.x, acc[4]), acc[5] = fmaf(f, a1.y, acc[5]), acc[6] = fmaf(f, a1.z, acc[6]), acc[7] = fmaf(f, a1.w, acc[7]);
      }
    } else {   // all loads from the other blocks on their way before the first is used; ranks past the last one read it again
      float ms[kMaxParts], ls[kMaxParts], v[kMaxParts][8];
#pragma unroll
      for (int w = 0; w < kMaxParts; ++w) {
        const int rank = min(w, parts - 1);
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ms[w]) : "r"(ptx::map_to_cta(&sh.m[0][n], rank)));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ls[w]) : "r"(ptx::map_to_cta(&sh.l[0][n], rank)));
        const uint32_t src = ptx::map_to_cta(&sh.o[0][n][d], rank);
#pragma unroll
        for (int x = 0; x < 8; x += 4)
          asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[w][x]), "=f"(v[w][x + 1]), "=f"(v[w][x + 2]), "=f"(v[w][x + 3]) : "r"(src + 4 * x));
      }
#pragma unroll
      for (int w = 0; w < kMaxParts; ++w) top = fmaxf(top, ms[w]);
#pragma unroll
      for (int w = 0; w < kMaxParts; ++w) {
        if (w < parts) {
          const float f = ex2(ms[w] - top);
          sum = fmaf(f, ls[w], sum);
#pragma unroll
          for (int x = 0; x < 8; ++x) acc[x] = fmaf(f, v[w][x], acc[x]);
        }
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // NaN stays
    const int tq = r / share;
    Pack<T> out;
#pragma unroll
    for (int x = 0; x < 8; ++x) out.v[x] = Elem<T>::from_f(tq < q_len ? acc[x] * inv : 0.f);
    st128(static_cast<T*>(a.out) + b * a.os_b + (hk * share + r - tq * share) * a.os_h + static_cast<int64_t>(tq) * a.os_t + d, out);
  }
  if (parts > 1) ptx::cluster_sync();   // nobody leaves while its sums are read
}

template <typename T, int D, int NT, int kWarps>
int launch(const Args& a, int ways, int parts, int64_t row_blocks, int64_t groups, cudaStream_t s) {
  const int64_t blocks = (groups + kWarps / ways - 1) / (kWarps / ways) * parts;
  OB_REQUIRE(groups <= 0x7fffffff && blocks <= 0x7fffffff, OASR_ERR_INVALID, "fmha_q4: too many rows for one call");
  static SmemLimit limit;
  constexpr int kRings = kWarps * Tile<D>::kStages * Tile<D>::kBytes, kMerge = sizeof(Merge<D, NT, kWarps>);
  constexpr int kSmem = kRings > kMerge ? kRings : kMerge;
  cudaError_t e = limit.raise(fmha_q4_kernel<T, D, NT, kWarps>, kSmem);
  if (e != cudaSuccess) return set_error(OASR_ERR_CUDA, "fmha_q4: shared memory limit: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = g_pdl ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, fmha_q4_kernel<T, D, NT, kWarps>, a, parts, ways, static_cast<int>(row_blocks), static_cast<int>(groups));
  return check_launch("fmha_q4 launch");
}

template <typename T, int D, int NT>
int launch(const Args& a, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.H / a.Hkv) * a.Tq, row_blocks = (rows + 8 * NT - 1) / (8 * NT);
  const int64_t groups = static_cast<int64_t>(a.B) * a.Hkv * row_blocks, tiles = (a.blocks_per_seq * a.block_size + 31) / 32;
  // Warps that share a group: until the SMs are full (down to two tiles each), and so many that none walks more than 32 tiles.  `tiles`
  // are the block table's, the only bound of the lengths that the host has: in a table wider than its sequences most warps find
  // nothing, and their blocks' start and end are what a call then takes (the two cases below in tables four times as wide: 179 ->
  // 228 us and 49 -> 49 us, 32 times: 228 and 238 us).  Fewer
  // leave the longest sequences of a ragged batch running alone, more pay a block's start and end (some 6 us of latency) more often:
  // 128 sequences of 500 to 8191 keys, 8 key heads of 128, take 186 / 176 / 189 us with 4 / 8 / 16 warps, 256 chunks of 16 rows over up
  // to 1001 keys, 8 heads of 64, take 60 / 50 / 52 us with 1 / 2 / 4.  Beyond eight, blocks of eight in a cluster.
  int splits = 1;
  while (splits < 8 * kMaxParts && (tiles > 32 * splits || (groups * splits < sm_count() * 16 && tiles > 2 * splits))) splits *= 2;
  if (splits <= 4) return launch<T, D, NT, 4>(a, splits, 1, row_blocks, groups, s);
  return launch<T, D, NT, 8>(a, 8, splits / 8, row_blocks, groups, s);
}

template <typename T, int D>
int run(const Args& a, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.H / a.Hkv) * a.Tq;
  if (rows <= 8) return launch<T, D, 1>(a, s);
  if constexpr (D == 64)
    if (rows > 16) return launch<T, D, 4>(a, s);
  return launch<T, D, 2>(a, s);
}

// Which form: measured times, as far as sizes tell.  The few-row form takes 3.66 ps (head_dim 128; 64: 1.46 ps) a row and key when it
// fills the GPU, up to twice that when it does not; the prompt form 2.5 us for 128 keys of a block of 256 rows, however many of them
// are there.  `keys` is the block table's width, as above.  In us, few-row against prompt form, bf16: 64 rows over 1000 keys, 128 groups of 128: 56 / 28, 8 groups: 14 / 26; 1024 groups of
// 64: 109 / 150; 512 rows over 1000 keys, 8 groups of 128: 45 / 37, 1024 groups: 1686 / 558; 64 rows over 8000 keys, 8 groups: 34 / 151.
bool prompt_is_faster(int64_t rows, int64_t heads, int64_t keys, int64_t D) {
  if (g_path != 0) return g_path == 2;
  if (rows <= 16) return false;
  const double few = 8e-6 + 1.3 * (D == 64 ? 1.46e-12 : 3.66e-12) * static_cast<double>(rows) * static_cast<double>(keys) * static_cast<double>(heads);
  const int64_t waves = ((rows + 255) / 256 * heads + sm_count() - 1) / sm_count();
  const double prompt = 6e-6 + 2.5e-6 * static_cast<double>(waves) * static_cast<double>((keys + 127) / 128);
  return prompt < few;
}

}  // namespace
}  // namespace fmha_q4
}  // namespace ob

extern "C" int oasr_b200_fmha_q4(void* out, const int64_t* out_strides, const void* q, const int64_t* q_strides, const void* k_codes,
                                 const void* k_scales, const void* v_codes, const void* v_scales, const int32_t* block_table,
                                 const int32_t* seqlens, const int32_t* seqstarts, const int32_t* q_lens, int64_t blocks_per_seq,
                                 int64_t block_size, int64_t num_blocks, int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t D,
                                 double scale, int causal, int dtype, void* stream) {
  using namespace ob;
  using namespace ob::fmha_q4;
  OB_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && Tq >= 0 && D > 0 && blocks_per_seq >= 0 && num_blocks > 0, OASR_ERR_INVALID, "fmha_q4: bad shape");
  OB_REQUIRE(H % Hkv == 0, OASR_ERR_INVALID, "fmha_q4: H (%lld) must be divisible by H_kv (%lld)", (long long)H, (long long)Hkv);
  OB_REQUIRE(D == 64 || D == 128, OASR_ERR_UNSUPPORTED, "fmha_q4: head_dim %lld is not supported (64 and 128 are)", (long long)D);
  OB_REQUIRE(block_size > 0 && block_size % 16 == 0, OASR_ERR_UNSUPPORTED, "fmha_q4: the block size must be a multiple of 16 (got %lld)",
             (long long)block_size);
  OB_REQUIRE(Hkv * block_size * D <= 0x7fffffff, OASR_ERR_INVALID, "fmha_q4: pages too large");
  // (a position and a whole tile more fit 32 bits)
  OB_REQUIRE(B <= 65535 && H <= 65535 && Tq <= 0x7fffff && blocks_per_seq * block_size <= 0x7fffff00, OASR_ERR_INVALID,
             "fmha_q4: batch, head count or length too large");
  // (a scale that is no number would pass for one of zero: scores and scale meet in fmaxf)
  OB_REQUIRE(std::isfinite(static_cast<float>(scale * 1.4426950408889634)), OASR_ERR_INVALID, "fmha_q4: softmax_scale must be a finite number");
  if (B == 0 || Tq == 0) return OASR_OK;
  OB_REQUIRE(out && out_strides && q && q_strides && k_codes && k_scales && v_codes && v_scales && (block_table || blocks_per_seq == 0) && seqlens, OASR_ERR_INVALID,
             "fmha_q4: null pointer argument");
  for (int i = 0; i < 3; ++i)
    OB_REQUIRE(out_strides[i] % 8 == 0 && q_strides[i] % 8 == 0, OASR_ERR_ALIGN, "fmha_q4: strides must be multiples of 8 elements");
  OB_REQUIRE(is_aligned(out, 16) && is_aligned(q, 16) && is_aligned(k_codes, 16) && is_aligned(v_codes, 16) && is_aligned(k_scales, 16) &&
                 is_aligned(v_scales, 16),
             OASR_ERR_ALIGN, "fmha_q4: operands must be 16-byte aligned");
  const Args a{out, q, static_cast<const uint32_t*>(k_codes), static_cast<const uint32_t*>(v_codes), k_scales, v_scales, block_table, seqlens,
               seqstarts, q_lens, q_strides[0], q_strides[1], q_strides[2], out_strides[0], out_strides[1], out_strides[2], blocks_per_seq,
               block_size, num_blocks, static_cast<int>(B), static_cast<int>(H), static_cast<int>(Hkv), static_cast<int>(Tq), causal != 0,
               static_cast<float>(scale * 1.4426950408889634)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (prompt_is_faster(H / Hkv * Tq, B * Hkv, blocks_per_seq * block_size, D)) return run_prompt(a, static_cast<int>(D), dtype, st);
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int { return D == 64 ? run<T_, 64>(a, st) : run<T_, 128>(a, st); });
}
