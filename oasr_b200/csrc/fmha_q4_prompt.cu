// Attention of long chunks over 4-bit pages (fmha_q4.cu has the formula, and the form for few rows): tcgen05 products.
//
// A block owns 256 query rows of one (sequence, key head), two tiles of 128, and walks the keys 128 at a time.  13 warps:
//   0-3, 4-7  softmax of the two tiles: a thread owns a row, reads its scores from tensor memory and writes its weights there;
//   8         issues the products: S = Q K^T into 128 columns of tensor memory per tile, O += P V into D columns per tile;
//   9-12      turn codes into 16-bit rows of K and V in shared memory (128-byte swizzle).
// The tiles run half a step apart: while one's softmax works, the tensor cores have the other's products.  Both share the
// converted keys and values, so a code is converted once for 256 rows.  Output stays in tensor memory; a row's maximum moves only
// when a score passes it by 2^8, and only then is the output scaled again.
// Weights take the place of the scores they were made of (16 bits for 32: the rounding that fmha_q4.cu explains) and are the A
// operand of the second product from there: a product with both operands in shared memory reads 128 bytes a clock, all there is,
// and the weights' way through it was a third of that traffic.  So S of step j + 1 waits for O of step j to be complete; the other
// tile's products fill the gap.
//
// Converted rows hold the exact values (q4.cuh).  Within an octet the dims lie in the order 0 4 1 5 2 6 3 7, the pairs that one mask
// of a code word gives; queries are stored in the same order, and the output's columns are put right when they are read.
// B200: 4001 rows over 4098 keys, causal, 32 heads of 128 over 8 key heads: 224 us (614 TFLOP/s; 236 us with the weights through shared
// memory).  A step of 128 keys takes 4.5k clocks: products 2.1k, a tile's softmax 2.9k, which its two warps a scheduler and 128
// registers a thread set.
// Shared memory at D = 128: Q 64 KB, K and V in five slots of 32 KB that follow one another K V K V.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "device_status.cuh"
#include "fmha_q4.cuh"
#include "q4.cuh"
#include "sm100_ptx.cuh"
#include "smem_limit.cuh"

namespace ob {
namespace fmha_q4 {
namespace {

constexpr int kMmaWarp = 8, kProducer = 9, kProducers = 4, kThreads = (kProducer + kProducers) * 32;
constexpr int kAtom = 128 * 128;   // 128 rows of 128 bytes
constexpr int kKeys = 128;

// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int D>
struct Smem {
  static constexpr int kAtoms = D / 64, kSlots = D == 128 ? 5 : 8;
  static constexpr int kQ = 0, kRing = kQ + 2 * kAtoms * kAtom, kBars = kRing + kSlots * kAtoms * kAtom;
  static constexpr int kNumBars = 2 * kSlots + 6;
  static constexpr int kTotal = kBars + kNumBars * 8 + 16, kDynamic = kTotal + 1024;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) fmha_q4_prompt_kernel(const Args a, const int row_blocks, uint32_t* status) {
  using S = Smem<D>;
  constexpr int G = D / 32;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescQK = ptx::umma_idesc_f16(kBf16, 128, kKeys, false, false);
  constexpr uint32_t kIdescPV = ptx::umma_idesc_f16(kBf16, 128, D, false, true);   // V: keys are its rows
  constexpr uint32_t kColS = 0, kColO = 256, kCols = 512;

  ptx::grid_dep_wait();
  // the last row blocks see the most keys under a causal mask: they start first
  const int heads = a.B * a.Hkv, rb = row_blocks - 1 - static_cast<int>(blockIdx.x) / heads;
  const int bh = static_cast<int>(blockIdx.x) % heads, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int share = a.H / a.Hkv, rows = share * a.Tq, row0 = rb * 256;
  const int len = max(a.seqlens[b], 0), q_len = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
  const int capacity = static_cast<int>(a.blocks_per_seq * a.block_size);
  const int start = a.seqstarts ? max(a.seqstarts[b], 0) : 0;
  auto limit_of = [&](int r) {   // keys that row r may see: [start, limit)
    int end = min(len, capacity);
    if (a.causal) end = static_cast<int>(min(static_cast<int64_t>(end), static_cast<int64_t>(len) - q_len + r / share + 1));
    return max(end, 0);
  };
  const int last_row = min(min(row0 + 256, rows), q_len * share) - 1;
  const int end = last_row >= row0 ? limit_of(last_row) : 0;
  const int tile0 = start / kKeys, tiles = max((end + kKeys - 1) / kKeys - tile0, 0);
  auto out_row = [&](int r) { return static_cast<T*>(a.out) + b * a.os_b + (hk * share + r % share) * a.os_h + static_cast<int64_t>(r / share) * a.os_t; };
  if (tiles == 0 || start >= end) {   // nothing to see: zero rows
    for (int i = threadIdx.x; i < min(256, rows - row0) * (D / 8); i += kThreads)
      *reinterpret_cast<uint4*>(out_row(row0 + i / (D / 8)) + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int streams = last_row >= row0 + 128 ? 2 : 1;   // row tiles with something in them

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kSlots;
  uint64_t* s_full = empty + S::kSlots;   // [2]  scores are there (and the output has all weights before)
  uint64_t* p_full = s_full + 2;          // [2]  weights are there, output is scaled
  uint64_t* o_done = s_full + 4;          // [2]  output has the weights
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 6);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* odd_values = tmem_slot + 2;   // some value scale is not finite

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kSlots; ++i) {
      ptx::mbar_init(&full[i], kProducers * 32);
      ptx::mbar_init(&empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      ptx::mbar_init(&s_full[x], 1);
      ptx::mbar_init(&p_full[x], 128);
      ptx::mbar_init(&o_done[x], 1);
    }
    *abort_flag = 0;
    *odd_values = 0;
    ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(tmem_slot, kCols);
    ptx::tmem_relinquish();
  }
  // queries, with the sign of the scale
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  for (int i = threadIdx.x; i < streams * 128 * (D / 8); i += kThreads) {
    const int r = i / (D / 8), o = i % (D / 8), rr = row0 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (rr < rows)
      v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs_b + (hk * share + rr % share) * a.qs_h +
                                          static_cast<int64_t>(rr / share) * a.qs_t + o * 8);
    const uint4 w = make_uint4(lows(v.x, v.z) ^ flip, highs(v.x, v.z) ^ flip, lows(v.y, v.w) ^ flip, highs(v.y, v.w) ^ flip);
    *reinterpret_cast<uint4*>(smem + S::kQ + ((r >> 7) * S::kAtoms + o / 8) * kAtom + (r & 127) * 128 + ((o & 7) ^ (r & 7)) * 16) = w;
  }
  ptx::fence_proxy_async_smem();
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dep_launch();   // only now: see sm100_ptx.cuh

  const int units = static_cast<int>(a.block_size) / 16, table_len = static_cast<int>(a.blocks_per_seq);
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  auto page_of = [&](int unit) {   // of 16 keys; -1: none
    const int blk = unit / units;
    const int page = blk < table_len ? table[blk] : -1;
    return page < a.num_blocks ? page : -1;
  };
  bool ok = true;
  float m = kEmpty, l = 0.f;

  if (warp == kMmaWarp) {
    const bool issuer = ptx::elect_one();
    const uint32_t base = ptx::smem_u32(smem);
    auto slot_of = [&](int h) { return base + S::kRing + (h % S::kSlots) * S::kAtoms * kAtom; };
    auto wait_full = [&](int h) { return ptx::mbar_wait(&full[h % S::kSlots], (h / S::kSlots) & 1, abort_flag); };
    auto scores = [&](int x, int j) {
      if (!issuer) return;
      const uint64_t ad = ptx::smem_desc_kmajor_sw128(base + S::kQ + x * S::kAtoms * kAtom), bd = ptx::smem_desc_kmajor_sw128(slot_of(2 * j));
#pragma unroll
      for (int kk = 0; kk < S::kAtoms * 4; ++kk) {
        const uint32_t off = ((kk / 4) * kAtom + (kk % 4) * 32) >> 4;
        ptx::umma_f16(tmem + kColS + x * 128, ad + off, bd + off, kIdescQK, kk > 0);
      }
      ptx::umma_commit(&s_full[x]);
      if (x == streams - 1) ptx::umma_commit(&empty[(2 * j) % S::kSlots]);
    };
    auto output = [&](int x, int j) {
      if (!issuer) return;
      const uint64_t bd = ptx::smem_desc_mnmajor_sw128(slot_of(2 * j + 1), kAtom, 1024);
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk)
        ptx::umma_f16_ts(tmem + kColO + x * 128, tmem + kColS + x * 128 + kk * 8, bd + ((kk * 2048) >> 4), kIdescPV, j > 0 || kk > 0);
      ptx::umma_commit(&o_done[x]);
      if (x == streams - 1) ptx::umma_commit(&empty[(2 * j + 1) % S::kSlots]);
    };
    ok = wait_full(0);
    ptx::tc_fence_after_sync();
    for (int x = 0; ok && x < streams; ++x) scores(x, 0);
    for (int j = 0; ok && j < tiles; ++j) {
      for (int x = 0; ok && x < streams; ++x) {
        if (x == 0) ok = wait_full(2 * j + 1);
        ok = ok && ptx::mbar_wait(&p_full[x], j & 1, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        output(x, j);
        if (j + 1 < tiles) {
          if (x == 0) ok = wait_full(2 * j + 2);
          // products into other columns are not bound to stay in order: the weights go only once they are used
          ok = ok && ptx::mbar_wait(&o_done[x], j & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          scores(x, j + 1);
        }
      }
    }
    if (!ok && issuer && status) atomicOr(status, kStatusFmhaMma);
    __syncwarp();
  } else if (warp >= kProducer) {
    // ---- codes -> rows.  A lane takes 16 bytes of codes (a quarter or half of a row) of `kPasses` rows of a tile
    constexpr int kLanes = D / 32, kPassRows = kProducers * 32 / kLanes, kPasses = kKeys / kPassRows;
    const int row_in_pass = (warp - kProducer) * (32 / kLanes) + lane / kLanes, piece = lane % kLanes;
    const uint32_t page_rows = static_cast<uint32_t>(a.Hkv * a.block_size), head_rows = static_cast<uint32_t>(hk * a.block_size);
    // Pages are asked for two tiles ahead and rows made of them one tile ahead, so that no load waits for another.  A lane's rows
    // of pass p lie in unit (16 keys of a page) 8 tile + unit0 + p * kPassRows / 16; quotient and remainder by the units of a
    // page are kept from tile to tile.
    const int first_unit = tile0 * 8 + (row_in_pass >> 4), step_blocks = 8 / units, step_units = 8 - step_blocks * units;
    int block[kPasses], unit[kPasses], page[kPasses];
    int64_t row[kPasses];      // of the pools
    uint32_t known = 0;        // bit p: that row has a page (one without reads row 0)
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      block[p] = (first_unit + p * (kPassRows / 16)) / units;
      unit[p] = first_unit + p * (kPassRows / 16) - block[p] * units;
    }
    auto ask = [&] {           // the pages of the next tile
#pragma unroll
      for (int p = 0; p < kPasses; ++p) page[p] = block[p] < table_len ? table[block[p]] : -1;
    };
    auto resolve = [&] {       // rows of the pages asked for, and on to the next tile
      known = 0;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const bool there = static_cast<uint32_t>(page[p]) < static_cast<uint32_t>(a.num_blocks);
        known |= (there ? 1u : 0u) << p;
        row[p] = there ? static_cast<int64_t>(page[p]) * page_rows + (head_rows + static_cast<uint32_t>(unit[p] * 16 + (row_in_pass & 15))) : 0;
        block[p] += step_blocks;
        unit[p] += step_units;
        if (unit[p] >= units) unit[p] -= units, ++block[p];
      }
    };
    struct Rows {
      uint4 w[kPasses];
      uint32_t s[kPasses][G / 2];
    } kr, vr;
    auto load = [&](Rows& r, const uint32_t* codes, const void* scales) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        r.w[p] = reinterpret_cast<const uint4*>(codes)[row[p] * kLanes + piece];
        const uint32_t* sc = static_cast<const uint32_t*>(scales) + row[p] * (G / 2);
#pragma unroll
        for (int i = 0; i < G / 2; ++i) r.s[p][i] = sc[i];
      }
    };
    auto convert = [&](const Rows& r, uint8_t* slot) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int kr_ = p * kPassRows + row_in_pass;
        uint8_t* dst = slot + kr_ * 128;
        const uint32_t word[4] = {r.w[p].x, r.w[p].y, r.w[p].z, r.w[p].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // word 4 piece + i: its octet, and its group's scale twice
          const int o = q4::octet_of_word(4 * piece + i, G);
          const uint32_t pair = r.s[p][G == 4 ? i / 2 : 0], s2 = __byte_perm(pair, pair, i & 1 ? 0x3232 : 0x1010), s4 = Op<T>::steep(s2);
          const uint32_t w = word[i], h = w >> 8;
          *reinterpret_cast<uint4*>(dst + (o / 8) * kAtom + ((o & 7) ^ (kr_ & 7)) * 16) =
              make_uint4(Op<T>::low(w, s2), Op<T>::second(w, s4), Op<T>::low(h, s2), Op<T>::second(h, s4));
        }
      }
    };
    auto hand_over = [&](int h, const Rows& r) {
      const int s = h % S::kSlots;
      if (h >= S::kSlots && !ptx::mbar_wait(&empty[s], (h / S::kSlots - 1) & 1, abort_flag)) return false;
      convert(r, smem + S::kRing + s * S::kAtoms * kAtom);
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&full[s]);
      return true;
    };
    ask();
    resolve();
    load(kr, a.k_codes, a.k_scales);
    load(vr, a.v_codes, a.v_scales);
    ask();
    for (int j = 0; ok && j < tiles; ++j) {
      // values that no row may see are zeros: a weight of zero does not undo a NaN; a NaN that some row sees is marked
      const int key0 = (tile0 + j) * kKeys;
      uint32_t usable = 0;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int key = key0 + p * kPassRows + row_in_pass;
        usable |= key >= start && key < end ? known & (1u << p) : 0u;
      }
      ok = hand_over(2 * j, kr);
      if (!ok) break;
      if (j + 1 < tiles) {
        resolve();
        load(kr, a.k_codes, a.k_scales);
        ask();
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int i = 0; i < G / 2; ++i) {
          const float lo = Op<T>::low_f(vr.s[p][i]), hi = Op<T>::high_f(vr.s[p][i]);
          const bool use = usable >> p & 1;
          if (use && !(fabsf(lo) < INFINITY && fabsf(hi) < INFINITY)) *odd_values = 1;
          if (!use || !(fabsf(lo) < INFINITY)) vr.s[p][i] &= 0xffff0000u;
          if (!use || !(fabsf(hi) < INFINITY)) vr.s[p][i] &= 0x0000ffffu;
        }
      ok = hand_over(2 * j + 1, vr);
      if (ok && j + 1 < tiles) load(vr, a.v_codes, a.v_scales);
    }
    if (!ok && lane == 0 && status) atomicOr(status, kStatusFmhaLoad);
    __syncwarp();
  } else if (warp / 4 < streams) {
    // ---- softmax of row tile x
    const int x = warp / 4, r = (warp & 3) * 32 + lane, rr = row0 + x * 128 + r;
    const bool valid = rr < rows && rr / share < q_len;
    const int limit = valid ? limit_of(rr) : 0x7fffffff;   // rows that nobody reads are not masked
    const float unit = fmaxf(fabsf(a.scale_log2), 1.2e-38f);   // a scale of zero leaves masked scores at -inf
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + kColS + x * 128, t_o = tmem + lanes + kColO + x * 128;
    auto ask = [&](int tile) {   // lane i < 8: the page of 16 keys, as the table has it (looked at a tile later)
      const int blk = (tile * 8 + lane) / units;
      return lane < 8 && blk < table_len ? table[blk] : -1;
    };
    int next_page = ask(tile0);
    for (int j = 0; j < tiles; ++j) {
      const int key0 = (tile0 + j) * kKeys;
      const uint32_t pages = __ballot_sync(0xffffffffu, static_cast<uint32_t>(next_page) < static_cast<uint32_t>(a.num_blocks)) & 0xffu;   // 16 keys each
      next_page = ask(tile0 + j + 1);
      ok = ptx::mbar_wait(&s_full[x], j & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      ptx::tc_fence_after_sync();
      const bool whole = __all_sync(0xffffffffu, key0 + kKeys <= limit) && key0 >= start && pages == 0xffu;
      auto seen = [&](int c) {
        const int key = key0 + c;
        return key >= start && key < limit && (pages >> (c >> 4) & 1);
      };
      float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll 1
      for (int c0 = 0; c0 < kKeys; c0 += 64) {
        uint32_t v[64];
        ptx::tmem_ld_32x64(t_s + c0, v);
        ptx::tmem_ld_wait();
        if (whole) {
#pragma unroll
          for (int i = 0; i < 64; i += 2) t0 = fmaxf(t0, __uint_as_float(v[i])), t1 = fmaxf(t1, __uint_as_float(v[i + 1]));
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (seen(c0 + i)) t0 = fmaxf(t0, __uint_as_float(v[i]));
        }
      }
      const float top = fmaxf(t0, t1) * unit;
      const bool raise = top > m + 8.f;
      if (__any_sync(0xffffffffu, raise)) {
        const float f = raise ? ex2(m - top) : 1.f;
        m = raise ? top : m;
        l *= f;
        if (j > 0) {
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t v[32];
            ptx::tmem_ld_32x32(t_o + c0, v);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
            ptx::tmem_st_32x32(t_o + c0, v);
          }
        }
      }
      const uint64_t unit2 = pair(unit, unit), minus_m = pair(-m, -m);
      uint64_t s0 = 0, s1 = 0;   // sums of two at a time
#pragma unroll 1
      for (int c0 = 0; c0 < kKeys; c0 += 32) {
        uint32_t v[32], packed[16];
        ptx::tmem_ld_32x32(t_s + c0, v);
        ptx::tmem_ld_wait();
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = seen(c0 + i) ? v[i] : 0xff800000u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 e = unpair(fma2(pair(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), unit2, minus_m));
          const float p0 = ex2(e.x), p1 = ex2(e.y);
          (i & 2 ? s1 : s0) = add2(i & 2 ? s1 : s0, pair(p0, p1));
          packed[i / 2] = Op<T>::pack(p0, p1);
        }
        ptx::tmem_st_32x16(t_s + c0 / 2, packed);   // columns whose scores are read
      }
      const float2 both = unpair(add2(s0, s1));
      l += both.x + both.y;
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      ptx::mbar_arrive(&p_full[x]);
    }
    if (ok) ok = ptx::mbar_wait(&o_done[x], (tiles - 1) & 1, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    ptx::tc_fence_after_sync();
    if (!ok && lane == 0 && status) atomicOr(status, kStatusFmhaSoftmax);
  }
  __syncthreads();
  if (warp < 8 && row0 + (warp / 4) * 128 < rows) {
    const int x = warp / 4, rr = row0 + x * 128 + (warp & 3) * 32 + lane;
    const bool there = rr < rows, valid = there && rr / share < q_len && x < streams && ok;
    uint32_t poison = 0;   // groups in which the row sees a NaN
    if (*odd_values && valid) {
      const int limit = limit_of(rr);
      for (int key = start; key < limit; ++key) {
        const int page = page_of(key >> 4);
        if (page < 0) continue;
        const T* sc = static_cast<const T*>(a.v_scales) +
                      ((static_cast<int64_t>(page) * a.Hkv + hk) * a.block_size + (key >> 4) % units * 16 + (key & 15)) * G;
#pragma unroll
        for (int i = 0; i < G; ++i)
          if (!(fabsf(Elem<T>::to_f(sc[i])) < INFINITY)) poison |= 1u << i;
      }
    }
    const float inv = !valid ? 0.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;   // NaN stays
    const uint32_t t_o = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + kColO + x * 128;
    T* out = out_row(there ? rr : 0);
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 32) {
      uint32_t v[32];
      if (x < streams && ok) {   // uniform in the warp
        ptx::tmem_ld_32x32(t_o + c0, v);
        ptx::tmem_ld_wait();
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float o = __uint_as_float(v[8 * q + (i < 4 ? 2 * i : 2 * i - 7)]);
          y[i] = !valid ? 0.f : poison >> (c0 / 32) & 1 ? __uint_as_float(0x7fffffffu) : o * inv;
        }
        if (there)
          *reinterpret_cast<uint4*>(out + c0 + 8 * q) = make_uint4(Op<T>::pack(y[0], y[1]), Op<T>::pack(y[2], y[3]), Op<T>::pack(y[4], y[5]), Op<T>::pack(y[6], y[7]));
      }
    }
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, kCols);
}

template <typename T, int D>
int launch(const Args& a, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.H / a.Hkv) * a.Tq, row_blocks = (rows + 255) / 256, blocks = row_blocks * a.B * a.Hkv;
  OB_REQUIRE(blocks <= 0x7fffffff, OASR_ERR_INVALID, "fmha_q4: too many rows for one call");
  static SmemLimit limit;
  const cudaError_t e = limit.raise(fmha_q4_prompt_kernel<T, D>, Smem<D>::kDynamic);
  if (e != cudaSuccess) return set_error(OASR_ERR_CUDA, "fmha_q4: shared memory limit: %s", cudaGetErrorString(e));
  launch_pdl(fmha_q4_prompt_kernel<T, D>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), Smem<D>::kDynamic, s, a, static_cast<int>(row_blocks),
             device_status_ptr());
  return check_launch("fmha_q4 launch");
}

}  // namespace

int run_prompt(const Args& a, int head_dim, int dtype, cudaStream_t stream) {
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int { return head_dim == 64 ? launch<T_, 64>(a, stream) : launch<T_, 128>(a, stream); });
}

}  // namespace fmha_q4
}  // namespace ob
