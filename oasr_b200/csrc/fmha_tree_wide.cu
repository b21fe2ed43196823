// Attention of a tree of drafted tokens over 16-bit pages when many rows share a key head (fmha_tree.cu has the formula, and the form for few
// rows): tcgen05 products, keys and values by TMA straight out of the pages.
//
// A block has 128 or 256 rows of one (sequence, key head) and walks its share of the keys 128 at a time.  19 warps:
//   0-7, 8-15 softmax of two streams: two threads to a row, each with 64 of a step's keys: they read their scores from tensor memory and write
//             weights there;
//   16        one thread issues the products: S = Q K^T into 128 columns of tensor memory per stream, O += P V into D columns per stream
//             (a whole warp that waits and votes together took 5.1k clocks a step for 2.7k of products);
//   18        looks through the values of tiles at the ends of the sequence and among the drafted keys before their product;
//   17        fetches tiles of keys and values: pieces of 16 to 128 rows (whatever power of two divides a page), 128-byte swizzle.
// The streams are the two halves of 256 rows over the same keys, or the same 128 rows over the even and the odd tiles (kKeys2), put together at
// the end.  They run half a step apart: while one's softmax works, the tensor cores have the other's products.  Weights take the place of the scores
// they were made of (16 bits for 32) and are the A operand of the second product from there.  What they are relative to (m) moves only when
// a score passes it by far (kLag).
// A piece without a page is fetched from behind the pool, which gives zeros.  Values that no row sees become zeros as they are looked through, and
// so do those that are not finite and that some rows may not see; the rows that do see one get it by hand at the end.
// Bound by the steps: 256 rows x 128 keys of 128 dims take 4.0k clocks, 2.0k of them products at the tensor cores' rate; the rest is what softmax and products
// hand over to one another.  8 trees of 61 over 4000 to 8191 keys, 32 heads over 8: 85 us, floor 32 (products and cache alike); the longest sequence's blocks
// have 32 steps, the mean is 21.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "device_status.cuh"
#include "fmha_tree.cuh"
#include "sm100_ptx.cuh"
#include "smem_limit.cuh"
#include "tma_host.cuh"

namespace ob {
namespace fmha_tree {
namespace {

constexpr int kMmaWarp = 16, kProducer = 17, kReader = 18, kThreads = 608;
constexpr int kAtom = 128 * 128;   // 128 rows of 128 bytes
constexpr int kKeys = 128;
constexpr int kMaxCluster = kMostOfCluster;

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
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ bool odd_word(uint32_t w) {   // one of two 16-bit values is not finite
  constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & kExponent) == kExponent || (w >> 16 & kExponent) == kExponent;
}

// Barrier of the two warps that share 32 rows: whether any of them says yes.
__device__ __forceinline__ bool any_of_rows(int id, bool yes) {
  uint32_t any;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, 64, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(any)
      : "r"(yes ? 1u : 0u), "r"(id)
      : "memory");
  return any != 0;
}

template <int D, bool kKeys2>
struct Smem {
  static constexpr int kAtoms = D / 64, kTiles = kKeys2 ? 1 : 2, kSlots = D == 64 ? 8 : kKeys2 ? 6 : 5;
  static constexpr int kQ = 0, kRing = kQ + kTiles * kAtoms * kAtom, kBars = kRing + kSlots * kAtoms * kAtom;
  static constexpr int kNumBars = 3 * kSlots + 6;
  static constexpr int kTops = kBars + kNumBars * 8 + 32, kTotal = kTops + 2 * 128 * 4, kDynamic = kTotal + 1024;
  static_assert(kDynamic <= 232448, "what a block may have");
};

template <typename T, int D, bool kKeys2>
__global__ void __launch_bounds__(kThreads, 1) fmha_tree_wide_kernel(const Args a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                     const int row_blocks, const int piece_rows, uint32_t* status) {
  using S = Smem<D, kKeys2>;
  constexpr int NR = kKeys2 ? 128 : 256;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescQK = ptx::umma_idesc_f16(kBf16, 128, kKeys, false, false);
  constexpr uint32_t kIdescPV = ptx::umma_idesc_f16(kBf16, 128, D, false, true);   // V: keys are its rows
  constexpr uint32_t kColS = 0, kColO = 256, kCols = 512;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kSlots;
  uint64_t* s_full = empty + S::kSlots;   // [2]  scores are there (and the output has all weights before)
  uint64_t* p_full = s_full + 2;          // [2]  weights are there, output is scaled
  uint64_t* o_done = s_full + 4;          // [2]  output has the weights
  uint64_t* looked = s_full + 6;          // [kSlots]  values are there and looked through
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(looked + S::kSlots);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* odd_values = tmem_slot + 2;   // a drafted key has a value that is not finite
  volatile uint32_t* drain_flag = tmem_slot + 3;

  // what needs nothing of the kernels before
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == kProducer) {
    if (lane == 0) {
      ptx::prefetch_tensormap(&k_map);
      ptx::prefetch_tensormap(&v_map);
      for (int i = 0; i < S::kSlots; ++i) {
        ptx::mbar_init(&full[i], 1);
        ptx::mbar_init(&empty[i], 1);
        ptx::mbar_init(&looked[i], 1);
      }
      for (int x = 0; x < 2; ++x) {
        ptx::mbar_init(&s_full[x], 1);
        ptx::mbar_init(&p_full[x], 256);
        ptx::mbar_init(&o_done[x], 1);
      }
      *abort_flag = 0;
      *odd_values = 0;
      *drain_flag = 0;
      ptx::fence_barrier_init();
    }
    __syncwarp();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(tmem_slot, kCols);
    ptx::tmem_relinquish();
  }

  ptx::grid_dep_wait();
  const int split = static_cast<int>(blockIdx.x) % a.splits, group = static_cast<int>(blockIdx.x) / a.splits, groups = static_cast<int>(gridDim.x) / a.splits;
  int at = group;
  const int rb = at % row_blocks;
  at /= row_blocks;
  const int hk = at % a.Hkv, b = at / a.Hkv;
  const int share = a.H / a.Hkv, rows = share * a.Tq, row0 = rb * NR;
  const Sequence seq(a, b);
  const int all0 = seq.start / kKeys, all1 = row0 < seq.live * share ? max((seq.end + kKeys - 1) / kKeys, all0) : all0;
  const int per = (all1 - all0 + a.splits - 1) / a.splits;
  const int tile0 = min(all0 + split * per, all1), tiles = min(tile0 + per, all1) - tile0;
  float* const part = a.parts ? a.parts + (static_cast<int64_t>(split) * groups + group) * part_floats<D>(NR) : nullptr;
  const bool cluster = a.splits > 1 && part == nullptr;   // the blocks that share the keys are a cluster, whose rank is `split`
  auto out_row = [&](int r) { return static_cast<T*>(a.out) + b * a.os_b + (hk * share + r % share) * a.os_h + static_cast<int64_t>(r / share) * a.os_t; };

  // After the walk, in the ring's place: sums of both halves of a row; kKeys2: the second stream's maxima and output, dims outside; in a cluster the
  // block's maxima, sums and output, dims outside.
  float* const sums = reinterpret_cast<float*>(smem + S::kRing);
  float* const other_m = sums + 512;
  float* const other = other_m + 128;
  float* const my_m = other + (kKeys2 ? D * 128 : 0);
  float* const my_l = my_m + NR;
  float* const my_o = my_l + NR;
  static_assert((640 + (kKeys2 ? D * 128 : 0) + NR * (D + 2)) * 4 <= S::kSlots * S::kAtoms * kAtom, "fits the ring");
  auto meet = [&] {   // the blocks of a cluster put their results together, each eight dims in turn
    ptx::cluster_sync();
    const int r = threadIdx.x % NR, ways = 512 / NR, rr = row0 + r;
    if (threadIdx.x < 512 && rr < rows) {
      auto of = [&](const float* p, int rank) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::map_to_cta(p, rank)));
        return v;
      };
      float f[kMaxCluster], top = kEmpty, sum = 0.f;
      const float unit = unit_of(a);
      uint32_t blocks = 0;   // those with keys; the others have left nothing but a maximum of -inf
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) f[x] = x < a.splits ? of(my_m + r, x) : -INFINITY, top = fmaxf(top, f[x]);
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        if (!(f[x] > -INFINITY)) continue;
        blocks |= 1u << x;
        f[x] = ex2((f[x] - top) * unit);
        sum = fmaf(f[x], of(my_l + r, x), sum);   // (a sum that is NaN, of a query or keys that are, counts whatever its maximum)
      }
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // NaN stays
      T* const out = out_row(rr);
      for (int c = split + a.splits * static_cast<int>(threadIdx.x / NR); c < D / 8; c += a.splits * ways) {
        float y[8] = {};
#pragma unroll
        for (int x = 0; x < kMaxCluster; ++x)
          if (blocks >> x & 1u)   // (a weight of zero too: it makes NaN of values that are not finite)
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = fmaf(f[x], of(my_o + (8 * c + i) * NR + r, x), y[i]);
        *reinterpret_cast<uint4*>(out + 8 * c) = make_uint4(pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv), pack2<T>(y[4] * inv, y[5] * inv),
                                                            pack2<T>(y[6] * inv, y[7] * inv));
      }
    }
    __syncwarp();
    ptx::cluster_sync();   // nobody leaves while its results are read
  };
  if (tiles == 0) {   // nothing to see: zero rows
    if (cluster) {
      for (int i = threadIdx.x; i < NR; i += kThreads) my_m[i] = -INFINITY;
    } else if (part) {
      for (int i = threadIdx.x; i < NR * (D + 2); i += kThreads) part[i] = i < NR ? kEmpty : 0.f;
    } else {
      for (int i = threadIdx.x; i < min(NR, rows - row0) * (D / 8); i += kThreads)
        *reinterpret_cast<uint4*>(out_row(row0 + i / (D / 8)) + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    if (warp == kMmaWarp) ptx::tmem_dealloc(*tmem_slot, kCols);
    if (cluster) meet();
    return;
  }
  // streams with something in them, and their steps
  const int streams = kKeys2 ? min(tiles, 2) : (min(rows, seq.live * share) > row0 + 128 ? 2 : 1);
  auto steps_of = [&](int x) { return kKeys2 ? (tiles - x + 1) / 2 : tiles; };
  auto tile_of = [&](int x, int j) { return kKeys2 ? 2 * j + x : j; };

  const int table_len = static_cast<int>(a.blocks_per_seq), block_size = static_cast<int>(a.block_size);
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  auto page_at = [&](int key) {   // -1: none
    const int blk = key / block_size;
    const int page = blk < table_len ? table[blk] : -1;
    return page < a.num_blocks ? page : -1;
  };
  // The producer's lane i fetches piece i / kAtoms of a tile, dims 64 (i % kAtoms) .. of it.  Pages are asked for a tile ahead; what the ring holds is on its
  // way before the queries are.
  const int pieces = kKeys / piece_rows * S::kAtoms, atom = lane % S::kAtoms, first = lane / S::kAtoms * piece_rows;
  int row_now = 0, row_next = 0;
  auto row_at = [&](int i) {
    const int key = (tile0 + i) * kKeys + first, page = lane < pieces && i < tiles ? page_at(key) : -1;
    return page >= 0 ? page * block_size + key % block_size : static_cast<int>(a.num_blocks * a.block_size);   // (behind the pool)
  };
  auto fetch = [&](int h) {
    const int slot = h % S::kSlots;
    if (h % 2 == 0) row_now = row_next, row_next = row_at(h / 2 + 1);
    if (lane == 0) ptx::mbar_expect_tx(&full[slot], S::kAtoms * kAtom);
    __syncwarp();
    if (lane < pieces)
      ptx::tma_load_3d(smem + S::kRing + slot * S::kAtoms * kAtom + atom * kAtom + first * 128, h % 2 ? &v_map : &k_map, atom * 64, hk, row_now, &full[slot]);
  };
  if (warp == kProducer) {
    row_next = row_at(0);
    for (int h = 0; h < min(S::kSlots, 2 * tiles); ++h) fetch(h);
  }
  // queries, with the sign of the scale
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  if (warp < 16) {
    constexpr int kLoads = S::kTiles * 128 * (D / 8) / 512;   // of a thread, all on their way at once
    uint4 v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = k * 512 + static_cast<int>(threadIdx.x), rr = row0 + i / (D / 8), tq = rr / share;
      v[k] = make_uint4(0, 0, 0, 0);
      if (rr < rows)
        v[k] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs_b + (hk * share + rr - tq * share) * a.qs_h + static_cast<int64_t>(tq) * a.qs_t)[i % (D / 8)];
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = k * 512 + static_cast<int>(threadIdx.x), r = i / (D / 8), o = i % (D / 8);
      *reinterpret_cast<uint4*>(smem + S::kQ + ((r >> 7) * S::kAtoms + o / 8) * kAtom + (r & 127) * 128 + ((o & 7) ^ (r & 7)) * 16) =
          make_uint4(v[k].x ^ flip, v[k].y ^ flip, v[k].z ^ flip, v[k].w ^ flip);
    }
  }
  ptx::fence_proxy_async_smem();
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dep_launch();   // only now: see sm100_ptx.cuh

  bool ok = true;
  float m = kEmpty, l = 0.f;

  // which use of its slot for values item h is
  auto value_use = [](int h) { return S::kSlots % 2 ? h / S::kSlots / 2 : h / S::kSlots; };
  // whether tile i has values that some row may not see as they are
  auto partial = [&](int i) {
    const int key0 = (tile0 + i) * kKeys;
    return key0 < seq.start || key0 + kKeys > min(seq.prefix, seq.end);
  };
  if (warp == kMmaWarp) {
    if (ptx::elect_one()) {
      const uint32_t base = ptx::smem_u32(smem);
      auto slot_of = [&](int h) { return base + S::kRing + (h % S::kSlots) * S::kAtoms * kAtom; };
      auto wait_full = [&](int h) { return ptx::mbar_wait(&full[h % S::kSlots], (h / S::kSlots) & 1, abort_flag); };
      // (a slot has keys and values in turn where their number is odd, and one kind where it is even)
      auto wait_looked = [&](int h) { return ptx::mbar_wait(&looked[h % S::kSlots], value_use(h) & 1, abort_flag); };
      auto scores = [&](int x, int h) {
        const uint64_t ad = ptx::smem_desc_kmajor_sw128(base + S::kQ + (kKeys2 ? 0 : x) * S::kAtoms * kAtom), bd = ptx::smem_desc_kmajor_sw128(slot_of(h));
#pragma unroll
        for (int kk = 0; kk < S::kAtoms * 4; ++kk) {
          const uint32_t off = ((kk / 4) * kAtom + (kk % 4) * 32) >> 4;
          ptx::umma_f16(tmem + kColS + x * 128, ad + off, bd + off, kIdescQK, kk > 0);
        }
        ptx::umma_commit(&s_full[x]);
        if (kKeys2 || x == streams - 1) ptx::umma_commit(&empty[h % S::kSlots]);
      };
      auto output = [&](int x, int h, bool more) {
        const uint64_t bd = ptx::smem_desc_mnmajor_sw128(slot_of(h), kAtom, 1024);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          ptx::umma_f16_ts(tmem + kColO + x * 128, tmem + kColS + x * 128 + kk * 8, bd + ((kk * 2048) >> 4), kIdescPV, more || kk > 0);
        ptx::umma_commit(&o_done[x]);
        if (kKeys2 || x == streams - 1) ptx::umma_commit(&empty[h % S::kSlots]);
      };
      for (int x = 0; ok && x < streams; ++x) {
        const int h = 2 * tile_of(x, 0);
        if (kKeys2 || x == 0) ok = wait_full(h);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        scores(x, h);
      }
      const int steps = steps_of(0);
      for (int j = 0; ok && j < steps; ++j) {
        for (int x = 0; ok && x < streams; ++x) {
          const int i = tile_of(x, j), next = tile_of(x, j + 1);
          if (i >= tiles) continue;
          if (kKeys2 || x == 0) ok = wait_looked(2 * i + 1);
          ok = ok && ptx::mbar_wait(&p_full[x], j & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          output(x, 2 * i + 1, j > 0);
          if (next >= tiles) continue;
          if (kKeys2 || x == 0) ok = wait_full(2 * next);
          // products into other columns are not bound to stay in order: the weights go only once they are used
          ok = ok && ptx::mbar_wait(&o_done[x], j & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          scores(x, 2 * next);
        }
      }
      if (!ok && status) atomicOr(status, kStatusFmhaMma);
    }
    __syncwarp();
  } else if (warp == kReader) {
    for (int i = 0; ok && i < tiles; ++i) {
      const int h = 2 * i + 1, key0 = (tile0 + i) * kKeys;
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&full[h % S::kSlots], (h / S::kSlots) & 1, abort_flag)) != 0;
      if (!ok) break;
      if (!partial(i)) {
        if (lane == 0) ptx::mbar_arrive(&looked[h % S::kSlots]);
        continue;
      }
      uint8_t* slot = smem + S::kRing + (h % S::kSlots) * S::kAtoms * kAtom;
      bool odd = false;
      for (int p = lane; p < kKeys * S::kAtoms * 8; p += 32) {
        const int key = key0 + p / 8 % kKeys;
        uint4* v = reinterpret_cast<uint4*>(slot + p * 16);   // (the order within a row does not matter here)
        if (key < seq.start || key >= seq.end) {
          *v = make_uint4(0, 0, 0, 0);
        } else if (key >= seq.prefix) {
          const uint4 w = *v;
          if (odd_word<T>(w.x) || odd_word<T>(w.y) || odd_word<T>(w.z) || odd_word<T>(w.w)) {
            odd = true;
            T* e = reinterpret_cast<T*>(v);
            for (int y = 0; y < 8; ++y)
              if (!(fabsf(Elem<T>::to_f(e[y])) < INFINITY)) e[y] = Elem<T>::from_f(0.f);
          }
        }
      }
      if (odd) *odd_values = 1;
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&looked[h % S::kSlots]);
    }
    if (!ok && lane == 0 && status) atomicOr(status, kStatusFmhaLoad);
    __syncwarp();
  } else if (warp == kProducer) {
    int h = min(S::kSlots, 2 * tiles);
    for (; ok && h < 2 * tiles; ++h) {
      const int slot = h % S::kSlots;
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&empty[slot], (h / S::kSlots - 1) & 1, abort_flag)) != 0;
      if (!ok) break;
      fetch(h);
    }
    // nothing may be on its way when the block ends
    if (!ok)
      for (int x = max(h - S::kSlots, 0); x < h; ++x) ptx::mbar_wait(&full[x % S::kSlots], (x / S::kSlots) & 1, drain_flag);
    if (!ok && lane == 0 && status) atomicOr(status, kStatusFmhaLoad);
    __syncwarp();
  } else if (warp / 8 < streams) {
    // ---- softmax of stream x, keys 64 half .. of each step
    const int x = warp / 8, half = warp >> 2 & 1, r = (warp & 3) * 32 + lane, rr = row0 + (kKeys2 ? 0 : x * 128) + r;
    const int tq = min(rr / share, a.Tq - 1);
    const uint32_t* const words = mask_row(a, b, tq);
    const float unit = unit_of(a);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + kColS + x * 128, t_o = tmem + lanes + kColO + x * 128 + half * (D / 2);
    float* const row_top = reinterpret_cast<float*>(smem + S::kTops) + x * 128 + r;
    const int steps = steps_of(x), rows_id = 1 + x * 4 + (warp & 3);
    // bits of the 32 keys from `key` on that the row sees, pages aside
    auto sees32 = [&](int key) {
      auto below = [](int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; };   // the first n bits
      uint32_t bits = below(seq.prefix - key);
      const int u = key - seq.prefix;   // the first one's node
      if (u + 32 > 0) {
        uint32_t tree;
        if (words == nullptr) {
          tree = below(tq + 1 - u);
        } else {
          const int w = u >> 5, off = u & 31;
          const uint32_t lo = w >= 0 && w < a.mask_words ? words[w] : 0u, hi = off && w + 1 >= 0 && w + 1 < a.mask_words ? words[w + 1] : 0u;
          tree = __funnelshift_r(lo, hi, off);
        }
        bits |= tree & below(seq.live - u) & ~below(-u);
      }
      return bits & below(seq.end - key) & ~below(seq.start - key);
    };
    // (Where a wait is given up the walk goes on with whatever is there: both warps of the rows meet at every barrier.)
    for (int j = 0; j < steps; ++j) {
      const int key0 = (tile0 + tile_of(x, j)) * kKeys + half * 64;
      // 16 keys a bit: those with a page.  (A piece without one has keys of zero, whose scores are no less than others.)
      const uint32_t pages = __ballot_sync(0xffffffffu, lane < 4 && page_at(key0 + lane * 16) >= 0);
      const bool whole = pages == 0xfu && key0 >= seq.start && key0 + 64 <= min(seq.prefix, seq.end);
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      if (!whole) {
#pragma unroll
        for (int w = 0; w < 2; ++w)
          seen[w] = sees32(key0 + 32 * w) & ((pages >> (2 * w) & 1u ? 0xffffu : 0u) | (pages >> (2 * w + 1) & 1u ? 0xffff0000u : 0u));
      }
      ok &= __all_sync(0xffffffffu, ptx::mbar_wait(&s_full[x], j & 1, abort_flag)) != 0;
      ptx::tc_fence_after_sync();
      uint32_t v[64];
      ptx::tmem_ld_32x64(t_s + half * 64, v);
      ptx::tmem_ld_wait();
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (!(seen[i / 32] >> (i % 32) & 1u)) v[i] = 0xff800000u;
      }
      float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 64; ++i) t[i & 3] = fmaxf(t[i & 3], __uint_as_float(v[i]));
      const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      ptx::tc_fence_before_sync();
      if (any_of_rows(rows_id, (top - m) * unit > kLag)) {   // (also: all scores of these rows are read, and weights may take their place)
        float both = top;   // of the row: there and back between its two threads
        if (half) *row_top = top;
        ptx::named_barrier_sync(rows_id, 64);
        if (!half) *row_top = both = fmaxf(top, *row_top);
        ptx::named_barrier_sync(rows_id, 64);
        if (half) both = *row_top;
        const bool raise = (both - m) * unit > kLag;
        const float f = raise ? ex2((m - both) * unit) : 1.f;
        m = raise ? both : m;
        l *= f;
        if (j > 0) {
          ptx::tc_fence_after_sync();
#pragma unroll 1
          for (int c0 = 0; c0 < D / 2; c0 += 16) {
            uint32_t o[16];
            ptx::tmem_ld_32x16(t_o + c0, o);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st_32x16(t_o + c0, o);
          }
        }
      }
      ptx::tc_fence_after_sync();
      const uint64_t unit2 = pair(unit, unit), minus_m = pair(-m, -m), below2 = pair(kBelow<T>, kBelow<T>);
      uint64_t s0 = 0, s1 = 0;   // sums of two at a time
#pragma unroll
      for (int c0 = 0; c0 < 64; c0 += 32) {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 e = unpair(fma2(add2(pair(__uint_as_float(v[c0 + i]), __uint_as_float(v[c0 + i + 1])), minus_m), unit2, below2));
          const float2 w = make_float2(ex2(e.x), ex2(e.y));
          (i & 2 ? s1 : s0) = add2(i & 2 ? s1 : s0, pair(w.x, w.y));
          packed[i / 2] = pack2<T>(w.x, w.y);
        }
        ptx::tmem_st_32x16(t_s + half * 32 + c0 / 2, packed);
      }
      const float2 both = unpair(add2(s0, s1));
      l += both.x + both.y;
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      ptx::mbar_arrive(&p_full[x]);
    }
    ok &= __all_sync(0xffffffffu, ptx::mbar_wait(&o_done[x], (steps - 1) & 1, abort_flag)) != 0;
    ptx::tc_fence_after_sync();
    if (!ok && lane == 0 && status) atomicOr(status, kStatusFmhaSoftmax);
  }
  __syncthreads();
  const bool done = *abort_flag == 0;
  if (warp < 16) {
    const int x = warp / 8, half = warp >> 2 & 1, r = (warp & 3) * 32 + lane;
    sums[(x * 2 + half) * 128 + r] = l;
    if (kKeys2 && x == 1 && streams == 2) {
      const uint32_t t_o = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + kColO + 128 + half * (D / 2);
#pragma unroll 1
      for (int c0 = 0; c0 < D / 2; c0 += 32) {
        uint32_t v[32];
        ptx::tmem_ld_32x32(t_o + c0, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) other[(half * (D / 2) + c0 + i) * 128 + r] = __uint_as_float(v[i]);
      }
      if (half == 0) other_m[r] = m;
    }
  }
  __syncthreads();
  const bool join = part || cluster;
  if (warp < (kKeys2 ? 8 : 16) && (join || row0 + (kKeys2 ? 0 : (warp / 8) * 128) < rows)) {
    const int x = warp / 8, half = warp >> 2 & 1, rs = (warp & 3) * 32 + lane, r = x * 128 + rs, rr = row0 + r;
    const bool there = rr < rows, valid = there && rr / share < seq.live && x < streams && done;
    l = sums[x * 256 + rs] + sums[x * 256 + 128 + rs];
    float f0 = 1.f, f1 = 0.f;
    if (kKeys2 && streams == 2) {
      const float unit = unit_of(a), top = fmaxf(m, other_m[rs]);
      f0 = ex2((m - top) * unit), f1 = ex2((other_m[rs] - top) * unit);
      m = top;
      l = fmaf(f0, l, f1 * (sums[256 + rs] + sums[384 + rs]));
    }
    const uint32_t t_o = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + kColO + x * 128;
    const float inv = !valid ? 0.f : join ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;   // NaN stays
    float *const to_m = part ? part : my_m, *const to_o = part ? part + 2 * NR : my_o;
    if (join && half == 0) to_m[r] = valid ? m : kEmpty, to_m[NR + r] = valid ? l : 0.f;
    const bool by_hand = *odd_values && valid;
    T* out = out_row(there ? rr : 0);
#pragma unroll 1
    for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
      uint32_t v[32];
      float y[32];
      if (x < streams && done) {   // uniform in the warp
        ptx::tmem_ld_32x32(t_o + c0, v);
        ptx::tmem_ld_wait();
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        y[i] = __uint_as_float(v[i]);
        if (kKeys2 && streams == 2) y[i] = fmaf(f0, y[i], f1 * other[(c0 + i) * 128 + rs]);
        y[i] = valid ? y[i] * inv : 0.f;
      }
      if (by_hand) {
        const int tq = rr / share;
        const uint32_t* const words = mask_row(a, b, tq);
        const int k0 = max(max(seq.prefix, seq.start), tile0 * kKeys), k1 = min(seq.end, (tile0 + tiles) * kKeys);
        for (int key = k0; key < k1; ++key) {
          const int page = page_at(key);
          if (page < 0 || !sees(a, words, tq, key - seq.prefix, seq.live)) continue;
          const T* vs = static_cast<const T*>(a.v) + ((static_cast<int64_t>(page) * block_size + key % block_size) * a.Hkv + hk) * D + c0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float e = Elem<T>::to_f(vs[i]);
            if (!(fabsf(e) < INFINITY)) y[i] += e;
          }
        }
      }
      if (join) {   // dims outside: the lanes' rows lie together
#pragma unroll
        for (int i = 0; i < 32; ++i) to_o[(c0 + i) * NR + r] = y[i];
      } else if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(out + c0 + 8 * i) = make_uint4(pack2<T>(y[8 * i], y[8 * i + 1]), pack2<T>(y[8 * i + 2], y[8 * i + 3]),
                                                                   pack2<T>(y[8 * i + 4], y[8 * i + 5]), pack2<T>(y[8 * i + 6], y[8 * i + 7]));
      }
    }
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, kCols);
  if (cluster) meet();
}

// Joins the partial results of a group's blocks, more than a cluster has: a block has 4 dims of 32 rows (the lanes), its warps an eighth of the
// parts each (16 dims: a part's loads fill the registers, and 74 parts take 7 us longer).
template <typename T, int D>
__global__ void __launch_bounds__(256) fmha_tree_wide_join_kernel(const Args a, const int row_blocks, const int NR, const int groups) {
  constexpr int kDims = 4, kWays = 8;
  __shared__ float outs[kWays][32][kDims + 1];
  __shared__ float tops[kWays][32], sums[kWays][32];
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int at = blockIdx.x;
  const int d0 = at % (D / kDims) * kDims;
  at /= D / kDims;
  const int n0 = at % (NR / 32) * 32, group = at / (NR / 32), rb = group % row_blocks, hk = group / row_blocks % a.Hkv, b = group / row_blocks / a.Hkv;
  const int share = a.H / a.Hkv, rows = share * a.Tq, r0 = rb * NR + n0;
  if (r0 >= rows) return;
  const int64_t part = part_floats<D>(NR), step = part * groups;
  const float* src = a.parts + group * part + n0 + lane;
  const float unit = unit_of(a);
  float top = kEmpty, sum = 0.f, acc[kDims] = {};
#pragma unroll 8
  for (int s = warp; s < a.splits; s += kWays) top = fmaxf(top, src[s * step]);
  constexpr int kBatch = 5;   // parts whose loads are on their way at once (74 parts: 31.9 us with the walk; 33.6 with 8, 34.4 as the compiler unrolls it)
#pragma unroll 1
  for (int s0 = warp; s0 < a.splits; s0 += kWays * kBatch) {
    float m[kBatch], l[kBatch], v[kBatch][kDims];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int s = s0 + x * kWays;
      const float* p = src + s * step;
      m[x] = s < a.splits ? p[0] : kEmpty, l[x] = s < a.splits ? p[NR] : 0.f;
#pragma unroll
      for (int i = 0; i < kDims; ++i) v[x][i] = s < a.splits ? p[(2 + d0 + i) * NR] : 0.f;
    }
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const float f = ex2((m[x] - top) * unit);
      sum = fmaf(f, l[x], sum);
#pragma unroll
      for (int i = 0; i < kDims; ++i) acc[i] = fmaf(f, v[x][i], acc[i]);
    }
  }
  tops[warp][lane] = top, sums[warp][lane] = sum;
#pragma unroll
  for (int i = 0; i < kDims; ++i) outs[warp][lane][i] = acc[i];
  __syncthreads();
  if (threadIdx.x < 32 * kDims) {
    const int n = threadIdx.x / kDims, d = threadIdx.x % kDims, r = r0 + n;
    if (r >= rows) return;
    float y = 0.f, all = 0.f, most = kEmpty;
#pragma unroll
    for (int w = 0; w < kWays; ++w) most = fmaxf(most, tops[w][n]);
#pragma unroll
    for (int w = 0; w < kWays; ++w) {
      const float f = ex2((tops[w][n] - most) * unit);
      y = fmaf(f, outs[w][n][d], y), all = fmaf(f, sums[w][n], all);
    }
    const int tq = r / share, live = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
    const float inv = all > 0.f ? 1.f / all : all == 0.f ? 0.f : all;   // NaN stays
    static_cast<T*>(a.out)[b * a.os_b + (hk * share + r - tq * share) * a.os_h + static_cast<int64_t>(tq) * a.os_t + d0 + d] = Elem<T>::from_f(tq < live ? y * inv : 0.f);
  }
}

template <typename T, int D, bool kKeys2>
int launch(const Args& a, int dtype, int64_t groups, int row_blocks, cudaStream_t s) {
  using S = Smem<D, kKeys2>;
  static SmemLimit limit;
  const cudaError_t e = limit.raise(fmha_tree_wide_kernel<T, D, kKeys2>, S::kDynamic);
  if (e != cudaSuccess) return set_error(OASR_ERR_CUDA, "fmha_tree: shared memory limit: %s", cudaGetErrorString(e));
  int piece = 16;
  while (piece < 128 && a.block_size % (2 * piece) == 0) piece *= 2;
  // (64 dims of a head, head, row of the pool)
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.Hkv), static_cast<uint64_t>(a.num_blocks * a.block_size)};
  const uint64_t strides[3] = {2, static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(a.Hkv) * D * 2};
  const uint32_t box[3] = {64, 1, static_cast<uint32_t>(piece)};
  CUtensorMap k_map, v_map;
  int rc = make_tensor_map(&k_map, tma_dtype(dtype), 3, a.k, dims, strides, box);
  if (rc == OASR_OK) rc = make_tensor_map(&v_map, tma_dtype(dtype), 3, a.v, dims, strides, box);
  if (rc != OASR_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * a.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kDynamic;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = g_pdl ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {static_cast<unsigned>(a.splits), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = a.parts == nullptr && a.splits > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, fmha_tree_wide_kernel<T, D, kKeys2>, a, k_map, v_map, row_blocks, piece, device_status_ptr());
  rc = check_launch("fmha_tree launch");
  if (rc != OASR_OK || a.parts == nullptr) return rc;
  constexpr int NR = kKeys2 ? 128 : 256;
  launch_pdl(fmha_tree_wide_join_kernel<T, D>, dim3(static_cast<unsigned>(groups * (NR / 32) * (D / 4))), dim3(256), 0, s, a, row_blocks, NR, static_cast<int>(groups));
  return check_launch("fmha_tree join launch");
}

}  // namespace

int run_wide(const Args& a, int head_dim, int dtype, int block_rows, int64_t groups, int row_blocks, cudaStream_t s) {
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int {
    if (head_dim == 64) return block_rows == 128 ? launch<T_, 64, true>(a, dtype, groups, row_blocks, s) : launch<T_, 64, false>(a, dtype, groups, row_blocks, s);
    return block_rows == 128 ? launch<T_, 128, true>(a, dtype, groups, row_blocks, s) : launch<T_, 128, false>(a, dtype, groups, row_blocks, s);
  });
}

}  // namespace fmha_tree
}  // namespace ob
