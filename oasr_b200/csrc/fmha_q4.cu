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
//   K   the lane holds words t G .. t G + G - 1 (an octet of each group) of keys 4 g .. 4 g + 3.  The operand is the code with
//       a magic exponent in front, 128 + n in bf16 (1024 + n in fp16): one LOP3 per two codes, exact.  The offset comes off in
//       the accumulator, which starts at -136 (-1032) sum(q) of the group; a group's sums are scaled in fp32 afterwards.
//   V   the lane holds words of keys 8 t .. 8 t + 7.  Long sums would drown under such an offset, so here the operand is
//       (n - 8) * scale, exact in the type (q4.cuh).
//   P   the scores' fragment is the transpose of what the second product reads: movmatrix.
// The running maximum moves only when a score passes it by 2^8 (weights stay below that, exact in either type): most tiles
// need one vote in the place of a reduction over the lanes.
// Every warp walks its own tiles with its own maximum, sum and output; the warps of a block, and the blocks of a cluster that
// share one (sequence, key head, rows), meet in shared memory at the end.
#include "common.cuh"
#include "q4.cuh"
#include "sm100_ptx.cuh"
#include "smem_limit.cuh"

namespace ob {
namespace {

struct Args {
  void* out;
  const void* q;
  const uint32_t *k_codes, *v_codes;
  const void *k_scales, *v_scales;
  const int32_t *block_table, *seqlens, *seqstarts, *q_lens;
  int64_t qs_b, qs_h, qs_t, os_b, os_h, os_t;
  int64_t blocks_per_seq, block_size, num_blocks;
  int B, H, Hkv, Tq, causal;
  float scale_log2;
};

constexpr int kWarps = 4;

template <typename T>
struct Op;
template <>
struct Op<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;   // 128
  static constexpr float kBias = 136.f;
  static __device__ __forceinline__ uint32_t centred(uint32_t w) {   // (128 + n) - 136
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&w), __nv_bfloat162(__float2bfloat16_rn(136.f), __float2bfloat16_rn(136.f)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Op<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;   // 1024
  static constexpr float kBias = 1032.f;
  static __device__ __forceinline__ uint32_t centred(uint32_t w) {
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&w), __half2(__float2half_rn(1032.f), __float2half_rn(1032.f)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
    const __half2 v = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// two 16-bit values (the low halves or the high halves of two words) as one
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

template <int G>
struct KTile {           // keys 4 g .. 4 g + 3
  uint32_t w[4][G];
  uint32_t s[4 * G / 2];  // their scales, two to a word
};
template <int G>
struct VTile {           // keys 8 t .. 8 t + 7
  uint32_t w[8][G / 2];
  uint32_t s[8 * G / 2];
};

template <int N>
__device__ __forceinline__ void ldg(const void* p, uint32_t* r) {
  if constexpr (N == 1) {
    r[0] = __ldg(static_cast<const uint32_t*>(p));
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(static_cast<const uint2*>(p));
    r[0] = v.x, r[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = __ldg(static_cast<const uint4*>(p) + i);
      r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w;
    }
  }
}

template <typename T, int D, int NT>
struct Merge {   // a warp's, and then the block's, maxima, sums and outputs
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  float o[kWarps][8 * NT][D + 4];
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32) fmha_q4_kernel(const Args a, const int parts, const int row_blocks) {
  constexpr int G = D / 32, W = D / 8, VW = G / 2;   // words of a row, of them a lane's in V
  constexpr int NR = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];
  Merge<T, D, NT>& sh = *reinterpret_cast<Merge<T, D, NT>*>(smem);
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int part = blockIdx.x % parts;
  int at = blockIdx.x / parts;
  const int rb = at % row_blocks;
  at /= row_blocks;
  const int hk = at % a.Hkv, b = at / a.Hkv;
  const int share = a.H / a.Hkv;
  const int rows = share * a.Tq, row0 = rb * NR;
  const int len = a.seqlens[b], q_len = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
  const int capacity = static_cast<int>(a.blocks_per_seq * a.block_size);
  const int start = a.seqstarts ? max(a.seqstarts[b], 0) : 0;

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

  // ---- queries as the second operand: column g, dims of octet t of each group
  uint32_t qf[NT][G][4];
  float bias[NT][G][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + n * 8 + g;
    const T* q = static_cast<const T*>(a.q) + b * a.qs_b + (hk * share + r % share) * a.qs_h + static_cast<int64_t>(r / share) * a.qs_t;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows) v = *reinterpret_cast<const uint4*>(q + k * 32 + t * 8);
      const T* x = reinterpret_cast<const T*>(&v);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += Elem<T>::to_f(x[i]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      bias[n][k][0] = -Op<T>::kBias * __shfl_sync(0xffffffffu, sum, 8 * t);
      bias[n][k][1] = -Op<T>::kBias * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      qf[n][k][0] = lows(v.x, v.z), qf[n][k][1] = highs(v.x, v.z);   // dims (0, 4), (1, 5) of the octet
      qf[n][k][2] = lows(v.y, v.w), qf[n][k][3] = highs(v.y, v.w);   // (2, 6), (3, 7)
    }
  }

  float o[NT][VW * 4][4] = {}, m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;

  const int units = static_cast<int>(a.block_size) / 16;   // halves of a tile are 16 keys of one page
  const int32_t* table = a.block_table + b * a.blocks_per_seq;
  const int step = kWarps * parts;
  const int tile_end = (end + 31) / 32;
  int tile = start / 32 + part * kWarps + warp;

  // pages of a tile's two halves; -1: none
  auto pages_of = [&](int i, int& p0, int& p1) {
    p0 = p1 = -1;
    if (i >= tile_end) return;
    const int u = 2 * i, blk = u / units;
    p0 = table[blk];                                                  // u * 16 < end <= capacity
    const int blk1 = u + 1 - blk * units < units ? blk : blk + 1;
    if (blk1 < a.blocks_per_seq) p1 = blk1 == blk ? p0 : table[blk1];
    if (p0 < 0 || p0 >= a.num_blocks) p0 = -1;
    if (p1 < 0 || p1 >= a.num_blocks) p1 = -1;
  };
  // first row of the half's 16 keys; a half without a page reads page 0 and is masked
  auto row_of = [&](int i, int half, int page) {
    const int u = 2 * i + half;
    return (static_cast<int64_t>(max(page, 0)) * a.Hkv + hk) * a.block_size + (u % units) * 16;
  };
  KTile<G> kt;
  VTile<G> vt;
  auto load_k = [&](int i, int p0, int p1) {
    const int half = g >> 2;
    const int64_t row = row_of(i, half, half ? p1 : p0) + (g & 3) * 4;
#pragma unroll
    for (int x = 0; x < 4; ++x) ldg<G>(a.k_codes + (row + x) * W + t * G, kt.w[x]);
    ldg<2 * G>(static_cast<const T*>(a.k_scales) + row * G, kt.s);
  };
  auto load_v = [&](int i, int p0, int p1) {
    const int half = t >> 1;
    const int64_t row = row_of(i, half, half ? p1 : p0) + (t & 1) * 8;
#pragma unroll
    for (int x = 0; x < 8; ++x) ldg<VW>(a.v_codes + (row + x) * W + g * VW, vt.w[x]);
    ldg<4 * G>(static_cast<const T*>(a.v_scales) + row * G, vt.s);
  };

  int p0, p1, n0, n1;
  pages_of(tile, p0, p1);
  pages_of(tile + step, n0, n1);
  if (tile < tile_end) {
    load_k(tile, p0, p1);
    load_v(tile, p0, p1);
  }
  for (; tile < tile_end; tile += step) {
    const int j0 = tile * 32;
    const bool whole = j0 >= start && j0 + 32 <= all_end && p0 >= 0 && p1 >= 0;   // nothing to mask
    int f0, f1;
    pages_of(tile + 2 * step, f0, f1);

    // ---- scores of keys 4 g + 2 i (+ 1), columns 2 t (+ 1)
    float s[NT][2][4] = {};
#pragma unroll
    for (int k = 0; k < G; ++k) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sc[2];   // scales of keys 4 g + 2 i, 4 g + 2 i + 1
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int e = (2 * i + x) * G + k;
          const uint32_t w = kt.s[e / 2];
          const unsigned short h = static_cast<unsigned short>(e & 1 ? w >> 16 : w);
          sc[x] = Elem<T>::to_f(*reinterpret_cast<const T*>(&h)) * a.scale_log2;
        }
        const uint32_t wa = kt.w[2 * i][k], wb = kt.w[2 * i + 1][k];
        uint32_t af[8];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          af[2 * n] = ((wa >> (4 * n)) & 0x000f000fu) | Op<T>::kMagic;
          af[2 * n + 1] = ((wb >> (4 * n)) & 0x000f000fu) | Op<T>::kMagic;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float c[4] = {bias[n][k][0], bias[n][k][1], bias[n][k][0], bias[n][k][1]};
          Op<T>::mma(c, af[0], af[1], af[2], af[3], qf[n][k][0], qf[n][k][1]);
          Op<T>::mma(c, af[4], af[5], af[6], af[7], qf[n][k][2], qf[n][k][3]);
          s[n][i][0] = fmaf(sc[0], c[0], s[n][i][0]);
          s[n][i][1] = fmaf(sc[0], c[1], s[n][i][1]);
          s[n][i][2] = fmaf(sc[1], c[2], s[n][i][2]);
          s[n][i][3] = fmaf(sc[1], c[3], s[n][i][3]);
        }
      }
    }
    if (tile + step < tile_end) load_k(tile + step, n0, n1);
    if (!whole) {
      const bool page = (g >> 2 ? p1 : p0) >= 0;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = j0 + 4 * g + 2 * i + (x >> 1);
            if (!page || j < start || j >= limit[n][x & 1]) s[n][i][x] = -INFINITY;
          }
    }

    // ---- weights
    float top[NT][2];
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = fmaxf(fmaxf(s[n][0][c], s[n][0][2 + c]), fmaxf(s[n][1][c], s[n][1][2 + c]));
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
          const float f = v == -INFINITY ? 1.f : ex2(m[n][c] - v);
          m[n][c] = v;
          l[n][c] *= f;
#pragma unroll
          for (int i = 0; i < VW * 4; ++i) o[n][i][c] *= f, o[n][i][2 + c] *= f;
        }
    }
    uint32_t pf[NT][4];   // block x: keys 4 g + x -> after the transpose columns are rows
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float e0 = ex2(s[n][x >> 1][(x & 1) * 2] - m0), e1 = ex2(s[n][x >> 1][(x & 1) * 2 + 1] - m1);
        l[n][0] += e0;
        l[n][1] += e1;
        pf[n][x] = transpose8x8(Op<T>::pack(e0, e1));
      }
    }

    // ---- output: dims of word(s) g, keys 8 t + x and 8 t + 4 + x of block x
    uint32_t vs[8 * VW];
    const int vgroup = (g * VW) % G;   // group of the lane's first word; the next word's group is the next one
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      // scales of key 8 t + x in the lane's groups: word x * G / 2 (+ which half)
      if constexpr (G == 2) vs[x] = vt.s[x];
      else vs[x] = vgroup ? vt.s[2 * x + 1] : vt.s[2 * x];
    }
    if (!whole) {   // a key that some row of the block does not see must not reach it as 0 * NaN: those rows' outputs take it by hand
      bool odd = false;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int j = j0 + 8 * t + x;
        const bool there = (t >> 1 ? p1 : p0) >= 0 && j >= start && j < end;
        unsigned short lo = static_cast<unsigned short>(vs[x]), hi = static_cast<unsigned short>(vs[x] >> 16);
        const float flo = Elem<T>::to_f(*reinterpret_cast<T*>(&lo)), fhi = Elem<T>::to_f(*reinterpret_cast<T*>(&hi));
        if (!there || !(fabsf(flo) < INFINITY)) odd |= there, vs[x] &= 0xffff0000u;
        if (!there || !(fabsf(fhi) < INFINITY)) odd |= there, vs[x] &= 0x0000ffffu;
      }
      if (__any_sync(0xffffffffu, odd)) {
        for (int x = 0; x < 32; ++x) {
          const int j = j0 + x, page = x >> 4 ? p1 : p0;
          if (page < 0 || j < start || j >= end) continue;
          const T* sc = static_cast<const T*>(a.v_scales) + (row_of(tile, x >> 4, page) + (x & 15)) * G;
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const float v = Elem<T>::to_f(sc[(g * VW + w) % G]);
            if (fabsf(v) < INFINITY) continue;
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
      uint32_t lo[4], hi[4], sp[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        lo[x] = lows(vt.w[x][w], vt.w[x + 4][w]);
        hi[x] = highs(vt.w[x][w], vt.w[x + 4][w]);
        // G = 2: the word's group is g % 2; G = 4: words 2 g, 2 g + 1 are the low and the high scale of the selected pair
        if constexpr (G == 2) sp[x] = g & 1 ? highs(vs[x], vs[x + 4]) : lows(vs[x], vs[x + 4]);
        else sp[x] = w ? highs(vs[x], vs[x + 4]) : lows(vs[x], vs[x + 4]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // dims 2 i, 2 i + 1 of the octet
        uint32_t d0[4], d1[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t src = i < 2 ? lo[x] : hi[x];
          d0[x] = Op<T>::mul(Op<T>::centred(((src >> (8 * (i & 1))) & 0x000f000fu) | Op<T>::kMagic), sp[x]);
          d1[x] = Op<T>::mul(Op<T>::centred(((src >> (8 * (i & 1) + 4)) & 0x000f000fu) | Op<T>::kMagic), sp[x]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          Op<T>::mma(o[n][w * 4 + i], d0[0], d1[0], d0[1], d1[1], pf[n][0], pf[n][1]);
          Op<T>::mma(o[n][w * 4 + i], d0[2], d1[2], d0[3], d1[3], pf[n][2], pf[n][3]);
        }
      }
    }
    if (tile + step < tile_end) load_v(tile + step, n0, n1);
    p0 = n0, p1 = n1, n0 = f0, n1 = f1;
  }

  // ---- the warps of the block meet, then the blocks of the cluster
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float v = l[n][c];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      const int r = n * 8 + 2 * t + c;
      if (g == 0) sh.m[warp][r] = v == v ? m[n][c] : 0.f, sh.l[warp][r] = v;   // a NaN never became the maximum, but has a say
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
        const float f = sh.m[w][r] == -INFINITY ? 0.f : ex2(sh.m[w][r] - top);
        const float4 v = *reinterpret_cast<const float4*>(&sh.o[w][r][d]);
        if (sh.m[w][r] != -INFINITY) acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
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
      for (int w = 0; w < kWarps; ++w)
        if (sh.m[w][r] != -INFINITY) sum = fmaf(sh.l[w][r], ex2(sh.m[w][r] - top), sum);
      sh.m[0][r] = top, sh.l[0][r] = sum;
    }
    ptx::cluster_sync();
  }
  const int ways = parts > 1 ? parts : kWarps;
  auto remote = [&](const float* p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::map_to_cta(p, rank)) : "memory");
    return v;
  };
  for (int i = part * kWarps * 32 + threadIdx.x; i < NR * (D / 8); i += parts * kWarps * 32) {
    const int n = i / (D / 8), d = i % (D / 8) * 8, r = row0 + n;
    if (r >= rows) continue;
    float ms[8], top = -INFINITY, sum = 0.f, acc[8] = {};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < ways) {
        ms[w] = parts > 1 ? remote(&sh.m[0][n], w) : sh.m[w & (kWarps - 1)][n];
        top = fmaxf(top, ms[w]);
      }
    }
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < ways && ms[w] != -INFINITY) {
        const float f = ex2(ms[w] - top);
        sum = fmaf(f, parts > 1 ? remote(&sh.l[0][n], w) : sh.l[w & (kWarps - 1)][n], sum);
        const float* src = parts > 1 ? &sh.o[0][n][d] : &sh.o[w & (kWarps - 1)][n][d];
        float v[8];
        if (parts > 1) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
            asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[4 * x]), "=f"(v[4 * x + 1]), "=f"(v[4 * x + 2]), "=f"(v[4 * x + 3])
                         : "r"(ptx::map_to_cta(src + 4 * x, w)) : "memory");
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = src[x];
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] = fmaf(f, v[x], acc[x]);
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // NaN stays
    Pack<T> out;
#pragma unroll
    for (int x = 0; x < 8; ++x) out.v[x] = Elem<T>::from_f(r / share < q_len ? acc[x] * inv : 0.f);
    st128(static_cast<T*>(a.out) + b * a.os_b + (hk * share + r % share) * a.os_h + static_cast<int64_t>(r / share) * a.os_t + d, out);
  }
  if (parts > 1) ptx::cluster_sync();   // nobody leaves while its sums are read
}

template <typename T, int D, int NT>
int launch(const Args& a, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.H / a.Hkv) * a.Tq, row_blocks = (rows + 8 * NT - 1) / (8 * NT);
  const int64_t groups = static_cast<int64_t>(a.B) * a.Hkv * row_blocks, tiles = (a.blocks_per_seq * a.block_size + 31) / 32;
  int parts = 1;   // few groups: a cluster each, down to two tiles a warp
  while (parts < 8 && groups * parts < sm_count() * 3 && tiles > 2 * kWarps * parts) parts *= 2;
  OB_REQUIRE(groups * parts <= 0x7fffffff, OASR_ERR_INVALID, "fmha_q4: too many rows for one call");
  static SmemLimit limit;
  constexpr int kSmem = sizeof(Merge<T, D, NT>);
  cudaError_t e = limit.raise(fmha_q4_kernel<T, D, NT>, kSmem);
  if (e != cudaSuccess) return set_error(OASR_ERR_CUDA, "fmha_q4: shared memory limit: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * parts));
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
  cudaLaunchKernelEx(&cfg, fmha_q4_kernel<T, D, NT>, a, parts, static_cast<int>(row_blocks));
  return check_launch("fmha_q4 launch");
}

template <typename T, int D>
int run(const Args& a, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.H / a.Hkv) * a.Tq;
  if (rows <= 8) return launch<T, D, 1>(a, s);
  if constexpr (D == 64)
    if (rows > 16) return launch<T, D, 4>(a, s);
  return launch<T, D, 2>(a, s);
}

}  // namespace
}  // namespace ob

extern "C" int oasr_b200_fmha_q4(void* out, const int64_t* out_strides, const void* q, const int64_t* q_strides, const void* k_codes,
                                 const void* k_scales, const void* v_codes, const void* v_scales, const int32_t* block_table,
                                 const int32_t* seqlens, const int32_t* seqstarts, const int32_t* q_lens, int64_t blocks_per_seq,
                                 int64_t block_size, int64_t num_blocks, int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t D,
                                 double scale, int causal, int dtype, void* stream) {
  using namespace ob;
  OB_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && Tq >= 0 && D > 0 && blocks_per_seq >= 0 && num_blocks > 0, OASR_ERR_INVALID, "fmha_q4: bad shape");
  OB_REQUIRE(H % Hkv == 0, OASR_ERR_INVALID, "fmha_q4: H (%lld) must be divisible by H_kv (%lld)", (long long)H, (long long)Hkv);
  OB_REQUIRE(D == 64 || D == 128, OASR_ERR_UNSUPPORTED, "fmha_q4: head_dim %lld is not supported (64 and 128 are)", (long long)D);
  OB_REQUIRE(block_size > 0 && block_size % 16 == 0, OASR_ERR_UNSUPPORTED, "fmha_q4: the block size must be a multiple of 16 (got %lld)",
             (long long)block_size);
  OB_REQUIRE(B <= 65535 && H <= 65535 && Tq <= 0x7fffff && blocks_per_seq * block_size <= 0x7fffffff, OASR_ERR_INVALID,
             "fmha_q4: batch, head count or length too large");
  if (B == 0 || Tq == 0) return OASR_OK;
  OB_REQUIRE(out && out_strides && q && q_strides && k_codes && k_scales && v_codes && v_scales && block_table && seqlens, OASR_ERR_INVALID,
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
  return OB_DISPATCH_HALF(dtype, T_, [&]() -> int { return D == 64 ? run<T_, 64>(a, st) : run<T_, 128>(a, st); });
}
